"""Schemas of the torch.ops of the windowed attention."""
import torch

from infer_b200 import infer_ops  # noqa: F401 - registers the ops


def test_window_is_optional_in_decode_as_in_prefill():
    """A model calls one op for all of its layers, those without a window with None."""
    for name in ("paged_attn_decode_window", "paged_attn_prefill_window"):
        args = {a.name: str(a.type) for a in getattr(torch.ops._C, name).default._schema.arguments}
        assert args["window"] == "Optional[int]" and args["sinks"] == "int", name
