"""What a pool handle refuses before any library or CUDA call, on tensors that only look like CUDA ones."""
import pytest
import torch

from infer_b200 import ops


class Fake:
    """Shape, type, strides and device of a tensor, without its memory."""

    def __init__(self, shape, dtype, device="cuda:0"):
        self.like, self.device = torch.empty(shape, dtype=dtype, device="meta"), torch.device(device)
        self.shape, self.dtype, self.is_cuda = self.like.shape, dtype, self.device.type == "cuda"

    def dim(self):
        return self.like.dim()

    def is_contiguous(self):
        return self.like.is_contiguous()


@pytest.fixture
def no_library(monkeypatch):
    def load():
        raise AssertionError("the checks come before the library")
    monkeypatch.setattr(ops._lib, "load", load)


def test_pools_and_scales_live_on_one_gpu(no_library):
    k = Fake((2, 256, 4, 128), torch.uint8)
    one = Fake((2, 4), torch.float32)
    with pytest.raises(AssertionError):                                   # these are fine
        ops.KVPool(k, k, one, one)
    for other in ("cpu", "cuda:1"):
        elsewhere = Fake((2, 4), torch.float32, other)
        for scales in ((elsewhere, one), (one, elsewhere)):
            with pytest.raises(ValueError, match="GPU"):
                ops.KVPool(k, k, *scales)
    with pytest.raises(ValueError, match="same GPU"):
        ops.KVPool(k, Fake((2, 256, 4, 128), torch.uint8, "cuda:1"), one, one)
    b = Fake((2, 256, 4, 128), torch.bfloat16)
    with pytest.raises(ValueError, match="same GPU"):
        ops.KVPool(b, Fake((2, 256, 4, 128), torch.bfloat16, "cuda:1"))
