// Host side of the torch ops whose calls are short: argument checks, output tensors, stream and device, then the C ABI.
//
// A decode step's rotary_append or load_kvcache runs 2-4 us on the GPU; checked and launched from Python through ctypes the
// call cost the host 12-14 us (an output tensor 2.4, the current stream 3.1, a ctypes call with 18 arguments 1.6, every
// look at a tensor's type, shape or address 0.1), from here 5-6.  The module is bound to libinfer_b200.so by address, so
// that there is one library in the process, the one that infer_b200/_lib.py has loaded.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <climits>
#include <stdexcept>
#include <string>

#include "../../include/infer_b200.h"
#include "../../include/infer_b200_selftest.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using std::string;

// ------------------------------------------------------------------ the library's entry points
struct Library {
    decltype(&infer_kv_load) kv_load = nullptr;
    decltype(&infer_rotary_append) rotary_append = nullptr;
    decltype(&infer_rotary_embed) rotary_embed = nullptr;
    decltype(&infer_paged_decode_window) decode_window = nullptr;
    decltype(&infer_paged_decode_append_window) decode_append_window = nullptr;
    decltype(&infer_paged_prefill_window_columns) prefill_window = nullptr;
    decltype(&infer_selftest_paged_decode_window) decode_window_test = nullptr;
    decltype(&infer_selftest_paged_prefill_window) prefill_window_test = nullptr;
    decltype(&infer_strerror) strerror = nullptr;
    decltype(&infer_last_cuda_error) last_cuda_error = nullptr;
} lib;

// What the windowed calls are routed to while a test makes the kernels' waits run out (0, 0: the product entry points).
struct {
    uint32_t wait_limit = 0;
    int stall_producer = 0;
} wait_test;

template <class F>
void bind_one(F& f, const pybind11::dict& d, const char* name) {
    f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}

void bind_library(const pybind11::dict& d) {
    bind_one(lib.kv_load, d, "infer_kv_load");
    bind_one(lib.rotary_append, d, "infer_rotary_append");
    bind_one(lib.rotary_embed, d, "infer_rotary_embed");
    bind_one(lib.decode_window, d, "infer_paged_decode_window");
    bind_one(lib.decode_append_window, d, "infer_paged_decode_append_window");
    bind_one(lib.prefill_window, d, "infer_paged_prefill_window_columns");
    bind_one(lib.decode_window_test, d, "infer_selftest_paged_decode_window");
    bind_one(lib.prefill_window_test, d, "infer_selftest_paged_prefill_window");
    bind_one(lib.strerror, d, "infer_strerror");
    bind_one(lib.last_cuda_error, d, "infer_last_cuda_error");
}

// ------------------------------------------------------------------ checks
[[noreturn]] void refuse(const char* what, const string& why) { throw std::runtime_error(string(what) + ": " + why); }

void check(int rc, const char* what) {
    if (rc == INFER_OK) return;
    string why = lib.strerror(rc);
    if (rc == INFER_ERR_CUDA) why += " [cudaError " + std::to_string(lib.last_cuda_error()) + "]";
    refuse(what, why);
}

string shape_of(at::IntArrayRef s) {
    string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

bool on(const Tensor& t, int64_t device) { return t.is_cuda() && t.get_device() == device; }

// Rows [T, H, 128] of bf16 with contiguous heads on GPU `device`; returns their pitch in elements.
int64_t rows(const char* what, const char* name, const Tensor& x, int64_t device) {
    if (x.scalar_type() != at::kBFloat16 || x.dim() != 3 || x.size(2) != 128 || !on(x, device))
        refuse(what, string(name) + " must be a bf16 CUDA tensor [T, H, 128] on cuda:" + std::to_string(device));
    if (x.stride(2) != 1 || (x.size(1) > 1 && x.stride(1) != 128)) refuse(what, string(name) + " must have contiguous heads");
    return x.size(0) > 1 ? x.stride(0) : x.size(1) * 128;     // torch may report any stride for a dimension of one
}

void same_shape(const char* what, const char* name, const Tensor& x, at::IntArrayRef shape) {
    if (x.sizes() != shape) refuse(what, string(name) + " must be " + shape_of(shape));
}

template <class T>
const T* vector(const char* what, const char* name, const Tensor& x, int64_t n, at::ScalarType type, const char* type_name,
                int64_t device) {
    if (x.scalar_type() != type || !on(x, device) || x.numel() != n || !x.is_contiguous())
        refuse(what, string(name) + " must be a contiguous " + type_name + " tensor of " + std::to_string(n) + " values on cuda:" +
                         std::to_string(device));
    return static_cast<const T*>(x.data_ptr());
}

// A table of int32 rows of contiguous entries on the device, one per sequence; returns their pitch in entries.
int64_t table_rows(const char* what, const Tensor& t, int64_t batch, int64_t device) {
    if (t.scalar_type() != at::kInt || !on(t, device)) refuse(what, "block_table must be an int32 CUDA tensor on cuda:" + std::to_string(device));
    if (t.dim() != 2 || t.size(0) < batch || t.stride(1) != 1)
        refuse(what, "block_table must have a row of contiguous entries per sequence");
    return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1);     // torch may report any stride for a dimension of one
}

// window and sinks as the library takes them, 0 = no window
std::pair<int, int> window_of(const char* what, std::optional<int64_t> window, int64_t sinks) {
    if (!window) {
        if (sinks) refuse(what, "sinks without a window (every key is visible)");
        return {0, 0};
    }
    if (*window < 1 || sinks < 0) refuse(what, "window must be at least 1 and sinks at least 0");
    return {int(std::min<int64_t>(*window, INT_MAX)), int(std::min<int64_t>(sinks, INT_MAX))};
}

const infer_kv_pool_t* pool_at(uintptr_t handle) { return reinterpret_cast<const infer_kv_pool_t*>(handle); }

// The device made current for the call, and its current stream.
struct Launch {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit Launch(int64_t device)
        : guard(static_cast<c10::DeviceIndex>(device)),
          stream(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()) {}
};

Tensor new_rows(at::IntArrayRef shape, int64_t device) {
    return at::empty(shape, at::TensorOptions().dtype(at::kBFloat16).device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
}

// ------------------------------------------------------------------ the ops
std::pair<Tensor, Tensor> load_kvcache(uintptr_t pool, int64_t device, int64_t n_kv_heads, const Tensor& slot_mapping,
                                       const OptTensor& k_out, const OptTensor& v_out) {
    const char* what = "load_kvcache";
    const int64_t n = slot_mapping.numel();
    const auto* slots = vector<int32_t>(what, "slot_mapping", slot_mapping, n, at::kInt, "int32", device);
    const int64_t shape[3] = {n, n_kv_heads, 128};
    Tensor k = k_out ? *k_out : new_rows(shape, device), v = v_out ? *v_out : new_rows(shape, device);
    const int64_t k_pitch = rows(what, "k_out", k, device), v_pitch = rows(what, "v_out", v, device);
    same_shape(what, "k_out", k, shape);
    same_shape(what, "v_out", v, shape);
    Launch l(device);
    check(lib.kv_load(pool_at(pool), k.data_ptr(), v.data_ptr(), k_pitch, v_pitch, slots, n, l.stream), what);
    return {k, v};
}

struct Rotary {
    int64_t t, q_pitch, k_pitch, q_out_pitch;
    const int64_t* positions;
    const double* inv_freq;
    int rot_dim;
    Tensor q_out;
};

Rotary rotary_args(const char* what, const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq,
                   const OptTensor& q_out, int64_t device) {
    Rotary r;
    r.q_pitch = rows(what, "q", q, device);
    r.k_pitch = rows(what, "k", k, device);
    r.t = q.size(0);
    if (k.size(0) != r.t) refuse(what, "q and k must have the same number of rows");
    r.positions = vector<int64_t>(what, "positions", positions, r.t, at::kLong, "int64", device);
    r.inv_freq = vector<double>(what, "inv_freq", inv_freq, inv_freq.numel(), at::kDouble, "float64", device);
    r.rot_dim = int(std::min<int64_t>(2 * inv_freq.numel(), INT_MAX));
    r.q_out = q_out ? *q_out : new_rows(q.sizes(), device);
    r.q_out_pitch = rows(what, "q_out", r.q_out, device);
    same_shape(what, "q_out", r.q_out, q.sizes());
    return r;
}

Tensor rotary_append(uintptr_t pool, int64_t device, int64_t n_kv_heads, const Tensor& q, const Tensor& k, const Tensor& v,
                     const Tensor& positions, const Tensor& inv_freq, const Tensor& slot_mapping, bool interleaved, double factor,
                     const OptTensor& q_out) {
    const char* what = "rotary_append";
    const Rotary r = rotary_args(what, q, k, positions, inv_freq, q_out, device);
    const int64_t v_pitch = rows(what, "v", v, device);
    if (v.sizes() != k.sizes() || k.size(1) != n_kv_heads) refuse(what, "k and v must have q's rows and the pool's heads");
    const auto* slots = vector<int32_t>(what, "slot_mapping", slot_mapping, r.t, at::kInt, "int32", device);
    Launch l(device);
    check(lib.rotary_append(pool_at(pool), r.q_out.data_ptr(), r.q_out_pitch, q.data_ptr(), k.data_ptr(), v.data_ptr(), r.q_pitch,
                            r.k_pitch, v_pitch, r.positions, r.inv_freq, r.rot_dim, interleaved, float(factor), slots, r.t,
                            int(q.size(1)), l.stream),
          what);
    return r.q_out;
}

std::pair<Tensor, Tensor> rotary_embedding(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq,
                                           bool interleaved, double factor, const OptTensor& q_out, const OptTensor& k_out) {
    const char* what = "rotary_embedding";
    const int64_t device = q.is_cuda() ? q.get_device() : 0;
    const Rotary r = rotary_args(what, q, k, positions, inv_freq, q_out, device);
    Tensor ko = k_out ? *k_out : new_rows(k.sizes(), device);
    const int64_t k_out_pitch = rows(what, "k_out", ko, device);
    same_shape(what, "k_out", ko, k.sizes());
    Launch l(device);
    check(lib.rotary_embed(r.q_out.data_ptr(), ko.data_ptr(), r.q_out_pitch, k_out_pitch, q.data_ptr(), k.data_ptr(), r.q_pitch,
                           r.k_pitch, r.positions, r.inv_freq, r.rot_dim, interleaved, float(factor), r.t, int(q.size(1)),
                           int(k.size(1)), l.stream),
          what);
    return {r.q_out, ko};
}

// Decode over a window, with the step's rows appended when key and value are given.  q and out may be pinned host tensors.
Tensor decode_window(uintptr_t pool, int64_t device, int64_t n_kv_heads, const Tensor& q, const OptTensor& key, const OptTensor& value,
                     const Tensor& lens, const Tensor& table, double scale, const OptTensor& out, const Tensor& ws,
                     std::optional<int64_t> window, int64_t sinks) {
    const char* what = key ? "paged_attn_decode_append" : "paged_attn_decode";
    const auto [win, sink] = window_of(what, window, sinks);
    auto reachable = [&](const char* name, const Tensor& t) {
        if (!on(t, device) && !t.is_pinned()) refuse(what, string(name) + " must live on the pools' GPU or in pinned host memory");
    };
    if (q.scalar_type() != at::kBFloat16 || !q.is_contiguous() || q.dim() < 3 || q.size(-1) != 128 ||
        q.numel() != q.size(0) * q.size(-2) * 128)
        refuse(what, "q must be contiguous bf16 [B, Hq, 128]");
    reachable("q", q);
    const int64_t b = q.size(0);
    Tensor o = out ? *out : new_rows(q.sizes(), device);
    if (o.scalar_type() != at::kBFloat16 || !o.is_contiguous() || o.numel() != q.numel())
        refuse(what, "out must be contiguous bf16 in the shape of q");
    reachable("out", o);
    if (lens.scalar_type() != at::kInt || !on(lens, device) || lens.numel() != b || !lens.is_contiguous())
        refuse(what, "cache_seqlens must be an int32 CUDA tensor with a length per sequence on cuda:" + std::to_string(device));
    const int64_t table_pitch = table_rows(what, table, b, device);
    if (ws.scalar_type() != at::kByte || !on(ws, device) || !ws.is_contiguous()) refuse(what, "workspace must be a contiguous uint8 CUDA tensor");
    Launch l(device);
    const auto* cl = static_cast<const int32_t*>(lens.data_ptr());
    const auto* bt = static_cast<const int32_t*>(table.data_ptr());
    int64_t pitch[2] = {0, 0};
    if (key) {
        const Tensor* kv[2] = {&*key, &*value};
        for (int i = 0; i < 2; ++i) {
            const Tensor& t = *kv[i];
            const char* name = i ? "value" : "key";
            if (t.scalar_type() != at::kBFloat16 || t.dim() != 3 || t.size(0) != b || t.size(1) != n_kv_heads || t.size(2) != 128 ||
                t.stride(2) != 1 || (n_kv_heads > 1 && t.stride(1) != 128))
                refuse(what, string(name) + " must be bf16 [B, Hkv, 128] with contiguous heads");
            reachable(name, t);
            pitch[i] = b > 1 ? t.stride(0) : n_kv_heads * 128;
        }
    }
    if (wait_test.wait_limit || wait_test.stall_producer) {
        check(lib.decode_window_test(pool_at(pool), o.data_ptr(), q.data_ptr(), key ? key->data_ptr() : nullptr,
                                     key ? value->data_ptr() : nullptr, pitch[0], pitch[1], cl, bt, table_pitch, int(b), int(q.size(-2)),
                                     float(scale), win, sink, ws.data_ptr(), size_t(ws.numel()), l.stream, wait_test.wait_limit,
                                     wait_test.stall_producer),
              what);
    } else if (!key) {
        check(lib.decode_window(pool_at(pool), o.data_ptr(), q.data_ptr(), cl, bt, table_pitch, int(b), int(q.size(-2)), float(scale),
                                win, sink, ws.data_ptr(), size_t(ws.numel()), l.stream),
              what);
    } else {
        check(lib.decode_append_window(pool_at(pool), o.data_ptr(), q.data_ptr(), key->data_ptr(), value->data_ptr(), pitch[0], pitch[1],
                                       cl, bt, table_pitch, int(b), int(q.size(-2)), float(scale), win, sink, ws.data_ptr(),
                                       size_t(ws.numel()), l.stream),
              what);
    }
    return o.sizes() == q.sizes() ? o : o.view(q.sizes());
}

Tensor prefill_window(uintptr_t pool, int64_t device, const Tensor& q, const Tensor& cu_q, const Tensor& cu_k, int64_t max_q,
                      int64_t max_k, double scale, const Tensor& table, const OptTensor& out, std::optional<int64_t> window,
                      int64_t sinks) {
    const char* what = "paged_attn_prefill";
    const auto [win, sink] = window_of(what, window, sinks);
    if (q.scalar_type() != at::kBFloat16 || q.dim() != 3 || q.size(2) != 128 || !q.is_contiguous() || !on(q, device))
        refuse(what, "q must be contiguous bf16 [total_q, Hq, 128] on the pools' device, cuda:" + std::to_string(device));
    Tensor o = out ? *out : new_rows(q.sizes(), device);
    if (o.scalar_type() != at::kBFloat16 || o.sizes() != q.sizes() || !o.is_contiguous() || !on(o, device))
        refuse(what, "out must be contiguous bf16 in the shape of q and on its device");
    for (const Tensor* t : {&cu_q, &cu_k})
        if (t->scalar_type() != at::kInt || !on(*t, device))
            refuse(what, string(t == &cu_q ? "cu_seqlens_q" : "cu_seqlens_k") + " must be an int32 CUDA tensor on cuda:" + std::to_string(device));
    const int64_t batch = cu_q.numel() - 1;
    if (batch < 0 || cu_k.numel() != batch + 1 || !cu_q.is_contiguous() || !cu_k.is_contiguous())
        refuse(what, "cu_seqlens_q and cu_seqlens_k must be contiguous, batch + 1 values each");
    const int64_t table_pitch = table_rows(what, table, batch, device);
    if (batch > INT_MAX || max_q > INT_MAX || max_k > INT_MAX || max_q < 0 || max_k < 0) check(INFER_ERR_GEOMETRY, what);
    Launch l(device);
    const auto* cq = static_cast<const int32_t*>(cu_q.data_ptr());
    const auto* ck = static_cast<const int32_t*>(cu_k.data_ptr());
    const auto* bt = static_cast<const int32_t*>(table.data_ptr());
    const int hq = int(q.size(1));
    if (wait_test.wait_limit || wait_test.stall_producer)
        check(lib.prefill_window_test(pool_at(pool), o.data_ptr(), q.data_ptr(), q.size(0), cq, ck, bt, table_pitch, table.size(1),
                                      int(batch), int(max_q), int(max_k), hq, float(scale), win, sink, l.stream, wait_test.wait_limit,
                                      wait_test.stall_producer),
              what);
    else
        check(lib.prefill_window(pool_at(pool), o.data_ptr(), q.data_ptr(), q.size(0), cq, ck, bt, table_pitch, table.size(1), int(batch),
                                 int(max_q), int(max_k), hq, float(scale), win, sink, l.stream),
              what);
    return o;
}

}  // namespace

PYBIND11_MODULE(_host_ops, m) {
    m.def("bind_library", &bind_library);
    m.def("set_wait_test", [](uint32_t wait_limit, int stall_producer) {
        wait_test.wait_limit = wait_limit;
        wait_test.stall_producer = stall_producer;
    });
    m.def("load_kvcache", &load_kvcache);
    m.def("rotary_append", &rotary_append);
    m.def("rotary_embedding", &rotary_embedding);
    m.def("decode_window", &decode_window);
    m.def("prefill_window", &prefill_window);
}
