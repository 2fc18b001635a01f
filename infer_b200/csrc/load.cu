// Rows of the page pools read back as bf16: the inverse of the append kernels (append.cu).
//
//   out[i][h] = pool[slot_mapping[i]][h]                              bf16 pools: the bytes
//   out[i][h] = bf16(float(byte) * scale[slot / block_size][h])       e4m3 pools: the product is taken in 32 bits
//                                                                     and rounded once, to the type of the result
// A slot outside the pool (negative: the padding of a captured batch) gives a row of zeros.
//
// Bound by HBM: per row and head 128 elements read and 256 bytes written, for K and for V.  Eight lanes take one (row,
// head), sixteen elements per lane: 32-byte stores (and, for bf16, loads), which need the addresses at 32 bytes; two
// 16-byte ones otherwise.  32768 rows of 8 heads out of an e4m3 pool: 34.9 us with a cold L2, 5.77 TB/s of the bytes that
// have to move (32.8-34.6 in a graph); 40.5 us with 16-byte stores, 43 us with eight elements per lane and four rows of
// sixteen lanes each in flight.  Two to four units per lane gain nothing (34.6-35.6 us) and cost a small call a microsecond.
#include "common.cuh"

namespace ib {

struct LoadArgs {
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const float* k_scale;            // null for bf16 pools
    const float* v_scale;
    __nv_bfloat16* k_out;
    __nv_bfloat16* v_out;
    int64_t k_pitch, v_pitch;        // elements between output rows
    const int32_t* slot_mapping;
    int64_t n_units;                 // n_tokens * n_kv_heads
    int64_t num_slots;
    int n_kv_heads;
    int block_size;
};

// eight e4m3 bytes times a scale, rounded to bf16
__device__ __forceinline__ uint4 dequantise8(uint32_t a, uint32_t b, float scale) {
    uint32_t h[4];
    e4m3x4_to_f16x2x2(a, h[0], h[1]);
    e4m3x4_to_f16x2x2(b, h[2], h[3]);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        o[i] = pack_bf16(f.x * scale, f.y * scale);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <bool FP8, bool WIDE>
__global__ void __launch_bounds__(256) kv_load_kernel(LoadArgs a) {
    const int lane8 = threadIdx.x & 7;
    const int64_t u = int64_t(blockIdx.x) * 32 + (threadIdx.x >> 3);       // (row, head) of this group of lanes
    if (u >= a.n_units) return;
    const int64_t tok = a.n_units <= 0x7fffffff ? int64_t(uint32_t(u) / uint32_t(a.n_kv_heads)) : u / a.n_kv_heads;
    const int head = int(u - tok * a.n_kv_heads);
    const int64_t slot = a.slot_mapping[tok];
    Bytes32 k{}, v{};
    if (slot >= 0 && slot < a.num_slots) {
        const int64_t at = ((slot * a.n_kv_heads + head) * 8 + lane8) * 16;      // sixteen elements
        if constexpr (FP8) {
            const uint4 kr = __ldg(reinterpret_cast<const uint4*>(a.k_cache + at));
            const uint4 vr = __ldg(reinterpret_cast<const uint4*>(a.v_cache + at));
            const int64_t page = uint32_t(slot) / uint32_t(a.block_size);
            const float ks = __ldg(a.k_scale + page * a.n_kv_heads + head), vs = __ldg(a.v_scale + page * a.n_kv_heads + head);
            k.lo = dequantise8(kr.x, kr.y, ks);
            k.hi = dequantise8(kr.z, kr.w, ks);
            v.lo = dequantise8(vr.x, vr.y, vs);
            v.hi = dequantise8(vr.z, vr.w, vs);
        } else {
            k = load32<WIDE>(a.k_cache + at * 2);
            v = load32<WIDE>(a.v_cache + at * 2);
        }
    }
    store32<WIDE>(a.k_out + tok * a.k_pitch + head * kHeadDim + lane8 * 16, k);
    store32<WIDE>(a.v_out + tok * a.v_pitch + head * kHeadDim + lane8 * 16, v);
}

}  // namespace ib

extern "C" int infer_kv_load(const infer_kv_pool_t* pool, void* k_out, void* v_out, int64_t k_row_stride, int64_t v_row_stride,
                             const int32_t* slot_mapping, int64_t n_tokens, void* stream_) {
    using namespace ib;
    if (!pool) return INFER_ERR_NULL;
    if (n_tokens < 0) return INFER_ERR_GEOMETRY;
    if (n_tokens == 0) return INFER_OK;
    if (!k_out || !v_out || !slot_mapping) return INFER_ERR_NULL;
    const int64_t row = int64_t(pool->n_kv_heads) * kHeadDim;
    if (k_row_stride < row || v_row_stride < row) return INFER_ERR_STRIDE;
    if (!aligned16(k_out) || !aligned16(v_out) || k_row_stride % 8 || v_row_stride % 8) return INFER_ERR_ALIGN;
    LoadArgs a;
    a.k_cache = static_cast<const uint8_t*>(pool->k_cache);
    a.v_cache = static_cast<const uint8_t*>(pool->v_cache);
    a.k_scale = pool->k_scale;
    a.v_scale = pool->v_scale;
    a.k_out = static_cast<__nv_bfloat16*>(k_out);
    a.v_out = static_cast<__nv_bfloat16*>(v_out);
    a.k_pitch = k_row_stride;
    a.v_pitch = v_row_stride;
    a.slot_mapping = slot_mapping;
    a.n_units = n_tokens * pool->n_kv_heads;
    a.num_slots = pool->num_slots;
    a.n_kv_heads = pool->n_kv_heads;
    a.block_size = pool->block_size;
    const cudaStream_t st = static_cast<cudaStream_t>(stream_);
    const int64_t blocks = (a.n_units + 31) / 32;
    if (blocks > 0x7fffffff) return INFER_ERR_GEOMETRY;
    const bool fp8 = pool->dtype == INFER_KV_E4M3;
    auto at32 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; };
    const bool wide = at32(k_out) && at32(v_out) && k_row_stride % 16 == 0 && v_row_stride % 16 == 0 &&
                      (fp8 || (at32(pool->k_cache) && at32(pool->v_cache)));
    if (fp8 && wide) kv_load_kernel<true, true><<<unsigned(blocks), 256, 0, st>>>(a);
    else if (fp8) kv_load_kernel<true, false><<<unsigned(blocks), 256, 0, st>>>(a);
    else if (wide) kv_load_kernel<false, true><<<unsigned(blocks), 256, 0, st>>>(a);
    else kv_load_kernel<false, false><<<unsigned(blocks), 256, 0, st>>>(a);
    return check_launch();
}
