// Rows of the page pools read back as bf16: the inverse of the append kernels (append.cu).
//
//   out[i][h] = pool[slot_mapping[i]][h]                              bf16 pools: the bytes
//   out[i][h] = bf16(float(byte) * scale[slot / block_size][h])       e4m3 pools: the product is taken in 32 bits
//                                                                     and rounded once, to the type of the result
// A slot outside the pool (negative: the padding of a captured batch) gives a row of zeros.
//
// Bound by HBM: per row and head 128 elements read and 256 bytes written, for K and for V.  Sixteen lanes take one
// (row, head): eight elements per lane, so a store instruction of a warp covers two whole 256-byte rows and a load two
// whole 128-byte (e4m3) or 256-byte (bf16) ones.  A lane first looks up the slots and scales of kUnits units, then
// issues all 2 * kUnits row loads, then converts and stores.
#include <type_traits>

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

constexpr int kLoadUnits = 4;

// eight e4m3 bytes times a scale, rounded to bf16
__device__ __forceinline__ uint4 dequantise8(uint2 raw, float scale) {
    uint32_t h[4];
    e4m3x4_to_f16x2x2(raw.x, h[0], h[1]);
    e4m3x4_to_f16x2x2(raw.y, h[2], h[3]);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        o[i] = pack_bf16(f.x * scale, f.y * scale);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <bool FP8>
__global__ void __launch_bounds__(256) kv_load_kernel(LoadArgs a) {
    using Raw = typename std::conditional<FP8, uint2, uint4>::type;      // eight elements
    const int lane16 = threadIdx.x & 15;
    const int64_t group = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
    const int64_t groups = (int64_t(gridDim.x) * blockDim.x) >> 4;
    for (int64_t u0 = group; u0 < a.n_units; u0 += groups * kLoadUnits) {
        int64_t tok[kLoadUnits];
        int head[kLoadUnits];
        int64_t slot[kLoadUnits];
        Raw k[kLoadUnits], v[kLoadUnits];
        float ks[kLoadUnits], vs[kLoadUnits];
#pragma unroll
        for (int i = 0; i < kLoadUnits; ++i) {
            const int64_t u = u0 + i * groups;
            tok[i] = -1;
            slot[i] = -1;
            if (u < a.n_units) {
                tok[i] = a.n_units <= 0x7fffffff ? int64_t(uint32_t(u) / uint32_t(a.n_kv_heads)) : u / a.n_kv_heads;
                head[i] = int(u - tok[i] * a.n_kv_heads);
                const int64_t s = a.slot_mapping[tok[i]];
                if (s >= 0 && s < a.num_slots) slot[i] = s;
            }
        }
#pragma unroll
        for (int i = 0; i < kLoadUnits; ++i) {
            k[i] = Raw{};
            v[i] = Raw{};
            ks[i] = vs[i] = 0.f;
            if (slot[i] >= 0) {
                const int64_t row = slot[i] * a.n_kv_heads + head[i];
                k[i] = __ldg(reinterpret_cast<const Raw*>(a.k_cache) + row * 16 + lane16);
                v[i] = __ldg(reinterpret_cast<const Raw*>(a.v_cache) + row * 16 + lane16);
                if (FP8) {
                    const int64_t page = uint32_t(slot[i]) / uint32_t(a.block_size);
                    ks[i] = __ldg(a.k_scale + page * a.n_kv_heads + head[i]);
                    vs[i] = __ldg(a.v_scale + page * a.n_kv_heads + head[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kLoadUnits; ++i) {
            if (tok[i] < 0) continue;
            uint4 ko, vo;
            if constexpr (FP8) {
                ko = dequantise8(k[i], ks[i]);
                vo = dequantise8(v[i], vs[i]);
            } else {
                ko = k[i];
                vo = v[i];
            }
            *reinterpret_cast<uint4*>(a.k_out + tok[i] * a.k_pitch + head[i] * kHeadDim + lane16 * 8) = ko;
            *reinterpret_cast<uint4*>(a.v_out + tok[i] * a.v_pitch + head[i] * kHeadDim + lane16 * 8) = vo;
        }
    }
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
    int64_t blocks = (a.n_units + 15) / 16;                                  // sixteen units per block and turn
    const int64_t cap = int64_t(pool->sm_count) * 8;
    if (blocks > cap) blocks = cap;
    if (pool->dtype == INFER_KV_E4M3) kv_load_kernel<true><<<unsigned(blocks), 256, 0, st>>>(a);
    else kv_load_kernel<false><<<unsigned(blocks), 256, 0, st>>>(a);
    return check_launch();
}
