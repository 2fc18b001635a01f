// Rotary positions for q and k, with the KV append folded in.
//
// A head's first rot_dim dims are rotated in pairs (x_a, x_b) by the angle t = position * inv_freq[i] of pair i:
//     x_a' = f (x_a cos t - x_b sin t),   x_b' = f (x_b cos t + x_a sin t)
// with (a, b) = (i, i + rot_dim / 2) (half layout) or (2i, 2i + 1) (interleaved); the dims behind rot_dim stay as they
// are.  f is the factor by which context scaling methods enlarge q and k.
//
// There is no table of cosines: a position of a million times a frequency near 1 has lost a tenth of a radian in 32
// bits, so the turns position * inv_freq / 2 pi are taken in 64 bits, whole turns are dropped there, and sincospif gets
// the remainder in [-1/2, 1/2] turns, exact to half a unit of 32 bits.  A warp computes the rot_dim / 2 angles of its
// token once, two per lane, and hands them round with shuffles.  The rotation runs in 32 bits and rounds once to bf16.
//
// Bound by HBM: (Hq + 2 Hkv) rows of 256 bytes read, as many written.  Eight lanes per head, two 16-byte chunks of
// eight dims per lane, chosen so that a pair never leaves its lane: in the half layout lane s < rot_dim / 16 owns chunks
// s and s + rot_dim / 16, the other lanes two adjacent chunks of the untouched tail; in the interleaved layout lane s owns
// the adjacent chunks 2s and 2s + 1, which it moves with 32-byte loads and stores where the addresses allow.
// Measured (32q/8kv heads): 32768 tokens half layout 125-128 us (6.3-6.4 TB/s of the bytes that have to move, 0.97 of the copy
// peak); 5001 tokens of 64q/8kv heads interleaved, half a head rotated: see kRotQuads.
#include "common.cuh"

namespace ib {

struct RotaryArgs {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;          // null: q and k are rotated, nothing is appended
    __nv_bfloat16* q_out;
    __nv_bfloat16* k_out;            // rotated k rows, or the K pool when appending
    __nv_bfloat16* v_out;            // the V pool when appending
    int64_t q_pitch, k_pitch, v_pitch, q_out_pitch, k_out_pitch;   // elements between token rows
    const int64_t* positions;
    const double* inv_freq;          // [rot_dim / 2] radians per position
    const int32_t* slot_mapping;     // null without append
    int64_t n_tokens;
    int64_t num_slots;
    int n_q_heads;
    int n_kv_heads;
    int rot_chunks;                  // rot_dim / 16: chunks of eight pairs
    float factor;
};

// Heads of one work item: four per load instruction, six or four instructions.  Swept, us at 6 / 5 / 4 / 3: half layout,
// 32768 tokens of 48 heads 128 / 139 / 137 / 132; interleaved, 5001 tokens of 80 heads 40.2 / 38.9 / 35.9 / 38.2 (four loads
// leave room for three blocks per SM; swept with 16-byte accesses, in a graph; the 32-byte ones take 35.3-35.6 there).
template <bool INTERLEAVED>
constexpr int kRotQuads = INTERLEAVED ? 4 : 6;

template <bool INTERLEAVED, bool WIDE>
__global__ void __launch_bounds__(256, INTERLEAVED ? 3 : 2) rotary_append_kernel(RotaryArgs a) {
    constexpr int Q = kRotQuads<INTERLEAVED>;
    const bool append = a.v != nullptr;
    const int qk_heads = a.n_q_heads + a.n_kv_heads;
    const int heads = append ? qk_heads + a.n_kv_heads : qk_heads;
    const int batches = (heads + 4 * Q - 1) / (4 * Q);
    const int lane = threadIdx.x & 31, sub = lane & 7, grp = lane >> 3;
    const int m = a.rot_chunks;
    // the two chunks of eight dims of this lane, and whether they are rotated
    const bool rotated = sub < m;
    const int c0 = !INTERLEAVED && rotated ? sub : 2 * sub;
    const int c1 = !INTERLEAVED && rotated ? sub + m : 2 * sub + 1;
    const int64_t n_items = a.n_tokens * batches;
    const int64_t n_warps = (int64_t(gridDim.x) * blockDim.x) >> 5;
    // turns per position of pairs `lane` and `lane + 32`
    const double turns0 = lane < 8 * m ? a.inv_freq[lane] * 0.15915494309189535 : 0.0;
    const double turns1 = lane + 32 < 8 * m ? a.inv_freq[lane + 32] * 0.15915494309189535 : 0.0;
    for (int64_t item = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; item < n_items; item += n_warps) {
        const int64_t tok = item / batches;
        const int h0 = int(item - tok * batches) * 4 * Q;
        const int64_t slot = append ? int64_t(a.slot_mapping[tok]) : tok;
        const bool slot_ok = !append || (slot >= 0 && slot < a.num_slots);     // false: padding row of a captured batch
        const double pos = double(a.positions[tok]);
        // every load of the item before any arithmetic
        uint4 x[Q], y[Q];
        int h[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) {
            h[j] = h0 + 4 * j + grp;
            const int hh = min(h[j], heads - 1);                   // a lane group past the last head re-reads it and stores nothing
            const __nv_bfloat16* src = hh < a.n_q_heads ? a.q + tok * a.q_pitch + hh * kHeadDim
                                     : hh < qk_heads    ? a.k + tok * a.k_pitch + (hh - a.n_q_heads) * kHeadDim
                                                        : a.v + tok * a.v_pitch + (hh - qk_heads) * kHeadDim;
            if constexpr (INTERLEAVED) {
                const Bytes32 w = load32<WIDE>(src + 8 * c0);
                x[j] = w.lo;
                y[j] = w.hi;
            } else {
                x[j] = *reinterpret_cast<const uint4*>(src + 8 * c0);
                y[j] = *reinterpret_cast<const uint4*>(src + 8 * c1);
            }
        }
        // the token's angles: pairs lane and lane + 32; this lane's eight pairs are 8 sub .. 8 sub + 7 in either layout
        float cs[8], sn[8];
        {
            const double t0 = pos * turns0, t1 = pos * turns1;
            float s0, co0, s1, co1;
            sincospif(2.f * float(t0 - rint(t0)), &s0, &co0);
            sincospif(2.f * float(t1 - rint(t1)), &s1, &co1);
            s0 *= a.factor; co0 *= a.factor; s1 *= a.factor; co1 *= a.factor;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pair = 8 * sub + i;
                const float clo = __shfl_sync(0xffffffffu, co0, pair & 31), chi = __shfl_sync(0xffffffffu, co1, pair & 31);
                const float slo = __shfl_sync(0xffffffffu, s0, pair & 31), shi = __shfl_sync(0xffffffffu, s1, pair & 31);
                cs[i] = pair >= 32 ? chi : clo;
                sn[i] = pair >= 32 ? shi : slo;
            }
        }
#pragma unroll
        for (int j = 0; j < Q; ++j) {
            if (h[j] >= heads) continue;                           // uniform over the 8 lanes of a group
            if (h[j] < qk_heads && rotated) {
                uint32_t* xr = reinterpret_cast<uint32_t*>(&x[j]);
                uint32_t* yr = reinterpret_cast<uint32_t*>(&y[j]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&xr[i]));
                    const float2 w = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&yr[i]));
                    if (INTERLEAVED) {
                        xr[i] = pack_bf16(u.x * cs[i] - u.y * sn[i], u.y * cs[i] + u.x * sn[i]);
                        yr[i] = pack_bf16(w.x * cs[4 + i] - w.y * sn[4 + i], w.y * cs[4 + i] + w.x * sn[4 + i]);
                    } else {
                        xr[i] = pack_bf16(u.x * cs[2 * i] - w.x * sn[2 * i], u.y * cs[2 * i + 1] - w.y * sn[2 * i + 1]);
                        yr[i] = pack_bf16(w.x * cs[2 * i] + u.x * sn[2 * i], w.y * cs[2 * i + 1] + u.y * sn[2 * i + 1]);
                    }
                }
            }
            __nv_bfloat16* dst;
            if (h[j] < a.n_q_heads) {
                dst = a.q_out + tok * a.q_out_pitch + h[j] * kHeadDim;
            } else {
                if (!slot_ok) continue;
                dst = h[j] < qk_heads ? a.k_out + slot * a.k_out_pitch + (h[j] - a.n_q_heads) * kHeadDim
                                      : a.v_out + slot * a.k_out_pitch + (h[j] - qk_heads) * kHeadDim;
            }
            if constexpr (INTERLEAVED) {
                store32<WIDE>(dst + 8 * c0, Bytes32{x[j], y[j]});
            } else {
                *reinterpret_cast<uint4*>(dst + 8 * c0) = x[j];
                *reinterpret_cast<uint4*>(dst + 8 * c1) = y[j];
            }
        }
    }
}

static int rotary(RotaryArgs& a, const void* q_out, int64_t q_out_stride, const void* q, const void* k, int64_t q_stride,
                  int64_t k_stride, const int64_t* positions, const double* inv_freq, int rot_dim, int interleaved, float factor,
                  int64_t n_tokens, int n_q_heads, int n_kv_heads, int sm_count, cudaStream_t st) {
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.k = static_cast<const __nv_bfloat16*>(k);
    a.q_out = static_cast<__nv_bfloat16*>(const_cast<void*>(q_out));
    a.q_pitch = q_stride;
    a.k_pitch = k_stride;
    a.q_out_pitch = q_out_stride;
    a.positions = positions;
    a.inv_freq = inv_freq;
    a.n_tokens = n_tokens;
    a.n_q_heads = n_q_heads;
    a.n_kv_heads = n_kv_heads;
    a.rot_chunks = rot_dim / 16;
    a.factor = factor;
    const int heads = n_q_heads + (a.v ? 2 : 1) * n_kv_heads;
    const int per = 4 * (interleaved ? kRotQuads<true> : kRotQuads<false>);
    const int64_t items = n_tokens * ((heads + per - 1) / per);                            // one warp each
    int64_t blocks = (items + 7) / 8;
    const int64_t cap = int64_t(sm_count) * 16;                                            // grid-stride beyond that
    if (blocks > cap) blocks = cap;
    // 32-byte accesses of the interleaved layout: every row at a multiple of 32 bytes
    auto at32 = [](const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0 && stride % 16 == 0; };
    const bool wide = at32(a.q, a.q_pitch) && at32(a.k, a.k_pitch) && at32(a.v, a.v_pitch) && at32(a.q_out, a.q_out_pitch) &&
                      at32(a.k_out, a.k_out_pitch) && at32(a.v_out, a.k_out_pitch);
    if (!interleaved) rotary_append_kernel<false, false><<<unsigned(blocks), 256, 0, st>>>(a);
    else if (wide) rotary_append_kernel<true, true><<<unsigned(blocks), 256, 0, st>>>(a);
    else rotary_append_kernel<true, false><<<unsigned(blocks), 256, 0, st>>>(a);
    return check_launch();
}

static bool rotary_geometry_ok(int64_t n_tokens, int n_q_heads, int rot_dim) {
    return n_tokens >= 0 && n_q_heads > 0 && rot_dim >= 16 && rot_dim <= kHeadDim && rot_dim % 16 == 0;
}

}  // namespace ib

extern "C" {

int infer_rotary_append(const infer_kv_pool_t* pool, void* q_out, int64_t q_out_row_stride, const void* q, const void* k,
                        const void* v, int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride, const int64_t* positions,
                        const double* inv_freq, int rot_dim, int interleaved, float factor, const int32_t* slot_mapping,
                        int64_t n_tokens, int n_q_heads, void* stream_) {
    using namespace ib;
    if (!pool) return INFER_ERR_NULL;
    if (pool->dtype != INFER_KV_BF16) return INFER_ERR_DTYPE;
    if (!rotary_geometry_ok(n_tokens, n_q_heads, rot_dim)) return INFER_ERR_GEOMETRY;
    if (n_tokens == 0) return INFER_OK;
    if (!q_out || !q || !k || !v || !positions || !inv_freq || !slot_mapping) return INFER_ERR_NULL;
    const int64_t qrow = int64_t(n_q_heads) * kHeadDim, kvrow = int64_t(pool->n_kv_heads) * kHeadDim;
    if (q_row_stride < qrow || q_out_row_stride < qrow || k_row_stride < kvrow || v_row_stride < kvrow) return INFER_ERR_STRIDE;
    if (!aligned16(q_out) || !aligned16(q) || !aligned16(k) || !aligned16(v) || q_row_stride % 8 || q_out_row_stride % 8 ||
        k_row_stride % 8 || v_row_stride % 8)
        return INFER_ERR_ALIGN;
    RotaryArgs a{};
    a.v = static_cast<const __nv_bfloat16*>(v);
    a.v_pitch = v_row_stride;
    a.k_out = static_cast<__nv_bfloat16*>(pool->k_cache);
    a.v_out = static_cast<__nv_bfloat16*>(pool->v_cache);
    a.k_out_pitch = kvrow;
    a.slot_mapping = slot_mapping;
    a.num_slots = pool->num_slots;
    return rotary(a, q_out, q_out_row_stride, q, k, q_row_stride, k_row_stride, positions, inv_freq, rot_dim, interleaved, factor,
                  n_tokens, n_q_heads, pool->n_kv_heads, pool->sm_count, static_cast<cudaStream_t>(stream_));
}

int infer_rotary_embed(void* q_out, void* k_out, int64_t q_out_row_stride, int64_t k_out_row_stride, const void* q, const void* k,
                       int64_t q_row_stride, int64_t k_row_stride, const int64_t* positions, const double* inv_freq, int rot_dim,
                       int interleaved, float factor, int64_t n_tokens, int n_q_heads, int n_kv_heads, void* stream_) {
    using namespace ib;
    if (!rotary_geometry_ok(n_tokens, n_q_heads, rot_dim) || n_kv_heads <= 0) return INFER_ERR_GEOMETRY;
    if (n_tokens == 0) return INFER_OK;
    if (!q_out || !k_out || !q || !k || !positions || !inv_freq) return INFER_ERR_NULL;
    const int64_t qrow = int64_t(n_q_heads) * kHeadDim, kvrow = int64_t(n_kv_heads) * kHeadDim;
    if (q_row_stride < qrow || q_out_row_stride < qrow || k_row_stride < kvrow || k_out_row_stride < kvrow) return INFER_ERR_STRIDE;
    if (!aligned16(q_out) || !aligned16(k_out) || !aligned16(q) || !aligned16(k) || q_row_stride % 8 || q_out_row_stride % 8 ||
        k_row_stride % 8 || k_out_row_stride % 8)
        return INFER_ERR_ALIGN;
    int dev = 0, sm_count = 0;
    IB_CUDA(cudaGetDevice(&dev));
    IB_CUDA(cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev));
    RotaryArgs a{};
    a.k_out = static_cast<__nv_bfloat16*>(k_out);
    a.k_out_pitch = k_out_row_stride;
    return rotary(a, q_out, q_out_row_stride, q, k, q_row_stride, k_row_stride, positions, inv_freq, rot_dim, interleaved, factor,
                  n_tokens, n_q_heads, n_kv_heads, sm_count, static_cast<cudaStream_t>(stream_));
}

}  // extern "C"
