// Paged prefill attention with a sliding window and sinks over bf16 pools, and with or without them over e4m3 pools, on
// the 5th-generation tensor cores.
//
// Query i of a sequence (its position in the sequence) sees key j when j <= i and (i - j < window or j < sinks).
//     out_i = sum_j softmax_j(scale * q_i . k_j) v_j,    k_j = byte * k_scale[page(j), head] in an e4m3 pool, v_j likewise.
//
// The pipeline is that of prefill_tc.cu (two query tiles of 128 rows per CTA that share every 128-key tile, S and O in
// tensor memory, P written back to tensor memory, one softmax warpgroup per query tile with a row per thread, a lazy
// reference maximum).  What differs:
//
// Rows.  A query tile holds the query heads of ONE kv head over 128 / group consecutive tokens (row = token * group +
//   head), for any group size, loaded with one TMA box per half.  A chunk of 45 tokens with four heads per kv head fills
//   1.4 tiles instead of four a third full, and a tile spans few positions, so that a window cuts its key range close.
// Keys.  A CTA walks the tiles that hold a key visible to any of its rows: those of the sinks, then those from the start
//   of its first row's window on.  Block-table entries of other pages are never read.  V rows that no row of the CTA sees
//   are cleared before the tensor core reads them: P is 0 there, but 0 times a stale NaN is not.  bf16: up to 64 sinks go into
//   the rows of the window's first tile that lie in front of the window, where there are enough of them, instead of a tile of
//   their own (16 sequences of 2048 rows, a window of 200 and 20 sinks 173 -> 146 us, of 1024 and four 3-8 %); an e4m3
//   tile has one scale.
// Many CTAs.  A CTA that is done takes over one that has not been launched yet (clusterlaunchcontrol): barriers, tensor
//   memory and roles stay, and the Q and first K tiles of the next row block are loaded (and converted) while the softmax
//   warps finish the current one.  Launched one by one, a CTA cost about 6 us beyond its tiles, a third of the time of a
//   window of 1024 keys.
// Few rows.  When the (row block, kv head, sequence) triples do not fill the GPU, the key tiles of a row block are split over
//   the CTAs of a cluster (2 to 16), which join their parts through distributed shared memory: maxima and sums first, then
//   every CTA scales its accumulator and leaves it in shared memory, and the rows are summed in turn.  No scratch in global
//   memory, no second kernel.
// e4m3.  S = Q K^T runs on the raw bytes of K (kind::f8f6f4, no conversion): a bf16 value has 8 significant bits, so it is
//   the exact sum of two e4m3 values, its rounding to 4 bits and the rest.  The softmax warps split Q once per row block,
//   each row scaled by a power of two that puts its largest value into [2^7, 2^8); values 2^-10 below that lose bits of the
//   second part, an error of 2^-16 of the row's largest.  Two e4m3 products take the tensor core as long as one bf16
//   product.  P has to keep more bits than that, so V becomes f16: TMA brings its bytes (half of bf16's traffic) into two
//   staging slots and a fourth warpgroup turns them into operand tiles (e4m3 -> f16 is exact).  When K was converted as well the
//   kernel was 1.2-1.5 times slower than on a bf16 cache: the S products alone read shared memory at its full rate (128
//   bytes a clock), and every converted tile moves another 48 KiB through it.
//   The K scale of a tile's page and the row's power of two go into the factor of the softmax exponent.  The V scale goes
//   into P: P = 2^(x - m) * 2^bias * v_scale / v_ref, where v_ref is the largest V scale met so far within a factor of 8;
//   the row sum takes it out again with one multiplication per tile, the output multiplies by v_ref.  P in f16 then lies
//   below 2^(6 + 6 + 3) and keeps 11 bits down to 2^-20 of the row's maximum, where bf16 would keep 8.  A page whose V scale
//   is 2^-20 of v_ref or less loses bits of its values, which is an error of 2^-33 v_ref.
//
// Every wait is bounded; one that runs out raises the abort flag, every role drains to the common epilogue, tensor memory
// is freed and the status word of the prefill kernels is set.
#include <algorithm>
#include <atomic>
#include <mutex>

#include "prefill.cuh"
#include "tcgen05.cuh"

namespace ib {

constexpr int kPwRows = 128;                  // rows per query tile (= TMEM lanes)
constexpr int kPwKeys = 128;                  // keys per K/V tile
constexpr int kPwHalf = 128 * 128;            // bytes of one [128 rows][64 elems] swizzled sub-tile
constexpr int kPwTile = 2 * kPwHalf;          // 32 KiB: one Q, K or V tile of 16-bit elements
constexpr int kPwRaw = 128 * 128;             // 16 KiB: one K or V tile of e4m3 bytes
constexpr int kPwRing = 8;                    // entries of the tile ring: one lives from its K's load to its P V product, 7 tiles at most
// A tile's entry: whether some row of the CTA sees only part of it (2: and its first rows are the sinks), its first key; e4m3: k
// scale, what O is multiplied by in front of this tile (1 as a rule), what the V scale adds to the exponents of P, what takes it
// out of a row sum again, the V scale that O is expressed in from there on; the rows that some query sees, [0, sink_end) and
// [begin, end).
enum PwTileEntry { PT_CUT, PT_KEY0, PT_K_SCALE, PT_O_FACTOR, PT_UP, PT_DOWN, PT_V_REF, PT_SINK_END = 8, PT_BEGIN, PT_END, PT_INTS = 16 };
// a row block's entry in the ring of two: number of key tiles (-1: no more row blocks), whether the second query tile has
// rows, first row of q, rows and first key position of the sequence, first token of the block, kv head, part, windowed
enum PwItemEntry { PI_TILES, PI_TWO, PI_Q0, PI_LQ, PI_SHIFT, PI_TOK0, PI_KVH, PI_SPLIT, PI_WINDOWED, PI_INTS = 16 };
// tensor memory columns: S (shared by the two tiles) at 0, P of tile i at 128 + 64 i, O of tile i at 256 + 128 i
constexpr uint32_t kPwTmemP = 128, kPwTmemO = 256;
constexpr int kPwSoftmaxWarps = 8;
constexpr int kPwProducer = 8, kPwIssueS = 9, kPwIssuePV = 10;   // warp roles; 0-7 softmax, 11 idle, 12-15 converters (e4m3)

template <bool FP8>
struct PwCfg {
    static constexpr int k_stages = FP8 ? 2 : 3, v_stages = FP8 ? 3 : 2, raw_slots = FP8 ? 2 : 0;
    static constexpr int v_loads = FP8 ? raw_slots : v_stages;        // V tiles that TMA can have under way
    static constexpr int k_bytes = FP8 ? kPwRaw : kPwTile;            // of a stage
    static constexpr int threads = (kPwSoftmaxWarps + (FP8 ? 8 : 4)) * 32;
    static constexpr int q = 0;
    static constexpr int k = q + 2 * kPwTile;
    static constexpr int v = k + k_stages * k_bytes;
    static constexpr int raw = v + v_stages * kPwTile;
    static constexpr int bars = raw + raw_slots * kPwRaw;
    static constexpr int n_bars = 36;
    static constexpr int misc = bars + n_bars * 8;                    // tmem base, abort flag
    static constexpr int claim = misc + 16;                           // answer to a request for another row block
    static constexpr int ring = claim + 16;                           // [kPwRing][PT_INTS]
    static constexpr int items = ring + kPwRing * PT_INTS * 4;        // [2][PI_INTS]
    static constexpr int total = items + 2 * PI_INTS * 4;
    // the probabilities' exponent: how far the reference maximum may lag, and what is added to it
    static constexpr float lazy = FP8 ? 6.f : 8.f, bias = FP8 ? 6.f : 0.f;
};

enum PwBar { PW_Q_FULL = 0, PW_K_FULL = 1, PW_K_EMPTY = 5, PW_V_FULL = 9, PW_V_EMPTY = 12, PW_S_FULL = 15, PW_P_FULL = 17,
             PW_PV_DONE = 19, PW_DRAIN = 21, PW_S_FREE = 23, PW_RAW_FULL = 24, PW_RAW_EMPTY = 26, PW_Q_READY = 28, PW_Q_EMPTY = 30,
             PW_ITEM_FULL = 31, PW_ITEM_EMPTY = 33, PW_CLAIM = 35 };

// Asks for a thread block of this launch that has not started yet; the answer (16 bytes) arrives on the barrier.
__device__ __forceinline__ void claim_request(uint32_t answer, uint32_t bar) {
    mbar_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(answer), "r"(bar) : "memory");
}
// The answer: true and the block's indices, or false when every block has started.
__device__ __forceinline__ bool claim_result(uint32_t answer, int& x, int& y, int& z) {
    const uint4 w = ld_shared_v4(answer);
    const uint64_t lo = uint64_t(w.x) | uint64_t(w.y) << 32, hi = uint64_t(w.z) | uint64_t(w.w) << 32;
    uint32_t got, cx = 0, cy = 0, cz = 0;
    asm volatile(
        "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
        "mov.b128 r, {%4, %5};\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, r;\n\t}"
        : "=&r"(got), "=&r"(cx), "=&r"(cy), "=&r"(cz)
        : "l"(lo), "l"(hi)
        : "memory");
    x = int(cx);
    y = int(cy);
    z = int(cz);
    return got != 0;
}

struct PwParams {
    __nv_bfloat16* out;
    const int32_t* cu_q;
    const int32_t* cu_k;
    const int32_t* block_tables;
    int64_t bt_stride;       // entries from one row of the table to the next ...
    int64_t bt_columns;      // ... of which these are the table's own; none behind them is read
    const float* k_scale;
    const float* v_scale;
    int n_q_heads, n_kv_heads, group;
    int tokens;              // tokens per query tile: 128 / group
    int block_size, num_blocks;
    int window, sinks;       // window: 0x7fffffff = none
    float scale_log2;
    int splits;              // CTAs (of one cluster) that share the key tiles of a row block
    int out_at32;            // out is a multiple of 32
    int* status;             // may be null
    uint32_t wait_limit;
    int stall_producer;
};

// Boxes of 16, 32 and 64 token rows.
constexpr int kPwParts = 3;
template <bool FP8>
struct PwParts {
    CUtensorMap k[kPwParts], v[kPwParts];
};
template <>
struct PwParts<true> {};         // an e4m3 tile has one scale
__device__ __forceinline__ const CUtensorMap* part_of(const PwParts<false>& p, bool v) { return v ? p.v : p.k; }
__device__ __forceinline__ const CUtensorMap* part_of(const PwParts<true>&, bool) { return nullptr; }

// tc_wait for warps that wait most of the time and can be late: they sleep between looks, since their polling takes issue slots
// from the softmax warps (the converters polling like the others: 507 us, sleeping: 495 us for 148 x 8 row blocks).
__device__ __forceinline__ bool tc_wait_idle(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        __nanosleep(100);
    }
    *abort_flag = 1;
    return false;
}

// All threads of all CTAs of the cluster.  (No bound on the wait: every thread comes here whatever happened before, since the
// waits in front of it are bounded, and the CTAs of a cluster are resident together.)
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The place in the shared memory of CTA `rank` of the cluster that corresponds to `addr` in this one's.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// Row t of a Q tile, 128 bf16 in two halves of 64 dims, becomes two rows of 128 e4m3 values in the same place whose sum it is
// up to a power of two, which is returned (NaN for a row with a value that is not finite): the largest value goes into
// [2^7, 2^8), that of a row below 2^-119 less far up, by 2^126.  (The power in two factors would lift those as well: 74.6 -> 79.1
// us for a call of few key tiles a row block, since nothing runs beside the split.)  Chunk x (of 16) holds eight bf16; result c
// (of 8) is the first parts of chunks 2c and 2c + 1, stored over chunk c, and their second parts, stored over chunk 8 + c.  The
// eight rows of a phase have a chunk at eight different banks.
// The split is arithmetic on bf16 bits: y = q * 2^-e * 2^-120 has the exponents of e4m3 (subnormal ones too), so the first part
// is y cut to three bits of mantissa, the second the difference, and the byte of either its sign and bits 10 .. 4.
__device__ __forceinline__ float split_q_row(uint32_t tile, int t) {
    auto chunk = [&](int x) { return tile + (x >> 3) * kPwHalf + swz128(t, x & 7); };
    uint4 w[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) w[x] = ld_shared_v4(chunk(x));
    __nv_bfloat162 top2[4];                                // largest magnitudes, NaN if there is one
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const uint32_t v[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v[k]));
            top2[k] = x == 0 ? m : __hmax2_nan(top2[k], m);
        }
    }
    const __nv_bfloat162 all = __hmax2_nan(__hmax2_nan(top2[0], top2[1]), __hmax2_nan(top2[2], top2[3]));
    const uint32_t top = __bfloat16_as_ushort(__hmax_nan(__low2bfloat16(all), __high2bfloat16(all))) & 0x7fffu;
    const int e = top == 0 ? 0 : max(int(top >> 7) - 127 - 7, -126);
    const uint32_t down = uint32_t(127 - e) << 7 | uint32_t(127 - e) << 23, tiny = 0x03800380u;      // 2^-e and 2^-120, twice
    auto bytes = [](uint32_t y0, uint32_t y1) {            // e4m3 of four bf16 scaled by 2^-120
        const uint32_t b0 = (y0 & 0x80008000u) | ((y0 << 4) & 0x7fff7fffu);
        const uint32_t b1 = (y1 & 0x80008000u) | ((y1 << 4) & 0x7fff7fffu);
        return __byte_perm(b0, b1, 0x7531);
    };
    auto as2 = [](const uint32_t& v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
    auto bits = [](const __nv_bfloat162& v) { return *reinterpret_cast<const uint32_t*>(&v); };
    auto split8 = [&](const uint4& q, uint32_t& h0, uint32_t& h1, uint32_t& l0, uint32_t& l1) {
        const uint32_t v[4] = {q.x, q.y, q.z, q.w};
        uint32_t y[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            y[k] = bits(__hmul2_rn(__hmul2_rn(as2(v[k]), as2(down)), as2(tiny)));
            const uint32_t h = y[k] & 0xfff0fff0u;
            l[k] = bits(__hsub2_rn(as2(y[k]), as2(h)));
        }
        h0 = bytes(y[0], y[1]);
        h1 = bytes(y[2], y[3]);
        l0 = bytes(l[0], l[1]);
        l1 = bytes(l[2], l[3]);
    };
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        uint4 h, l;
        split8(w[2 * c], h.x, h.y, l.x, l.y);
        split8(w[2 * c + 1], h.z, h.w, l.z, l.w);
        st_shared_v4(chunk(c), h);
        st_shared_v4(chunk(8 + c), l);
    }
    return __uint_as_float(top < 255u << 7 ? uint32_t(127 + e) << 23 : 0x7fffffffu);
}

template <bool FP8>
__global__ void __launch_bounds__(PwCfg<FP8>::threads, 1) prefill_window_kernel(PwParams p, const __grid_constant__ CUtensorMap map_q,
                                                                                const __grid_constant__ CUtensorMap map_k,
                                                                                const __grid_constant__ CUtensorMap map_v,
                                                                                const __grid_constant__ PwParts<FP8> parts) {
    using C = PwCfg<FP8>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem);
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem + C::misc);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::misc + 4);
    volatile int* s_ring = reinterpret_cast<volatile int*>(smem + C::ring);
    volatile int* s_item = reinterpret_cast<volatile int*>(smem + C::items);
    auto bar = [&](int which, int idx = 0) { return base + uint32_t(C::bars) + uint32_t(which + idx) * 8; };

    // The roles of the third warpgroup sit in the first four hardware warps (see prefill_tc.cu), the converters in the last.
    const int hw = int(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int warp = hw < 4 ? hw + kPwSoftmaxWarps : hw < 12 ? hw - 4 : hw;

    // the producer's first look-ups, under the set-up below (thread 0 is the producer)
    int seq_q0 = 0, seq_q1 = 0, seq_k0 = 0, seq_k1 = 0;
    if (threadIdx.x == 0) {
        seq_q0 = p.cu_q[blockIdx.z];
        seq_q1 = p.cu_q[blockIdx.z + 1];
        seq_k0 = p.cu_k[blockIdx.z];
        seq_k1 = p.cu_k[blockIdx.z + 1];
        mbar_init(bar(PW_Q_FULL), 1);
        mbar_init(bar(PW_Q_READY, 0), 4);
        mbar_init(bar(PW_Q_READY, 1), 4);
        mbar_init(bar(PW_Q_EMPTY), 1);
        mbar_init(bar(PW_CLAIM), 1);
        for (int i = 0; i < C::k_stages; ++i) {
            mbar_init(bar(PW_K_FULL, i), 1);
            mbar_init(bar(PW_K_EMPTY, i), 1);
        }
        for (int i = 0; i < C::v_stages; ++i) {
            mbar_init(bar(PW_V_FULL, i), FP8 ? 4 : 1);
            mbar_init(bar(PW_V_EMPTY, i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(PW_S_FULL, i), 1);
            mbar_init(bar(PW_P_FULL, i), 128);
            mbar_init(bar(PW_PV_DONE, i), 1);
            mbar_init(bar(PW_DRAIN, i), 1);
            mbar_init(bar(PW_RAW_FULL, i), 1);
            mbar_init(bar(PW_RAW_EMPTY, i), 4);
            mbar_init(bar(PW_ITEM_FULL, i), 1);
            mbar_init(bar(PW_ITEM_EMPTY, i), kPwSoftmaxWarps + 2 + (FP8 ? 4 : 0));     // every warp that reads the entry
        }
        mbar_init(bar(PW_S_FREE), 128);                     // the warpgroup that copied the S buffer to registers
        *s_abort = 0;
        fence_mbar_init();
        fence_proxy_async();
    }
    if (warp == kPwIssueS) {
        // all 512 columns (one CTA per SM by shared-memory use)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(base + uint32_t(C::misc)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *s_tmem, 0);   // warp-uniform by construction
    bool ok = true;
    // Every role walks the row blocks that the producer publishes, with counters that run on from block to block (a
    // barrier's phase is the count of its uses).
    auto item_wait = [&](int item) -> const volatile int* {
        if (!tc_wait(bar(PW_ITEM_FULL, item & 1), (item >> 1) & 1, s_abort, p.wait_limit)) ok = false;
        return s_item + (item & 1) * PI_INTS;
    };
    auto item_done = [&](int item) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(PW_ITEM_EMPTY, item & 1));
    };

    // Register budget.  bf16: 384 threads x 168 at launch = 72 for the third warpgroup and 216 for the softmax ones.
    // e4m3: 512 x 128 = 56 for roles and converters, 200 for softmax.
    if (hw < 4) {
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;" ::: "memory");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
        if (warp == kPwProducer) {
            // ============================================================= row blocks and TMA
            if (lane == 0) {
                tma_prefetch_desc(&map_q);
                tma_prefetch_desc(&map_k);
                tma_prefetch_desc(&map_v);
                int item = 0, q_loads = 0, kc = 0, vc = 0;       // published row blocks, Q loads, K and V tiles
                uint32_t claims = 0;
                bool asked = false, stalled = false;             // asked: an answer is outstanding
                int bx = blockIdx.x, by = blockIdx.y, b = blockIdx.z;
                while (ok) {
                    const int kvh = by / p.splits, split = by - kvh * p.splits;
                    const int q0 = seq_q0, lq = seq_q1 - q0, lk = seq_k1 - seq_k0;
                    const int shift = lk - lq;                              // position of the first query row
                    const int tok0 = (int(gridDim.x) - 1 - bx) * 2 * p.tokens;     // longest rows first
                    auto ask = [&] {
                        fence_proxy_async();                                // the last answer has been read
                        claim_request(base + C::claim, bar(PW_CLAIM));
                        asked = true;
                    };
                    if (tok0 < lq) {
                        // key tiles: [0, n_sink) and [n_sink + skip, last]; list entry x is tile x below n_sink, x + skip behind
                        const int pos_lo = shift + tok0, pos_hi = shift + min(lq, tok0 + 2 * p.tokens) - 1;
                        const bool windowed = p.window < lk;
                        const int first_key = windowed ? max(pos_lo - p.window + 1, 0) : 0;
                        const int sinks = windowed ? min(p.sinks, lk) : 0;
                        int n_sink = (sinks + kPwKeys - 1) / kPwKeys;
                        int skip = max(first_key / kPwKeys - n_sink, 0);
                        if (skip == 0) n_sink = 0;
                        // sinks in the rows of the window's first tile that lie in front of the window: 0, or 16, 32, 64 rows
                        int sink_rows = 0;
                        if (!FP8 && sinks > 0 && sinks <= 64 && first_key >= kPwKeys) {
                            const int rows = sinks <= 16 ? 16 : sinks <= 32 ? 32 : 64;
                            if (rows <= first_key % kPwKeys) {
                                sink_rows = rows;
                                n_sink = 0;
                                skip = first_key / kPwKeys;
                            }
                        }
                        const int n_all = pos_hi < 0 ? 0 : pos_hi / kPwKeys + 1 - skip;
                        const int per_split = (n_all + p.splits - 1) / p.splits;
                        const int x0 = min(n_all, split * per_split), n = min(n_all, x0 + per_split) - x0;
                        auto tile_at = [&](int j) { return x0 + j < n_sink ? x0 + j : x0 + j + skip; };
                        const bool two = tok0 + p.tokens < lq;
                        if (n > 0 && !p.stall_producer) {
                            if (!tc_wait(bar(PW_Q_EMPTY), (q_loads & 1) ^ 1, s_abort, p.wait_limit)) { ok = false; break; }
                            const int n_q = two ? 2 : 1;
                            mbar_expect_tx(bar(PW_Q_FULL), n_q * 2 * p.tokens * p.group * 128);
                            for (int i = 0; i < n_q; ++i)
                                for (int half = 0; half < 2; ++half)
                                    tma_load_3d(base + C::q + i * kPwTile + half * kPwHalf, &map_q, bar(PW_Q_FULL), half * 64,
                                                kvh * p.group, q0 + tok0 + i * p.tokens);
                            ++q_loads;
                        }
                        if (!tc_wait(bar(PW_ITEM_EMPTY, item & 1), ((item >> 1) & 1) ^ 1, s_abort, p.wait_limit)) { ok = false; break; }
                        volatile int* e = s_item + (item & 1) * PI_INTS;
                        e[PI_TILES] = n;
                        e[PI_TWO] = two;
                        e[PI_Q0] = q0;
                        e[PI_LQ] = lq;
                        e[PI_SHIFT] = shift;
                        e[PI_TOK0] = tok0;
                        e[PI_KVH] = kvh;
                        e[PI_SPLIT] = split;
                        e[PI_WINDOWED] = windowed;
                        mbar_arrive(bar(PW_ITEM_FULL, item & 1));
                        ++item;
                        if (n > 0 && p.stall_producer) {                    // self-test: nothing is loaded, every wait runs out
                            stalled = true;
                            break;
                        }
                        if (n > 0) {
                            const int32_t* table = p.block_tables + int64_t(b) * p.bt_stride;
                            auto page_at = [&](int key) {                   // -1: outside of the table or of the pool
                                const int idx = key / p.block_size;
                                const int page = idx < p.bt_columns ? table[idx] : -1;
                                return page >= 0 && page < p.num_blocks ? page : -1;
                            };
                            auto page_of = [&](int j) { return page_at(j < n ? tile_at(j) * kPwKeys : 0); };
                            auto scale_of = [&](const float* scale, int page) {
                                return FP8 && page >= 0 ? scale[int64_t(page) * p.n_kv_heads + kvh] : 0.f;
                            };
                            // a page is looked up two tiles ahead and its scales one tile ahead: neither load is waited for
                            const int sink_page = sink_rows > 0 && x0 == 0 ? page_at(0) : -1;
                            int page = page_of(0), page_next = page_of(1), v_slot = 0;
                            float k_scale = scale_of(p.k_scale, page), v_scale = scale_of(p.v_scale, page);
                            constexpr int lag = FP8 ? 0 : 1;
                            // a tile of K or V; the window's first with the sinks in its first rows
                            auto load = [&](uint32_t dst, const CUtensorMap* map, const CUtensorMap* part, uint32_t full, int j, int from) {
                                if constexpr (FP8) {
                                    tma_load_3d(dst, map, full, 0, kvh, from);
                                } else if (x0 + j > 0 || sink_rows == 0) {
                                    tma_load_3d(dst, map, full, 0, kvh, from);
                                    tma_load_3d(dst + kPwHalf, map, full, 64, kvh, from);
                                } else {
                                    for (int half = 0; half < 2; ++half, dst += kPwHalf) {
                                        int i = sink_rows >> 5;             // 16, 32, 64: 0, 1, 2
                                        tma_load_3d(dst, &part[i], full, half * 64, kvh, sink_page >= 0 ? sink_page * p.block_size : -kPwKeys);
                                        for (int r = sink_rows; r < kPwKeys; r *= 2, ++i)
                                            tma_load_3d(dst + r * 128, &part[i], full, half * 64, kvh, from + r);
                                    }
                                }
                            };
                            float v_ref = 0.f;                              // e4m3: V scale that O is expressed in, 0 = none yet
                            // order K0, K1, V0, K2, V1, ...: K of the next tile is needed before V of this one.  e4m3: K0, V0, K1,
                            // V1, ...: V has the conversion in front of it
                            for (int j = 0; j < n + lag && ok; ++j) {
                                int slot = 0;
                                if (j < n) {
                                    const int tile = tile_at(j), key0 = tile * kPwKeys;
                                    // a page outside of the pool gives rows of zeros (TMA fills what lies outside of the tensor)
                                    slot = page >= 0 ? page * p.block_size + key0 % p.block_size : -kPwKeys;
                                    page = page_next;
                                    page_next = page_of(j + 2);
                                    const float k_scale_next = scale_of(p.k_scale, page), v_scale_next = scale_of(p.v_scale, page);
                                    const int s = kc % C::k_stages;
                                    if (!tc_wait(bar(PW_K_EMPTY, s), ((kc / C::k_stages) & 1) ^ 1, s_abort, p.wait_limit)) {
                                        ok = false;
                                        break;
                                    }
                                    // the copy first; the tile's entry is written while it runs and released by the arrival below,
                                    // without which the barrier cannot complete
                                    load(base + C::k + s * C::k_bytes, &map_k, part_of(parts, false), bar(PW_K_FULL, s), j, slot);
                                    volatile int* t = s_ring + (kc % kPwRing) * PT_INTS;
                                    t[PT_KEY0] = key0;
                                    t[PT_CUT] = key0 + kPwKeys - 1 > pos_lo || (windowed && key0 <= pos_hi - p.window && key0 + kPwKeys > sinks);
                                    t[PT_SINK_END] = sinks - key0;
                                    if (!FP8 && x0 + j == 0 && sink_rows > 0) {
                                        t[PT_CUT] = 2;
                                        t[PT_SINK_END] = sinks;
                                    }
                                    t[PT_BEGIN] = first_key - key0;
                                    t[PT_END] = pos_hi + 1 - key0;
                                    if constexpr (FP8) {
                                        float o_factor = 1.f, ratio = 1.f;
                                        if (j == 0) v_ref = 0.f;
                                        if (v_ref == 0.f) v_ref = v_scale;              // O is 0 so far
                                        else if (v_scale > 8.f * v_ref) {
                                            o_factor = v_ref / v_scale;
                                            v_ref = v_scale;
                                        }
                                        if (v_scale > 0.f) ratio = fmaxf(v_scale / v_ref, 1e-18f);
                                        else t[PT_SINK_END] = t[PT_BEGIN] = t[PT_END] = 0;     // a scale of 0: values of 0
                                        t[PT_K_SCALE] = __float_as_int(k_scale);
                                        t[PT_UP] = __float_as_int(C::bias + log2f(ratio));
                                        t[PT_DOWN] = __float_as_int(1.f / ratio);
                                        t[PT_O_FACTOR] = __float_as_int(o_factor);
                                        t[PT_V_REF] = __float_as_int(v_ref);
                                    }
                                    k_scale = k_scale_next;
                                    v_scale = v_scale_next;
                                    mbar_expect_tx(bar(PW_K_FULL, s), C::k_bytes);
                                    ++kc;
                                }
                                if (FP8) v_slot = slot;
                                if (j >= lag && ok) {
                                    const int s = vc % C::v_loads;
                                    if (tc_wait(bar(FP8 ? PW_RAW_EMPTY : PW_V_EMPTY, s), ((vc / C::v_loads) & 1) ^ 1, s_abort, p.wait_limit)) {
                                        const uint32_t full = bar(FP8 ? PW_RAW_FULL : PW_V_FULL, s);
                                        const uint32_t dst = FP8 ? base + C::raw + s * kPwRaw : base + C::v + s * kPwTile;
                                        mbar_expect_tx(full, C::k_bytes);
                                        load(dst, &map_v, part_of(parts, true), full, j - lag, v_slot);
                                        ++vc;
                                    } else ok = false;
                                }
                                v_slot = slot;
                                if (ok && !asked && p.splits == 1 && j + 2 >= n) ask();      // two tiles before the last load: the answer is there in time
                            }
                        }
                    }
                    if (!ok || p.splits > 1) break;                         // (a cluster stays with its one row block)
                    if (!asked) ask();
                    if (!tc_wait(bar(PW_CLAIM), claims & 1, s_abort, p.wait_limit)) { ok = false; break; }
                    ++claims;
                    asked = false;
                    if (!claim_result(base + C::claim, bx, by, b)) break;
                    seq_q0 = p.cu_q[b];
                    seq_q1 = p.cu_q[b + 1];
                    seq_k0 = p.cu_k[b];
                    seq_k1 = p.cu_k[b + 1];
                }
                if (ok && !stalled) {
                    if (tc_wait(bar(PW_ITEM_EMPTY, item & 1), ((item >> 1) & 1) ^ 1, s_abort, p.wait_limit)) {
                        s_item[(item & 1) * PI_INTS + PI_TILES] = -1;
                        mbar_arrive(bar(PW_ITEM_FULL, item & 1));
                    }
                }
                // never leave with a copy (or an answer) in flight: wait (bounded) for everything that was armed
                if (asked) mbar_wait(bar(PW_CLAIM), claims & 1, p.wait_limit);
                if (q_loads > 0) mbar_wait(bar(PW_Q_FULL), (q_loads - 1) & 1, p.wait_limit);
                for (int j = max(0, kc - C::k_stages); j < kc; ++j)
                    mbar_wait(bar(PW_K_FULL, j % C::k_stages), (j / C::k_stages) & 1, p.wait_limit);
                for (int j = max(0, vc - C::v_loads); j < vc; ++j)
                    mbar_wait(bar(FP8 ? PW_RAW_FULL : PW_V_FULL, j % C::v_loads), (j / C::v_loads) & 1, p.wait_limit);
            }
        } else if (warp == kPwIssueS) {
            // ============================================================= MMA issue: the S products
            // S_0(0) S_1(0) S_0(1) S_1(1) ...: each once the warpgroup of the previous one has copied the S buffer (S_FREE)
            constexpr uint32_t idesc_s = tc_idesc(false, FP8);
            const uint64_t q_desc0 = tc_desc(base + C::q, 16), k_desc0 = tc_desc(base + C::k, 16);
            int n_s = 0;                               // S products issued so far
            auto issue_s = [&](int i, int stage) {     // S = Q_i K^T  (K_FULL of that stage already awaited)
                if (n_s > 0 && !tc_wait(bar(PW_S_FREE), (n_s - 1) & 1, s_abort, p.wait_limit)) { ok = false; return; }
                ++n_s;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t qd = q_desc0 + uint64_t(i * (kPwTile >> 4));
                    const uint64_t kd = k_desc0 + uint64_t(stage * (C::k_bytes >> 4));
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t off = ((kk >> 2) * kPwHalf + (kk & 3) * 32) >> 4;
                        // e4m3: the two parts of Q lie where bf16 has the two halves of the dims, K is the same for both
                        if constexpr (FP8) tc_mma_f8(tmem, qd + off, kd + ((kk & 3) * 32 >> 4), idesc_s, kk > 0);
                        else tc_mma(tmem, qd + off, kd + off, idesc_s, kk > 0);
                    }
                    tc_commit(bar(PW_S_FULL, i));
                }
                __syncwarp();
            };
            int q_uses = 0, q1_uses = 0, ks = 0, kph = 0;                               // stage and phase of the next K tile
            for (int item = 0; ok; ++item) {
                const volatile int* e = item_wait(item);
                if (!ok) break;
                const int n = e[PI_TILES];
                const bool two = e[PI_TWO] != 0;
                if (n < 0) break;
                if (n > 0) {
                    if (!tc_wait(bar(FP8 ? PW_Q_READY : PW_Q_FULL), q_uses & 1, s_abort, p.wait_limit)) { ok = false; break; }
                    for (int j = 0; j < n && ok; ++j) {
                        if (!tc_wait(bar(PW_K_FULL, ks), kph, s_abort, p.wait_limit)) { ok = false; break; }
                        issue_s(0, ks);
                        if (FP8 && j == 0 && ok && two && !tc_wait(bar(PW_Q_READY, 1), q1_uses++ & 1, s_abort, p.wait_limit)) ok = false;
                        if (ok && two) issue_s(1, ks);
                        if (!ok) break;
                        if (elect_one()) {                                    // all S(j) are issued
                            tc_commit(bar(PW_K_EMPTY, ks));
                            if (j == n - 1) tc_commit(bar(PW_Q_EMPTY));
                        }
                        __syncwarp();
                        if (++ks == C::k_stages) { ks = 0; kph ^= 1; }
                    }
                    ++q_uses;
                }
                item_done(item);
            }
            // all tensor-core work issued by this warp must have retired before TMEM is freed
            if (elect_one()) tc_commit(bar(PW_DRAIN, 0));
            __syncwarp();
            mbar_wait(bar(PW_DRAIN, 0), 0, p.wait_limit);
        } else if (warp == kPwIssuePV) {
            // ============================================================= MMA issue: the P V products
            constexpr uint32_t idesc_pv = tc_idesc(true, FP8);
            const uint64_t v_desc0 = tc_desc(base + C::v, kPwHalf);
            int uses0 = 0, uses1 = 0;                        // products of either query tile so far
            auto issue_pv = [&](int i, int stage, int j, int& uses) {   // O_i += P_i V  (V_FULL of that stage already awaited)
                if (!tc_wait(bar(PW_P_FULL, i), uses & 1, s_abort, p.wait_limit)) { ok = false; return; }
                ++uses;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t vd = v_desc0 + uint64_t(stage * (kPwTile >> 4));
                    const uint32_t p_tmem = tmem + kPwTmemP + i * 64;
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)     // 16 keys: 8 packed columns of P, 16 rows of V
                        tc_mma_ts(tmem + kPwTmemO + i * 128, p_tmem + kk * 8, vd + uint32_t(kk * 16 * 128 >> 4), idesc_pv,
                                  (j > 0 || kk > 0) ? 1u : 0u);
                    tc_commit(bar(PW_PV_DONE, i));
                }
                __syncwarp();
            };
            int vc = 0, vs = 0, vph = 0;                     // V tiles so far, stage and phase of the next
            for (int item = 0; ok; ++item) {
                const volatile int* e = item_wait(item);
                if (!ok) break;
                const int n = e[PI_TILES];
                const bool two = e[PI_TWO] != 0;
                if (n < 0) break;
                for (int j = 0; j < n && ok; ++j, ++vc) {
                    if (!tc_wait(bar(PW_V_FULL, vs), vph, s_abort, p.wait_limit)) { ok = false; break; }
                    if constexpr (!FP8) {
                        // clear the rows that nobody sees (e4m3: the converters did)
                        const volatile int* t = s_ring + (vc % kPwRing) * PT_INTS;
                        const int sink_end = t[PT_SINK_END], begin = t[PT_BEGIN], end = t[PT_END];
                        if (end < kPwKeys || begin > max(sink_end, 0)) {
                            uint8_t* vt = smem + C::v + vs * kPwTile;
                            for (int x = lane; x < kPwKeys * 8; x += 32) {
                                const int r = x >> 3;
                                if (r < sink_end || (r >= begin && r < end)) continue;
                                *reinterpret_cast<uint4*>(vt + x * 16) = make_uint4(0, 0, 0, 0);
                                *reinterpret_cast<uint4*>(vt + kPwHalf + x * 16) = make_uint4(0, 0, 0, 0);
                            }
                            fence_proxy_async();
                            __syncwarp();
                        }
                    }
                    issue_pv(0, vs, j, uses0);
                    if (ok && two) issue_pv(1, vs, j, uses1);
                    if (!ok) break;
                    if (elect_one()) tc_commit(bar(PW_V_EMPTY, vs));              // all products with V_j are issued
                    __syncwarp();
                    if (++vs == C::v_stages) { vs = 0; vph ^= 1; }
                }
                item_done(item);
            }
            if (elect_one()) tc_commit(bar(PW_DRAIN, 1));
            __syncwarp();
            mbar_wait(bar(PW_DRAIN, 1), 0, p.wait_limit);
        }
    } else if (FP8 && hw >= 12) {
        // ================================================================= converters: V bytes -> f16
        if constexpr (FP8) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 56;" ::: "memory");
            const int t = int(threadIdx.x) - 12 * 32;                         // 0 .. 127
            // A thread's chunk of V: 16 dims (4 bytes of the lane number, low bits) of rows row0, row0 + 16, ...; the eight lanes
            // of a phase take four chunks of one half of the dims in rows m and m ^ 5, whose swizzles put them at eight
            // different banks both where they are read and where they are written.
            const int row0 = (t >> 6) * 8 + (((t >> 4) & 3) ^ (t & 4 ? 5 : 0)), c0 = ((t >> 3) & 1) * 4 + (t & 3);
            const uint32_t src0 = base + C::raw + swz128(row0, c0);
            const uint32_t dst0 = base + C::v + (c0 >> 2) * kPwHalf + swz128(row0, (c0 & 3) * 2);
            int vc = 0, vs = 0, vph = 0;
            for (int item = 0; ok; ++item) {
                const volatile int* ie = item_wait(item);
                if (!ok) break;
                const int n = ie[PI_TILES];
                if (n < 0) break;
                for (int j = 0; j < n && ok; ++j, ++vc) {
                    const int s = vc % C::raw_slots;
                    if (!tc_wait_idle(bar(PW_RAW_FULL, s), (vc / C::raw_slots) & 1, s_abort, p.wait_limit) ||
                        !tc_wait_idle(bar(PW_V_EMPTY, vs), vph ^ 1, s_abort, p.wait_limit)) {
                        ok = false;
                        break;
                    }
                    const volatile int* e = s_ring + (vc % kPwRing) * PT_INTS;
                    const int sink_end = e[PT_SINK_END], begin = e[PT_BEGIN], end = e[PT_END];
                    const uint32_t src = src0 + s * kPwRaw, dst = dst0 + vs * kPwTile;
                    const bool partly = end < kPwKeys || begin > max(sink_end, 0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint4 w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = ld_shared_v4(src + (h * 4 + i) * 16 * 128);
                        if (partly) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int r = row0 + (h * 4 + i) * 16;
                                if (!(r < sink_end || (r >= begin && r < end))) w[i] = make_uint4(0, 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 lo, hi;                                    // sixteen dims: two chunks of eight f16
                            e4m3x4_to_f16x2x2(w[i].x, lo.x, lo.y);
                            e4m3x4_to_f16x2x2(w[i].y, lo.z, lo.w);
                            e4m3x4_to_f16x2x2(w[i].z, hi.x, hi.y);
                            e4m3x4_to_f16x2x2(w[i].w, hi.z, hi.w);
                            st_shared_v4(dst + (h * 4 + i) * 16 * 128, lo);
                            st_shared_v4((dst ^ 16) + (h * 4 + i) * 16 * 128, hi);
                        }
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(PW_V_FULL, vs));
                        mbar_arrive(bar(PW_RAW_EMPTY, s));
                    }
                    if (++vs == C::v_stages) { vs = 0; vph ^= 1; }
                }
                item_done(item);
            }
        }
    } else {
        // ================================================================= softmax, one row per thread
        if constexpr (FP8) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;" ::: "memory");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;" ::: "memory");
        const int g = warp >> 2;                                   // query tile of this warpgroup
        const int r = (warp & 3) * 32 + lane;                      // row in the tile == TMEM lane
        const uint32_t lane_sel = uint32_t((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lane_sel;                   // the S buffer is shared by the two tiles
        const uint32_t p_addr = tmem + lane_sel + kPwTmemP + g * 64;
        const uint32_t o_addr = tmem + lane_sel + kPwTmemO + g * 128;
        int tiles = 0, uses = 0, q_uses = 0;                       // key tiles so far: of the CTA, of this query tile; Q loads so far
        float m_ref = -INFINITY, l_run = 0.f;                      // reference maximum (log2 domain), row sum
        float unit = 1.f;                                          // e4m3: V scale that O is expressed in
        int blocks = 0;                                            // row blocks so far

        for (int item = 0; ok; ++item) {
        const volatile int* ie = item_wait(item);
        if (!ok) break;
        const int n_all = ie[PI_TILES];
        if (n_all < 0) break;
        if (n_all == 0 && p.splits == 1) {                         // nothing is visible here: zeros
            const int tok0 = ie[PI_TOK0], q0 = ie[PI_Q0], head0 = ie[PI_KVH] * p.group;
            const int rows = min(ie[PI_LQ] - tok0, 2 * p.tokens) * p.group;
            for (int i = warp * 32 + lane; i < rows * 16; i += kPwSoftmaxWarps * 32) {
                const int x = i >> 4;
                const int64_t row = int64_t(q0 + tok0 + x / p.group) * p.n_q_heads + head0 + x % p.group;
                reinterpret_cast<uint4*>(p.out + row * kHeadDim)[i & 15] = make_uint4(0, 0, 0, 0);
            }
        }
        m_ref = -INFINITY;
        l_run = 0.f;
        float c_row = p.scale_log2;
        int left = g == 0 || ie[PI_TWO] ? n_all : 0;
        if (left == 0) tiles += n_all;                             // this query tile has no rows
        const bool any_tile = left > 0;
        if (FP8 && any_tile) {
            // this thread's row of Q: one row block's tiles take 256 threads 1.8 us; by the converters, four warps that also
            // yield to these, they took 6.5
            if (!tc_wait(bar(PW_Q_FULL), q_uses & 1, s_abort, p.wait_limit)) ok = false;
            if (ok) {
                c_row = p.scale_log2 * split_q_row(base + C::q + g * kPwTile, r);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(PW_Q_READY, g));
            }
        }

        for (; left > 0; --left, ++uses, ++tiles) {
            if (ok && !tc_wait(bar(PW_S_FULL, g), uses & 1, s_abort, p.wait_limit)) ok = false;
            if (!ok) continue;
            tc_fence_after();
            const bool first = left == ie[PI_TILES];
            // the tile's entry, early: its latency passes under the loads of S
            const volatile int* e = s_ring + (tiles % kPwRing) * PT_INTS;
            const uint4 head = ld_shared_v4(base + C::ring + (tiles % kPwRing) * (PT_INTS * 4));      // CUT, KEY0, K_SCALE, O_FACTOR
            float c_tile = FP8 ? c_row * __uint_as_float(head.z) : c_row;
            uint32_t sv[128];                                      // the whole row of S in registers
            tc_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
            tc_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
            tc_ld32(s_addr + 64, *reinterpret_cast<uint32_t(*)[32]>(&sv[64]));
            tc_ld32(s_addr + 96, *reinterpret_cast<uint32_t(*)[32]>(&sv[96]));
            tc_wait_ld();
            // the row is in registers: the tensor core may overwrite the S buffer
            tc_fence_before();
            mbar_arrive(bar(PW_S_FREE));
            if (__any_sync(0xffffffffu, head.x != 0 || (FP8 && c_tile == 0.f))) {
                if (FP8 && c_tile == 0.f) {                        // a K scale of 0: scores of 0
#pragma unroll
                    for (int i = 0; i < 128; ++i) sv[i] = 0u;
                    c_tile = 1.f;
                }
                // keys behind a row's own position, or in front of its window and behind the sinks: -infinity
                const int tile_tok = ie[PI_TOK0] + g * p.tokens;   // first token of the query tile
                const int pos = ie[PI_SHIFT] + min(tile_tok + r / p.group, min(ie[PI_LQ], tile_tok + p.tokens) - 1);
                const int sinks = !FP8 && head.x == 2 ? p.sinks : p.sinks - int(head.y);      // from the tile's first row on
                const int start = ie[PI_WINDOWED] ? pos - p.window + 1 : -0x40000000;
                auto low_bits = [](int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; };
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int k0 = int(head.y) + w * 32;
                    const uint32_t seen = low_bits(pos + 1 - k0) & (~low_bits(start - k0) | low_bits(sinks - w * 32));
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(seen & (1u << i))) sv[w * 32 + i] = 0xff800000u;
                }
            }
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 128; i += 8) {
                mx0 = fmax3(mx0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                mx1 = fmax3(mx1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
                mx2 = fmax3(mx2, __uint_as_float(sv[i + 4]), __uint_as_float(sv[i + 5]));
                mx3 = fmax3(mx3, __uint_as_float(sv[i + 6]), __uint_as_float(sv[i + 7]));
            }
            const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * c_tile;    // -inf: this row sees none of the tile
            // move the reference only when the maximum outgrew it by more than 2^lazy
            const bool move = mx > m_ref + C::lazy || (m_ref == -INFINITY && mx > -INFINITY);
            const float o_factor = FP8 ? __uint_as_float(head.w) : 1.f;
            if (__any_sync(0xffffffffu, move || (FP8 && o_factor != 1.f))) {
                const float m_new = move ? mx : m_ref;
                const float alpha = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - m_new);
                if (!first) {
                    // O is whole once the P V product of the previous tile has retired; the next cannot start before P_FULL below
                    if (!tc_wait(bar(PW_PV_DONE, g), (uses - 1) & 1, s_abort, p.wait_limit)) { ok = false; continue; }
                    tc_fence_after();
                    const float f = alpha * o_factor;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {                  // sixteen columns at a time: S is still in registers
                        uint32_t v[16];
                        tc_ld16(o_addr + c * 16, v);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                        tc_st16(o_addr + c * 16, v);
                    }
                    tc_wait_st();
                }
                l_run *= alpha;
                m_ref = m_new;
            }
            float up = m_ref == -INFINITY ? 0.f : -m_ref;          // added to the exponent
            if constexpr (FP8) up += __int_as_float(e[PT_UP]);
            // the tensor core must be done reading P of the previous key tile (long since, as a rule)
            if (!first && !tc_wait(bar(PW_PV_DONE, g), (uses - 1) & 1, s_abort, p.wait_limit)) { ok = false; continue; }
            // P = exp2(S * c + up) as packed 16-bit values
            uint64_t rsa = pk2(0.f, 0.f), rsb = pk2(0.f, 0.f);
            const uint64_t c2 = pk2(c_tile, c_tile), up2 = pk2(up, up);
            auto pair = [&](int c, uint64_t& sum) {
                const uint64_t x2 = ffma2(pk2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), c2, up2);
                float e0, e1;
                upk2(x2, e0, e1);
                e0 = fast_exp2(e0);
                e1 = fast_exp2(e1);
                sum = fadd2(sum, pk2(e0, e1));
                return FP8 ? pack_f16(e0, e1) : pack_bf16(e0, e1);
            };
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t pk[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) pk[i] = pair(h * 64 + 2 * i, i & 1 ? rsb : rsa);
                tc_st32(p_addr + h * 32, pk);
            }
            float rs0, rs1, rs2, rs3;
            upk2(rsa, rs0, rs1);
            upk2(rsb, rs2, rs3);
            l_run = fmaf((rs0 + rs1) + (rs2 + rs3), FP8 ? __int_as_float(e[PT_DOWN]) : 1.f, l_run);
            if constexpr (FP8) unit = __int_as_float(e[PT_V_REF]);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(bar(PW_P_FULL, g));                        // (the tile's entry may be gone from here on)
        }
        // where the row goes (worked out while the last P V product runs)
        const int tok = ie[PI_TOK0] + g * p.tokens + r / p.group;
        const bool live = r < p.tokens * p.group && tok < ie[PI_LQ];      // rows behind the tokens of the tile or the sequence hold anything
        const int64_t row = int64_t(ie[PI_Q0] + tok) * p.n_q_heads + ie[PI_KVH] * p.group + r % p.group;
        const bool any = l_run != 0.f;                              // a row that sees nothing gives zeros
        const float f = any ? unit / l_run : 0.f;
        // O is complete once the last P V has retired
        if (any_tile && ok && !tc_wait(bar(PW_PV_DONE, g), (uses - 1) & 1, s_abort, p.wait_limit)) ok = false;
        if (any_tile && ok && p.splits == 1) {
            tc_fence_after();
            uint32_t v[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32(o_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
            tc_wait_ld();
            if (!any) {
#pragma unroll
                for (int i = 0; i < 128; ++i) v[i] = 0u;
            }
            // two lanes write a row of either together, 64 bytes next to each other: a store touches 16 lines instead of 32 (16
            // sequences of 2048 rows, a window of 1024: e4m3 354 -> 335 us, bf16 286 -> 281; ten rows 7.1 -> 7.4; four
            // lanes, 128 bytes, 346 and 283: the exchange costs more)
            uint32_t w[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) w[i] = pack_bf16(__uint_as_float(v[2 * i]) * f, __uint_as_float(v[2 * i + 1]) * f);
            const bool odd = lane & 1;
            const int64_t at = live ? row : -1, other = __shfl_xor_sync(0xffffffffu, at, 1);
            const int64_t row_even = odd ? other : at, row_odd = odd ? at : other;
#pragma unroll
            for (int c = 0; c < 64; c += 16) {                     // words c .. c + 7 are the even lane's to write, c + 8 .. the odd one's
                uint32_t own[8], got[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    own[i] = odd ? w[c + 8 + i] : w[c + i];
                    got[i] = __shfl_xor_sync(0xffffffffu, odd ? w[c + i] : w[c + 8 + i], 1);
                }
                auto put = [&](int64_t r, const uint32_t* x) {
                    if (r < 0) return;
                    __nv_bfloat16* dst = p.out + r * kHeadDim + 2 * c + (odd ? 16 : 0);
                    const Bytes32 y = {make_uint4(x[0], x[1], x[2], x[3]), make_uint4(x[4], x[5], x[6], x[7])};
                    if (p.out_at32) store32<true>(dst, y);
                    else store32<false>(dst, y);
                };
                uint32_t first[8], second[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    first[i] = odd ? got[i] : own[i];              // of the even lane's row
                    second[i] = odd ? own[i] : got[i];
                }
                put(row_even, first);
                put(row_odd, second);
            }
            tc_fence_before();
        }
        ++blocks;
        q_uses += ie[PI_TILES] > 0;
        item_done(item);
        }

        if (p.splits > 1) {
            // ------------------------------------------------------------- joins the parts of the cluster's row block
            // maximum and sum of a row: over this query tile's Q, which no product needs any more
            const uint32_t ml = base + C::q + g * kPwTile + r * 8;
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(ml), "f"(m_ref), "f"(l_run) : "memory");
            cluster_sync();                                        // (and every product of this CTA has retired)
            const volatile int* ie = s_item;
            const int tile_rows = p.tokens * p.group;
            int tok0 = 0, rank = 0, rows = 0;                      // a cluster whose row block lies behind its sequence joins nothing
            if (blocks > 0) {
                tok0 = ie[PI_TOK0];
                rank = ie[PI_SPLIT];
                rows = min(ie[PI_LQ] - tok0, 2 * p.tokens) * p.group;
            }
            const uint32_t o_part = base + C::k;                   // [256][128] f32, 16-byte chunks swizzled by the row
            if (r < tile_rows && g * tile_rows + r < rows) {
                float m_all = -INFINITY, l_all = 0.f;
                for (int k = 0; k < p.splits; ++k) {
                    const float2 x = ld_cluster_f2(cluster_addr(ml, k));
                    if (x.y != 0.f) m_all = fmaxf(m_all, x.x);     // a sum of 0: this part of the keys is hidden from the row
                }
                for (int k = 0; k < p.splits; ++k) {
                    const float2 x = ld_cluster_f2(cluster_addr(ml, k));
                    if (x.y != 0.f) l_all = fmaf(x.y, fast_exp2(x.x - m_all), l_all);
                }
                m_ref = l_run != 0.f ? fast_exp2(m_ref - m_all) * unit / l_all : 0.f;      // factor of this part
            }
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t v[32];
                tc_ld32(o_addr + c * 32, v);
                tc_wait_ld();
                if (r >= tile_rows || g * tile_rows + r >= rows) continue;
                const uint32_t dst = o_part + (g * kPwRows + r) * 512;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint4 w;
                    w.x = l_run != 0.f ? __float_as_uint(__uint_as_float(v[4 * i]) * m_ref) : 0u;
                    w.y = l_run != 0.f ? __float_as_uint(__uint_as_float(v[4 * i + 1]) * m_ref) : 0u;
                    w.z = l_run != 0.f ? __float_as_uint(__uint_as_float(v[4 * i + 2]) * m_ref) : 0u;
                    w.w = l_run != 0.f ? __float_as_uint(__uint_as_float(v[4 * i + 3]) * m_ref) : 0u;
                    st_shared_v4(dst + (((c * 8 + i) ^ (r & 31)) << 4), w);
                }
            }
            tc_fence_before();
            cluster_sync();
            // rows in turn over the CTAs and their warps, four dims per lane
            for (int x = rank + p.splits * warp; x < rows; x += p.splits * kPwSoftmaxWarps) {
                const int t = x / tile_rows, xr = x - t * tile_rows;
                const uint32_t src = o_part + (t * kPwRows + xr) * 512 + ((lane ^ (xr & 31)) << 4);
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < p.splits; ++k) {
                    const float4 v = ld_cluster_f4(cluster_addr(src, k));
                    o.x += v.x;
                    o.y += v.y;
                    o.z += v.z;
                    o.w += v.w;
                }
                const int64_t row = int64_t(ie[PI_Q0] + tok0 + x / p.group) * p.n_q_heads + ie[PI_KVH] * p.group + x % p.group;
                *reinterpret_cast<uint2*>(p.out + row * kHeadDim + lane * 4) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
            }
            cluster_sync();                                        // nobody leaves while another CTA reads its shared memory
        }
    }
    if (p.splits > 1 && (hw < 4 || hw >= 12)) {                    // the other warps' share of the three barriers
        __syncwarp();
        cluster_sync();
        cluster_sync();
        cluster_sync();
    }

    // ===================================================================== common epilogue
    tc_fence_before();
    __syncthreads();
    if (warp == kPwIssueS) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (threadIdx.x == 0 && *s_abort && p.status) atomicExch(p.status, 0x5AFE0006);
}

// What a launch over clusters needs to know of a device: how many clusters of 2 .. 16 CTAs fit at a time (their sizes do not
// divide the GPCs evenly: 74, 45, 33, 26, 22, 15, 15, 15, 11 and 7 from 11 CTAs on).
constexpr int kPwMaxSplits = 16;
struct PwDevice {
    std::atomic<bool> ready{false};
    int clusters[kPwMaxSplits + 1] = {};
    int sm_count = 0;
};

// The launch configuration; attr has to outlive it.
static cudaLaunchConfig_t prefill_config(dim3 grid, int threads, int smem, int splits, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    if (splits > 1) {
        attr->id = cudaLaunchAttributeClusterDimension;
        attr->val.clusterDim.x = 1;
        attr->val.clusterDim.y = splits;
        attr->val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    return cfg;
}

// Shared-memory limit and cluster counts of the current device, looked up once.
template <bool FP8>
static int prefill_device(const PwDevice** out) {
    static PwDevice devices[64];
    static std::mutex mutex;
    int dev = 0;
    IB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) {
        set_cuda_error(cudaErrorInvalidDevice);
        return INFER_ERR_CUDA;
    }
    PwDevice& d = devices[dev];
    *out = &d;
    if (d.ready.load(std::memory_order_acquire)) return INFER_OK;
    std::lock_guard<std::mutex> lock(mutex);
    if (d.ready.load(std::memory_order_relaxed)) return INFER_OK;       // another thread was first: its counts may be in use by now
    const int smem = PwCfg<FP8>::total + 1024;
    IB_CUDA(cudaFuncSetAttribute(prefill_window_kernel<FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    IB_CUDA(cudaFuncSetAttribute(prefill_window_kernel<FP8>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    IB_CUDA(cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev));
    for (int size = 2; size <= kPwMaxSplits; ++size) {
        cudaLaunchAttribute attr;
        const cudaLaunchConfig_t cfg = prefill_config(dim3(1, size, 1), PwCfg<FP8>::threads, smem, size, nullptr, &attr);
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, prefill_window_kernel<FP8>, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            n = 0;
        }
        d.clusters[size] = n;
    }
    d.ready.store(true, std::memory_order_release);
    return INFER_OK;
}

// Over how many CTAs the key tiles of a row block are spread: the number that an estimate of the time makes best.  Measured,
// e4m3, us, with the choice in brackets:
//     rows behind keys (heads)          1        2      4      5      7      8      10
//     45 behind 300 (32 / 8)          [12.8]  17.1   13.6   14.3   15.3   14.1   15.8
//     45 behind 600                    17.7   19.6   15.8   16.6   15.4  [14.3]  15.9
//     45 behind 8000                  106.8   63.7   37.0   33.3   28.5  [25.5]  25.8
//     4 x 60 behind 9900 (18 / 3)     131.4   78.3   45.5  [41.5]  66.7   59.2   75.3     a second wave from 6 on
//     8 x 16 behind 1500 (32 / 8)      23.3  [20.8]  31.6   42.9   66.9   63.2   84.0
//     2 x 200 behind 900 (40 / 8)     [23.5]  26.1   39.1   52.6   87.7   78.8  109.2
//     1200, 4 x 1 behind 8000 (8 / 2) 123.3  [73.4]  88.7  100.1  135.3  125.9  163.5     most row blocks lie behind their sequence
static int prefill_splits(const PwDevice& d, int64_t blocks, int64_t empty, int64_t max_k, int tokens, int window, int sinks) {
    int64_t tiles = (max_k + kPwKeys - 1) / kPwKeys;
    if (window > 0) {
        const int64_t seen = (int64_t(window) + 2 * tokens + kPwKeys - 1) / kPwKeys + 1 + (int64_t(sinks) + kPwKeys - 1) / kPwKeys;
        if (seen < tiles) tiles = seen;
    }
    // us: a key tile, the set-up, a row block, a join at least, a cluster whose row block lies behind its sequence; a cluster
    // whose size is no power of two and one of more than eight CTAs start later
    constexpr double kTile = 1.5, kFirst = 6., kNext = 2., kJoin = 3.5, kEmpty = 3., kOdd = 1., kWide = 1.5;
    const int64_t turns = (blocks + d.sm_count - 1) / d.sm_count;
    double best = kFirst + double(turns) * (double(tiles) * kTile + kNext);
    int splits = 1;
    for (int s = 2; s <= kPwMaxSplits; ++s) {
        if (d.clusters[s] <= 0) continue;
        const int64_t waves = (blocks + d.clusters[s] - 1) / d.clusters[s];
        const double one = kFirst + kNext + kJoin + 6. / s + double((tiles + s - 1) / s) * kTile + (s & (s - 1) ? kOdd : 0.) + (s > 8 ? kWide : 0.);
        const double t = double(waves) * one + double(empty) / d.clusters[s] * kEmpty;
        if (t < best) {
            best = t;
            splits = s;
        }
    }
    return splits;
}

template <bool FP8>
static int launch_prefill_window(PwParams& p, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                                 const PwParts<FP8>& parts, int64_t total_q, int max_q, int max_k, int window, int batch, cudaStream_t st) {
    const PwDevice* d = nullptr;
    const int rc = prefill_device<FP8>(&d);
    if (rc != INFER_OK) return rc;
    const int64_t row_blocks = (int64_t(max_q) + 2 * p.tokens - 1) / (2 * p.tokens);
    // row blocks that hold rows: no more than this, whatever the lengths
    const int64_t filled = std::min(row_blocks * batch, total_q / (2 * p.tokens) + batch);
    p.splits = prefill_splits(*d, filled * p.n_kv_heads, (row_blocks * batch - filled) * p.n_kv_heads, max_k, p.tokens, window, p.sinks);
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = prefill_config(dim3(unsigned(row_blocks), p.n_kv_heads * p.splits, batch), PwCfg<FP8>::threads,
                                                  PwCfg<FP8>::total + 1024, p.splits, st, &attr);
    IB_CUDA(cudaLaunchKernelEx(&cfg, prefill_window_kernel<FP8>, PwParams(p), mq, mk, mv, parts));
    return check_launch();
}

static int paged_prefill_window(const infer_kv_pool_t* pool, void* out, const void* q, int64_t total_q, const int32_t* cu_seqlens_q,
                                const int32_t* cu_seqlens_k, const int32_t* block_tables, int64_t bt_stride, int64_t bt_columns,
                                int batch, int max_seqlen_q, int max_seqlen_k, int n_q_heads, float softmax_scale, int window, int sinks,
                                cudaStream_t st, uint32_t wait_limit, int stall_producer) {
    if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY) || window < 0 || sinks < 0) return INFER_ERR_GEOMETRY;
    if (!pool || !out || !q || !cu_seqlens_q || !cu_seqlens_k || !block_tables) return INFER_ERR_NULL;
    if (batch < 0 || n_q_heads <= 0 || n_q_heads % pool->n_kv_heads != 0 || n_q_heads / pool->n_kv_heads > kPwRows || bt_stride <= 0 ||
        max_seqlen_q < 0 || max_seqlen_k < 0 || batch > 65535 || n_q_heads > 65535 || total_q < 0 ||
        total_q > int64_t(batch) * max_seqlen_q || total_q >= (int64_t(1) << 31) || bt_columns < 0)
        return INFER_ERR_GEOMETRY;
    if (!aligned16(out) || !aligned16(q)) return INFER_ERR_ALIGN;
    if (total_q == 0 || batch == 0) return INFER_OK;
    PwParams p{};
    p.out = static_cast<__nv_bfloat16*>(out);
    p.out_at32 = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
    p.cu_q = cu_seqlens_q;
    p.cu_k = cu_seqlens_k;
    p.block_tables = block_tables;
    p.bt_stride = bt_stride;
    p.bt_columns = bt_columns;
    p.k_scale = pool->k_scale;
    p.v_scale = pool->v_scale;
    p.n_q_heads = n_q_heads;
    p.n_kv_heads = pool->n_kv_heads;
    p.group = n_q_heads / pool->n_kv_heads;
    p.tokens = kPwRows / p.group;
    p.block_size = pool->block_size;
    p.num_blocks = int(pool->num_blocks);
    p.window = window > 0 ? window : 0x7fffffff;
    p.sinks = sinks;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    p.status = prefill_status_word();
    p.wait_limit = wait_limit;
    p.stall_producer = stall_producer;
    CUtensorMap mq;   // q [total_q, Hq, 128]: a box is one kv head's query heads of `tokens` tokens; zeros past total_q
    int rc = encode_map_3d(&mq, q, 2, kHeadDim, uint64_t(n_q_heads), uint64_t(total_q), 256, uint64_t(n_q_heads) * 256, 64,
                           uint32_t(p.group), uint32_t(p.tokens));
    if (rc != INFER_OK) return rc;
    if (pool->dtype == INFER_KV_E4M3)
        return launch_prefill_window<true>(p, mq, pool->maps[3].k, pool->maps[3].v, PwParts<true>{}, total_q, max_seqlen_q,
                                           max_seqlen_k, window, batch, st);
    PwParts<false> parts;
    for (int i = 0; i < kPwParts; ++i) {
        parts.k[i] = pool->maps[i].k;
        parts.v[i] = pool->maps[i].v;
    }
    return launch_prefill_window<false>(p, mq, pool->maps[3].k, pool->maps[3].v, parts, total_q, max_seqlen_q, max_seqlen_k, window,
                                           batch, st);
}

}  // namespace ib

extern "C" {

int infer_paged_prefill_window(const infer_kv_pool_t* pool, void* out, const void* q, int64_t total_q, const int32_t* cu_seqlens_q,
                               const int32_t* cu_seqlens_k, const int32_t* block_tables, int64_t bt_stride, int batch,
                               int max_seqlen_q, int max_seqlen_k, int n_q_heads, float softmax_scale, int window, int sinks,
                               void* stream_) {
    return infer_paged_prefill_window_columns(pool, out, q, total_q, cu_seqlens_q, cu_seqlens_k, block_tables, bt_stride, bt_stride, batch,
                                              max_seqlen_q, max_seqlen_k, n_q_heads, softmax_scale, window, sinks, stream_);
}

int infer_paged_prefill_window_columns(const infer_kv_pool_t* pool, void* out, const void* q, int64_t total_q,
                                       const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, const int32_t* block_tables,
                                       int64_t bt_stride, int64_t bt_columns, int batch, int max_seqlen_q, int max_seqlen_k,
                                       int n_q_heads, float softmax_scale, int window, int sinks, void* stream_) {
    return ib::paged_prefill_window(pool, out, q, total_q, cu_seqlens_q, cu_seqlens_k, block_tables, bt_stride, bt_columns, batch,
                                    max_seqlen_q, max_seqlen_k, n_q_heads, softmax_scale, window, sinks,
                                    static_cast<cudaStream_t>(stream_), ib::kDefaultWaitLimit, 0);
}

int infer_selftest_paged_prefill_window(const infer_kv_pool_t* pool, void* out, const void* q, int64_t total_q,
                                        const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, const int32_t* block_tables,
                                        int64_t bt_stride, int64_t bt_columns, int batch, int max_seqlen_q, int max_seqlen_k,
                                        int n_q_heads, float softmax_scale, int window, int sinks, void* stream_,
                                        uint32_t wait_limit, int stall_producer) {
    return ib::paged_prefill_window(pool, out, q, total_q, cu_seqlens_q, cu_seqlens_k, block_tables, bt_stride, bt_columns, batch,
                                    max_seqlen_q, max_seqlen_k, n_q_heads, softmax_scale, window, sinks,
                                    static_cast<cudaStream_t>(stream_), wait_limit ? wait_limit : ib::kDefaultWaitLimit,
                                    stall_producer);
}

}  // extern "C"
