// Attention of prompt portions over the key/value cache in 8 bits (kv8.cuh) on tcgen05: bfloat16, head sizes 64 and 128, pages of 8..64
// tokens, two tiles of 128 query rows a CTA.
//
// s_j = scale (q . code_j) ks_j, out = sum_j p_j vs_j code'_j / sum_j p_j.  The exponentials bound it (128 x 128 of them for every pair of
// products of 128 x 128 x d), so nothing of the 8 bits is left to the threads that compute them:
// * four warps of their own turn codes into float16 numbers, code * (scale / reference), in the layout of the tensor core's operands, 32 keys
//   each of a tile of 128, while the softmax of the tile before runs.  The reference is the power of two above the largest scale of the 32
//   keys, which is left to the softmax as one factor for 32 columns.  A number is rounded once to 11 bits (keys; their scale goes in as
//   a sum of two float16) or, with its scale, twice (values); half a step is 2^-11 of the number, an eighth of what bfloat16 keys and
//   values lose.  (Scales applied to scores and weights in float32 by the softmax's threads: two reads of shared memory and
//   two multiplications for every four scores, 3 % of the time.)
// * 32 keys whose scales lie further apart than 2^11, and values beyond 2^45 or 2^-45, have a power of two each.  A row's weights then go by the
//   largest score and reference among the keys that it sees, its sum by the scores alone, an exponential each: what a row does not see, or
//   gives no weight, takes no bits from what it does.  Steps of such keys take four times as long (km_apart: 1,325 us if all of the portion
//   below are); all others pay 2 % of the time for looking (309 and 315 us).
// * each of these warps asks for its keys' codes of the next tile as soon as it has converted the last ones, and both operands have two
//   places, so that the conversion runs a tile ahead of the products.
// * a row whose key or value is no number makes its scores so and leaves its values zero: a weight of zero stays zero in the sums of the
//   rows that do not see it.
// * queries are multiplied by the power of two that brings a row's largest number to 2^14..2^15 (kv8_few.cu).
// * a row's exponentials refer to R = (largest score + log2 of its value reference) - 10: a weight 2^(s - R) reference is at most 2^14
//   before R is raised, and is rounded once to float16.  Both sums carry the factor, which cancels.  R is raised, and the sums so far
//   rescaled (the output in TMEM), only when it has been outgrown by 2^4.
// * a row belongs to one thread, which reads its scores from TMEM twice, 32 at a time, for the maximum and for the weights.  The weights
//   go back to TMEM in the scores' place, as the second product's left operand; O lives in TMEM too.  One query tile's softmax runs
//   beside the other's products: its own next scores follow its outputs in the tensor core's order, which is all that keeps them off
//   the weights.
// * work is cut evenly (as in kv8_few.cu): a step is a tile of keys of one double tile and key/value head, CTA c of C walks steps c N / C to
//   (c + 1) N / C.  What a CTA has of a double tile that others share goes to scratch, and whoever brings its last piece merges them, in
//   the order of the keys.  (Whole double tiles a CTA: 228 items of 2,048 tokens and 28 heads are two rounds on 148 SMs where 1.5 would do.)
// Measured: 2,048 tokens behind 6,144, 28 heads of 128 on 4: 315 us, 668 TFLOP/s, 0.41 of the measured bf16 rate; the bfloat16 cache's kernel
// takes 270 us (both a pass among others; alone 330 and 289).  Latency bounds it: half of the issue slots stay empty and the tensor pipe is
// active a third of the time, with 13 warps an SM (128 registers a thread) waiting for TMEM reads and for each other's results.
// Barrier waits are bounded (HFB_ERR_WAIT, TMEM freed; tc_ptx.cuh).
#include <cuda_fp16.h>

#include <type_traits>

#include "kv8.cuh"
#include "tc_ptx.cuh"

static thread_local cudaError_t g_launch_err = cudaSuccess;      // what the last launch_pdl returned

namespace hfb {
int *error_word();

constexpr int KM_ROWS = 128, KM_KEYS = 128, KM_THREADS = 416, KM_TMEM_COLS = 512;
// Fewest steps (a tile's start and end counted) that are worth a CTA of their own: a piece costs its merge 64 KB or 128 KB of reads by one CTA.
// With 3 | 5 | 8, 28 heads of 128 on 4: 64 tokens of each of four requests of 1,024 tokens 43 | 49 | 57 us, a prompt of 500 41 | 51 | 56; 64 tokens
// behind 8,192 94 | 80 | 77, but those go to the kernel of few queries.
constexpr int KM_MIN_STEPS = 3;
constexpr uint32_t KM_SUB = 128 * 64 * 2;           // one swizzled sub-tile: 128 rows of 64 float16

struct Kv8ManyParams {
    Kv8Params a;
    int per, n_tiles, tile_cost, settled;            // tokens per query tile, double tiles in all, steps that a tile's start and end are reckoned as
    float *part_o, *part_ml;                         // pieces of double tiles: [CTAs, 2, 2, D / 4, 128, 4] and [CTAs, 2, 2, 128, 4]
    int *counters;                                   // ... one per (double tile, head, query tile), zero between launches
};

template <int D> constexpr uint32_t km_smem() { return 6 * (D / 64) * KM_SUB + 2 * KM_KEYS * D + 128 + 256 + 4 * KM_KEYS; }

__device__ __forceinline__ uint32_t km_off(int row, int c16)
{
    return (uint32_t)(c16 >> 3) * KM_SUB + (uint32_t)row * 128u + (uint32_t)(((c16 & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ uint32_t km_codes(uint32_t w, uint32_t selector)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x64646464u), "r"(selector));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));                // 1024 + byte - 1152
    return r;
}
__device__ __forceinline__ uint32_t km_pack(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float km_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void km_st16(uint32_t taddr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                   "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
// D = A B or D += A B.  Of an operand descriptor only the low word differs from product to product; the high word is the layout (8-row groups
// 1,024 bytes apart, 128-byte swizzle).  A single thread issues the products, and every instruction it spends on one is time the
// tensor core may have to wait for.
constexpr uint32_t KM_DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
template <bool ADD> __device__ __forceinline__ void km_mma_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t idesc)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(a), "r"(b), "r"(idesc), "n"(KM_DESC_HIGH), "n"(ADD ? 1 : 0) : "memory");
}
// ... with A in TMEM (a row a lane, two numbers a column)
__device__ __forceinline__ void km_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%2, %4};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(idesc), "n"(KM_DESC_HIGH), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void km_store16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float km_load1(uint32_t addr)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 km_load4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
// Waits for what has been asked of TMEM, and ties the registers to the wait: nothing that reads them may move in front of it.
__device__ __forceinline__ void km_wait(uint32_t (&v)[32])
{
#define KM_REGS(o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
    asm volatile("tcgen05.wait::ld.sync.aligned;" : KM_REGS(0), KM_REGS(8)::"memory");
    asm volatile("" : KM_REGS(16), KM_REGS(24)::"memory");
#undef KM_REGS
}

// Exponent field of the power of two above a scale; of none (zero), that of one.
__device__ __forceinline__ uint32_t km_above(float scale) { return scale > 0.f ? min((__float_as_uint(scale) >> 23) + 1u, 253u) : 127u; }
// 32 keys share their references unless one of their scales is below the largest one's by more than a factor of 2^KM_APART: up to there
// no number code * scale, down to the code 1, leaves float16's normal range, and a key's second float16 is good to 2^-13.
// ... and unless the values' reference is beyond 2^KM_RANGE or its inverse: within, a score's exponential relative to the largest weight, whatever
// the quarters of a row's keys are scaled by, stays in float32 as long as it counts (down to 2^-46 of the largest).
constexpr uint32_t KM_APART = 11, KM_RANGE = 45;

// The steps whose keys have references of their own, one for all of the row's 128 scores: the largest score, and the largest with its value's
// reference; or (WEIGHTS) the weights into their place, and the sum of the exponentials, each relative to the largest so far.  For what
// models don't do: it may be slow, and stays out of the way of the other steps' registers and instructions.
struct KmRow {
    uint32_t tmem, exponents, present;               // where the scores, the keys' exponents and the bits of the keys there are (0: no row) lie
    float by, cap, slope;
    int key0, pos, lo;
};
template <bool WEIGHTS> __device__ __noinline__ float2 km_apart(KmRow r, float minus, float l_minus)
{
    float2 out = WEIGHTS ? make_float2(0.f, 0.f) : make_float2(-INFINITY, -INFINITY);
#pragma unroll 1
    for (int n = 0; n < 16; n++) {                   // eight scores a time
        uint32_t raw[8], ex[4], pk[4], there;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(ex[0]), "=r"(ex[1]), "=r"(ex[2]), "=r"(ex[3]) : "r"(r.exponents + 16u * n));
        there = r.present ? (__float_as_uint(km_load1(r.present + 4u * (n >> 2))) | __float_as_uint(km_load1(r.present + 16u + 4u * (n >> 2)))) >> (8 * (n & 3)) : 0u;
        __syncwarp();
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]), "=r"(raw[7]) : "r"(r.tmem + 8 * n));
        tmem_wait_ld();
        float before = 0.f;
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const int key = r.key0 + 8 * n + c;
            const uint32_t e = ex[c >> 1] >> (16 * (c & 1));
            float x = __uint_as_float(raw[c]) * r.by * __uint_as_float((e & 255u) << 23);
            const float log = (float)(e >> 8 & 255u) - 127.f;
            if (r.cap > 0.f) x = r.cap * tanh_fast(x);
            x = fmaf(r.slope, (float)(key - r.pos), x);
            if (!(there >> c & 1u) || key < r.lo || key > r.pos) x = -INFINITY;
            if (!WEIGHTS) { out.x = fmaxf(out.x, x); out.y = fmaxf(out.y, x + log); continue; }
            const float w = km_ex2(x + (log + minus));
            out.x += km_ex2(x + l_minus);
            if (c & 1) pk[c / 2] = km_pack(before, w);
            before = w;
        }
        if (WEIGHTS) {
            __syncwarp();
            asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(r.tmem + 4 * n), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]) : "memory");
        }
    }
    return out;
}

// A wait of a whole warp: its lanes look for the phase one by one, and go on together.  Lane 0's release behind it may begin the phase
// after next, in which a lane that still looked would never find the one it looks for; and where a wait runs out for one lane no
// other may go on to what the warp does as one.
__device__ __forceinline__ bool km_wait_warp(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *err)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err));
}

template <int D>
__global__ void __launch_bounds__(KM_THREADS, 1)
kv8_many_kernel(Kv8ManyParams f, int *err)
{
    const Kv8Params &p = f.a;
    extern __shared__ __align__(1024) uint8_t km_raw[];
    const uint32_t base = (smem_u32(km_raw) + 1023u) & ~1023u;
    uint8_t *gen = km_raw + (base - smem_u32(km_raw));
    constexpr uint32_t HT = (D / 64) * KM_SUB;       // a [128 x D] float16 operand: Q, K or V
    const uint32_t sQ = base, sK = base + 2 * HT, sV = base + 4 * HT;         // (keys and values: two each)
    const uint32_t stK = base + 6 * HT, stV = stK + KM_KEYS * D;         // codes of the next keys and values
    // [2][16]: per quarter of a tile the keys' reference, log2 of the values', the keys there are, or in the next four those of a quarter "apart"
    const uint32_t sS = stV + KM_KEYS * D;
    const uint32_t bars = sS + 128, sE = bars + 256; // sE [2][128]: exponents of a key's references (key, value), a byte each
    const uint32_t q_ready = bars, s_full = bars + 16, p_ready = bars + 32, pv_done = bars + 48;                          // + 8 * query tile
    const uint32_t k_full = bars + 144, k_empty = bars + 160, v_full = bars + 176, v_empty = bars + 192;                  // + 8 * place
    const uint32_t sc_full = bars + 208, sc_empty = bars + 64;                                                            // + 8 * buffer
    volatile uint32_t *tmem_slot = (volatile uint32_t *)(gen + (bars - base) + 224);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (!f.settled) pdl_wait();                      // nothing is read that the kernels in front may still write
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(q_ready + 8 * i, 4); mbar_init(s_full + 8 * i, 1); mbar_init(p_ready + 8 * i, 4); mbar_init(pv_done + 8 * i, 1);
            mbar_init(k_full + 8 * i, 4); mbar_init(v_full + 8 * i, 4); mbar_init(k_empty + 8 * i, 1); mbar_init(v_empty + 8 * i, 1);
            mbar_init(sc_full + 8 * i, 4); mbar_init(sc_empty + 8 * i, 8);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    // ---- this CTA's steps -------------------------------------------------------------------------------------------------------
    const int r = p.H / p.G, bs = p.block_size;
    struct Tile { int seq, t0, nt, pos_last, lo_first, kt_lo, n_kt0, n_kt; };
    auto tile_of = [&](int i) {
        Tile x;
        x.seq = p.tile_seq[i]; x.t0 = p.tile_t0[i];
        x.nt = max(1, min(p.tile_nt[i], 2 * f.per));                     // (what the tile has places for)
        x.pos_last = p.positions[x.t0 + x.nt - 1];
        x.lo_first = mask_lo(p.positions[x.t0], p.window);
        x.kt_lo = x.lo_first / KM_KEYS;
        x.n_kt0 = max(1, p.positions[x.t0 + min(x.nt, f.per) - 1] / KM_KEYS + 1 - x.kt_lo);
        x.n_kt = max(x.n_kt0, x.pos_last / KM_KEYS + 1 - x.kt_lo);
        return x;
    };
    int *scan = (int *)(gen + (sV - base));                              // (the values' place, still free)
    const int each = (f.n_tiles + KM_THREADS - 1) / KM_THREADS, i0 = min((int)threadIdx.x * each, f.n_tiles), i1 = min(i0 + each, f.n_tiles);
    int mine = 0;
    for (int i = i0; i < i1; i++) mine += tile_of(i).n_kt + f.tile_cost;
    int up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, up, o); if (lane >= o) up += v; }
    if (lane == 31) scan[warp] = up;
    __syncthreads();
    int before = up - mine, per_head = 0;
    for (int w = 0; w < KM_THREADS / 32; w++) { if (w < warp) before += scan[w]; per_head += scan[w]; }
    const long long total = (long long)per_head * p.G;
    const int ctas = (int)max(1ll, min((long long)gridDim.x, total / KM_MIN_STEPS)), cta = blockIdx.x;
    if (cta >= ctas) return;
    auto start_of = [&](int c) { return total * c / ctas; };
    const long long x_start = start_of(cta), x_end = start_of(cta + 1);
    if ((long long)before * p.G <= x_start && x_start < (long long)(before + mine) * p.G) {
        int i = i0, at = before;
        for (;; i++) {
            const int n = tile_of(i).n_kt + f.tile_cost;
            if ((long long)(at + n) * p.G > x_start) break;
            at += n;
        }
        scan[32] = i; scan[33] = at;
    }
    __syncthreads();
    const int first_tile = scan[32], first_before = scan[33];
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void *)tmem_slot)), "r"(KM_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (f.settled) pdl_wait();
    pdl_trigger();

    // A piece: steps off .. off + n_kt of one double tile and head; n_kt0, n_kt1: how many of them the two query tiles take part in.
    // Every role walks the same ones.
    struct Item { int g, seq, t0, nt0, nt1, pos_last, lo_first, kt_lo, n_kt0, n_kt1, n_kt, tile, all; long long first; };
    struct Walk { long long x; int tile, before; };
    auto item_of = [&](Walk &w, Item &it) -> bool {
        for (;;) {
            if (w.x >= x_end) return false;
            const Tile tl = tile_of(w.tile);
            const int n = tl.n_kt + f.tile_cost;
            const long long t_first = (long long)w.before * p.G;
            if (w.x >= t_first + (long long)n * p.G) { w.before += n; w.tile++; continue; }
            it.g = (int)((w.x - t_first) / n);
            it.first = t_first + (long long)it.g * n + f.tile_cost;      // (the tile's own steps lie behind the empty ones)
            const long long begin = max(w.x, it.first);
            w.x = min(x_end, it.first + tl.n_kt);
            const int off = (int)(begin - it.first);
            it.n_kt = (int)max(0ll, w.x - begin);
            if (it.n_kt == 0) continue;
            it.tile = w.tile; it.all = tl.n_kt;
            it.seq = tl.seq; it.t0 = tl.t0; it.pos_last = tl.pos_last; it.lo_first = tl.lo_first; it.kt_lo = tl.kt_lo + off;
            it.nt0 = min(tl.nt, f.per); it.nt1 = tl.nt - it.nt0;         // tokens of the two query tiles
            it.n_kt0 = max(0, min(it.n_kt, tl.n_kt0 - off));
            it.n_kt1 = it.nt1 > 0 ? it.n_kt : 0;
            return true;
        }
    };

    if (warp == 12) {
        if (lane == 0) {
            // ---- tensor-core issue ------------------------------------------------------------------------------------------------
            constexpr uint32_t F16 = (1u << 7) | (1u << 10);             // (the operands' type bits of bfloat16: clear for float16)
            constexpr uint32_t idesc_s = bf16_idesc(KM_ROWS, KM_KEYS, false) & ~F16, idesc_pv = bf16_idesc(KM_ROWS, D, true) & ~F16;
            const uint32_t tS0 = tmem_base, tO0 = tmem_base + 256;
            // the descriptors' low words, made once
            uint32_t dq[2][D / 16], dk[2][D / 16], dv[2][KM_KEYS / 16];
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    const uint32_t o = (uint32_t)(kk >> 2) * KM_SUB + (uint32_t)(kk & 3) * 32u + u * HT;
                    dq[u][kk] = (uint32_t)sw128_desc(sQ + o);
                    dk[u][kk] = (uint32_t)sw128_desc(sK + o);
                }
#pragma unroll
                for (int kk = 0; kk < KM_KEYS / 16; kk++) dv[u][kk] = (uint32_t)sw128_desc_mn(sV + u * HT + kk * 2048u, KM_SUB);
            }
            auto issue_s = [&](int i, uint32_t place) {
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    const uint32_t b = place ? dk[1][kk] : dk[0][kk];
                    if (kk == 0) km_mma_ss<false>(tS0 + i * 128, dq[i][kk], b, idesc_s);
                    else km_mma_ss<true>(tS0 + i * 128, dq[i][kk], b, idesc_s);
                }
                tc_commit(s_full + 8 * i);
            };
            auto issue_pv = [&](int i, uint32_t place, bool accumulate) {
#pragma unroll
                for (int kk = 0; kk < KM_KEYS / 16; kk++)                // (two weights a column of TMEM)
                    km_mma_ts(tO0 + i * D, tS0 + i * 128 + kk * 8, place ? dv[1][kk] : dv[0][kk], idesc_pv, (accumulate || kk > 0) ? 1u : 0u);
                tc_commit(pv_done + 8 * i);
            };
            bool ok = true;
            uint32_t gs = 0, g_tile0 = 0, g_tile1 = 0, q_uses0 = 0, q_uses1 = 0;      // steps so far, per query tile, and pieces per query tile
            Walk walk = {x_start, first_tile, first_before};
            for (Item it; ok && item_of(walk, it);) {
                if (it.n_kt0 > 0) ok = mbar_wait(q_ready, q_uses0++ & 1, abort_flag, err);
                if (ok && it.n_kt1 > 0) ok = mbar_wait(q_ready + 8, q_uses1++ & 1, abort_flag, err);
                if (ok) ok = mbar_wait(k_full + 8 * (gs & 1), (gs >> 1) & 1, abort_flag, err);
                if (ok) {
                    tc_fence_after();
                    if (it.n_kt0 > 0) issue_s(0, gs & 1);
                    if (it.n_kt1 > 0) issue_s(1, gs & 1);
                    tc_commit(k_empty + 8 * (gs & 1));
                }
                for (int j = 0; j < it.n_kt && ok; j++, gs++) {
                    const uint32_t here = gs & 1, next = here ^ 1;
                    ok = mbar_wait(v_full + 8 * here, (gs >> 1) & 1, abort_flag, err);
                    if (ok && j + 1 < it.n_kt) ok = mbar_wait(k_full + 8 * next, ((gs + 1) >> 1) & 1, abort_flag, err);
                    // per query tile: the outputs of step j, then the scores of step j + 1 in the place of the weights
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int n = i ? it.n_kt1 : it.n_kt0;
                        if (ok && j < n) {
                            ok = mbar_wait(p_ready + 8 * i, ((i ? g_tile1 : g_tile0) + j) & 1, abort_flag, err);
                            if (ok) {
                                tc_fence_after();
                                issue_pv(i, here, j > 0);
                                if (j + 1 < n) issue_s(i, next);
                            }
                        }
                    }
                    if (!ok) break;
                    tc_commit(v_empty + 8 * here);
                    if (j + 1 < it.n_kt) tc_commit(k_empty + 8 * next);
                }
                g_tile0 += it.n_kt0; g_tile1 += it.n_kt1;
            }
            // nothing of this CTA's is in flight once the last release of V has landed
            if (ok && gs > 0) mbar_wait(v_empty + 8 * ((gs - 1) & 1), ((gs - 1) >> 1) & 1, abort_flag, err);
        }
    } else if (warp >= 8) {
        // ---- codes into operands: a warp has a quarter of a tile's keys, a lane one of them ----------------------------------------
        const int row = (warp - 8) * 32 + lane;
        // this thread's key: code * (hi + lo) with `both`, else code * hi
        auto convert = [&](uint32_t from, uint32_t to, __half2 hi, __half2 lo, auto both) {
            auto number = [&](uint32_t word, uint32_t selector) {
                const uint32_t bits = km_codes(word, selector);
                const __half2 c = *(const __half2 *)&bits, r = decltype(both)::value ? __hfma2(c, hi, __hmul2(c, lo)) : __hmul2(c, hi);
                return *(const uint32_t *)&r;
            };
#pragma unroll 2
            for (int c = 0; c < D / 16; c++) {
                uint4 w;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                             : "r"(from + (uint32_t)row * D + (uint32_t)kv8_piece(row % bs, c, D) * 16u) : "memory");
                km_store16(to + km_off(row, 2 * c), number(w.x, 0x4140), number(w.x, 0x4342), number(w.y, 0x4140), number(w.y, 0x4342));
                km_store16(to + km_off(row, 2 * c + 1), number(w.z, 0x4140), number(w.z, 0x4342), number(w.w, 0x4140), number(w.w, 0x4342));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        bool ok = true;
        uint32_t gs = 0;                                                  // steps of the items before
        Walk walk = {x_start, first_tile, first_before};
        for (Item it; ok && item_of(walk, it);) {
            const int32_t *table = p.block_table + (size_t)it.seq * p.max_blocks;
            // the page of this thread's key in step j; -1 where there is none to be read (behind the last, passed by every row's mask, no page)
            auto page_of = [&](int j) {
                const int key = (it.kt_lo + j) * KM_KEYS + row, blk = key / bs;
                if (j >= it.n_kt || key > it.pos_last || key < it.lo_first) return -1;
                const int page = blk < p.max_blocks ? table[blk] : -1;
                if (page < 0 || page >= p.num_pages) { atomicOr(err, HFB_ERR_PAGE); return -1; }
                return page;
            };
            const int in_page = row % bs;                                 // (tiles begin on pages)
            auto record_of = [&](int page) { return p.cache + ((size_t)page * p.G + it.g) * p.record; };
            // the warp's 32 keys' codes, 16 bytes a lane, neighbouring lanes neighbouring bytes (zeros of keys that are not there: their scales are)
            auto fetch = [&](int page, int skip, uint32_t to) {
#pragma unroll
                for (int n = 0; n < D / 16; n++) {
                    const int at = n * 32 + lane, r_q = at / (D / 16), r_tile = (warp - 8) * 32 + r_q;
                    const int its = __shfl_sync(0xffffffffu, page, r_q);
                    const uint8_t *src = record_of(max(its, 0)) + skip + (r_tile % bs) * D + at % (D / 16) * 16;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 ::"r"(to + (uint32_t)(warp - 8) * 32u * D + at * 16u), "l"(src), "r"(its >= 0 ? 16 : 0) : "memory");
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            // ... behind a piece's last step nothing, but a group all the same, for the count: the next piece's first copies go to the same
            // places, and nothing orders two copies to one place but a wait
            auto fetch_next = [&](bool any, int page, int skip, uint32_t to) {
                if (any) fetch(page, skip, to);
                else asm volatile("cp.async.commit_group;" ::: "memory");
            };
            auto fetched = [&] { asm volatile("cp.async.wait_group 1;" ::: "memory"); __syncwarp(); };       // (all but the last)
            auto scales_of = [&](int page) {
                if (page < 0) return make_float2(0.f, 0.f);
                const float *s = (const float *)(record_of(page) + 2 * bs * D) + in_page;
                return make_float2(s[0], s[bs]);
            };
            int page = page_of(0);
            fetch(page, 0, stK);
            fetch(page, bs * D, stV);
            float2 sc = scales_of(page);
            bool there = page >= 0;
            page = page_of(1);
            for (int j = 0; j < it.n_kt && ok; j++) {
                const uint32_t g = gs + j, b = g & 1, ph = (g >> 1) & 1, at = sS + b * 64u + 4u * (warp - 8);
                // the references: powers of two above the largest scales (maxima pass by what is no number)
                const float k_scale = fmaxf(sc.x, 0.f), v_scale = fmaxf(sc.y, 0.f);
                uint32_t kf = km_above(warp_max(k_scale)), vf = km_above(warp_max(v_scale));
                const bool number = sc.x == sc.x && sc.y == sc.y;
                // ... for all 32 keys, unless they are so far apart that float16 would lose the smaller ones, or so large or small that a row's weights
                // and exponentials could not go by one reference: then every key has its own.  (Rows of zeros, which have the least scale there is, don't
                // count, nor do those with them whose largest number is below 1.5e-36.)
                auto far_below = [&](float scale, uint32_t f) { return scale > 1.17549435e-38f && km_above(scale) + KM_APART < f; };
                const bool apart = __any_sync(0xffffffffu, there && number && (far_below(k_scale, kf) || far_below(v_scale, vf))) ||
                                   vf + KM_RANGE < 127u || vf > 127u + KM_RANGE;
                const uint32_t k_ref = kf, v_ref = vf;
                if (apart && there && number) { kf = km_above(k_scale); vf = km_above(v_scale); }
                const float ks = number ? sc.x * __uint_as_float((254u - kf) << 23) : __uint_as_float(0x7fc00000u);
                const __half k_hi = __float2half_rn(ks), k_lo = __float2half_rn(ks - __half2float(k_hi));
                const __half v_hi = __float2half_rn(number ? sc.y * __uint_as_float((254u - vf) << 23) : 0.f);
                const uint32_t present = __ballot_sync(0xffffffffu, there);
                ok = km_wait_warp(sc_empty + 8 * b, ph ^ 1, abort_flag, err);
                if (!ok) break;
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(sE + 2u * (b * KM_KEYS + row)), "h"((unsigned short)(kf | vf << 8)) : "memory");
                __syncwarp();
                if (lane == 0) {
                    asm volatile("st.shared.f32 [%0], %1;\n\tst.shared.f32 [%0 + 16], %2;\n\tst.shared.u32 [%0 + 32], %3;\n\tst.shared.u32 [%0 + 48], %4;"
                                 ::"r"(at), "f"(__uint_as_float(k_ref << 23)), "f"((float)v_ref - 127.f), "r"(apart ? 0u : present), "r"(apart ? present : 0u) : "memory");
                    mbar_arrive(sc_full + 8 * b);
                }
                if (!km_wait_warp(k_empty + 8 * b, ph ^ 1, abort_flag, err)) { ok = false; break; }
                fetched();
                convert(stK, sK + b * HT, __half2half2(k_hi), __half2half2(k_lo), std::true_type());
                if (lane == 0) mbar_arrive(k_full + 8 * b);
                fetch_next(j + 1 < it.n_kt, page, 0, stK);                // (of step j + 1)
                sc = scales_of(page);
                if (!km_wait_warp(v_empty + 8 * b, ph ^ 1, abort_flag, err)) { ok = false; break; }
                fetched();
                convert(stV, sV + b * HT, __half2half2(v_hi), __half2half2(v_hi), std::false_type());
                if (lane == 0) mbar_arrive(v_full + 8 * b);
                fetch_next(j + 1 < it.n_kt, page, bs * D, stV);
                there = page >= 0;
                page = page_of(j + 2);
            }
            gs += it.n_kt;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ---- softmax and output: one thread per row -------------------------------------------------------------------------------
        const float log2e = 1.4426950408889634f;
        const int i = warp >> 2;                                         // query tile
        const int row = (warp & 3) * 32 + lane;                          // TMEM lane = row; a warp reads its own quarter
        const int tl = row / r, hl = row % r;
        const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tS = lane_base + i * 128, tO = lane_base + 256 + i * D;
        uint32_t g_mine = 0, gs = 0;                                     // this query tile's steps so far, and the item's
        bool ok = true;
        Walk walk = {x_start, first_tile, first_before};
        for (Item it; ok && item_of(walk, it);) {
            const int n_mine = i ? it.n_kt1 : it.n_kt0, nt_mine = i ? it.nt1 : it.nt0, t_first = it.t0 + i * f.per;
            const bool valid = tl < nt_mine;
            const size_t th = ((size_t)(t_first + (valid ? tl : 0)) * p.H + it.g * r + hl) * D;
            float unit = 0.f;                                            // from a product's sum to a score in the exponent's base 2
            if (n_mine > 0) {
                // the tile's products of the item before are done (their scores have all been waited for)
                const uint4 *src = (const uint4 *)((const __nv_bfloat16 *)p.q + th);
                uint4 raw[D / 8];
                unsigned top = 0;
#pragma unroll
                for (int c = 0; c < D / 8; c++) {
                    raw[c] = valid ? src[c] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
                    for (int u = 0; u < 4; u++) top = max(top, max(w[u] & 0x7fffu, (w[u] >> 16) & 0x7fffu));
                }
                const unsigned field = min(268u - (top >> 7), 253u);
                const float by = __uint_as_float(field << 23);
                unit = p.scale * log2e * __uint_as_float((254u - field) << 23);
#pragma unroll
                for (int c = 0; c < D / 8; c++) {
                    const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
                    uint32_t h[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) h[u] = km_pack(__uint_as_float(w[u] << 16) * by, __uint_as_float(w[u] & 0xffff0000u) * by);
                    km_store16(sQ + i * HT + km_off(row, c), h[0], h[1], h[2], h[3]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_ready + 8 * i);
            }
            const int pos = valid ? p.positions[t_first + tl] : -1;
            const int lo = mask_lo(pos, p.window);
            const float slope2 = (p.slopes && valid) ? p.slopes[it.g * r + hl] * log2e : 0.f;
            const float hscale = (p.head_scales && valid) ? p.head_scales[it.g * r + hl] : 1.f;
            const bool capped = p.softcap > 0.f, finished = capped || p.slopes || p.head_scales;     // (scores are finished in place)
            const float cap_in = capped ? unit * hscale / (p.softcap * log2e) : 0.f, cap2 = p.softcap * log2e;
            // which of 32 keys from key0 on the row sees, those from `lo` to `pos`, as bits
            auto seen = [&](int key0) {
                const int from = min(max(lo - key0, 0), 32), to = min(max(pos + 1 - key0, 0), 32);
                return (to > 31 ? 0xffffffffu : (1u << to) - 1u) & (from > 31 ? 0u : 0xffffffffu << from);
            };
            float ref = -INFINITY, l = 0.f;                              // what the exponentials refer to, their sum
            // `two`: weights and sum have references of their own, the sum l_ref
            bool two = false;
            float l_ref = -INFINITY;
            for (int j = 0; j < it.n_kt && ok; j++) {
                const uint32_t b = (gs + j) & 1, sc_ph = ((gs + j) >> 1) & 1, s_at = sS + b * 64u;
                if (!km_wait_warp(sc_full + 8 * b, sc_ph, abort_flag, err)) { ok = false; break; }
                if (j >= n_mine) {                                       // (the other query tile's step)
                    if (lane == 0) mbar_arrive(sc_empty + 8 * b);
                    continue;
                }
                const uint32_t ph = (g_mine + j) & 1;                    // (O holds everything up to the step before once these scores are there)
                const int key0 = (it.kt_lo + j) * KM_KEYS;
                if (!km_wait_warp(s_full + 8 * i, ph, abort_flag, err)) { ok = false; break; }
                tc_fence_after();
                // a step without options in which every row sees every key, as most are (rows beyond the tile's tokens go with those)
                const float4 there4 = km_load4(s_at + 32u);
                const bool full = (__float_as_uint(there4.x) & __float_as_uint(there4.y) & __float_as_uint(there4.z) & __float_as_uint(there4.w)) == 0xffffffffu;
                const bool open = __all_sync(0xffffffffu, !valid || (key0 + KM_KEYS - 1 <= pos && key0 >= lo)) && full && !finished && !two;
                bool apart = two;                                        // (keys with references of their own are not among `there4`)
                if (!open) {
                    const float4 own = km_load4(s_at + 48u);
                    apart = apart || (__float_as_uint(own.x) | __float_as_uint(own.y) | __float_as_uint(own.z) | __float_as_uint(own.w)) != 0u;
                }
                const float by_head = unit * hscale;
                // (loops over the quarters of a tile stay loops: eight warps of these run beside four that convert, and unrolled their
                // instructions do not stay in the caches: when that was tried, 410 us for the portion named above against 358)
                auto load32 = [&](int q, uint32_t (&raw)[32]) { tmem_ld16(tS + 32 * q, raw); tmem_ld16(tS + 32 * q + 16, raw + 16); };
                auto k_ref = [&](int q) { return km_load1(s_at + 4u * q); };
                auto v_log = [&](int q) { return km_load1(s_at + 16u + 4u * q); };
                // 32 finished scores (options, masks) in the exponent's base 2.  (What a step does not have costs it nothing: a capped step in which
                // every row sees every key is as long as its special functions, three a score.)
                auto finish = [&](int q, uint32_t (&raw)[32], uint32_t sees) {
                    const float in = (capped ? cap_in : by_head) * k_ref(q);
                    if (capped) {
#pragma unroll
                        for (int c = 0; c < 32; c++) raw[c] = __float_as_uint(cap2 * tanh_fast(__uint_as_float(raw[c]) * in));
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c++) raw[c] = __float_as_uint(__uint_as_float(raw[c]) * in);
                    }
                    if (p.slopes) {
                        const float far = (float)(key0 + 32 * q - pos);
#pragma unroll
                        for (int c = 0; c < 32; c++) raw[c] = __float_as_uint(fmaf(slope2, far + (float)c, __uint_as_float(raw[c])));
                    }
                    if (__any_sync(0xffffffffu, sees != 0xffffffffu)) {
#pragma unroll
                        for (int c = 0; c < 32; c++) raw[c] = sees >> c & 1u ? raw[c] : 0xff800000u;
                    }
                };
                auto row_of = [&] {
                    return KmRow{tS, sE + 2u * b * KM_KEYS, valid ? s_at + 32u : 0u, capped ? cap_in : by_head, capped ? cap2 : 0.f, slope2, key0, pos, lo};
                };
                auto sees_of = [&](int q) { return valid ? seen(key0 + 32 * q) & __float_as_uint(km_load1(s_at + 32u + 4u * q)) : 0u; };
                float mx = -INFINITY, ms = -INFINITY;                    // the row's largest weight (`apart`: and score), in the exponent's base 2
                uint32_t ra[32], rb[32];
                if (apart) {
                    const float2 most = km_apart<false>(row_of(), 0.f, 0.f);
                    ms = most.x; mx = most.y;
                } else if (open) {
                    // (the next 32 are on their way while these are worked on)
                    auto largest = [&](int q, const uint32_t (&raw)[32]) {
                        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 32; c += 2)
                            top[(c >> 1) & 3] = fmaxf(top[(c >> 1) & 3], fmaxf(__uint_as_float(raw[c]), __uint_as_float(raw[c + 1])));
                        mx = fmaxf(mx, fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), unit * k_ref(q), v_log(q)));
                    };
                    load32(0, ra);
                    km_wait(ra);
#pragma unroll 1
                    for (int q = 0; q < 4; q += 2) {
                        load32(q + 1, rb);
                        largest(q, ra);
                        km_wait(rb);
                        load32((q + 2) & 3, ra);                         // (the last time: for the weights)
                        largest(q + 1, rb);
                        km_wait(ra);
                    }
                } else {
                    // without slopes, factors and a cap keep the order of the scores or turn it round: the largest is found first, and finished alone
                    const float way = hscale < 0.f ? -1.f : 1.f;
#pragma unroll 1
                    for (int q = 0; q < 4; q++) {
                        __syncwarp();
                        load32(q, ra);
                        km_wait(ra);
                        float top = -INFINITY;
                        if (p.slopes) {
                            finish(q, ra, sees_of(q));
#pragma unroll
                            for (int c = 0; c < 32; c++) top = fmaxf(top, __uint_as_float(ra[c]));
                        } else {
                            const uint32_t sees = sees_of(q);
                            if (__all_sync(0xffffffffu, sees == 0xffffffffu)) {
#pragma unroll
                                for (int c = 0; c < 32; c++) top = fmaxf(top, __uint_as_float(ra[c]) * way);
                            } else {
#pragma unroll
                                for (int c = 0; c < 32; c++) top = fmaxf(top, sees >> c & 1u ? __uint_as_float(ra[c]) * way : -INFINITY);
                            }
                            if (top != -INFINITY) top = capped ? cap2 * tanh_fast(top * way * cap_in * k_ref(q)) : top * way * by_head * k_ref(q);
                        }
                        mx = fmaxf(mx, top + v_log(q));
                    }
                }
                mx -= 10.f;
                // raise the reference only when it has been outgrown by 2^4 (or there was none yet)
                const float before = ref;
                float corr = 1.f;
                if (mx > ref + 4.f || (ref == -INFINITY && mx > -INFINITY)) {
                    corr = ref == -INFINITY ? 0.f : km_ex2(ref - mx);
                    ref = mx;
                }
                if (j > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; c++) {
                        uint32_t ov[16];
                        tmem_ld16(tO + 16 * c, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * corr);
                        km_st16(tO + 16 * c, ov);
                    }
                }
                const float minus = ref == -INFINITY ? 0.f : -ref;
                const f32pair one2 = pair_of(1.f, 1.f);
                float step_sum = 0.f;
                // weights 2^(score + log2 of the values' reference - R), over scores that have been read; the sum goes without that reference
                auto weights = [&](int q, const uint32_t (&raw)[32], bool scaled) {
                    const float factor = scaled ? 1.f : unit * k_ref(q), log = v_log(q);
                    const f32pair a2 = pair_of(factor, factor), m2 = pair_of(log + minus, log + minus);
                    f32pair sum[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
                    uint32_t pk[16];
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float2 x = halves(fma2(pair_of(__uint_as_float(raw[c]), __uint_as_float(raw[c + 1])), a2, m2));
                        const float e0 = km_ex2(x.x), e1 = km_ex2(x.y);
                        sum[(c >> 1) & 1] = fma2(pair_of(e0, e1), one2, sum[(c >> 1) & 1]);
                        pk[c / 2] = km_pack(e0, e1);
                    }
                    km_st16(tS + 16 * q, pk);
                    const float2 s0 = halves(sum[0]), s1 = halves(sum[1]);
                    step_sum = fmaf((s0.x + s0.y) + (s1.x + s1.y), __uint_as_float((uint32_t)(127.f - log) << 23), step_sum);
                };
                __syncwarp();
                if (apart) {
                    // the sum's own reference: that of the weights until here, then kept such that the sum is near one
                    auto near_one = [&] {
                        const int e = l > 0.f && l < 1e38f ? (int)(__float_as_uint(l) >> 23) - 127 : 0;
                        l *= __uint_as_float((uint32_t)(127 - e) << 23);
                        l_ref += (float)e;
                    };
                    if (!two) { l_ref = before; near_one(); }
                    if (ms > l_ref + 4.f || (l_ref == -INFINITY && ms > -INFINITY)) {
                        if (l_ref != -INFINITY) l *= km_ex2(l_ref - ms);
                        l_ref = ms;
                    }
                    l += km_apart<true>(row_of(), minus, l_ref == -INFINITY ? 0.f : -l_ref).x;
                    near_one();
                    // one reference does again where the two are as near each other, in every row of the warp, as steps of one reference bring them
                    const float gap = ref == -INFINITY ? 0.f : l_ref - ref;
                    two = !__all_sync(0xffffffffu, gap > 10.f - KM_RANGE && gap < KM_RANGE);
                    if (!two) l *= km_ex2(gap);
                } else if (open) {
#pragma unroll 1
                    for (int q = 0; q < 4; q += 2) {
                        load32(q + 1, rb);
                        weights(q, ra, false);
                        km_wait(rb);
                        if (q == 0) load32(2, ra);
                        weights(q + 1, rb, false);
                        if (q == 0) km_wait(ra);
                    }
                } else {
#pragma unroll 1
                    for (int q = 0; q < 4; q++) {
                        __syncwarp();
                        load32(q, ra);
                        km_wait(ra);
                        finish(q, ra, sees_of(q));
                        __syncwarp();
                        weights(q, ra, true);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sc_empty + 8 * b);
                if (!apart) l = fmaf(l, corr, step_sum);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + 8 * i);
            }
            gs += it.n_kt;
            g_mine += n_mine;
            if (ok && n_mine > 0) ok = km_wait_warp(pv_done + 8 * i, (g_mine - 1) & 1, abort_flag, err);
            {
                // (a wait that ran out ends the walk of the query tile's warps together: none may be left at a barrier)
                int all;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, %2, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                             : "=r"(all) : "r"((int)ok), "r"(1 + i) : "memory");
                ok = all;
            }
            if (!ok || nt_mine <= 0) continue;
            tc_fence_after();
            // the sink is one more term of the whole sum, and joins it where that is made: what one piece's exponentials refer to may lie hundreds
            // below it (with slopes a tile's oldest keys do), out of float32's range
            const bool sink = p.sinks || p.zero_sink;
            if (!two) l_ref = ref;
            const float sk = p.sinks && valid ? p.sinks[it.g * r + hl] * log2e : 0.f;
            // the pieces of this double tile and head: of CTAs c_first .. c_first + pieces - 1, each its first but for the first one's last
            const int c_first = (int)(((it.first + 1) * ctas - 1) / total), pieces = (int)(((it.first + it.all) * ctas - 1) / total) - c_first + 1;
            uint4 *dst = (uint4 *)((__nv_bfloat16 *)p.out + th);
            if (pieces == 1) {
                const float top = sink ? fmaxf(l_ref, sk) : l_ref;
                if (sink) l = fmaf(l, exp2f(l_ref - top), exp2f(sk - top));
                const float inv = l == 0.f ? 0.f : (ref == -INFINITY ? 1.f : exp2f(ref - top)) / l;
#pragma unroll 1
                for (int c = 0; c < D / 16; c += 4) {                    // four reads of 16 columns under way together
                    uint32_t ov[64];
#pragma unroll
                    for (int u = 0; u < 4; u++) tmem_ld16(tO + 16 * (c + u), ov + 16 * u);   // all lanes take part, valid row or not
                    tmem_wait_ld();
                    if (valid) {
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            __nv_bfloat162 h[8];
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                h[e] = __floats2bfloat162_rn(__uint_as_float(ov[16 * u + 2 * e]) * inv, __uint_as_float(ov[16 * u + 2 * e + 1]) * inv);
                            dst[2 * (c + u)] = *(uint4 *)&h[0];
                            dst[2 * (c + u) + 1] = *(uint4 *)&h[4];
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();
                continue;
            }
            auto place_of = [&](int c) { return (size_t)((c * 2 + (start_of(c) >= it.first ? 0 : 1)) * 2 + i); };
            {
                float4 *po = (float4 *)f.part_o + place_of(cta) * (D / 4) * 128 + row;
                if (n_mine > 0) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; c++) {
                        uint32_t ov[16];
                        tmem_ld16(tO + 16 * c, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 4; u++)
                            po[(4 * c + u) * 128] = make_float4(__uint_as_float(ov[4 * u]), __uint_as_float(ov[4 * u + 1]), __uint_as_float(ov[4 * u + 2]), __uint_as_float(ov[4 * u + 3]));
                    }
                    tc_fence_before();
                } else {
                    for (int c = 0; c < D / 4; c++) po[c * 128] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                ((float4 *)f.part_ml)[place_of(cta) * 128 + row] = make_float4(ref, l_ref, l, 0.f);
            }
            int *flag = (int *)(gen + (bars - base) + 232 + 4 * i);
            asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
            if ((threadIdx.x & 127) == 0) {
                __threadfence();                                         // (after the barrier: it covers the four warps' stores)
                int *cnt = f.counters + ((size_t)it.tile * p.G + it.g) * 2 + i;
                const int last = atomicAdd(cnt, 1) == pieces - 1;
                if (last) *cnt = 0;
                *(volatile int *)flag = last;
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
            if (!*(volatile int *)flag || !valid) continue;              // (the flag is written again behind two barriers)
            __threadfence();
            float top = sink ? sk : -INFINITY, sum = 0.f;
            auto sums_of = [&](int c) { return __ldcg((const float4 *)f.part_ml + place_of(c_first + c) * 128 + row); };
            for (int c = 0; c < pieces; c++) top = fmaxf(top, sums_of(c).y);
            if (sink) sum = exp2f(sk - top);
            for (int c = 0; c < pieces; c++) {
                const float4 m = sums_of(c);
                sum += m.z * (m.y == -INFINITY ? 1.f : exp2f(m.y - top));              // (zero, or no number)
            }
            const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll 1
            for (int c = 0; c < D / 4; c += 8) {
                float4 acc[8];
#pragma unroll
                for (int u = 0; u < 8; u++) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < pieces; k++) {
                    const size_t at = place_of(c_first + k);
                    const float own = sums_of(k).x, e = own == -INFINITY ? 0.f : exp2f(own - top) * inv;
                    const float4 *po = (const float4 *)f.part_o + (at * (D / 4) + c) * 128 + row;
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const float4 v = __ldcg(po + u * 128);
                        acc[u].x += v.x * e; acc[u].y += v.y * e; acc[u].z += v.z * e; acc[u].w += v.w * e;
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; u += 2) {
                    __nv_bfloat162 h[4] = {__floats2bfloat162_rn(acc[u].x, acc[u].y), __floats2bfloat162_rn(acc[u].z, acc[u].w),
                                           __floats2bfloat162_rn(acc[u + 1].x, acc[u + 1].y), __floats2bfloat162_rn(acc[u + 1].z, acc[u + 1].w)};
                    dst[(c + u) / 2] = *(uint4 *)h;
                }
            }
        }
    }

    // ---- teardown -------------------------------------------------------------------------------------------------------------------
    tc_fence_before();
    __syncthreads();
    if (*abort_flag != 0 && threadIdx.x == 0)                            // a wait ran out: products still in flight end before their operands go away
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(KM_TMEM_COLS) : "memory");
    }
}

template <int D>
static int launch_kv8_many(const Kv8ManyParams &f, int grid, cudaStream_t st)
{
    constexpr uint32_t smem = km_smem<D>() + 1024;                       // (the tiles begin on a multiple of 1,024)
    static_assert(smem <= 227 * 1024, "the tiles do not fit");
    static bool configured[64] = {false};                                // (the opt-in is a property of the function on one device)
    if (!configured[current_device()]) {
        cudaError_t e = cudaFuncSetAttribute(kv8_many_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return fail(HFB_ECUDA, "kv8_attention_many: cannot opt in to %u bytes of shared memory: %s", smem, cudaGetErrorString(e));
        configured[current_device()] = true;
    }
    g_launch_err = launch_pdl(kv8_many_kernel<D>, dim3(grid), dim3(KM_THREADS), smem, st, f, error_word());
    return check_pdl_launch(g_launch_err, "kv8_attention_many");
}

}  // namespace hfb

using namespace hfb;

extern "C" size_t hfb_kv8_attention_many_scratch(int ctas, int d) { return (size_t)ctas * 4 * 128 * (d + 4) * sizeof(float); }

extern "C" int hfb_kv8_attention_many(const void *q, const void *cache, const int32_t *block_table, int max_blocks, const int32_t *positions,
                                      const int32_t *tile_seq, const int32_t *tile_t0, const int32_t *tile_nt, int n_tiles, int ctas, int tile_cost, int settled, int block_size,
                                      int64_t num_pages, int window, float scale, void *out, void *scratch,
                                      size_t scratch_bytes, int *counters, int counters_len, int H, int G, int d, const float *sinks, int zero_sink,
                                      const float *slopes, const float *head_scales, float softcap, hfb_stream s)
{
    if (n_tiles <= 0) return HFB_OK;
    if (d != 64 && d != 128) return fail(HFB_ENOTSUP, "kv8_attention_many: head size %d (64 and 128 only)", d);
    if (H <= 0 || G <= 0 || H % G || H / G > KM_ROWS || max_blocks <= 0 || num_pages < 0)
        return fail(HFB_EINVAL, "kv8_attention_many: bad arguments (H=%d G=%d)", H, G);
    if (block_size < 8 || block_size > 64 || 64 % block_size) return fail(HFB_ENOTSUP, "kv8_attention_many: pages of %d tokens (8, 16, 32 and 64)", block_size);
    if (!(scale > 0.f)) return fail(HFB_ENOTSUP, "kv8_attention_many: the factor on the scores must be positive");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache) & 15) return fail(HFB_EINVAL, "kv8_attention_many: misaligned arrays");
    if (ctas < 1 || tile_cost < 0 || !scratch || ((uintptr_t)scratch & 15) || scratch_bytes < hfb_kv8_attention_many_scratch(ctas, d) || !counters ||
        (long long)counters_len < (long long)n_tiles * G * 2)
        return fail(HFB_EINVAL, "kv8_attention_many: %d CTAs need scratch and counters", ctas);
    Kv8ManyParams f = {};
    f.a.q = q; f.a.cache = (const uint8_t *)cache; f.a.out = out; f.a.block_table = block_table; f.a.positions = positions;
    f.a.tile_seq = tile_seq; f.a.tile_t0 = tile_t0; f.a.tile_nt = tile_nt; f.a.max_blocks = max_blocks; f.a.block_size = block_size;
    f.a.record = kv8_record_bytes(block_size, d); f.a.window = window; f.a.H = H; f.a.G = G; f.a.num_pages = num_pages; f.a.scale = scale;
    f.a.sinks = sinks; f.a.slopes = slopes; f.a.head_scales = head_scales; f.a.zero_sink = zero_sink; f.a.softcap = softcap > 0.f ? softcap : 0.f;
    f.per = KM_ROWS / (H / G); f.n_tiles = n_tiles; f.tile_cost = tile_cost; f.settled = settled;
    f.counters = counters;
    f.part_o = (float *)scratch; f.part_ml = (float *)scratch + (size_t)ctas * 4 * 128 * d;
    const int grid = ctas;
    return d == 128 ? launch_kv8_many<128>(f, grid, (cudaStream_t)s) : launch_kv8_many<64>(f, grid, (cudaStream_t)s);
}
