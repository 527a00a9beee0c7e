// Attention of few queries over the key/value cache in 8 bits (kv8.cuh): bfloat16, head sizes 64 and 128, pages of 8..64 tokens.
//
// What bounds it is reading the cache: d + 4 bytes a key, and as many a value.  A warp of its own keeps the copies going, one bulk copy per page
// and head (codes and scales of keys and values are one record), several tiles of 64 keys ahead of the warps that compute.
//
// Between the copy and the tensor core every byte has to become a 16-bit number, so that is what the layout serves:
// * A code's byte, code + 128, is a float16 number as it stands: with a zero byte above it the subnormal (code + 128) 2^-24.  A key
//   needs no more than that permutation of bytes, since q . (code + 128) = q . code + 128 sum(q), and the sum of a query's numbers is
//   known; the term is of the size that the largest scores have, so that float32 loses nothing that it would hold of those.
//   (Taken off the values in the same way it would be large beside an average of many; a value becomes 0x6400 | byte = 1024 + byte,
//   minus 1152: half a subtraction a number more.)  The scales stay out of the operands: a key's multiplies its score in float32, a
//   value's its weight.
// * Scores are computed as S^T = K Q^T and outputs as O^T = V^T P^T: the cache fills the 16 rows of mma.m16n8k16, the (token, head)
//   pairs that share it the 8 columns, so that up to eight of them cost one product and not half an empty one.  The numbers of
//   a K word (four neighbours of a row) go to places k = 2c, 2c+1, 2c+8, 2c+9 of one product, and the queries are loaded
//   in that order.  A transposing ldmatrix of value bytes gives two neighbouring numbers of two keys; the even ones make the product's
//   rows 0..7, the odd ones 8..15, so that a thread ends up with neighbours of the output.
// * A query row is multiplied by the power of two that brings its largest number to 2^14..2^15: float16 then holds every number
//   of it that matters exactly (eight bits, down to 2^-31 of the largest).
// * A weight goes into the second product as p * (scale of the value / reference scale) * 2^10, p relative to a reference maximum.  The
//   references are raised, and the sums so far rescaled, only when a score exceeds its by more than 2^4 or a scale by more than a
//   factor of two: the product is 2^15 at most, and is rounded once to float16 (11 bits; weights down to 2^-24 of the largest at
//   full precision, 2^-34 at all).  (Raised whenever a maximum grows, one of eight columns' did in more than half of the steps.)
// * The scales' reference is all columns', whatever each of them sees.  Where a scale lies more than 2^12 below it, the step's second product
//   is made up to four times, for weights of 2^-24 of each other: down to 2^-91 of the largest they keep their 11 bits, beside keys that
//   their token does not see or gives no weight.
//
// Measured (28 heads of 128 on 4): 64 requests of up to 8,192 tokens 70 us, 0.60 of the measured bandwidth (the bfloat16 cache's kernel, which
// reads twice the bytes, 108 us); eight of up to 32,768 tokens 43 us, 0.49 (59).  About 15 us of each are the start of a launch, its
// first copies and its merges, which a launch that follows another one on the stream hides in part.
//
// Work is cut evenly: all steps (64 keys of one tile and key/value head) stand in one row, a tile's behind `tile_cost` empty ones
// for its queries and its merge, and CTA c of C walks steps c N / C to (c + 1) N / C.  The copies run ahead from one tile's keys into the next
// one's, its queries included.  What a CTA has of a tile that others share goes to scratch, where a CTA has two places (a first and a last
// piece); the CTA that brings a tile's last piece merges them, in the order of the keys whoever it is.
#include <cuda_fp16.h>

#include "attention_common.cuh"
#include "kv8.cuh"
#include "tc_ptx.cuh"

static thread_local cudaError_t g_launch_err = cudaSuccess;      // what the last launch_pdl returned

namespace hfb {
int *error_word();

constexpr int KF_MAX_TILES = 2048;
constexpr float KF_APART = 0.000244140625f;          // 2^-12: value scales up to here below the reference go into the weights all at once

struct Kv8FewParams {
    Kv8Params a;
    float *part_o, *part_ml;             // pieces of tiles that several CTAs share: [CTAs, 2, columns, D] and [CTAs, 2, columns, 2]
    int *counters;                       // ... one per (tile, group of heads), zero between launches
    int n_tiles, min_steps, tile_cost;   // fewest steps that are worth a CTA; steps that beginning and ending a tile is reckoned as
    int kv_share;                        // neighbouring groups of heads that read the same key/value head (a.G counts the groups)
    int settled;                         // rows before the step's positions need no wait
};

__device__ __forceinline__ void bulk_prefetch(const void *src, uint32_t bytes)
{
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Two bytes of a word of codes (named by the selector, whose nibbles 4 name a zero) as two float16 numbers (code + 128) 2^-24.
__device__ __forceinline__ uint32_t bytes_f16(uint32_t w, uint32_t selector)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(selector));
    return r;
}
// Two bytes of a word of codes (named by the selector) as two float16 numbers.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t selector)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0x64646464u), "r"(selector));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));                // 1152
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// (the first product of a sum)
__device__ __forceinline__ void mma_f16_first(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D: head size; NT: columns (token, head) of a tile in eights; STAGES: tiles of 64 keys in flight; OPTS: a cap or slopes.  Two groups of four
// computing warps take the tiles in turn, a warp has 16 keys of each.
template <int D, int NT, int STAGES, bool OPTS, int CTAS>
__global__ void __launch_bounds__(32 * 9, CTAS)
kv8_few_kernel(Kv8FewParams f, int *err)
{
    const Kv8Params &p = f.a;
    // (a stage belongs to one of the two groups of warps: one that took turns on it could find the phase before its own complete)
    static_assert(STAGES % 2 == 0, "the groups of warps have stages of their own");
    constexpr int WARPS = 8, GROUP = WARPS / 2, THREADS = 32 * (WARPS + 1);
    constexpr int COLS = 8 * NT, CH = D / 16, OROW = D + 4;  // (rows of the merge buffer in different banks)
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
    uint8_t *gen = smem_raw + (base - smem_u32(smem_raw));
    const int bs = p.block_size, pages = ABN / bs;
    const uint32_t stage_bytes = (uint32_t)pages * p.record;
    // barriers, page masks and flags; the merge buffer; the tiles' first steps; the stages
    const uint32_t full0 = base, empty0 = base + 8 * STAGES;
    volatile uint32_t *page_mask = (volatile uint32_t *)(gen + 16 * STAGES);
    volatile int *abort_flag = (volatile int *)(gen + 20 * STAGES), *last_flag = abort_flag + 1;
    int *scan = (int *)(gen + 128);                           // [WARPS + 1], 9 at most
    // two slots for coming pieces: a barrier each for their queries' arrival and release, the tile's numbers, the queries
    const uint32_t q_full = base + 192, q_empty = base + 208;
    constexpr uint32_t Q_BYTES = COLS * D * 2, SLOT = 128 + Q_BYTES;
    float *mo = (float *)(gen + 256 + 2 * SLOT), *ml = mo + WARPS * COLS * OROW, *mv = ml + WARPS * COLS * 2;
    enum { I_T0, I_NT, I_POS_FIRST, I_POS_LAST, I_KT, I_LEN, I_HEADS, I_BEGINS, I_COUNTER, I_PIECES, I_PLACE, I_FIRST, I_FIRST_PLACE, I_POSITIONS = 16 };
    int *first_step = (int *)(mv + WARPS);                        // [n_tiles + 1]
    const uint32_t tiles0 = (base + 256 + 2 * SLOT + WARPS * (COLS * (OROW + 2) + 1) * 4 + 4 * (f.n_tiles + 1) + 127u) & ~127u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (!f.settled) pdl_wait();                               // nothing is read that the kernels in front may still write
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) { mbar_init(q_full + 8 * s, 1); mbar_init(q_empty + 8 * s, WARPS); }
        for (int s = 0; s < STAGES; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, GROUP); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }

    // The steps of one key/value head before each tile: every tile has one at least, which writes its zeros.
    struct Tile { int seq, t0, nt, pos_first, pos_last, lo_first, kt_lo, n; };
    auto tile_of = [&](int i) {
        Tile x;
        x.seq = p.tile_seq[i]; x.t0 = p.tile_t0[i];
        x.nt = max(1, min(p.tile_nt[i], COLS / (p.H / p.G)));      // (what the tile has places for)
        x.pos_first = p.positions[x.t0]; x.pos_last = p.positions[x.t0 + x.nt - 1];
        x.lo_first = mask_lo(x.pos_first, p.window);
        x.kt_lo = x.lo_first / ABN;
        x.n = x.pos_last < 0 ? 1 : max(1, x.pos_last / ABN + 1 - x.kt_lo);
        return x;
    };
    {
        const int each = (f.n_tiles + THREADS - 1) / THREADS, i0 = min((int)threadIdx.x * each, f.n_tiles), i1 = min(i0 + each, f.n_tiles);
        int sum = 0;
        for (int i = i0; i < i1; i++) { first_step[i] = sum; sum += tile_of(i).n + f.tile_cost; }
        int up = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, up, o); if (lane >= o) up += v; }
        if (lane == 31) scan[warp] = up;
        __syncthreads();
        int before = up - sum;
        for (int w = 0; w < warp; w++) before += scan[w];
        for (int i = i0; i < i1; i++) first_step[i] += before;
        if (threadIdx.x == THREADS - 1) first_step[f.n_tiles] = before + sum;
    }
    __syncthreads();
    const int groups = p.G, r = p.H / groups;
    const long long total = (long long)first_step[f.n_tiles] * groups;
    const int ctas = (int)max(1ll, min((long long)gridDim.x, total / f.min_steps)), cta = blockIdx.x;
    if (cta >= ctas) return;
    auto start_of = [&](int c) { return total * c / ctas; };
    const long long x_end = start_of(cta + 1);

    // A piece: steps off .. off + len of one tile and head, whose own steps begin at `first` (len 0: nothing but empty ones).
    struct Piece { int tile, g, n, off, len; long long first; };
    int tile_at = 0;
    auto piece_at = [&](long long &x, Piece &it) {
        if (tile_at == 0 || first_step[tile_at] * (long long)groups > x) {           // (the first one: search)
            int lo = 0, hi = f.n_tiles - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if ((long long)first_step[mid] * groups <= x) lo = mid; else hi = mid - 1;
            }
            tile_at = lo;
        }
        while ((long long)first_step[tile_at + 1] * groups <= x) tile_at++;
        const long long t_first = (long long)first_step[tile_at] * groups;
        it.tile = tile_at;
        const int all = first_step[tile_at + 1] - first_step[tile_at];
        it.tile = tile_at;
        it.n = all - f.tile_cost;
        it.g = (int)((x - t_first) / all);
        it.first = t_first + (long long)it.g * all + f.tile_cost;
        const long long begin = max(x, it.first);
        x = min(x_end, it.first + it.n);
        it.off = (int)(begin - it.first);
        it.len = (int)max(0ll, x - begin);
    };

    if (warp == WARPS) {
        // ---- the copying warp: the lanes look up 32 pages at a time, and each asks for its page -------------------------------
        const int tiles_per_round = 32 / pages, kv_heads = groups / f.kv_share;
        bool ok = true;
        int js = 0, number = 0;
        if (f.settled) {
            // what was written before the step may be on its way into L2 while the kernel in front still runs
            Piece it;
            long long x = start_of(cta);
            piece_at(x, it);
            const Tile tl = tile_of(it.tile);
            const int key0 = (tl.kt_lo + it.off) * ABN + lane * bs, blk = key0 / bs;
            if (lane < min(it.len, STAGES) * pages && key0 + bs <= tl.pos_first && key0 + bs > tl.lo_first && blk < p.max_blocks) {
                const long long page = p.block_table[(size_t)tl.seq * p.max_blocks + blk];
                if (page >= 0 && page < p.num_pages) bulk_prefetch(p.cache + ((size_t)page * kv_heads + it.g / f.kv_share) * p.record, p.record);
            }
            pdl_wait();
        }
        for (long long x = start_of(cta); x < x_end && ok;) {
            Piece it;
            piece_at(x, it);
            if (it.len == 0) continue;
            const Tile tl = tile_of(it.tile);
            {
                const int slot = number & 1;
                int *info = (int *)(gen + 256 + slot * SLOT);
                if (lane == 0) ok = mbar_wait(q_empty + 8 * slot, ((number >> 1) & 1) ^ 1, abort_flag, err);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (lane == 0) {
                    // the piece for the computing warps; of a tile's pieces only the first can be its CTA's last
                    const int c_first = (int)(((it.first + 1) * ctas - 1) / total);
                    info[I_T0] = tl.t0; info[I_NT] = tl.nt; info[I_POS_FIRST] = tl.pos_first; info[I_POS_LAST] = tl.pos_last;
                    info[I_KT] = tl.kt_lo + it.off; info[I_LEN] = it.len; info[I_HEADS] = it.g * r; info[I_BEGINS] = it.off == 0;
                    info[I_COUNTER] = it.tile * groups + it.g;
                    info[I_PIECES] = (int)(((it.first + it.n) * ctas - 1) / total) - c_first + 1;
                    info[I_PLACE] = cta * 2 + (start_of(cta) >= it.first ? 0 : 1);
                    info[I_FIRST] = c_first;
                    info[I_FIRST_PLACE] = c_first * 2 + (start_of(c_first) >= it.first ? 0 : 1);
                }
                if (lane < 16) info[I_POSITIONS + lane] = lane < tl.nt ? p.positions[tl.t0 + lane] : -1;
                __syncwarp();
                const uint32_t bytes = (uint32_t)r * D * 2;
                if (lane == 0) mbar_arrive_expect_tx(q_full + 8 * slot, tl.nt * bytes);
                __syncwarp();
                if (lane < tl.nt)
                    bulk_load(base + 256 + slot * SLOT + 128 + lane * bytes, (const __nv_bfloat16 *)p.q + ((size_t)(tl.t0 + lane) * p.H + it.g * r) * D,
                              bytes, q_full + 8 * slot);
                number++;
            }
            const int32_t *table = p.block_table + (size_t)tl.seq * p.max_blocks;
            const int kv_g = it.g / f.kv_share, kt_first = tl.kt_lo + it.off, kt_end = kt_first + it.len;
            for (int kt0 = kt_first; kt0 < kt_end && ok; kt0 += tiles_per_round) {
                const int key0 = kt0 * ABN + lane * bs, blk = key0 / bs;
                const bool wanted = lane < tiles_per_round * pages && kt0 + lane / pages < kt_end && key0 <= tl.pos_last && key0 + bs > tl.lo_first;
                const long long page = wanted && blk < p.max_blocks ? table[blk] : -1;
                const bool there = page >= 0 && page < p.num_pages;
                if (wanted && !there) atomicOr(err, HFB_ERR_PAGE);
                const uint32_t have = __ballot_sync(0xffffffffu, there);
                const uint8_t *src = p.cache + ((size_t)(there ? page : 0) * kv_heads + kv_g) * p.record;
                for (int t = 0; t < tiles_per_round && kt0 + t < kt_end && ok; t++, js++) {
                    const int s = js % STAGES;
                    const uint32_t mine = (have >> (t * pages)) & ((1u << pages) - 1u);
                    if (lane == 0) {
                        ok = mbar_wait(empty0 + 8 * s, ((js / STAGES) & 1) ^ 1, abort_flag, err);
                        if (ok) {
                            page_mask[s] = mine;
                            mbar_arrive_expect_tx(full0 + 8 * s, __popc(mine) * p.record);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (ok && there && lane / pages == t)
                        bulk_load(tiles0 + s * stage_bytes + (lane % pages) * p.record, src, p.record, full0 + 8 * s);
                }
            }
        }
        // the end of the row
        if (lane == 0 && ok && mbar_wait(q_empty + 8 * (number & 1), ((number >> 1) & 1) ^ 1, abort_flag, err)) {
            ((int *)(gen + 256 + (number & 1) * SLOT))[I_LEN] = 0;
            mbar_arrive(q_full + 8 * (number & 1));
        }
    } else {
        // ---- the computing warps --------------------------------------------------------------------------------------------
        if (f.settled) pdl_wait();                            // the queries come from the kernel in front
        pdl_trigger();
        const float log2e = 1.4426950408889634f, cap2 = p.softcap * log2e;
        const bool capped = p.softcap > 0.f;
        const int c4 = lane & 3, row8 = lane >> 2;
        const int kbase = (warp % GROUP) * 16, group = warp / GROUP;
        // ldmatrix: lanes 0..7 and 8..15 name the rows of two eights of keys, the upper lanes the same rows one piece further; this lane
        // holds the scores of the keys `row8` and `row8 + 8` of the warp's sixteen
        const int turn = D == 128 ? lane & 7 : (lane & 7) >> 1;
        uint32_t piece[CH / 2], s_at[2];
        const int kk = kbase + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int c = 0; c < CH / 2; c++)
            piece[c] = (uint32_t)(kk / bs) * p.record + (uint32_t)(kk % bs) * D + (uint32_t)((2 * c + (lane >> 4)) ^ turn) * 16u;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int k = kbase + 8 * u + row8;
            s_at[u] = (uint32_t)(k / bs) * p.record + 2u * bs * D + 4u * (k % bs);
        }
        const uint32_t v_codes = (uint32_t)bs * D, v_scales = 4u * bs;
        const uint32_t all_pages = (1u << pages) - 1u;
        int js = 0;

        for (int number = 0;; number++) {
            const int *info = (const int *)(gen + 256 + (number & 1) * SLOT);
            bool ok = mbar_wait(q_full + 8 * (number & 1), (number >> 1) & 1, abort_flag, err);
            {
                // (a wait that ran out ends the walk of all warps together: none may be left at a barrier)
                int all;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                             : "=r"(all) : "r"((int)ok), "n"(32 * WARPS) : "memory");
                if (!all) break;
            }
            const int len = info[I_LEN], nt = info[I_NT], heads = info[I_HEADS];
            if (len == 0) break;
            const int pos_first = info[I_POS_FIRST], pos_last = info[I_POS_LAST], kt_first = info[I_KT];
            const int lo_first = mask_lo(pos_first, p.window), lo_last = mask_lo(pos_last, p.window);
            uint32_t qf[CH][NT][2];
            float fac[NT][2], off[NT][2], slope[NT][2];
            int pos[NT][2], lo[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                // this lane's share of column 8 n + lane / 4: numbers 16 c + 4 (lane % 4) + 0..3
                const int col = 8 * n + row8, tok = col / r, hl = col % r;
                const bool valid = tok < nt;
                const uint8_t *src = (const uint8_t *)(info + 32) + (valid ? col : 0) * D * 2 + 8 * c4;
                uint2 raw[CH];
                unsigned top = 0;
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    raw[c] = valid ? *(const uint2 *)(src + 32 * c) : make_uint2(0, 0);
                    top = max(top, max(max(raw[c].x & 0x7fffu, (raw[c].x >> 16) & 0x7fffu), max(raw[c].y & 0x7fffu, (raw[c].y >> 16) & 0x7fffu)));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const unsigned field = min(268u - (top >> 7), 253u);              // exponent field of the power of two
                const float by = __uint_as_float(field << 23), back = __uint_as_float((254u - field) << 23);
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < CH; c++) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t w = u ? raw[c].y : raw[c].x;
                        qf[c][n][u] = pack_f16(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xffff0000u) * by);
                        const float2 q = __half22float2(*(const __half2 *)&qf[c][n][u]);
                        sum += q.x + q.y;
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const float hs = p.head_scales && valid ? p.head_scales[heads + hl] : 1.f;
                const float unit = (capped ? p.scale * hs / p.softcap : p.scale * hs * log2e) * back, own_off = -128.f * sum * unit;
                const float own = unit * 16777216.f;
                const float sl = p.slopes && valid ? p.slopes[heads + hl] * log2e : 0.f;
                const int ps = valid ? info[I_POSITIONS + tok] : -1;
#pragma unroll
                for (int i = 0; i < 2; i++) {                 // ... and of the columns whose scores it will hold
                    fac[n][i] = __shfl_sync(0xffffffffu, own, 4 * (2 * c4 + i));
                    off[n][i] = __shfl_sync(0xffffffffu, own_off, 4 * (2 * c4 + i));
                    slope[n][i] = __shfl_sync(0xffffffffu, sl, 4 * (2 * c4 + i));
                    pos[n][i] = __shfl_sync(0xffffffffu, ps, 4 * (2 * c4 + i));
                    lo[n][i] = mask_lo(pos[n][i], p.window);
                }
            }
            float o[CH][NT][4], m[NT][2], l[NT][2], vm = 0.f, rv = 0.f;           // rv = 1 / vm
#pragma unroll
            for (int n = 0; n < NT; n++) {
                m[n][0] = m[n][1] = -INFINITY;
                l[n][0] = l[n][1] = 0.f;
#pragma unroll
                for (int c = 0; c < CH; c++) o[c][n][0] = o[c][n][1] = o[c][n][2] = o[c][n][3] = 0.f;
            }
            const int skip = (js ^ group) & 1;
            for (int j = skip; j < len; j += 2) {
                const int kt = kt_first + j, s = (js + j) % STAGES;
                ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, ((js + j) / STAGES) & 1, abort_flag, err)) && ok;   // (lanes go on together)
                if (!ok) continue;
                const uint32_t st = tiles0 + s * stage_bytes, sv = st + v_codes;
                const uint8_t *sg = gen + (tiles0 - base) + s * stage_bytes;
                const uint32_t mask = page_mask[s];
                // (two sums a score, of the even and the odd pieces of a row: a chain of products half as long)
                float sc[NT][4], sd[NT][4];
#pragma unroll
                for (int c = 0; c < CH / 2; c++) {
                    uint32_t w0, w1, w2, w3;
                    ldsm_x4(st + piece[c], w0, w1, w2, w3);
                    const uint32_t a0 = bytes_f16(w0, 0x4140), a1 = bytes_f16(w1, 0x4140), a2 = bytes_f16(w0, 0x4342), a3 = bytes_f16(w1, 0x4342);
                    const uint32_t b0 = bytes_f16(w2, 0x4140), b1 = bytes_f16(w3, 0x4140), b2 = bytes_f16(w2, 0x4342), b3 = bytes_f16(w3, 0x4342);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (c == 0) {
                            mma_f16_first(sc[n], a0, a1, a2, a3, qf[0][n][0], qf[0][n][1]);
                            mma_f16_first(sd[n], b0, b1, b2, b3, qf[1][n][0], qf[1][n][1]);
                        } else {
                            mma_f16(sc[n], a0, a1, a2, a3, qf[2 * c][n][0], qf[2 * c][n][1]);
                            mma_f16(sd[n], b0, b1, b2, b3, qf[2 * c + 1][n][0], qf[2 * c + 1][n][1]);
                        }
                    }
                }
                float ks[2], vs[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    ks[u] = *(const float *)(sg + s_at[u]);
                    vs[u] = *(const float *)(sg + s_at[u] + v_scales);
                }
                // a tile wholly inside every row's range, with all of its pages, needs no mask
                const bool edge = kt * ABN + ABN - 1 > pos_first || kt * ABN < lo_last || mask != all_pages;
                if (edge) {
                    // (rows behind the request's last, those that every token's mask has passed and missing pages hold anything)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int k = kbase + 8 * u + row8;
                        if (kt * ABN + k > pos_last || kt * ABN + k < lo_first || !(mask >> (k / bs) & 1u)) { ks[u] = 0.f; vs[u] = vm; }
                    }
                }
                const float vs_top = fmaxf(vs[0], vs[1]);
                const float vs_low = fminf(vs[0], vs[1]);
                bool apart = false;
                if (__any_sync(0xffffffffu, vs_top > 2.f * vm || vs_low < KF_APART * vm)) {
                    if (__any_sync(0xffffffffu, vs_top > 2.f * vm)) {
                        float v = fmaxf(vm, vs_top);
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                        const float shrink = vm / v;
#pragma unroll
                        for (int c = 0; c < CH; c++)
#pragma unroll
                            for (int n = 0; n < NT; n++) { o[c][n][0] *= shrink; o[c][n][1] *= shrink; o[c][n][2] *= shrink; o[c][n][3] *= shrink; }
                        vm = v;
                        rv = 1.0f / v;
                    }
                    apart = __any_sync(0xffffffffu, vs_low < KF_APART * vm);
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[n][e] = fmaf(sc[n][e] + sd[n][e], fac[n][e & 1], off[n][e & 1]) * ks[e >> 1];
                if (OPTS) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int key = kt * ABN + kbase + 8 * (e >> 1) + row8;
                            if (capped) sc[n][e] = cap2 * tanh_fast(sc[n][e]);
                            sc[n][e] = fmaf(slope[n][e & 1], (float)(key - pos[n][e & 1]), sc[n][e]);
                        }
                }
                if (edge) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int k = kbase + 8 * (e >> 1) + row8, key = kt * ABN + k;
                            if (key > pos[n][e & 1] || key < lo[n][e & 1] || !(mask >> (k / bs) & 1u)) sc[n][e] = -INFINITY;
                        }
                }
                float top[NT][2];
                bool grew = false;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        top[n][i] = fmaxf(sc[n][i], sc[n][2 + i]);
                        grew |= top[n][i] > m[n][i] + 4.f;
                    }
                if (__any_sync(0xffffffffu, grew)) {
                    // a maximum has outgrown its reference somewhere in the warp: rescale what has been summed so far
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float v = fmaxf(m[n][i], top[n][i]);
                            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                            const float corr = fast_exp2(m[n][i] - (v == -INFINITY ? 0.f : v));
                            l[n][i] *= corr;
#pragma unroll
                            for (int c = 0; c < CH; c++) { o[c][n][i] *= corr; o[c][n][2 + i] *= corr; }
                            m[n][i] = v;
                        }
                }
                const float vn0 = vs[0] * rv * 1024.f, vn1 = vs[1] * rv * 1024.f;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = e & 1;
                        const bool none = edge && sc[n][e] == -INFINITY;
                        const float q = fast_exp2(sc[n][e] - (m[n][i] == -INFINITY ? 0.f : m[n][i]));
                        l[n][i] += q;
                        sc[n][e] = q * (e < 2 ? vn0 : vn1);
                        if (none) sc[n][e] = 0.f;                            // (a value that is no number, for a row that does not see it)
                    }
                }
                // the weights in float16: all at once, or those down to 2^-24 of the largest there can be, the next 2^-24 with the sums so far (and
                // themselves) 2^24 times as large, and so on
                int times = 0;
#pragma unroll 1
                for (;;) {
                    uint32_t pf[NT][2];
                    bool more = false;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (apart) {
                            float w[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const bool small = sc[n][e] < 0.001953125f;           // 2^-9
                                w[e] = small ? 0.f : sc[n][e];
                                sc[n][e] = small ? sc[n][e] * 16777216.f : 0.f;
                                more |= sc[n][e] != 0.f;
                            }
                            pf[n][0] = transpose8(pack_f16(w[0], w[1]));
                            pf[n][1] = transpose8(pack_f16(w[2], w[3]));
                        } else {
                            pf[n][0] = transpose8(pack_f16(sc[n][0], sc[n][1]));
                            pf[n][1] = transpose8(pack_f16(sc[n][2], sc[n][3]));
                        }
                    }
#pragma unroll
                    for (int c = 0; c < CH / 2; c++) {
                        uint32_t w0, w1, w2, w3;
                        ldsm_x4_t(sv + piece[c], w0, w1, w2, w3);
                        const uint32_t a0 = codes_f16(w0, 0x4240), a1 = codes_f16(w0, 0x4341), a2 = codes_f16(w1, 0x4240), a3 = codes_f16(w1, 0x4341);
                        const uint32_t b0 = codes_f16(w2, 0x4240), b1 = codes_f16(w2, 0x4341), b2 = codes_f16(w3, 0x4240), b3 = codes_f16(w3, 0x4341);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            mma_f16(o[2 * c][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                            mma_f16(o[2 * c + 1][n], b0, b1, b2, b3, pf[n][0], pf[n][1]);
                        }
                    }
                    if (!apart) break;
                    more = __any_sync(0xffffffffu, more) && times < 3;
                    const float by = more ? 16777216.f : __uint_as_float((uint32_t)(127 - 24 * times) << 23);
#pragma unroll
                    for (int c = 0; c < CH; c++)
#pragma unroll
                        for (int n = 0; n < NT; n++) { o[c][n][0] *= by; o[c][n][1] *= by; o[c][n][2] *= by; o[c][n][3] *= by; }
                    if (!more) break;
                    times++;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty0 + 8 * s);
            }
            js += len;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 4);
                    l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 8);
                    l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 16);
                    // ---- merge the warps (they saw disjoint keys) in warp order
                    const int col = 8 * n + 2 * c4 + i;
#pragma unroll
                    for (int c = 0; c < CH; c++)
                        *(float2 *)(mo + (warp * COLS + col) * OROW + 16 * c + 2 * row8) = make_float2(o[c][n][i], o[c][n][2 + i]);
                    if (row8 == 0) *(float2 *)(ml + (warp * COLS + col) * 2) = make_float2(m[n][i], l[n][i]);
                }
            if (lane == 0) mv[warp] = vm;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
            const int rows = nt * r, t0 = info[I_T0], pieces = info[I_PIECES], place = info[I_PLACE];
            const bool whole = pieces == 1;
            float top_v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) top_v = fmaxf(top_v, mv[w]);
            for (int idx = threadIdx.x; idx < rows * (D / 4); idx += 32 * WARPS) {
                const int row = idx / (D / 4), q4 = idx % (D / 4);
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < WARPS; w++) top = fmaxf(top, ml[(w * COLS + row) * 2]);
                float denom = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < WARPS; w++) {
                    const float mw = ml[(w * COLS + row) * 2];
                    const float e = mw == -INFINITY ? 0.f : fast_exp2(mw - top);
                    denom += ml[(w * COLS + row) * 2 + 1] * (mw == -INFINITY ? 1.f : e);       // (zero, or no number)
                    const float fo = mv[w] == 0.f ? 0.f : e * (mv[w] / top_v);
                    const float4 v = *(const float4 *)(mo + (w * COLS + row) * OROW + 4 * q4);
                    acc.x += v.x * fo; acc.y += v.y * fo; acc.z += v.z * fo; acc.w += v.w * fo;
                }
                const float unit = top_v * (1.f / 1024.f);
                acc.x *= unit; acc.y *= unit; acc.z *= unit; acc.w *= unit;
                const int head = heads + row % r;
                if ((p.sinks || p.zero_sink) && info[I_BEGINS]) {
                    // the sink joins the first piece's sum as one more score; the merge of the pieces carries it like any other
                    const float sk = p.sinks ? p.sinks[head] * log2e : 0.f;
                    const float t = fmaxf(top, sk);
                    const float e = top == -INFINITY ? 0.f : exp2f(top - t);
                    denom = denom * (top == -INFINITY ? 1.f : e) + exp2f(sk - t);
                    acc.x *= e; acc.y *= e; acc.z *= e; acc.w *= e;
                    top = t;
                }
                if (whole) {
                    const float inv = denom == 0.f ? 0.f : 1.0f / denom;
                    *(uint2 *)((__nv_bfloat16 *)p.out + ((size_t)(t0 + row / r) * p.H + head) * D + 4 * q4) =
                        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
                } else {
                    *(float4 *)(f.part_o + ((size_t)place * COLS + row) * D + 4 * q4) = acc;
                    if (q4 == 0) *(float2 *)(f.part_ml + ((size_t)place * COLS + row) * 2) = make_float2(top, denom);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");    // the buffer is free again
            // ---- merge the pieces: whoever stored its piece last, in the order of the keys ----------------------------------------
            bool last = false;
            const int c_first = info[I_FIRST], first_place = info[I_FIRST_PLACE];
            if (!whole) {
                if (threadIdx.x == 0) {
                    __threadfence();                          // (after the barrier: it covers every thread's stores)
                    int *cnt = f.counters + info[I_COUNTER];
                    const int is = atomicAdd(cnt, 1) == pieces - 1;
                    if (is) *cnt = 0;
                    *last_flag = is;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
                last = *last_flag;                            // (written again behind two barriers)
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(q_empty + 8 * (number & 1));
            if (!last) continue;
            __threadfence();
            for (int idx = threadIdx.x; idx < rows * (D / 4); idx += 32 * WARPS) {
                const int row = idx / (D / 4), q4 = idx % (D / 4);
                float top = -INFINITY, denom = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int c = 0; c < pieces; c += 8) {         // eight reads in flight
                    float2 w[8];
                    float4 v[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        // (of the pieces only the first can be its CTA's last)
                        const size_t at = (size_t)(c + i == 0 ? first_place : (c_first + c + i) * 2) * COLS + row;
                        w[i] = c + i < pieces ? __ldcg((const float2 *)(f.part_ml + at * 2)) : make_float2(-INFINITY, 0.f);
                        v[i] = c + i < pieces ? __ldcg((const float4 *)(f.part_o + at * D) + q4) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    float t = top;
#pragma unroll
                    for (int i = 0; i < 8; i++) t = fmaxf(t, w[i].x);
                    if (top != -INFINITY) { const float e = exp2f(top - t); denom *= e; acc.x *= e; acc.y *= e; acc.z *= e; acc.w *= e; }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float e = w[i].x == -INFINITY ? 0.f : exp2f(w[i].x - t);
                        denom += w[i].y * (w[i].x == -INFINITY ? 1.f : e);
                        acc.x += v[i].x * e; acc.y += v[i].y * e; acc.z += v[i].z * e; acc.w += v[i].w * e;
                    }
                    top = t;
                }
                const float inv = denom == 0.f ? 0.f : 1.0f / denom;
                *(uint2 *)((__nv_bfloat16 *)p.out + ((size_t)(t0 + row / r) * p.H + heads + row % r) * D + 4 * q4) =
                    make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
            }
        }
    }
    __syncthreads();
    if (*abort_flag != 0 && threadIdx.x == 0)                 // a wait ran out: copies still in flight land before the shared memory goes away
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    __syncthreads();
}

template <int D, int NT, int STAGES, int CTAS, bool OPTS>
static int launch_kv8_few_opts(const Kv8FewParams &f, int ctas, cudaStream_t st)
{
    constexpr int fixed = 128 + 256 + 2 * (128 + 8 * NT * D * 2) + 8 * (8 * NT * (D + 6) + 1) * 4 + 128;
    constexpr int most = fixed + 4 * (KF_MAX_TILES + 1) + STAGES * ABN * (2 * D + 8);
    const int smem = fixed + 4 * (f.n_tiles + 1) + STAGES * (ABN / f.a.block_size) * f.a.record;
    const auto kernel = kv8_few_kernel<D, NT, STAGES, OPTS, CTAS>;
    static bool configured[64] = {false};                     // (the opt-in is a property of the function on one device)
    if (!configured[current_device()]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return fail(HFB_ECUDA, "kv8_attention_few: cannot opt in to %d bytes of shared memory: %s", most, cudaGetErrorString(e));
        configured[current_device()] = true;
    }
    g_launch_err = launch_pdl(kernel, dim3(ctas), dim3(32 * 9), smem, st, f, error_word());
    return check_pdl_launch(g_launch_err, "kv8_attention_few");
}

template <int D, int NT, int STAGES, int CTAS>
static int launch_kv8_few(const Kv8FewParams &f, int ctas, cudaStream_t st)
{
    return f.a.slopes || f.a.softcap > 0.f ? launch_kv8_few_opts<D, NT, STAGES, CTAS, true>(f, ctas, st)
                                           : launch_kv8_few_opts<D, NT, STAGES, CTAS, false>(f, ctas, st);
}

}  // namespace hfb

using namespace hfb;

extern "C" size_t hfb_kv8_attention_few_scratch(int ctas, int d) { return (size_t)ctas * 2 * 16 * (d + 2) * sizeof(float); }
extern "C" int hfb_kv8_attention_few_tiles(void) { return KF_MAX_TILES; }

extern "C" int hfb_kv8_attention_few(const void *q, const void *cache, const int32_t *block_table, int max_blocks, const int32_t *positions,
                                     const int32_t *tile_seq, const int32_t *tile_t0, const int32_t *tile_nt, int n_tiles, int tile_tokens,
                                     int ctas, int min_steps, int tile_cost, int settled, int block_size, int64_t num_pages, int window, float scale, void *out,
                                     void *scratch, size_t scratch_bytes, int *counters, int counters_len, int H, int G, int d,
                                     const float *sinks, int zero_sink, const float *slopes, const float *head_scales, float softcap, hfb_stream s)
{
    if (n_tiles <= 0) return HFB_OK;
    if (d != 64 && d != 128) return fail(HFB_ENOTSUP, "kv8_attention_few: head size %d (64 and 128 only)", d);
    if (n_tiles > KF_MAX_TILES) return fail(HFB_ENOTSUP, "kv8_attention_few: %d tiles (%d at most)", n_tiles, KF_MAX_TILES);
    if (H <= 0 || G <= 0 || H % G || max_blocks <= 0 || num_pages < 0 || tile_tokens < 1)
        return fail(HFB_EINVAL, "kv8_attention_few: bad arguments (H=%d G=%d)", H, G);
    if (block_size < 8 || block_size > ABN || ABN % block_size) return fail(HFB_ENOTSUP, "kv8_attention_few: pages of %d tokens (8, 16, 32 and 64)", block_size);
    // more heads on a key/value head than a tile has columns: as several groups that read the same keys and values
    int share = 1;
    while (H / G > 16 * share || (H / G) % share) share++;
    const int groups = G * share, cols = tile_tokens * (H / groups);
    if (cols > 16 || (tile_tokens > 1 && share > 1)) return fail(HFB_EINVAL, "kv8_attention_few: tiles of %d tokens of %d heads", tile_tokens, H / groups);
    if (ctas < 1 || min_steps < 1 || tile_cost < 0) return fail(HFB_EINVAL, "kv8_attention_few: bad CTA count");
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 7) || ((uintptr_t)cache & 15) || ((uintptr_t)scratch & 15))
        return fail(HFB_EINVAL, "kv8_attention_few: misaligned arrays");
    if (!scratch || scratch_bytes < hfb_kv8_attention_few_scratch(ctas, d) || !counters || (long long)counters_len < (long long)n_tiles * groups)
        return fail(HFB_EINVAL, "kv8_attention_few: %d CTAs need scratch and counters", ctas);
    Kv8FewParams f = {};
    f.a.q = q; f.a.cache = (const uint8_t *)cache; f.a.out = out; f.a.block_table = block_table; f.a.positions = positions;
    f.a.tile_seq = tile_seq; f.a.tile_t0 = tile_t0; f.a.tile_nt = tile_nt; f.a.max_blocks = max_blocks; f.a.block_size = block_size;
    f.a.record = kv8_record_bytes(block_size, d); f.a.window = window; f.a.H = H; f.a.G = groups; f.a.num_pages = num_pages; f.a.scale = scale;
    f.a.sinks = sinks; f.a.slopes = slopes; f.a.head_scales = head_scales; f.a.zero_sink = zero_sink; f.a.softcap = softcap > 0.f ? softcap : 0.f;
    f.part_o = (float *)scratch; f.part_ml = (float *)scratch + (size_t)ctas * 2 * 16 * d;
    f.counters = counters; f.n_tiles = n_tiles; f.min_steps = min_steps; f.tile_cost = tile_cost; f.kv_share = share; f.settled = settled;
    cudaStream_t st = (cudaStream_t)s;
    if (d == 128) return cols <= 8 ? launch_kv8_few<128, 1, 4, 2>(f, ctas, st) : launch_kv8_few<128, 2, 4, 1>(f, ctas, st);
    return cols <= 8 ? launch_kv8_few<64, 1, 4, 2>(f, ctas, st) : launch_kv8_few<64, 2, 4, 2>(f, ctas, st);
}
