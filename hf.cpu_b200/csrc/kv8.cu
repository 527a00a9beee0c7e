// The key/value cache in 8 bits (kv8.cuh): rows written to it, pages read back, and attention over it, plain kernel.
#include "kv8.cuh"
#include "tc_ptx.cuh"

static thread_local cudaError_t g_launch_err = cudaSuccess;      // what the last launch_pdl returned

namespace hfb {
int *error_word();

// Code i of a word as a number: the byte under 2^23's exponent is 2^23 + code + 128.  (Conversions between whole numbers and floats run at a
// quarter of the additions' rate.)
__device__ __forceinline__ float kv8_number(uint32_t word, int i)
{
    return __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440u + i)) - 8388736.f;
}

// ---- write ---------------------------------------------------------------------------------------------------------------
// Rows q | k | v of a step: queries and keys are rotated; queries go out in the run's type, keys and values into the cache.
//
// A key is rotated to twice float32's precision and a value next to a border between two codes is made and divided again in float64: the
// products of a 24-bit number with the table's float32 are exact there, so that the codes are those of the definition and a row's
// codes don't depend on the kernel that made them.  (Plain float32 would move about one code in 10^5 to its neighbour.)  Queries are
// rotated as the other kernels rotate them.
//
// A row belongs to `lanes` (a power of two) neighbouring lanes, each with PER consecutive numbers of it.
struct Kv8WriteParams {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;          // elements from one token's rows to the next one's
    const float *cos_sin;
    const int32_t *positions, *slots;
    void *q_out;
    uint8_t *cache;
    long long cache_slots;
    int n_rot, n_positions, interleaved, T, H, G, d, block_size, record, lanes, turns;
};

template <typename T, int PER> struct alignas(sizeof(T) * PER) Kv8Pack { T e[PER]; };

// x c + y s in float64: exact products, one rounding.  (A pair's first number is turned with -s, its second with s; a number that is not
// turned has c = 1, s = y = 0.)
__device__ __forceinline__ double kv8_turned(float x, float y, float c, float s) { return fma((double)x, (double)c, (double)y * s); }
// The same in float32, rounded once from a sum of twice the precision (products and their errors, the sum and its error).
__device__ __forceinline__ float kv8_turned_f32(float x, float y, float c, float s)
{
    const float p = __fmul_rn(x, c), q = __fmul_rn(y, s), pe = __fmaf_rn(x, c, -p), qe = __fmaf_rn(y, s, -q);
    const float sum = __fadd_rn(p, q), part = __fsub_rn(sum, p);
    const float err = __fadd_rn(__fsub_rn(p, __fsub_rn(sum, part)), __fsub_rn(q, part));
    return __fadd_rn(sum, __fadd_rn(err, __fadd_rn(pe, qe)));
}
// What few numbers need stays out of the way of the others.  The whole number is read off the low bits (code + 1.5 * 2^23).
__device__ __noinline__ float kv8_code_at_border(float x, float y, float c, float s, float scale)
{
    return (float)rint(kv8_turned(x, y, c, s) / (double)scale) + 12582912.f;
}
__device__ __noinline__ float kv8_turned_tiny(float x, float y, float c, float s) { return (float)kv8_turned(x, y, c, s); }

// Every head of a token is turned by the same table row, so that a lane reads its (cos, sin) once; a block takes 8 * 32 / lanes heads at a
// time, `turns` times, with the next ones' rows on their way.
constexpr int KV8_WRITE_THREADS = 256, KV8_WRITE_WARPS = KV8_WRITE_THREADS / 32;

template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(KV8_WRITE_THREADS)
kv8_write_kernel(Kv8WriteParams p, int *err)
{
    // the successor may start once the kernel in front of this one is done: then all that was written to the cache before
    // this step is there for it, and its own wait covers what this kernel writes
    pdl_sync();
    const int lane = threadIdx.x & 31, per_warp = 32 / p.lanes, heads = p.H + 2 * p.G, t = blockIdx.x;
    const int sub = lane / p.lanes, l = lane % p.lanes, e0 = l * PER, half = p.n_rot / 2;
    // where the numbers' partners are; which numbers are turned, and which are their pairs' second (VEC: all of a lane's are turned or none)
    const int partner = p.interleaved ? e0 : e0 < half ? e0 + half : e0 - half;
    auto turned = [&](int i) { return (VEC ? e0 : e0 + i) < p.n_rot; };
    auto second = [&](int i) { return p.interleaved ? (i & 1) != 0 : (VEC ? e0 : e0 + i) >= half; };
    const int first_head = (blockIdx.y * p.turns * KV8_WRITE_WARPS + (threadIdx.x >> 5)) * per_warp + sub, step = KV8_WRITE_WARPS * per_warp;
    Kv8Pack<T, PER> a, b;                                    // the coming row's numbers and their partners
    auto load = [&](int head) {
        if (head >= heads || e0 >= p.d) return;
        const T *row = head < p.H ? (const T *)p.q + t * p.q_stride + (size_t)head * p.d
                     : head < p.H + p.G ? (const T *)p.k + t * p.k_stride + (size_t)(head - p.H) * p.d
                                        : (const T *)p.v + t * p.v_stride + (size_t)(head - p.H - p.G) * p.d;
        const bool rotate = e0 < p.n_rot && head < p.H + p.G;
        if (VEC) {                                           // (all of a lane's numbers are turned or none, all are first or all second)
            a = *(const Kv8Pack<T, PER> *)(row + e0);
            if (rotate && !p.interleaved) b = *(const Kv8Pack<T, PER> *)(row + partner);
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                a.e[i] = row[e0 + i];
                if (rotate && turned(i)) b.e[i] = row[p.interleaved ? (e0 + i) ^ 1 : second(i) ? e0 + i - half : e0 + i + half];
            }
        }
    };
    load(first_head);
    int slot = p.slots ? p.slots[t] : -1;
    float c[PER], s[PER];                                    // (s: of a pair's first number with the sign turned)
#pragma unroll
    for (int i = 0; i < PER; i++) { c[i] = 1.f; s[i] = 0.f; }
    if (p.n_rot > 0) {
        int pos = p.positions[t];
        if (pos < 0 || pos >= p.n_positions) { if (threadIdx.x == 0) atomicOr(err, HFB_ERR_POSITION); pos = 0; }
        const float2 *cs = (const float2 *)(p.cos_sin + (size_t)pos * p.n_rot);
        if (VEC) {
            if (e0 < p.n_rot) {
                cs += p.interleaved ? e0 / 2 : e0 < half ? e0 : e0 - half;
#pragma unroll
                for (int i = 0; i < PER; i += 2) {
                    if (p.interleaved) { const float2 v = cs[i / 2]; c[i] = c[i + 1] = v.x; s[i] = -v.y; s[i + 1] = v.y; }
                    else {
                        const float4 v = *(const float4 *)(cs + i);
                        c[i] = v.x; c[i + 1] = v.z;
                        s[i] = e0 < half ? -v.y : v.y; s[i + 1] = e0 < half ? -v.w : v.w;
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (turned(i)) {
                    const float2 v = cs[p.interleaved ? (e0 + i) / 2 : second(i) ? e0 + i - half : e0 + i];
                    c[i] = v.x;
                    s[i] = second(i) ? v.y : -v.y;
                }
        }
    }
    if (slot >= p.cache_slots) { if (threadIdx.x == 0) atomicOr(err, HFB_ERR_SLOT); slot = -1; }
    const int in_page = slot >= 0 ? slot % p.block_size : 0;
    uint8_t *page = p.cache + (size_t)(slot >= 0 ? slot / p.block_size : 0) * p.G * p.record;
    for (int n = 0; n < p.turns; n++) {
        const int head = first_head + n * step;
        const bool is_q = head < p.H, is_k = !is_q && head < p.H + p.G;
        const bool work = head < heads && e0 < p.d && (is_q || slot >= 0);
        const bool rotate = p.n_rot > 0 && (is_q || is_k);
        float x[PER], y[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            x[i] = to_f32(a.e[i]);
            y[i] = VEC && p.interleaved ? to_f32(a.e[i ^ 1]) : to_f32(b.e[i]);
        }
        if (n + 1 < p.turns) load(head + step);
        if (work && is_q) {
            Kv8Pack<T, PER> o;
#pragma unroll
            for (int i = 0; i < PER; i++)                    // (the arithmetic of rope_pair)
                o.e[i] = from_f32<T>(rotate && turned(i) ? __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i])) : x[i]);
            T *dst = (T *)p.q_out + ((size_t)t * p.H + head) * p.d + e0;
            if (VEC) *(Kv8Pack<T, PER> *)dst = o;
            else
#pragma unroll
                for (int i = 0; i < PER; i++) dst[i] = o.e[i];
        }
        if (!__any_sync(0xffffffffu, work && !is_q)) continue;
        // keys and values: every lane of the row takes part in finding its largest magnitude (as bits: NaN > inf > finite)
        float z[PER];
        unsigned top = 0;
        if (work && !is_q) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (!(rotate && turned(i))) y[i] = 0.f;
                z[i] = rotate && turned(i) ? kv8_turned_f32(x[i], y[i], c[i], s[i]) : x[i];
                top = max(top, __float_as_uint(z[i]) & 0x7fffffffu);
            }
        }
        for (int o = p.lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // (rows below 2^-80: the products' errors leave float32's range; above 2^120 their sums may)
        const bool wild = work && is_k && rotate && (top < (47u << 23) || top > (247u << 23));
        if (__any_sync(0xffffffffu, wild)) {
            if (wild) {
                top = 0;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    if (turned(i)) z[i] = kv8_turned_tiny(x[i], y[i], c[i], s[i]);
                    top = max(top, __float_as_uint(z[i]) & 0x7fffffffu);
                }
            }
            for (int o = p.lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (work && !is_q) {
            const bool finite = top < 0x7f800000u;
            const float scale = finite ? fmaxf(__fdiv_rn(__uint_as_float(top), 127.f), 1.17549435e-38f) : __uint_as_float(0x7fc00000u);
            const float inv = finite ? 1.0f / scale : 0.f;
            float r[PER];
            bool border = false;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                // (1.5 * 2^23 added: rounded to a whole number; u is off by at most 127 * 3 * 2^-24 = 2.3e-5)
                const float u = finite ? z[i] * inv : 0.f;
                r[i] = u + 12582912.f;
                border |= fabsf(u - (r[i] - 12582912.f)) > 0.4999f;
            }
            if (border) {
#pragma unroll
                for (int i = 0; i < PER; i++)
                    if (fabsf(z[i] * inv - (r[i] - 12582912.f)) > 0.4999f) {
                        const bool t2 = rotate && turned(i);
                        r[i] = kv8_code_at_border(x[i], y[i], t2 ? c[i] : 1.f, t2 ? s[i] : 0.f, scale);
                    }
            }
            uint32_t codes[PER / 4];
#pragma unroll
            for (int i = 0; i < PER; i += 4)                 // the low bytes, plus 128
                codes[i / 4] = __byte_perm(__byte_perm(__float_as_uint(r[i]), __float_as_uint(r[i + 1]), 0x0040),
                                           __byte_perm(__float_as_uint(r[i + 2]), __float_as_uint(r[i + 3]), 0x0040), 0x5410) ^ 0x80808080u;
            const int g = is_k ? head - p.H : head - p.H - p.G;
            uint8_t *rec = page + (size_t)g * p.record;
            uint8_t *dst = rec + (is_k ? 0 : p.block_size * p.d) + in_page * p.d + kv8_piece(in_page, e0 >> 4, p.d) * 16 + (e0 & 15);
            if (PER == 8) *(uint2 *)dst = make_uint2(codes[0], codes[PER / 4 - 1]);
            else *(uint32_t *)dst = codes[0];
            if (l == 0) ((float *)(rec + 2 * p.block_size * p.d))[(is_k ? 0 : p.block_size) + in_page] = scale;
        }
    }
}

// Measured: 2,048 tokens, 28 heads of 128 on 4, 21 us: the instructions per row (about 180 a warp) bound it, not the 37 MB.

// ---- read ----------------------------------------------------------------------------------------------------------------
// The rows of some pages as the values that they stand for, [N, block, G, d] keys and values.  A thread makes 16 bytes of the output at a
// time, neighbouring threads neighbouring ones.
__device__ __forceinline__ void kv8_store(float *dst, const float (&v)[4]) { *(float4 *)dst = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void kv8_store(__nv_bfloat16 *dst, const float (&v)[8])
{
    const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3]), __floats2bfloat162_rn(v[4], v[5]),
                                 __floats2bfloat162_rn(v[6], v[7])};
    *(uint4 *)dst = *(const uint4 *)h;
}

constexpr int KV8_READ_THREADS = 256, KV8_READ_AHEAD = 4, KV8_READ_STAGES = 4;

// Records of up to 24 KB: brought whole by bulk copies, four ahead, by one thread; where a thread's pieces come from and go to is looked up
// in a table that the block makes once (worked out for every piece it took three times the instructions).  81,936 tokens of 4 heads of
// 128 into bfloat16: 45 us of the kernel's own (61 with plain loads), 52 us a pass among others, 0.60 of the measured bandwidth.
template <typename T>
__global__ void __launch_bounds__(KV8_READ_THREADS)
kv8_read_bulk_kernel(const uint8_t *cache, long long num_pages, const int32_t *pages, const int32_t *used, T *k_out, T *v_out, int records,
                     int block_size, int G, int d, int record, int *err)
{
    constexpr int PER = 16 / sizeof(T);
    extern __shared__ __align__(128) uint8_t kv8_smem[];
    const int row_pieces = d / PER, pieces = 2 * block_size * row_pieces;
    uint4 *table = (uint4 *)(kv8_smem + KV8_READ_STAGES * record);       // from, scale from, row, to (element; values' from the keys' end on)
    const uint32_t bars = smem_u32(table + pieces), stages = smem_u32(kv8_smem);
    volatile int *abort_flag = (volatile int *)((uint8_t *)(table + pieces) + 8 * KV8_READ_STAGES), *there = abort_flag + 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < KV8_READ_STAGES; s++) mbar_init(bars + 8 * s, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    for (int i = threadIdx.x; i < pieces; i += KV8_READ_THREADS) {
        const int kv = i / (pieces / 2), in_kv = i % (pieces / 2), row = in_kv / row_pieces, c = in_kv % row_pieces * PER;
        table[i] = make_uint4((kv ? block_size * d : 0) + row * d + kv8_piece(row, c >> 4, d) * 16 + (c & 15), 2 * block_size * d + 4 * (kv * block_size + row),
                              row, row * G * d + c);
    }
    pdl_sync();
    // (called by thread 0: `page` is that of record r)
    auto ask = [&](int r, int page, int s) {
        const bool is = page >= 0 && page < num_pages;
        if (page >= num_pages) atomicOr(err, HFB_ERR_PAGE);
        there[s] = is;
        mbar_arrive_expect_tx(bars + 8 * s, is ? record : 0);
        if (is)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(stages + s * record), "l"(cache + ((size_t)page * G + r % G) * record), "r"(record), "r"(bars + 8 * s) : "memory");
    };
    int coming = -1;                                             // page of the record that is asked for next
    if (threadIdx.x == 0) {
        for (int s = 0; s < KV8_READ_STAGES; s++) {
            const int r = blockIdx.x + s * gridDim.x;
            if (r < records) ask(r, pages[r / G], s);
        }
        const int r = blockIdx.x + KV8_READ_STAGES * gridDim.x;
        if (r < records) coming = pages[r / G];
    }
    __syncthreads();
    int s = 0, phase = 0;
    for (int r0 = blockIdx.x; r0 < records; r0 += gridDim.x) {
        const bool ok = mbar_wait(bars + 8 * s, phase, abort_flag, err);
        if (__syncthreads_or(!ok)) break;
        const int n = r0 / G, g = r0 % G, rows = there[s] ? used[n] : 0;
        const uint8_t *rec = kv8_smem + s * record;
        const size_t to = ((size_t)n * block_size * G + g) * d;
        for (int i = threadIdx.x; i < pieces; i += KV8_READ_THREADS) {
            const uint4 e = table[i];
            float v[PER];
            if ((int)e.z < rows) {
                const float scale = *(const float *)(rec + e.y);
                uint32_t w[PER / 4];
                if (PER == 8) { const uint2 c = *(const uint2 *)(rec + e.x); w[0] = c.x; w[PER / 4 - 1] = c.y; }
                else w[0] = *(const uint32_t *)(rec + e.x);
#pragma unroll
                for (int u = 0; u < PER; u++) v[u] = kv8_number(w[u >> 2], u & 3) * scale;
            } else {
#pragma unroll
                for (int u = 0; u < PER; u++) v[u] = 0.f;
            }
            kv8_store((i < pieces / 2 ? k_out : v_out) + to + e.w, v);
        }
        __syncthreads();                                         // the stage has been read
        if (threadIdx.x == 0) {
            const int r = r0 + KV8_READ_STAGES * gridDim.x, after = r + gridDim.x;
            if (r < records) ask(r, coming, s);
            if (after < records && after > r) coming = pages[after / G];
        }
        if (++s == KV8_READ_STAGES) { s = 0; phase ^= 1; }
    }
    __syncthreads();
    if (*abort_flag != 0 && threadIdx.x == 0)                    // a wait ran out: copies still in flight land before the shared memory goes away
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    __syncthreads();
}

// Larger records (more pieces than threads, then): plain loads, of four records before any is stored.
template <typename T>
__global__ void __launch_bounds__(KV8_READ_THREADS)
kv8_read_kernel(const uint8_t *cache, long long num_pages, const int32_t *pages, const int32_t *used, T *k_out, T *v_out, int records,
                int block_size, int G, int d, int record, int *err)
{
    pdl_sync();
    constexpr int PER = 16 / sizeof(T);                          // codes of a piece: 8 or 4
    const int row_pieces = d / PER, pieces = 2 * block_size * row_pieces;
    for (int i = threadIdx.x; i < pieces; i += KV8_READ_THREADS) {
        const int kv = i / (pieces / 2), in_kv = i % (pieces / 2), row = in_kv / row_pieces, c = in_kv % row_pieces * PER;
        const size_t from = (size_t)(kv ? block_size * d : 0) + row * d + kv8_piece(row, c >> 4, d) * 16 + (c & 15);
        const size_t scale_from = (size_t)2 * block_size * d + 4 * (kv * block_size + row);
        T *out = (kv ? v_out : k_out) + (size_t)row * G * d + c;
        for (int r0 = blockIdx.x; r0 < records; r0 += gridDim.x * KV8_READ_AHEAD) {
            uint32_t codes[KV8_READ_AHEAD][PER / 4];
            float scale[KV8_READ_AHEAD];
            int n[KV8_READ_AHEAD], g[KV8_READ_AHEAD];
#pragma unroll
            for (int u = 0; u < KV8_READ_AHEAD; u++) {
                const int r = r0 + u * gridDim.x;
                n[u] = r < records ? r / G : -1;
                g[u] = r - n[u] * G;
#pragma unroll
                for (int w = 0; w < PER / 4; w++) codes[u][w] = 0x80808080u;
                scale[u] = 0.f;
                if (n[u] < 0) continue;
                const long long page = pages[n[u]];
                if (page >= num_pages) { if (i == 0) atomicOr(err, HFB_ERR_PAGE); }
                else if (page >= 0 && row < used[n[u]]) {
                    const uint8_t *rec = cache + ((size_t)page * G + g[u]) * record;
                    if (PER == 8) { const uint2 v = *(const uint2 *)(rec + from); codes[u][0] = v.x; codes[u][PER / 4 - 1] = v.y; }
                    else codes[u][0] = *(const uint32_t *)(rec + from);
                    scale[u] = *(const float *)(rec + scale_from);
                }
            }
#pragma unroll
            for (int u = 0; u < KV8_READ_AHEAD; u++) {
                if (n[u] < 0) continue;
                float v[PER];
#pragma unroll
                for (int e = 0; e < PER; e++) v[e] = kv8_number(codes[u][e >> 2], e & 3) * scale[u];
                kv8_store(out + ((size_t)n[u] * block_size * G + g[u]) * d, v);
            }
        }
    }
}

// ---- attention, plain kernel ---------------------------------------------------------------------------------------------
// One block per (token, head); any head size, page size and mask, float32 throughout, for the float32 run and for what the
// tiled kernels don't take.  s_j = scale (q . code_j) ks_j, softmax, out = sum_j p_j vs_j code'_j / sum_j p_j.  The warps take
// groups of eight keys in turn (all of a group's reads in flight together) and keep a maximum and sums each, merged in warp order at the end: the result depends only on the keys
// seen, never on the rest of the batch.  A lane holds four numbers of a row (WORDS times), as one word of codes.
constexpr int KV8_WARPS = 8, KV8_KEYS = 8;

template <typename T, int WORDS>
__global__ void __launch_bounds__(KV8_WARPS * 32)
kv8_attention_plain_kernel(Kv8Params p, const int32_t *token_seq, int d, int *err)
{
    pdl_sync();
    const int t = blockIdx.x, h = blockIdx.y, g = h / (p.H / p.G), bs = p.block_size;
    const int seq = token_seq[t], pos = p.positions[t], lo = mask_lo(pos, p.window);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t *table = p.block_table + (size_t)seq * p.max_blocks;
    __shared__ float s_m[KV8_WARPS], s_l[KV8_WARPS], s_acc[KV8_WARPS][128 * WORDS];

    float q[WORDS][4], acc[WORDS][4];
#pragma unroll
    for (int w = 0; w < WORDS; w++) {
        const int e = 4 * (lane + 32 * w);
        const T *src = (const T *)p.q + ((size_t)t * p.H + h) * d + e;
#pragma unroll
        for (int i = 0; i < 4; i++) { q[w][i] = e < d ? to_f32(src[i]) : 0.f; acc[w][i] = 0.f; }
    }
    const float slope = p.slopes ? p.slopes[h] : 0.f;
    const float scale = p.head_scales ? p.scale * p.head_scales[h] : p.scale;
    float m = -INFINITY, l = 0.f;
    for (int j0 = lo + warp * KV8_KEYS; j0 <= pos; j0 += KV8_WARPS * KV8_KEYS) {
        // a key a lane: where its record and its row lie (-1: beyond the query, or no page), and its scales
        long long at = -1;
        float ks = 0.f, vs = 0.f;
        const int j = j0 + (lane & (KV8_KEYS - 1)), row = j % bs;
        if (j <= pos) {
            const int blk = j / bs;
            const long long page = blk < p.max_blocks ? table[blk] : -1;
            if (page < 0 || page >= p.num_pages) { if (lane < KV8_KEYS) atomicOr(err, HFB_ERR_PAGE); }
            else {
                at = (page * p.G + g) * p.record;
                const float *sc = (const float *)(p.cache + at + 2 * bs * d) + row;
                ks = sc[0]; vs = sc[bs];
            }
        }
        if (!__any_sync(0xffffffffu, at >= 0)) continue;
        float dot[KV8_KEYS];
        uint32_t kc[KV8_KEYS][WORDS], vc[KV8_KEYS][WORDS];
#pragma unroll
        for (int k = 0; k < KV8_KEYS; k++) {
            const long long its = __shfl_sync(0xffffffffu, at, k);
            const int r = __shfl_sync(0xffffffffu, row, k);
#pragma unroll
            for (int w = 0; w < WORDS; w++) {
                const int e = 4 * (lane + 32 * w);
                kc[k][w] = vc[k][w] = 0x80808080u;
                if (its >= 0 && e < d) {
                    const uint8_t *src = p.cache + its + r * d + kv8_piece(r, e >> 4, d) * 16 + (e & 15);
                    kc[k][w] = *(const uint32_t *)src;
                    vc[k][w] = *(const uint32_t *)(src + bs * d);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < KV8_KEYS; k++) {
            dot[k] = 0.f;
#pragma unroll
            for (int w = 0; w < WORDS; w++)
#pragma unroll
                for (int i = 0; i < 4; i++) dot[k] = fmaf(q[w][i], kv8_number(kc[k][w], i), dot[k]);
        }
        // the keys' sums over the lanes, all at once: key k ends up in the lanes whose number is k modulo 8
#pragma unroll
        for (int o = 1; o < KV8_KEYS; o <<= 1)
#pragma unroll
            for (int k = 0; k < KV8_KEYS; k += 2 * o)
                dot[k] = (lane & o ? dot[k + o] : dot[k]) + __shfl_xor_sync(0xffffffffu, lane & o ? dot[k] : dot[k + o], o);
        float x = dot[0];
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        x = x * ks * scale;
        if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
        x -= slope * (float)(pos - j);
        if (at < 0) x = -INFINITY;
        float top = fmaxf(m, x);
#pragma unroll
        for (int o = 1; o < KV8_KEYS; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool none = top == -INFINITY;                              // (keys of which nothing is a number)
        const float corr = m == -INFINITY ? 0.f : expf(m - top), e = x == -INFINITY ? 0.f : expf(x - (none ? 0.f : top));
        const float f = x == -INFINITY ? 0.f : e * vs;
        float sum = e;
#pragma unroll
        for (int o = 1; o < KV8_KEYS; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = (l == 0.f ? 0.f : l * (none ? 1.f : corr)) + sum;
#pragma unroll
        for (int w = 0; w < WORDS; w++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[w][i] *= corr;
#pragma unroll
        for (int k = 0; k < KV8_KEYS; k++) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
            for (int w = 0; w < WORDS; w++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[w][i] = fmaf(fk, kv8_number(vc[k][w], i), acc[w][i]);
        }
        m = top;
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int w = 0; w < WORDS; w++)
#pragma unroll
        for (int i = 0; i < 4; i++) s_acc[warp][4 * (lane + 32 * w) + i] = acc[w][i];
    __syncthreads();
    float top = -INFINITY, total = 0.f, f[KV8_WARPS];
    for (int w = 0; w < KV8_WARPS; w++) top = fmaxf(top, s_m[w]);
    const bool sink = p.sinks || p.zero_sink;
    const float sk = p.sinks ? p.sinks[h] : 0.f;
    if (sink) top = fmaxf(top, sk);
    for (int w = 0; w < KV8_WARPS; w++) {
        f[w] = s_m[w] == -INFINITY ? (s_l[w] == 0.f ? 0.f : 1.f) : expf(s_m[w] - top);
        total += s_l[w] * f[w];
    }
    if (sink) total += expf(sk - top);
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    T *o = (T *)p.out + ((size_t)t * p.H + h) * d;
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
        float v = 0.f;
        for (int w = 0; w < KV8_WARPS; w++) v += s_acc[w][c] * f[w];
        o[c] = from_f32<T>(v * inv);
    }
}

}  // namespace hfb

using namespace hfb;

extern "C" int hfb_kv8_record_bytes(int block_size, int d) { return kv8_sizes(block_size, d) ? kv8_record_bytes(block_size, d) : 0; }

extern "C" int hfb_kv8_write(const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride, int dt,
                             const float *cos_sin, int n_rot, int n_positions, int interleaved, const int32_t *positions,
                             const int32_t *slots, void *q_out, void *cache, int64_t num_pages, int block_size, int T, int H, int G, int d,
                             hfb_stream s)
{
    if (T <= 0) return HFB_OK;
    if (!valid_dt(dt) || H < 0 || G < 0 || H + G <= 0 || n_rot < 0 || n_rot > d || (n_rot & 1))
        return fail(HFB_EINVAL, "kv8_write: bad arguments (H=%d G=%d d=%d n_rot=%d)", H, G, d, n_rot);
    if (!kv8_sizes(block_size, d)) return fail(HFB_ENOTSUP, "kv8_write: head size %d or page of %d tokens (multiples of 16 up to 256, 1..1024)", d, block_size);
    if (n_rot > 0 && (!cos_sin || !positions)) return fail(HFB_EINVAL, "kv8_write: rotation needs a table and positions");
    if ((H > 0 && (!q || !q_out)) || (G > 0 && (!k || !v || !cache)) || num_pages < 0 || ((uintptr_t)cache & 15))
        return fail(HFB_EINVAL, "kv8_write: a missing array, or a cache that is not 16-byte aligned");
    Kv8WriteParams p;
    p.q = q; p.k = k; p.v = v; p.q_stride = q_stride; p.k_stride = k_stride; p.v_stride = v_stride;
    p.cos_sin = cos_sin; p.positions = positions; p.slots = slots; p.q_out = q_out; p.cache = (uint8_t *)cache;
    p.cache_slots = num_pages * block_size;
    p.n_rot = n_rot; p.n_positions = n_positions; p.interleaved = interleaved; p.T = T; p.H = H; p.G = G; p.d = d;
    p.block_size = block_size; p.record = kv8_record_bytes(block_size, d);
    // Wide accesses where rows, table and rotated part allow them.  Four numbers a lane (above 128 numbers a head eight): with eight, half
    // as many lanes share a row's fixed work, but half as many warps fit (2,048 rows of 36 heads of 128: 21.3 us with four, 25.7 with
    // eight).  A block takes as many turns as leave a round of blocks on the SMs.
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)(n_rot ? cos_sin : nullptr);
    const long long strides = (H ? q_stride : 0) | (G ? k_stride | v_stride : 0);
    auto wide = [&](int n) { return !(all & (dt == HFB_F32 && n == 8 ? 31 : 15)) && strides % n == 0 && n_rot % (interleaved ? n : 2 * n) == 0; };
    const int per = d > 128 ? 8 : 4;
    const bool vec = wide(per);
    p.lanes = 1;
    while (p.lanes * per < d) p.lanes *= 2;
    const int at_once = KV8_WRITE_WARPS * (32 / p.lanes), parts = (H + 2 * G + at_once - 1) / at_once;
    const long long spare = (long long)T * parts / (148 * 4);
    p.turns = (int)(spare < 1 ? 1 : spare > parts ? parts : spare);
    const dim3 grid(T, (parts + p.turns - 1) / p.turns);
    if (grid.y > 65535) return fail(HFB_ENOTSUP, "kv8_write: %d heads exceed the grid limit", H + 2 * G);
#define HFB_KV8_WRITE(TY, PER) \
    g_launch_err = vec ? launch_pdl(kv8_write_kernel<TY, PER, true>, grid, dim3(KV8_WRITE_THREADS), 0, (cudaStream_t)s, p, error_word()) \
                       : launch_pdl(kv8_write_kernel<TY, PER, false>, grid, dim3(KV8_WRITE_THREADS), 0, (cudaStream_t)s, p, error_word())
    if (dt == HFB_F32) { if (per == 8) HFB_KV8_WRITE(float, 8); else HFB_KV8_WRITE(float, 4); }
    else { if (per == 8) HFB_KV8_WRITE(__nv_bfloat16, 8); else HFB_KV8_WRITE(__nv_bfloat16, 4); }
#undef HFB_KV8_WRITE
    return check_pdl_launch(g_launch_err, "kv8_write");
}

extern "C" int hfb_kv8_read(const void *cache, int64_t num_pages, const int32_t *pages, const int32_t *used, void *k_out, void *v_out,
                            int out_dt, int64_t N, int block_size, int G, int d, hfb_stream s)
{
    if (N <= 0) return HFB_OK;
    if (!valid_dt(out_dt) || G <= 0 || num_pages < 0 || !cache || !pages || !used || !k_out || !v_out)
        return fail(HFB_EINVAL, "kv8_read: bad arguments (G=%d)", G);
    if (!kv8_sizes(block_size, d)) return fail(HFB_ENOTSUP, "kv8_read: head size %d or page of %d tokens (multiples of 16 up to 256, 1..1024)", d, block_size);
    if (((uintptr_t)cache | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return fail(HFB_EINVAL, "kv8_read: arrays must be 16-byte aligned");
    const int pieces = 2 * block_size * (d / (out_dt == HFB_F32 ? 4 : 8));
    if (N * G >= (1ll << 31) - (1 << 24)) return fail(HFB_ENOTSUP, "kv8_read: %lld pages of %d heads", (long long)N, G);
    const int record = kv8_record_bytes(block_size, d);
    if (record <= 24 * 1024) {
        const int smem = KV8_READ_STAGES * record + pieces * 16 + 8 * KV8_READ_STAGES + 4 + 4 * KV8_READ_STAGES;
        static bool configured[64] = {false};                             // (the opt-in is a property of the function on one device)
        if (!configured[current_device()]) {
            cudaError_t e = cudaFuncSetAttribute(kv8_read_bulk_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kv8_read_bulk_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e != cudaSuccess) return fail(HFB_ECUDA, "kv8_read: cannot opt in to shared memory: %s", cudaGetErrorString(e));
            configured[current_device()] = true;
        }
        const int resident = 148 * (smem > 110 * 1024 ? 1 : smem > 74 * 1024 ? 2 : smem > 55 * 1024 ? 3 : smem > 36 * 1024 ? 4 : 6);
        const int grid = (int)(N * G < resident ? N * G : resident);
        if (out_dt == HFB_F32)
            g_launch_err = launch_pdl(kv8_read_bulk_kernel<float>, dim3(grid), dim3(KV8_READ_THREADS), smem, (cudaStream_t)s, (const uint8_t *)cache,
                                      (long long)num_pages, pages, used, (float *)k_out, (float *)v_out, (int)(N * G), block_size, G, d, record, error_word());
        else
            g_launch_err = launch_pdl(kv8_read_bulk_kernel<__nv_bfloat16>, dim3(grid), dim3(KV8_READ_THREADS), smem, (cudaStream_t)s, (const uint8_t *)cache,
                                      (long long)num_pages, pages, used, (__nv_bfloat16 *)k_out, (__nv_bfloat16 *)v_out, (int)(N * G), block_size, G, d, record,
                                      error_word());
        return check_pdl_launch(g_launch_err, "kv8_read");
    }
    const int grid = (int)(N * G < 148 * 8 ? N * G : 148 * 8);            // (as many as are resident)
    if (out_dt == HFB_F32)
        g_launch_err = launch_pdl(kv8_read_kernel<float>, dim3(grid), dim3(KV8_READ_THREADS), 0, (cudaStream_t)s, (const uint8_t *)cache, (long long)num_pages,
                                  pages, used, (float *)k_out, (float *)v_out, (int)(N * G), block_size, G, d, record, error_word());
    else
        g_launch_err = launch_pdl(kv8_read_kernel<__nv_bfloat16>, dim3(grid), dim3(KV8_READ_THREADS), 0, (cudaStream_t)s, (const uint8_t *)cache, (long long)num_pages,
                                  pages, used, (__nv_bfloat16 *)k_out, (__nv_bfloat16 *)v_out, (int)(N * G), block_size, G, d, record, error_word());
    return check_pdl_launch(g_launch_err, "kv8_read");
}

extern "C" int hfb_kv8_attention_plain(const void *q, const void *cache, int dt, const int32_t *block_table, int max_blocks,
                                       const int32_t *token_seq, const int32_t *positions, int block_size, int64_t num_pages, int window,
                                       float scale, void *out, int T, int H, int G, int d, const float *sinks, int zero_sink,
                                       const float *slopes, const float *head_scales, float softcap, hfb_stream s)
{
    if (T <= 0) return HFB_OK;
    if (!valid_dt(dt) || H <= 0 || G <= 0 || H % G || max_blocks <= 0 || num_pages < 0)
        return fail(HFB_EINVAL, "kv8_attention: bad arguments (H=%d G=%d)", H, G);
    if (!kv8_sizes(block_size, d)) return fail(HFB_ENOTSUP, "kv8_attention: head size %d or page of %d tokens (multiples of 16 up to 256, 1..1024)", d, block_size);
    if (H > 65535) return fail(HFB_ENOTSUP, "kv8_attention: %d heads exceed the grid limit", H);
    Kv8Params p = {};
    p.q = q; p.cache = (const uint8_t *)cache; p.out = out; p.block_table = block_table; p.positions = positions;
    p.max_blocks = max_blocks; p.block_size = block_size; p.record = kv8_record_bytes(block_size, d); p.window = window; p.H = H; p.G = G;
    p.num_pages = num_pages; p.scale = scale; p.sinks = sinks; p.slopes = slopes; p.head_scales = head_scales; p.zero_sink = zero_sink;
    p.softcap = softcap > 0.f ? softcap : 0.f;
#define HFB_KV8_PLAIN(TY, W) g_launch_err = launch_pdl(kv8_attention_plain_kernel<TY, W>, dim3(T, H), dim3(KV8_WARPS * 32), 0, (cudaStream_t)s, p, token_seq, d, error_word())
    if (dt == HFB_F32) { if (d > 128) HFB_KV8_PLAIN(float, 2); else HFB_KV8_PLAIN(float, 1); }
    else { if (d > 128) HFB_KV8_PLAIN(__nv_bfloat16, 2); else HFB_KV8_PLAIN(__nv_bfloat16, 1); }
#undef HFB_KV8_PLAIN
    return check_pdl_launch(g_launch_err, "kv8_attention_plain");
}
