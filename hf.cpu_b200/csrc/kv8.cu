// The key/value cache in 8 bits (kv8.cuh): rows written to it, pages read back, and attention over it, plain kernel.
#include "kv8.cuh"

static thread_local cudaError_t g_launch_err = cudaSuccess;      // what the last launch_pdl returned

namespace hfb {
int *error_word();

// ---- write ---------------------------------------------------------------------------------------------------------------
// Rows q | k | v of a step: queries and keys are rotated; queries go out in the run's type, keys and values into the cache.
//
// A key is rotated in float64 and a value next to a border between two codes is divided in float64: the products of a 24-bit
// number with the table's float32 are exact there, so that the codes are those of the definition and a row's codes don't
// depend on the kernel that made them.  (float32 would move about one code in 10^5 to its neighbour.)  Queries are rotated as
// the other kernels rotate them.
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

// (cos, sin) of the pairs that PER numbers from e0 on belong to, and whether each number is its pair's second.
template <typename T, int PER, bool VEC>
__device__ __forceinline__ void kv8_load(const T *row, int e0, const Kv8WriteParams &p, bool rotate, const float *cs, float (&x)[PER],
                                         float (&y)[PER], float (&c)[PER], float (&s)[PER], unsigned &second, unsigned &turned)
{
    // x: the numbers; y: their partners; bit i of `turned`: number i is rotated; of `second`: it is its pair's second
    second = turned = 0;
    const int half = p.n_rot / 2;
    if (VEC) {
        const Kv8Pack<T, PER> a = *(const Kv8Pack<T, PER> *)(row + e0);
#pragma unroll
        for (int i = 0; i < PER; i++) x[i] = to_f32(a.e[i]);
        if (rotate && e0 < p.n_rot) {                    // (a lane's numbers are all rotated or all not, and all first or all second)
            turned = (1u << PER) - 1u;
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < PER; i += 2) {
                    y[i] = x[i + 1]; y[i + 1] = x[i];
                    const float2 t = *(const float2 *)(cs + e0 + i);
                    c[i] = c[i + 1] = t.x; s[i] = s[i + 1] = t.y;
                    second |= 2u << i;
                }
            } else {
                const bool up = e0 >= half;
                const int i0 = up ? e0 - half : e0;
                const Kv8Pack<T, PER> b = *(const Kv8Pack<T, PER> *)(row + (up ? i0 : e0 + half));
                if (up) second = turned;
#pragma unroll
                for (int i = 0; i < PER; i += 2) {
                    const float4 t = *(const float4 *)(cs + 2 * (i0 + i));
                    c[i] = t.x; s[i] = t.y; c[i + 1] = t.z; s[i + 1] = t.w;
                    y[i] = to_f32(b.e[i]); y[i + 1] = to_f32(b.e[i + 1]);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = e0 + i;
            x[i] = to_f32(row[e]);
            if (rotate && e < p.n_rot) {
                const int pair = p.interleaved ? e >> 1 : (e < half ? e : e - half);
                const bool up = p.interleaved ? e & 1 : e >= half;
                y[i] = to_f32(row[p.interleaved ? e ^ 1 : (up ? e - half : e + half)]);
                c[i] = cs[2 * pair]; s[i] = cs[2 * pair + 1];
                turned |= 1u << i;
                if (up) second |= 1u << i;
            }
        }
    }
}

template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(128)
kv8_write_kernel(Kv8WriteParams p, int *err)
{
    // the successor may start once the kernel in front of this one is done: then all that was written to the cache before
    // this step is there for it, and its own wait covers what this kernel writes
    pdl_sync();
    // a block takes a token's heads 4 * 32 / lanes at a time, `turns` times
    const int lane = threadIdx.x & 31, per_warp = 32 / p.lanes, heads = p.H + 2 * p.G, t = blockIdx.x;
    const int sub = lane / p.lanes, l = lane % p.lanes, e0 = l * PER;
    int slot = p.slots ? p.slots[t] : -1;
    const float *cs = nullptr;
    if (slot >= p.cache_slots) { if (threadIdx.x == 0) atomicOr(err, HFB_ERR_SLOT); slot = -1; }
    if (p.n_rot > 0) {
        int pos = p.positions[t];
        if (pos < 0 || pos >= p.n_positions) { if (threadIdx.x == 0) atomicOr(err, HFB_ERR_POSITION); pos = 0; }
        cs = p.cos_sin + (size_t)pos * p.n_rot;
    }
    const int in_page = slot >= 0 ? slot % p.block_size : 0;
    uint8_t *page = p.cache + (size_t)(slot >= 0 ? slot / p.block_size : 0) * p.G * p.record;
    for (int n = 0; n < p.turns; n++) {
        const int head = ((blockIdx.y * p.turns + n) * 4 + (threadIdx.x >> 5)) * per_warp + sub;
        const bool is_q = head < p.H, is_k = !is_q && head < p.H + p.G;
        const bool work = head < heads && e0 < p.d && (is_q || slot >= 0);
        float x[PER], y[PER], c[PER], s[PER];
        unsigned second = 0, turned = 0;
        if (work) {
            const bool rotate = p.n_rot > 0 && (is_q || is_k);
            const T *row = is_q ? (const T *)p.q + t * p.q_stride + (size_t)head * p.d
                         : is_k ? (const T *)p.k + t * p.k_stride + (size_t)(head - p.H) * p.d
                                : (const T *)p.v + t * p.v_stride + (size_t)(head - p.H - p.G) * p.d;
            kv8_load<T, PER, VEC>(row, e0, p, rotate, cs, x, y, c, s, second, turned);
        }
        if (work && is_q) {
            T o[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                float lo = x[i], hi = x[i];
                const bool up = second >> i & 1;
                if (turned >> i & 1) rope_pair(up ? y[i] : x[i], up ? x[i] : y[i], c[i], s[i], lo, hi);
                o[i] = from_f32<T>(up ? hi : lo);
            }
            T *dst = (T *)p.q_out + ((size_t)t * p.H + head) * p.d + e0;
            if (VEC) *(Kv8Pack<T, PER> *)dst = *(Kv8Pack<T, PER> *)o;
            else
#pragma unroll
                for (int i = 0; i < PER; i++) dst[i] = o[i];
        }
        // keys and values: every lane of the row takes part in finding its largest magnitude (as bits: NaN > inf > finite)
        double xd[PER];
        unsigned top = 0;
        if (work && !is_q) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                xd[i] = x[i];
                if (turned >> i & 1) {
                    // first: x c - y s; second: y s + x c with y the pair's first
                    const double a = (double)y[i] * s[i];
                    xd[i] = fma((double)x[i], (double)c[i], second >> i & 1 ? a : -a);
                }
                x[i] = (float)xd[i];
                top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
            }
        }
        for (int o = p.lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (work && !is_q) {
            const bool finite = top < 0x7f800000u;
            const float scale = finite ? fmaxf(__fdiv_rn(__uint_as_float(top), 127.f), 1.17549435e-38f) : __uint_as_float(0x7fc00000u);
            const float inv = finite ? 1.0f / scale : 0.f;
            uint32_t codes[PER / 4];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const float u = x[i] * inv;
                float code = rintf(u);
                // (u is off by at most 127 * 3 * 2^-24 = 2.3e-5)
                if (fabsf(fabsf(u - code) - 0.5f) < 1e-4f) code = (float)rint(xd[i] / (double)scale);
                const uint32_t b = finite ? (uint32_t)((int)code + 128) : 128u;
                if (i % 4 == 0) codes[i / 4] = b;
                else codes[i / 4] |= b << (8 * (i % 4));
            }
            const int g = is_k ? head - p.H : head - p.H - p.G;
            uint8_t *rec = page + (size_t)g * p.record;
            uint8_t *dst = rec + (is_k ? 0 : p.block_size * p.d) + in_page * p.d + kv8_piece(in_page, e0 >> 4, p.d) * 16 + (e0 & 15);
            if (PER == 8) *(uint2 *)dst = make_uint2(codes[0], codes[PER / 4 - 1]);
            else *(uint32_t *)dst = codes[0];
            if (l == 0) ((float *)(rec + 2 * p.block_size * p.d))[(is_k ? 0 : p.block_size) + in_page] = scale;
        }
    }
}

// ---- read ----------------------------------------------------------------------------------------------------------------
// The rows of some pages as the values that they stand for, [N, block, G, d] keys and values.  A thread takes 16 codes.
__device__ __forceinline__ float kv8_value(uint32_t word, int i, float scale)
{
    return (float)((int)(word >> (8 * i) & 255u) - 128) * scale;
}

// A block takes as many records at once as its threads have pieces for, and four times that many before it stores any: a thread has the same
// piece of each.
constexpr int KV8_READ_THREADS = 256, KV8_READ_AHEAD = 4;

template <typename T>
__global__ void __launch_bounds__(KV8_READ_THREADS)
kv8_read_kernel(const uint8_t *cache, long long num_pages, const int32_t *pages, const int32_t *used, T *k_out, T *v_out, int records,
                int block_size, int G, int d, int record, int *err)
{
    pdl_sync();
    const int row_pieces = d / 16, pieces = 2 * block_size * row_pieces, at_once = max(1, KV8_READ_THREADS / pieces);
    const int mine = threadIdx.x / pieces;                       // of the records at once (more pieces than threads: always 0)
    if (mine >= at_once) return;
    for (int i = threadIdx.x % pieces; i < pieces; i += KV8_READ_THREADS) {
        const int kv = i / (pieces / 2), in_kv = i % (pieces / 2), row = in_kv / row_pieces, c = in_kv % row_pieces;
        const size_t from = (size_t)(kv ? block_size * d : 0) + row * d + kv8_piece(row, c, d) * 16, scale_from = (size_t)2 * block_size * d + 4 * (kv * block_size + row);
        T *out = (kv ? v_out : k_out) + (size_t)row * G * d + c * 16;
        for (int r0 = blockIdx.x * at_once + mine; r0 < records; r0 += gridDim.x * at_once * KV8_READ_AHEAD) {
            uint4 codes[KV8_READ_AHEAD];
            float scale[KV8_READ_AHEAD];
            int n[KV8_READ_AHEAD], g[KV8_READ_AHEAD];
#pragma unroll
            for (int u = 0; u < KV8_READ_AHEAD; u++) {
                const int r = r0 + u * gridDim.x * at_once;
                n[u] = r < records ? r / G : -1;
                g[u] = r - n[u] * G;
                codes[u] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                scale[u] = 0.f;
                if (n[u] < 0) continue;
                const long long page = pages[n[u]];
                if (page >= num_pages) { if (i == 0) atomicOr(err, HFB_ERR_PAGE); }
                else if (page >= 0 && row < used[n[u]]) {
                    const uint8_t *rec = cache + ((size_t)page * G + g[u]) * record;
                    codes[u] = *(const uint4 *)(rec + from);
                    scale[u] = *(const float *)(rec + scale_from);
                }
            }
#pragma unroll
            for (int u = 0; u < KV8_READ_AHEAD; u++) {
                if (n[u] < 0) continue;
                const uint32_t w[4] = {codes[u].x, codes[u].y, codes[u].z, codes[u].w};
                T o[16];
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] = from_f32<T>(kv8_value(w[e >> 2], e & 3, scale[u]));
                uint4 *dst = (uint4 *)(out + ((size_t)n[u] * block_size * G + g[u]) * d);
#pragma unroll
                for (int e = 0; e < (int)sizeof(T); e++) dst[e] = ((const uint4 *)o)[e];
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
                for (int i = 0; i < 4; i++) dot[k] = fmaf(q[w][i], kv8_value(kc[k][w], i, 1.f), dot[k]);
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
                for (int i = 0; i < 4; i++) acc[w][i] = fmaf(fk, kv8_value(vc[k][w], i, 1.f), acc[w][i]);
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
    // Wide accesses where rows, table and rotated part allow them; bfloat16 rows then go eight numbers a lane (16 bytes), others four (above
    // 128 numbers a head eight).  A block takes as many turns as leave two rounds of blocks on the SMs.
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)(n_rot ? cos_sin : nullptr);
    const long long strides = (H ? q_stride : 0) | (G ? k_stride | v_stride : 0);
    auto wide = [&](int n) { return !(all & (dt == HFB_F32 && n == 8 ? 31 : 15)) && strides % n == 0 && n_rot % (interleaved ? n : 2 * n) == 0; };
    const int per = d > 128 || (dt == HFB_BF16 && wide(8)) ? 8 : 4;
    const bool vec = wide(per);
    p.lanes = 1;
    while (p.lanes * per < d) p.lanes *= 2;
    const int at_once = 4 * (32 / p.lanes), parts = (H + 2 * G + at_once - 1) / at_once;
    const long long spare = (long long)T * parts / (2 * 148 * 12);
    p.turns = (int)(spare < 1 ? 1 : spare > parts ? parts : spare);
    const dim3 grid(T, (parts + p.turns - 1) / p.turns);
    if (grid.y > 65535) return fail(HFB_ENOTSUP, "kv8_write: %d heads exceed the grid limit", H + 2 * G);
#define HFB_KV8_WRITE(TY, PER) \
    g_launch_err = vec ? launch_pdl(kv8_write_kernel<TY, PER, true>, grid, dim3(128), 0, (cudaStream_t)s, p, error_word()) \
                       : launch_pdl(kv8_write_kernel<TY, PER, false>, grid, dim3(128), 0, (cudaStream_t)s, p, error_word())
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
    const int pieces = 2 * block_size * (d / 16), at_once = pieces < KV8_READ_THREADS ? KV8_READ_THREADS / pieces : 1;
    if (N * G >= (1ll << 31) - (1 << 24)) return fail(HFB_ENOTSUP, "kv8_read: %lld pages of %d heads", (long long)N, G);
    const long long blocks = (N * G + at_once - 1) / at_once;
    const int grid = (int)(blocks < 148 * 8 ? blocks : 148 * 8);          // (as many as are resident)
    const int record = kv8_record_bytes(block_size, d);
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
