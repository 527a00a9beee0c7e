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
    int n_rot, n_positions, interleaved, T, H, G, d, block_size, record, lanes;
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
    const int lane = threadIdx.x & 31, per_warp = 32 / p.lanes, heads = p.H + 2 * p.G;
    const long long rows = (long long)p.T * heads;
    const int sub = lane / p.lanes, l = lane % p.lanes, e0 = l * PER;
    for (long long r0 = ((long long)blockIdx.x * 4 + (threadIdx.x >> 5)) * per_warp; r0 < rows; r0 += (long long)gridDim.x * 4 * per_warp) {
        const long long r = r0 + sub;
        const bool mine = r < rows && e0 < p.d;
        const int t = mine ? (int)(r / heads) : 0, head = mine ? (int)(r % heads) : 0;
        const bool is_q = head < p.H, is_k = !is_q && head < p.H + p.G;
        long long slot = -1;
        if (mine && !is_q) {
            slot = p.slots ? p.slots[t] : -1;
            if (slot >= p.cache_slots) { if (l == 0) atomicOr(err, HFB_ERR_SLOT); slot = -1; }
        }
        const bool work = mine && (is_q || slot >= 0);
        float x[PER], y[PER], c[PER], s[PER];
        unsigned second = 0, turned = 0;
        if (work) {
            const float *cs = nullptr;
            const bool rotate = p.n_rot > 0 && (is_q || is_k);
            if (rotate) {
                int pos = p.positions[t];
                if (pos < 0 || pos >= p.n_positions) { if (l == 0) atomicOr(err, HFB_ERR_POSITION); pos = 0; }
                cs = p.cos_sin + (size_t)pos * p.n_rot;
            }
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
            const int in_page = (int)(slot % p.block_size);
            uint8_t *rec = p.cache + ((size_t)(slot / p.block_size) * p.G + g) * p.record;
            uint8_t *dst = rec + (is_k ? 0 : p.block_size * p.d) + in_page * p.d + kv8_piece(in_page, e0 >> 4, p.d) * 16 + (e0 & 15);
#pragma unroll
            for (int i = 0; i < PER / 4; i++) ((uint32_t *)dst)[i] = codes[i];
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

template <typename T>
__global__ void __launch_bounds__(256)
kv8_read_kernel(const uint8_t *cache, long long num_pages, const int32_t *pages, const int32_t *used, T *k_out, T *v_out, long long N,
                int block_size, int G, int d, int record, int *err)
{
    pdl_sync();
    const int pieces = d / 16;
    const long long items = N * G * 2 * block_size * pieces;
    for (long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x; it < items; it += (long long)gridDim.x * blockDim.x) {
        const int c = (int)(it % pieces);
        long long rest = it / pieces;
        const int row = (int)(rest % block_size);
        rest /= block_size;
        const int kv = (int)(rest & 1);
        rest >>= 1;
        const int g = (int)(rest % G);
        const long long n = rest / G;
        const long long page = pages[n];
        uint4 codes = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        float scale = 0.f;
        if (page >= num_pages) { if (c == 0 && row == 0) atomicOr(err, HFB_ERR_PAGE); }
        else if (page >= 0 && row < used[n]) {
            const uint8_t *rec = cache + ((size_t)page * G + g) * record;
            codes = *(const uint4 *)(rec + (kv ? block_size * d : 0) + row * d + kv8_piece(row, c, d) * 16);
            scale = ((const float *)(rec + 2 * block_size * d))[kv * block_size + row];
        }
        T o[16];
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = from_f32<T>(kv8_value(i < 4 ? codes.x : i < 8 ? codes.y : i < 12 ? codes.z : codes.w, i & 3, scale));
        uint4 *dst = (uint4 *)((kv ? v_out : k_out) + ((n * block_size + row) * G + g) * d + c * 16);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) dst[i] = ((const uint4 *)o)[i];
    }
}

// ---- attention, plain kernel ---------------------------------------------------------------------------------------------
// One block per (token, head); any head size, page size and mask, float32 throughout, for the float32 run and for what the
// tiled kernels don't take.  s_j = scale (q . code_j) ks_j, softmax, out = sum_j p_j vs_j code'_j / sum_j p_j.  The warps take
// groups of eight keys in turn and keep a maximum and sums each, merged in warp order at the end: the result depends only on the keys
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
        float s[KV8_KEYS], vs[KV8_KEYS];
        uint32_t vc[KV8_KEYS][WORDS];
#pragma unroll
        for (int k = 0; k < KV8_KEYS; k++) {
            const int j = j0 + k, blk = j / bs, row = j % bs;
            const long long page = j <= pos && blk < p.max_blocks ? table[blk] : -1;
            const bool there = page >= 0 && page < p.num_pages;
            if (j <= pos && !there && lane == 0) atomicOr(err, HFB_ERR_PAGE);
            const uint8_t *rec = p.cache + ((size_t)(there ? page : 0) * p.G + g) * p.record;
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < WORDS; w++) {
                const int e = 4 * (lane + 32 * w);
                vc[k][w] = 0x80808080u;
                if (there && e < d) {
                    const int at = row * d + kv8_piece(row, e >> 4, d) * 16 + (e & 15);
                    const uint32_t kc = *(const uint32_t *)(rec + at);
                    vc[k][w] = *(const uint32_t *)(rec + bs * d + at);
#pragma unroll
                    for (int i = 0; i < 4; i++) x = fmaf(q[w][i], kv8_value(kc, i, 1.f), x);
                }
            }
            const float *sc = (const float *)(rec + 2 * bs * d);
            vs[k] = there ? sc[bs + row] : 0.f;
            x = warp_sum(x) * (there ? sc[row] : 0.f) * scale;
            if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
            x -= slope * (float)(pos - j);
            s[k] = there ? x : -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < KV8_KEYS; k++) top = fmaxf(top, s[k]);
        if (top == -INFINITY) {
            bool any = false;                                            // (a key of which nothing is a number counts)
#pragma unroll
            for (int k = 0; k < KV8_KEYS; k++) any |= s[k] != s[k];
            if (!any) continue;
        }
        const float corr = m == -INFINITY ? 0.f : expf(m - top);
        l *= corr;
#pragma unroll
        for (int w = 0; w < WORDS; w++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[w][i] *= corr;
#pragma unroll
        for (int k = 0; k < KV8_KEYS; k++) {
            const float e = s[k] == -INFINITY ? 0.f : expf(s[k] - top);
            l += e;
            const float f = s[k] == -INFINITY ? 0.f : e * vs[k];
#pragma unroll
            for (int w = 0; w < WORDS; w++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[w][i] = fmaf(f, kv8_value(vc[k][w], i, 1.f), acc[w][i]);
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
    const int per = d > 128 ? 8 : 4;
    p.lanes = 1;
    while (p.lanes * per < d) p.lanes *= 2;
    const long long rows = (long long)T * (H + 2 * G), blocks = (rows + 4 * (32 / p.lanes) - 1) / (4 * (32 / p.lanes));
    const int grid = (int)(blocks < (1 << 20) ? blocks : (1 << 20));
    // wide accesses where rows, table and rotated part allow them
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)(n_rot ? cos_sin : nullptr);
    const long long strides = (H ? q_stride : 0) | (G ? k_stride | v_stride : 0);
    const bool vec = !(all & 31 & (dt == HFB_F32 ? 4 * per - 1 : (2 * per - 1) | 15)) && strides % per == 0 && n_rot % (interleaved ? per : 2 * per) == 0;
#define HFB_KV8_WRITE(TY, PER) \
    g_launch_err = vec ? launch_pdl(kv8_write_kernel<TY, PER, true>, dim3(grid), dim3(128), 0, (cudaStream_t)s, p, error_word()) \
                       : launch_pdl(kv8_write_kernel<TY, PER, false>, dim3(grid), dim3(128), 0, (cudaStream_t)s, p, error_word())
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
    const long long items = N * G * 2 * block_size * (d / 16), blocks = (items + 255) / 256;
    const int grid = (int)(blocks < (1 << 20) ? blocks : (1 << 20));
    const int record = kv8_record_bytes(block_size, d);
    if (out_dt == HFB_F32)
        g_launch_err = launch_pdl(kv8_read_kernel<float>, dim3(grid), dim3(256), 0, (cudaStream_t)s, (const uint8_t *)cache, (long long)num_pages,
                                  pages, used, (float *)k_out, (float *)v_out, (long long)N, block_size, G, d, record, error_word());
    else
        g_launch_err = launch_pdl(kv8_read_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, (cudaStream_t)s, (const uint8_t *)cache, (long long)num_pages,
                                  pages, used, (__nv_bfloat16 *)k_out, (__nv_bfloat16 *)v_out, (long long)N, block_size, G, d, record, error_word());
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
