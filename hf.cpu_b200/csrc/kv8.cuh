// The key/value cache in 8 bits: how a page is laid out, and the parameters its attention kernels share.
//
// A row (a token's key or value of one key/value head, d numbers) is held as d codes from -127 to 127 and one float32 scale:
//     scale = max(top / 127, 2^-126), top = the largest magnitude of the row in float32;  code = round to nearest even (x / scale).
// A row with a value that float32 cannot hold as a finite number has the scale NaN and reads as NaN.  The scale belongs to one
// token and head: one for a whole page would have to be raised, and the page's earlier tokens rounded a second time, whenever
// a larger token arrives, so that what the cache holds would depend on how a prompt was cut into steps, and a page that
// several requests share would be written to.  It costs 8 bytes a token and head (3 % at d = 128).
//
// A page's rows of one head lie together in one record: [block][d] key codes, [block][d] value codes, [block] key scales,
// [block] value scales, filled up to a multiple of 16 bytes; record (page, g) is the (page * G + g)-th.  One untiled bulk copy
// brings a record into shared memory.  A byte is code + 128.  The 16-byte pieces of a row stand in an order that depends on the
// row (kv8_piece): eight rows' pieces c then lie in different banks, as ldmatrix wants them, without a copy that swizzles.
#pragma once
#include "common.cuh"

namespace hfb {

__host__ __device__ inline int kv8_record_bytes(int block_size, int d) { return (2 * block_size * d + 8 * block_size + 15) / 16 * 16; }

// Where piece `c` of row `row` stands (the rule is its own inverse).
__host__ __device__ __forceinline__ int kv8_piece(int row, int c, int d)
{
    return d % 128 == 0 ? c ^ (row & 7) : d % 64 == 0 ? c ^ ((row >> 1) & 3) : c;
}

// Head sizes and pages the cache takes.
inline bool kv8_sizes(int block_size, int d) { return block_size >= 1 && block_size <= 1024 && d >= 16 && d <= 256 && d % 16 == 0; }

struct Kv8Params {
    const void *q;
    const uint8_t *cache;
    void *out;
    const int32_t *block_table, *positions, *tile_seq, *tile_t0, *tile_nt;
    int max_blocks, block_size, record, window, H, G;
    long long num_pages;
    float scale;
    // options, as the other attention kernels have them: a sink per head [H] or one of score zero; slopes [H], slope * (query
    // position - key position) off every score; a factor per head [H] on the scaled score; score <- softcap * tanh(score / softcap)
    const float *sinks, *slopes, *head_scales;
    int zero_sink;
    float softcap;
};

}  // namespace hfb
