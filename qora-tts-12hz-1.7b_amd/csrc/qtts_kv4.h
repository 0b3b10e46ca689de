// qtts_kv4.h — the 4-bit cache of many sequences (qtts_kv4.hip): layout of a
// page's block, argument structs of the kernels, and the index rules that the
// host and the kernels share.
#pragma once
#include "qtts_device.h"

namespace qtts {

// A block holds 64 positions of one kv head, 72 D bytes (D = head_dim).  Both
// code parts are laid out as the matrix instructions of the attention read
// them: 16 rows of K (positions p % 4 == t) follow each other, so a wave's
// 16-byte loads cover them without a gap; of V, four positions' codes of one
// group of four columns make 8 bytes, so that two positions' codes for one
// column lie 16 bits apart and unpack into a pair of f16 with one mask.  Every
// 16-bit unit and every byte of K belongs to one position: rows are stored
// without reading what is there.
constexpr int KV4_PAGE = 64;
__host__ __device__ constexpr int kv4_block(int D) { return 72 * D; }
__host__ __device__ constexpr int kv4_k_at(int D, int p) { return ((p & 3) * 16 + (p >> 2)) * (D / 2); }
__host__ __device__ constexpr int kv4_v_at(int D, int p, int unit) { return 32 * D + ((p >> 2) * (D / 4) + unit) * 8 + (p & 3) * 2; }
__host__ __device__ constexpr int kv4_ks_at(int D, int p, int g) { return 64 * D + (g * KV4_PAGE + p) * 2; }
__host__ __device__ constexpr int kv4_vs_at(int D, int p, int g) { return 68 * D + (g * KV4_PAGE + p) * 2; }

struct Kv4Pages {
    uint8_t *base;
    int64_t n_pages, stride;
    int32_t heads;
};

struct Kv4Tables {
    const int32_t *cached, *fresh, *free_pages;
    int32_t *table, *row_start, *lengths, *positions, *status;
    int64_t *slots;
    int64_t n_free, table_stride, n_rows;
    int32_t n_seqs, max_pages;
};
constexpr int KV4_MAX_SEQS = 4096;   // of one tables call: their row and page sums lie in LDS

struct QkNormRope {
    const void *q, *k, *v;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const uint16_t *q_norm, *k_norm;
    const float *cos, *sin;
    int64_t max_pos;
    const int32_t *positions;
    const int64_t *slots;
    Kv4Pages cache;
    int32_t rows, group, kv_heads;   // group: query heads per kv head
    float eps;
    int32_t vec;                     // every pointer and stride lets four elements move at once
};

struct Kv4Attn {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    Kv4Pages cache;
    const int32_t *row_start, *lengths, *table;
    int64_t table_stride;
    float *part;                     // splits > 1: [tile][kv head][split] {W maxima, W sums}, then the rows
    int64_t part_rows;               // floats before the rows
    int32_t rows, n_seqs, max_pages, group;
    int32_t window, chunk, splits;   // pages of a workgroup, most workgroups of a tile
    float scale;
    int32_t vec;
};

// The work of a sequence is cut into tiles of W columns, a column being a
// (row, query head of the kv head) pair in that order.  A tile's number is found
// without a sum over all sequences: blocks of 64 sequences begin at tile
// row_start[b] * group / W + b, since c columns starting at column s need at most
// (s + c) / W - s / W + 1 tiles; within a block tiles are numbered without gaps
// (numbers that no tile has, spread evenly among the others, left the card half
// idle: workgroups go round XCDs and their parts by number).
constexpr int KV4_W = 16, KV4_WIDE = 128;
__host__ __device__ constexpr int64_t kv4_first_tile(int64_t row, int group, int b, int W) { return row * group / W + b; }

hipError_t enqueue_kv4_tables(const Kv4Tables &a, hipStream_t s);
hipError_t enqueue_qk_norm_rope(const QkNormRope &a, int dtype, int D, bool store, hipStream_t s);
hipError_t enqueue_kv4_gather(const Kv4Pages &c, int D, const int64_t *slots, int n, int dtype, void *K, void *V, hipStream_t s);
struct Kv4Cut {
    int width, chunk, splits;
    int64_t parts;                   // partial results that the workspace holds; 0: nothing is split
};
Kv4Cut kv4_attn_cut(bool f32, int64_t rows, int n_seqs, int group, int kv_heads, int64_t max_len, int window);
hipError_t enqueue_kv4_attn(const Kv4Attn &a, int dtype, int D, int width, hipStream_t s);

}  // namespace qtts
