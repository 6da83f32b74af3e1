// Host-only side of the projections and their adapters: argument validation,
// buffer sizes and the choice of kernels. Plain C++ (no HIP headers), as host.h.
//
// The projections of a decoder layer (kappa/qwen3/linear.py:10-25, the q, k, v and o
// einsums over to_compute_dtype weights) and low-rank adapters beside them, which the
// reference does not have.
#pragma once

#include "host.h"

namespace kmoe {

constexpr int kLinearInPad = 128;      // packed weights: `in` to a multiple of this (128 bytes of int8)
constexpr int kLinearOutPad = 32;      // and `out` to one of this (two column groups)
constexpr int kLoraRankPad = 32;       // ranks of one step of the expanding product
constexpr int kLoraMaxRank = 256;
constexpr int kLoraMaxAdapters = 1024;
constexpr int kLoraSortBlock = 512;    // tokens per block of the sort
constexpr int kLinearDecodeTokens = 64;  // above: always tiles
constexpr int kSplitSteps = 8;         // 128-byte steps of the rows that a block of the two-launch form takes

}  // namespace kmoe

namespace kmoe_host {

inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline int64_t padded_in(int64_t in) { return round_up(in, kmoe::kLinearInPad); }
inline int64_t padded_out(int64_t out) { return round_up(out, kmoe::kLinearOutPad); }
inline int64_t padded_rank(int64_t rank) { return round_up(rank, kmoe::kLoraRankPad); }

// Elements of a row that one 128-byte step of the kernels covers
inline int64_t step_of(kmoe_dtype x) { return enum_value(x) == KMOE_DTYPE_I8 ? 128 : 64; }
// Whether the kernels read x where it is: whole steps, rows on 16-byte boundaries.
// Other rows are copied into the workspace first, padded with zeros.
bool linear_rows_fit(const kmoe_linear_weight& w, const void* x, kmoe_dtype x_dtype, int64_t x_stride);

// Which kernels a call runs (linear.hip): one launch in which every block reads all rows and
// its columns' weights, two launches (partial sums, then their sum and the adapters'
// part), or tiles of rows and columns.
enum class LinearForm { kOne, kSplit, kTiles };
LinearForm linear_form(const kmoe_linear_weight& w, int64_t tokens, kmoe_dtype x_dtype, bool lora);

// Column groups (16 columns) that a block of the one launch takes; cgs: groups of the packed weights
int decode_groups(int64_t cgs);

// The tiles' size, rows x columns; converts: bf16 rows with int8 weights
enum class LinearTile { k32x64, k64x64, k64x128, k128x128, k256x256 };
LinearTile linear_tile(int64_t tokens, int64_t cgs, bool converts, bool lora);

// The blocks of the 256 x 256 tiles: the first `whole` take one each (a multiple of 8, those past
// the last nothing), the others a quarter
struct LinearRounds {
  int64_t whole, blocks;
};
LinearRounds linear_rounds(int64_t tiles);

// The adapters' inner products above 64 tokens, per 16 rows: groups of 16 ranks that a block
// sums at a time (1, 2 or 4), and how many blocks share the adapters (y) and the groups (z)
struct LoraShrink {
  int groups;
  unsigned y, z;
};
LoraShrink lora_shrink(int64_t tokens, int64_t rank, int64_t adapters);

// Byte offsets of the workspace: the copied rows (0, where they are copied), partial sums
// (two-launch form), the adapters' inner values.
struct LinearSpace {
  size_t part, u, total;
};
LinearSpace linear_space(const kmoe_linear_weight& w, int64_t tokens, kmoe_dtype x_dtype, const kmoe_lora* lora,
                         bool copied);
// The largest of any call of up to `tokens` rows
size_t linear_most_bytes(const kmoe_linear_weight& w, int64_t tokens, kmoe_dtype x_dtype, const kmoe_lora* lora);

kmoe_status check_linear_weight(const kmoe_linear_weight* w, bool buffers);
kmoe_status check_lora(const kmoe_lora* lora, bool buffers);

kmoe_status validate_linear_pack_bytes(const kmoe_linear_weight* packed, size_t* values, size_t* scale);
kmoe_status validate_linear_pack(const kmoe_weight* w, const kmoe_linear_weight* packed);
kmoe_status validate_lora_pack_bytes(const kmoe_lora* lora, size_t* a, size_t* b);
kmoe_status validate_lora_pack(const kmoe_lora* lora, int64_t first, int64_t count, int64_t rank, const void* a,
                               const void* b, const float* factor);
kmoe_status validate_lora_sort_bytes(const kmoe_lora_batch* batch, size_t* bytes);
kmoe_status validate_lora_sort(const int32_t* adapter, const kmoe_lora_batch* batch, const void* scratch,
                               size_t scratch_bytes);
kmoe_status validate_linear_workspace_bytes(const kmoe_linear_weight* w, int64_t tokens, kmoe_dtype x_dtype,
                                            const kmoe_lora* lora, size_t* bytes);
kmoe_status validate_linear_call_bytes(const kmoe_linear_weight* w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                                       int64_t x_stride, const kmoe_lora* lora, size_t* bytes);
kmoe_status validate_linear(const kmoe_linear_weight* w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                            int64_t x_stride, const float* x_scale, const kmoe_lora* lora,
                            const kmoe_lora_batch* batch, const void* out, const void* workspace,
                            size_t workspace_bytes, LinearSpace* space);
// That out and the workspace overlap neither x's rows nor each other (tokens > 0, the call valid otherwise)
kmoe_status validate_linear_apart(const kmoe_linear_weight& w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                                  int64_t x_stride, const void* out, const void* workspace, const LinearSpace& space);

}  // namespace kmoe_host
