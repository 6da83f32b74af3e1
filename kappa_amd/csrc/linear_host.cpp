// Host-only side of the projections and their adapters (see linear.h). No HIP call
// is made here; the entry points in linear_api.hip run these checks first.
#include "linear.h"

#include <algorithm>

namespace kmoe_host {

namespace {

constexpr int64_t kMostIn = (int64_t)1 << 16;  // int8 sums stay inside i32
constexpr int64_t kMostOut = (int64_t)1 << 20;
constexpr int64_t kMostTokens = (int64_t)1 << 20;  // the sort's blocks read each other's counts
constexpr int64_t kMostRowBytes = (int64_t)1 << 32;  // 32-bit load offsets

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

kmoe_status check_tokens(int64_t tokens) {
  if (tokens < 0) return fail(KMOE_ERR_INVALID_ARG, "tokens must be >= 0 (got %lld)", (long long)tokens);
  if (tokens > kMostTokens) return fail(KMOE_ERR_UNSUPPORTED, "tokens %lld too large", (long long)tokens);
  return KMOE_OK;
}

kmoe_status check_x_dtype(const kmoe_linear_weight& w, kmoe_dtype x_dtype) {
  const int x = enum_value(x_dtype);
  if (x != KMOE_DTYPE_BF16 && x != KMOE_DTYPE_I8)
    return fail(KMOE_ERR_INVALID_ARG, "x must be BF16 or I8 rows");
  if (x == KMOE_DTYPE_I8 && enum_value(w.dtype) != KMOE_DTYPE_I8)
    return fail(KMOE_ERR_INVALID_ARG, "8-bit rows need int8 weights");
  return KMOE_OK;
}

kmoe_status check_beside(const kmoe_linear_weight& w, const kmoe_lora& l) {
  if (l.in_features != w.in_features || l.out_features != w.out_features)
    return fail(KMOE_ERR_INVALID_ARG, "the adapters are [%lld, %lld], the weights [%lld, %lld]",
                (long long)l.in_features, (long long)l.out_features, (long long)w.in_features,
                (long long)w.out_features);
  return KMOE_OK;
}

}  // namespace

bool linear_rows_fit(const kmoe_linear_weight& w, const void* x, kmoe_dtype x_dtype, int64_t x_stride) {
  return w.in_features % step_of(x_dtype) == 0 && aligned16(x) &&
         x_stride * (int64_t)dtype_size(x_dtype) % 16 == 0;
}

// Blocks that share the reduction of a row in the two-launch form: each leaves its partial sums
static int64_t split_parts(const kmoe_linear_weight& w, kmoe_dtype x_dtype) {
  return (padded_in(w.in_features) / step_of(x_dtype) + kmoe::kSplitSteps - 1) / kmoe::kSplitSteps;
}

LinearForm linear_form(const kmoe_linear_weight& w, int64_t tokens, kmoe_dtype x_dtype, bool lora) {
  if (tokens > kmoe::kLinearDecodeTokens) return LinearForm::kTiles;
  // The partial sums of two launches stay below 64 MB: where they are more, tiles are as fast or
  // faster for the most part, and the workspace would grow with in x out (34 GB at the limits).
  // us (two launches, tiles), bf16 / bf16 x int8 / int8, 16 adapters of rank 16:
  //   64 x 2048 -> 151936 (156, 156, 78 MB)   215, 149 / 180, 103 / 132, 103
  //   64 x 4096 -> 65536  (134, 134, 67 MB)   163, 125 / 133,  77 /  89,  72
  //   64 x 4096 -> 32768   (67,  67, 34 MB)    87,  85 /  73,  52 /  52,  52
  //   64 x 8192 -> 28672  (117, 117, 59 MB)   138, 146 / 116,  83 /  76,  80
  //   64 x 4096 -> 9216    (19,  19,  9 MB)    32,  40 /  28,  30 /  22,  23
  //   24 x 2048 -> 16384  (6.3, 6.3, 3 MB)     23,  22 /  18,  20 /  15,  18
  //    8 x 2048 -> 5120                      10.6, 14.8 / 8.9, 15.9 / 9.1, 12.5
  // without adapters, 16 x 16384 -> 32768 (67, 67, 34 MB) 221, 184 / 112, 96 / 102, 96; 16 x 32768 ->
  // 16384 (the same) 187, 179 / 109, 122 / 97, 93; one row of it 164, 179 / 91, 121 / 85, 92.
  const int64_t sums = split_parts(w, x_dtype) * tokens * padded_out(w.out_features) * 4;
  const LinearForm two = sums < ((int64_t)64 << 20) ? LinearForm::kSplit : LinearForm::kTiles;
  if (lora) return two;
  // Above 16 rows the one launch grows with the 16-row groups times the column groups, the tiles
  // do not. us (one or two launches, tiles), bf16 / bf16 x int8 / int8:
  //   17 x 4096 -> 9216   (1152)   23.7, 14.0 /  18.0, 15.2 /  12.7, 9.2
  //   32 x 2048 -> 6144    (768)    9.1,  9.6 /   7.6, 10.1 /   6.3, 7.1
  //   48 x 2048 -> 5120    (960)   10.6,  9.7 /   9.4, 10.2 /   7.2, 7.1
  //   64 x 2048 -> 5120   (1280)   12.8,  9.8 /  11.5, 10.6 /   8.3, 7.2
  //   64 x 4096 -> 2048    (512)   12.3, 14.0 /  10.8, 15.2 /  12.0, 8.6
  //   64 x 2048 -> 151936 (37984)  210,   114 /   188, 68   /   134, 65
  // Up to 16 rows the one launch (one row -> 151936 93, 102 / 51, 55 / 49, 53), but where its blocks
  // (of two column groups) make a full round of 256 CUs and a small one: 4096 -> 9216, one row
  // 18.6, 13.5 / 10.3, 14.6 / 9.2, 8.7. Wider ones stay with it for one row's sake, though 16 rows
  // are faster in tiles up to about 1300 groups: 2048 -> 12288 (768), one row 10.8, 10.0 / 7.3, 9.4 /
  // 6.7, 7.0, 16 rows 13.0, 10.8 / 9.1, 9.7 / 8.0, 7.6; 2048 -> 24576 (1536) 17.5, 19.4 / 11.5, 11.5 /
  // 10.1, 10.9 and 19.0, 20.3 / 15.1, 11.8 / 11.9, 11.0.
  const bool converts = enum_value(x_dtype) == KMOE_DTYPE_BF16 && enum_value(w.dtype) == KMOE_DTYPE_I8;
  const int64_t rows = (tokens + 15) / 16, columns = padded_out(w.out_features) / 16;
  if (rows > 1 ? rows * columns > (converts ? 1024 : 896) : !converts && columns > 512 && columns < 768)
    return LinearForm::kTiles;
  // Every block of the one launch reads all rows: two launches above 256 KB of them. us (one,
  // two), bf16 rows and int8 weights: 64 x 4096 -> 2048 18.4, 10.9; 64 x 8192 -> 4096 33.8, 23.6;
  // but 24 x 2048 -> 5120 6.6, 9.1; one row 2048 -> 5120 4.4, 6.8.
  const int64_t row_bytes = (w.in_features + 63) / 64 * 64 * (int64_t)dtype_size(x_dtype);
  return rows * 16 * row_bytes > 256 * 1024 ? two : LinearForm::kOne;
}

int decode_groups(int64_t cgs) {
  // One column group per block while that is no more than a block per CU (one row 8192 ->
  // 4096 7.7 us, two groups 10.8); above, two, which share the rows (24 x 2048 -> 5120 6.6, one 8.9)
  return cgs <= 256 ? 1 : 2;
}

// The tile by how many there are, against 256 CUs. Times in us of tiles of 32 x 64, 64 x 64,
// 64 x 128, 128 x 128 and 256 x 256, for n tiles of 128 x 128 (m of 256 x 256):
//   1024 -> 512, 1024 rows (n = 32)  bf16 x int8   6.2   7.4   9.9  13.8  28.4
//   4096 -> 2048, 333 (48)           bf16 x int8  19.6  18.6  26.8  39.3  83.6
//   2560 -> 6144, 200 / 512 (96, 192)       bf16  19.7 / 35.5, 16.4 / 26.6, 23.0 / 25.3, 27.5 / 28.0
//   4096 -> 2048, 1500 (192)         bf16 x int8  46.6  34.5  37.2  39.9  84.3
//   2048 -> 5120, 700 (240)          bf16 x int8  28.8  25.2  22.5  24.6  48.8
//   4096 -> 9216, 333 / 512 (216, 288)      int8  32.7 / 42.6, 26.2 / 33.3, 22.0 / 29.3, 25.3 / 33.3
//   2560 -> 6144, 1024 (384)                bf16  62.3  48.6  39.4  40.3  59.3
//   2048 -> 5120, 1500 (480)                bf16  63.7  47.9  43.0  34.7  51.2
//   2048 -> 5120, 2048 (640; m = 160) bf16 x int8 74.6  55.5  47.9  48.6  55.3
//   2560 -> 6144, 2048 (768; m = 192)       bf16 119.7  93.6  74.2  70.1  64.2
//   4096 -> 9216, 2048 (1152; m = 288)      int8 153.3 111.7  90.2  87.6  75.6 (quarters in the last round)
// A tile is not much taller than the rows: 64 rows 2048 -> 151936 in tiles of 256 rows 152 us,
// of 64 114; 300 x 4096 -> 9216 in tiles of 256 46.9, of 128 37.7; but 160 x 2048 -> 151936 166, 182.
// With adapters, of which a low tile meets fewer, 32 x 64 up to 96 tiles of 128 x 128: 128 rows
// of as many requests, 64 adapters of rank 64, 2048 -> 5120 37.0 in tiles of 64, 29.2 of 32.
LinearTile linear_tile(int64_t tokens, int64_t cgs, bool converts, bool lora) {
  const int64_t tm = (tokens + 255) / 256, tn = (cgs + 15) / 16;
  const int64_t mid = ((tokens + 127) / 128) * ((cgs + 7) / 8);
  if (tm * tn >= 176 && tm * 256 * 3 <= tokens * 5) return LinearTile::k256x256;
  if (mid >= 400 && tokens > 64) return LinearTile::k128x128;
  if (mid >= (converts ? 224 : 144) && tokens > 32) return LinearTile::k64x128;
  if (mid > (lora ? 96 : 32) && tokens > 32) return LinearTile::k64x64;
  return LinearTile::k32x64;
}

LinearRounds linear_rounds(int64_t tiles) {
  // what is left after the whole rounds goes in quarters, unless those would take four rounds
  const int64_t rest = tiles % 256;
  if (tiles > 256 && rest <= 192) return {tiles - rest, tiles - rest + (4 * rest + 7) / 8 * 8};
  const int64_t whole = (tiles + 7) / 8 * 8;
  return {whole, whole};
}

LoraShrink lora_shrink(int64_t tokens, int64_t rank, int64_t adapters) {
  // one block per CU: what the tiles leave of them goes to the groups, then to the adapters (up to
  // two per CU was no faster for 128 rows and cost 4096 rows 2 us)
  const int64_t tiles = (tokens + 15) / 16, groups = (rank + 15) / 16, room = std::max<int64_t>(256 / tiles, 1);
  const int64_t ng = groups <= room ? 1 : (groups <= 2 ? 2 : 4);
  const int64_t z = std::min((groups + ng - 1) / ng, room), y = std::min({room / z, (int64_t)16, adapters});
  return {(int)ng, (unsigned)y, (unsigned)z};
}

LinearSpace linear_space(const kmoe_linear_weight& w, int64_t tokens, kmoe_dtype x_dtype, const kmoe_lora* lora,
                         bool copied) {
  const size_t T = (size_t)tokens, in = (size_t)padded_in(w.in_features);
  const bool splits = linear_form(w, tokens, x_dtype, lora) == LinearForm::kSplit;
  const size_t parts = (size_t)split_parts(w, x_dtype);
  LinearSpace s;
  s.part = copied ? align256(T * in * dtype_size(x_dtype)) : 0;
  s.u = s.part + (splits ? align256(parts * T * (size_t)padded_out(w.out_features) * 4) : 0);
  // f32 per token and rank, or two bf16
  s.total = s.u + (lora ? align256(T * (size_t)padded_rank(lora->rank) * 4) : 0);
  return s;
}

size_t linear_most_bytes(const kmoe_linear_weight& w, int64_t tokens, kmoe_dtype x_dtype, const kmoe_lora* lora) {
  size_t most = linear_space(w, tokens, x_dtype, lora, true).total;
  // fewer tokens may hold partial sums where these do not
  for (int64_t t = 1; t <= kmoe::kLinearDecodeTokens && t < tokens; ++t) {
    const size_t s = linear_space(w, t, x_dtype, lora, true).total;
    if (s > most) most = s;
  }
  return most;
}

kmoe_status check_linear_weight(const kmoe_linear_weight* w, bool buffers) {
  if (!w) return fail(KMOE_ERR_INVALID_ARG, "the packed weights are NULL");
  const int t = enum_value(w->dtype);
  if (t != KMOE_DTYPE_BF16 && t != KMOE_DTYPE_I8)
    return fail(KMOE_ERR_INVALID_ARG, "packed weights are BF16 or I8");
  if (w->in_features < 1 || w->out_features < 1)
    return fail(KMOE_ERR_INVALID_ARG, "in_features and out_features must be >= 1");
  if (w->in_features > kMostIn || w->out_features > kMostOut)
    return fail(KMOE_ERR_UNSUPPORTED, "weights [%lld, %lld] too large", (long long)w->in_features,
                (long long)w->out_features);
  if (buffers && (!w->values || !w->scale))
    return fail(KMOE_ERR_INVALID_ARG, "packed weights: every buffer must be non-NULL");
  if (buffers && (!aligned16(w->values) || !aligned16(w->scale)))
    return fail(KMOE_ERR_INVALID_ARG, "packed weights: the buffers must be 16-byte aligned");
  return KMOE_OK;
}

kmoe_status check_lora(const kmoe_lora* l, bool buffers) {
  if (!l) return fail(KMOE_ERR_INVALID_ARG, "lora is NULL");
  if (l->num_adapters < 1 || l->rank < 1 || l->in_features < 1 || l->out_features < 1)
    return fail(KMOE_ERR_INVALID_ARG, "num_adapters, rank, in_features and out_features must be >= 1");
  if (l->num_adapters > kmoe::kLoraMaxAdapters)
    return fail(KMOE_ERR_UNSUPPORTED, "num_adapters %lld exceeds %d", (long long)l->num_adapters,
                kmoe::kLoraMaxAdapters);
  if (l->rank > kmoe::kLoraMaxRank)
    return fail(KMOE_ERR_UNSUPPORTED, "rank %lld exceeds %d", (long long)l->rank, kmoe::kLoraMaxRank);
  if (l->in_features > kMostIn || l->out_features > kMostOut)
    return fail(KMOE_ERR_UNSUPPORTED, "adapters [%lld, %lld] too large", (long long)l->in_features,
                (long long)l->out_features);
  if (buffers && (!l->a || !l->b || !l->factor))
    return fail(KMOE_ERR_INVALID_ARG, "adapters: every buffer must be non-NULL");
  if (buffers && (!aligned16(l->a) || !aligned16(l->b)))
    return fail(KMOE_ERR_INVALID_ARG, "adapters: the buffers must be 16-byte aligned");
  return KMOE_OK;
}

kmoe_status validate_linear_pack_bytes(const kmoe_linear_weight* p, size_t* values, size_t* scale) {
  KMOE_TRY(check_linear_weight(p, false));
  if (!values || !scale) return fail(KMOE_ERR_INVALID_ARG, "kmoe_linear_pack_bytes: NULL result");
  const size_t out = (size_t)padded_out(p->out_features);
  *values = (size_t)padded_in(p->in_features) * out * dtype_size(p->dtype);
  *scale = 4 * out;
  return KMOE_OK;
}

kmoe_status validate_linear_pack(const kmoe_weight* w, const kmoe_linear_weight* p) {
  KMOE_TRY(check_weight(w, "the projection's"));
  KMOE_TRY(check_linear_weight(p, true));
  if (enum_value(w->dtype) != enum_value(p->dtype))
    return fail(KMOE_ERR_INVALID_ARG, "kmoe_linear_pack: the weights are BF16 or I8, as the packed copy");
  return KMOE_OK;
}

kmoe_status validate_lora_pack_bytes(const kmoe_lora* l, size_t* a, size_t* b) {
  KMOE_TRY(check_lora(l, false));
  if (!a || !b) return fail(KMOE_ERR_INVALID_ARG, "kmoe_lora_pack_bytes: NULL result");
  const size_t per = 2 * (size_t)padded_rank(l->rank) * (size_t)l->num_adapters;
  *a = per * (size_t)padded_in(l->in_features);
  *b = per * (size_t)padded_out(l->out_features);
  return KMOE_OK;
}

kmoe_status validate_lora_pack(const kmoe_lora* l, int64_t first, int64_t count, int64_t rank, const void* a,
                               const void* b, const float* factor) {
  KMOE_TRY(check_lora(l, true));
  if (first < 0 || count < 0 || first > l->num_adapters || count > l->num_adapters - first)
    return fail(KMOE_ERR_INVALID_ARG, "kmoe_lora_pack: %lld slots from %lld on, of %lld", (long long)count,
                (long long)first, (long long)l->num_adapters);
  if (rank < 1 || rank > l->rank)
    return fail(KMOE_ERR_INVALID_ARG, "kmoe_lora_pack: rank %lld is not in [1, %lld]", (long long)rank,
                (long long)l->rank);
  if (count > 0 && (!a || !b || !factor)) return fail(KMOE_ERR_INVALID_ARG, "kmoe_lora_pack: NULL buffer");
  return KMOE_OK;
}

namespace {

kmoe_status check_batch(const kmoe_lora_batch* b, bool buffers) {
  if (!b) return fail(KMOE_ERR_INVALID_ARG, "batch is NULL");
  KMOE_TRY(check_tokens(b->tokens));
  if (b->num_adapters < 1) return fail(KMOE_ERR_INVALID_ARG, "num_adapters must be >= 1");
  if (b->num_adapters > kmoe::kLoraMaxAdapters)
    return fail(KMOE_ERR_UNSUPPORTED, "num_adapters %lld exceeds %d", (long long)b->num_adapters,
                kmoe::kLoraMaxAdapters);
  if (buffers && (!b->adapter || !b->order || !b->sorted || !b->offsets))
    return fail(KMOE_ERR_INVALID_ARG, "batch: every buffer must be non-NULL");
  return KMOE_OK;
}

size_t sort_bytes(const kmoe_lora_batch& b) {
  const size_t blocks = ((size_t)b.tokens + kmoe::kLoraSortBlock - 1) / kmoe::kLoraSortBlock;
  return 4 * blocks * (size_t)(b.num_adapters + 1);
}

}  // namespace

kmoe_status validate_lora_sort_bytes(const kmoe_lora_batch* b, size_t* bytes) {
  KMOE_TRY(check_batch(b, false));
  if (!bytes) return fail(KMOE_ERR_INVALID_ARG, "bytes is NULL");
  *bytes = sort_bytes(*b);
  return KMOE_OK;
}

kmoe_status validate_lora_sort(const int32_t* adapter, const kmoe_lora_batch* b, const void* scratch,
                               size_t scratch_bytes) {
  KMOE_TRY(check_batch(b, true));
  if (b->tokens > 0 && !adapter) return fail(KMOE_ERR_INVALID_ARG, "kmoe_lora_sort: NULL buffer");
  if (b->tokens > 0 && (!scratch || scratch_bytes < sort_bytes(*b)))
    return fail(KMOE_ERR_WORKSPACE_TOO_SMALL, "kmoe_lora_sort: scratch of %zu bytes is smaller than the %zu required",
                scratch_bytes, sort_bytes(*b));
  return KMOE_OK;
}

kmoe_status validate_linear_workspace_bytes(const kmoe_linear_weight* w, int64_t tokens, kmoe_dtype x_dtype,
                                            const kmoe_lora* lora, size_t* bytes) {
  KMOE_TRY(check_linear_weight(w, false));
  KMOE_TRY(check_tokens(tokens));
  KMOE_TRY(check_x_dtype(*w, x_dtype));
  if (lora) {
    KMOE_TRY(check_lora(lora, false));
    KMOE_TRY(check_beside(*w, *lora));
  }
  if (!bytes) return fail(KMOE_ERR_INVALID_ARG, "bytes is NULL");
  *bytes = linear_most_bytes(*w, tokens, x_dtype, lora);
  return KMOE_OK;
}

kmoe_status validate_linear_call_bytes(const kmoe_linear_weight* w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                                       int64_t x_stride, const kmoe_lora* lora, size_t* bytes) {
  KMOE_TRY(validate_linear_workspace_bytes(w, tokens, x_dtype, lora, bytes));
  if (x_stride < 0 || x_stride > kMostRowBytes) return fail(KMOE_ERR_INVALID_ARG, "x_stride %lld", (long long)x_stride);
  *bytes = tokens > 0 ? linear_space(*w, tokens, x_dtype, lora, !linear_rows_fit(*w, x, x_dtype, x_stride)).total : 0;
  return KMOE_OK;
}

kmoe_status validate_linear(const kmoe_linear_weight* w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                            int64_t x_stride, const float* x_scale, const kmoe_lora* lora,
                            const kmoe_lora_batch* batch, const void* out, const void* workspace,
                            size_t workspace_bytes, LinearSpace* space) {
  KMOE_TRY(check_linear_weight(w, true));
  KMOE_TRY(check_tokens(tokens));
  KMOE_TRY(check_x_dtype(*w, x_dtype));
  if (x_stride < w->in_features && tokens > 0)
    return fail(KMOE_ERR_INVALID_ARG, "x_stride %lld is smaller than in_features %lld", (long long)x_stride,
                (long long)w->in_features);
  if ((enum_value(x_dtype) == KMOE_DTYPE_I8) != (x_scale != nullptr) && tokens > 0)
    return fail(KMOE_ERR_INVALID_ARG, "x_scale comes with I8 rows, and with those only");
  if (!lora != !batch) return fail(KMOE_ERR_INVALID_ARG, "lora and batch come together");
  if (lora) {
    KMOE_TRY(check_lora(lora, true));
    KMOE_TRY(check_beside(*w, *lora));
    KMOE_TRY(check_batch(batch, true));
    if (batch->tokens != tokens || batch->num_adapters != lora->num_adapters)
      return fail(KMOE_ERR_INVALID_ARG,
                  "the batch holds %lld tokens of %lld adapters; the call has %lld tokens and %lld adapters",
                  (long long)batch->tokens, (long long)batch->num_adapters, (long long)tokens,
                  (long long)lora->num_adapters);
  }
  const int64_t size = (int64_t)dtype_size(x_dtype);
  const int64_t row = (kMostRowBytes - 1) / (tokens > 0 ? tokens : 1);  // bytes of a row and what follows it
  if (tokens > 0 && (x_stride > kMostRowBytes || x_stride * size > row || padded_in(w->in_features) * size > row))
    return fail(KMOE_ERR_UNSUPPORTED, "x must span less than 4 GiB");
  if (tokens > 0 && (!x || !out)) return fail(KMOE_ERR_INVALID_ARG, "kmoe_linear: x and out must be non-NULL");
  *space = linear_space(*w, tokens, x_dtype, lora, tokens > 0 && !linear_rows_fit(*w, x, x_dtype, x_stride));
  if (tokens > 0 && ((!workspace && space->total > 0) || workspace_bytes < space->total))
    return fail(KMOE_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes is smaller than the %zu required",
                workspace_bytes, space->total);
  if (tokens > 0 && !aligned16(workspace))
    return fail(KMOE_ERR_INVALID_ARG, "kmoe_linear: the workspace must be 16-byte aligned");
  return KMOE_OK;
}

namespace {

// n bytes at p against `rows` stretches of `row` bytes, `pitch` >= row apart from x on
bool meets(const void* p, size_t n, const void* x, size_t rows, size_t row, size_t pitch) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(x);
  if (n == 0 || rows * row == 0 || a + n <= b) return false;
  // the first row that ends behind p; it or none
  const size_t first = a >= b + row ? (a - b - row) / pitch + 1 : 0;
  return first < rows && b + first * pitch < a + n;
}

}  // namespace

kmoe_status validate_linear_apart(const kmoe_linear_weight& w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                                  int64_t x_stride, const void* out, const void* workspace, const LinearSpace& space) {
  const size_t size = dtype_size(x_dtype), rows = (size_t)tokens, row = (size_t)w.in_features * size;
  const size_t pitch = (size_t)x_stride * size, n = 2 * rows * (size_t)w.out_features;
  if (meets(out, n, x, rows, row, pitch) || meets(out, n, workspace, 1, space.total, space.total))
    return fail(KMOE_ERR_INVALID_ARG, "kmoe_linear: out must not overlap x or the workspace");
  if (meets(workspace, space.total, x, rows, row, pitch))
    return fail(KMOE_ERR_INVALID_ARG, "kmoe_linear: the workspace must not overlap x");
  return KMOE_OK;
}

}  // namespace kmoe_host
