// Projections of a decoder layer, y = x W, and the low-rank adapters of many requests
// beside them: token t of adapter a adds factor_a (x_t A_a) B_a.
//
// Reference: the q, k, v and o einsums (kappa/qwen3/linear.py:10-25) over
// to_compute_dtype weights (kappa/qwen3/quant.py:34-38); it has no adapters. The
// scale of int8 weights multiplies the f32 sum of the products with the integers, so
// nothing is rounded between the operands and the output.
//
// Three kinds of products (Kind): bf16 rows with bf16 or int8 weights on
// v_mfma_f32_16x16x32_bf16 (int8 becomes bf16 in registers, exactly), and int8 rows
// with int8 weights on v_mfma_i32_16x16x64_i8, whose sums are exact.
#include <type_traits>

#include "common.h"
#include "expert_dev.h"
#include "linear_launch.h"

namespace kmoe {

namespace {

constexpr int kBB = 0;  // bf16 rows, bf16 weights
constexpr int kBI = 1;  // bf16 rows, int8 weights
constexpr int kII = 2;  // int8 rows, int8 weights

struct LinearArgs {
  const char* x;      // rows, 16-byte aligned
  uint32_t row_bytes;
  const float* xs;    // the rows' scales (kII)
  const char* w;
  const float* ws;
  uint16_t* out;
  int T, N, kc;       // kc: 64-deep chunks
  int cgs;            // column groups (16 columns) of the packed weights
  size_t cg_bytes;    // bytes of one
  // adapters
  const int32_t* adapter;  // NULL: none
  const int32_t* order;
  const int32_t* sorted;
  const int32_t* offsets;
  const char* a;      // [L][rank/16][in/64][2][4][16][8]
  const char* b;      // [L][out/16][rank/32][4][16][8]
  const float* factor;
  int rank, rp, kcp;  // rank, rank padded, 64-deep chunks of the packed A
  floatx4* part;      // up to 64 tokens: [splits][T][out/4] partial sums
  void* u;            // up to 64 tokens f32 [T][rp]; above, bf16 [T][rp/32][hi 32 | lo 32] in sorted order
};

__device__ __forceinline__ int32x4 as_i32x4(const uint4 v) { return __builtin_bit_cast(int32x4, v); }

__device__ __forceinline__ void unpack8(const uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// four output columns of one row; vec: rows on 8-byte boundaries
__device__ __forceinline__ void store4(uint16_t* __restrict__ row, int col, int N, bool vec, const float* v) {
  if (vec && col + 4 <= N) {
    *reinterpret_cast<uint2*>(row + col) = uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < N) row[col + j] = f32_to_bf16_bits(v[j]);
}

}  // namespace

// ---------------------------------------------------------------------------
// Load time: weights and adapters into the layouts of include/kmoe.h, one 16-byte
// piece per thread (16 neighbouring threads read 16 neighbouring columns).
// ---------------------------------------------------------------------------

// bf16 [K][N] (or its `mats` copies, one after the other) -> [N/16][K/64][2][4][16][8], zeros outside
__global__ __launch_bounds__(256) void k_pack_bf16(int64_t mats, int K, int N, int Kp, int Np,
                                                   const uint16_t* __restrict__ src, uint16_t* __restrict__ dst) {
  const int64_t per = (int64_t)Kp * Np / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < mats * per; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / per, p = i - m * per;
    const int c = p & 15, q = (p >> 4) & 3, st = (p >> 6) & 1;
    const int64_t cell = p >> 7;
    const int kc = (int)(cell % (Kp >> 6)), n = (int)(cell / (Kp >> 6)) * 16 + c;
    const int k0 = kc * 64 + 16 * q + 8 * st;
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n < N && k0 + j < K) v[j >> 1] |= (uint32_t)src[(m * K + k0 + j) * N + n] << (16 * (j & 1));
    reinterpret_cast<uint4*>(dst)[i] = uint4{v[0], v[1], v[2], v[3]};
  }
}

// int8 [K][N] -> [N/16][K/16][16][16], zeros outside
__global__ __launch_bounds__(256) void k_pack_i8(int K, int N, int Kp, int Np, const uint8_t* __restrict__ src,
                                                 uint8_t* __restrict__ dst) {
  const int64_t pieces = (int64_t)Kp * Np / 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
    const int c = i & 15;
    const int64_t cell = i >> 4;
    const int k0 = (int)(cell % (Kp >> 4)) * 16, n = (int)(cell / (Kp >> 4)) * 16 + c;
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (n < N && k0 + j < K) v[j >> 2] |= (uint32_t)src[(int64_t)(k0 + j) * N + n] << (8 * (j & 3));
    reinterpret_cast<uint4*>(dst)[i] = uint4{v[0], v[1], v[2], v[3]};
  }
}

// the scales of N columns in f32; kind: kmoe_scale_kind
__global__ __launch_bounds__(256) void k_pack_scale(int N, int Np, int kind, int s_bf16, const void* __restrict__ s,
                                                    float* __restrict__ dst) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= Np) return;
  float v = 1.0f;
  if (kind != KMOE_SCALE_NONE) {
    const int i = kind == KMOE_SCALE_CHANNEL ? min(n, N - 1) : 0;
    v = s_bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(s)[i]) : reinterpret_cast<const float*>(s)[i];
  }
  dst[n] = v;
}

// B [count][R][N] -> slots of [N/16][rp/32][4][16][8], zeros outside
__global__ __launch_bounds__(256) void k_pack_lora_b(int64_t count, int R, int N, int rp, int Np,
                                                     const uint16_t* __restrict__ src, uint16_t* __restrict__ dst) {
  const int64_t per = (int64_t)rp * Np / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count * per; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / per, p = i - m * per;
    const int c = p & 15, r8 = (p >> 4) & 3;
    const int64_t cell = p >> 6;
    const int r0 = (int)(cell % (rp >> 5)) * 32 + 8 * r8, n = (int)(cell / (rp >> 5)) * 16 + c;
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n < N && r0 + j < R) v[j >> 1] |= (uint32_t)src[(m * R + r0 + j) * N + n] << (16 * (j & 1));
    reinterpret_cast<uint4*>(dst)[i] = uint4{v[0], v[1], v[2], v[3]};
  }
}

__global__ __launch_bounds__(256) void k_copy_f32(int64_t n, const float* __restrict__ src, float* __restrict__ dst) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) dst[i] = src[i];
}

// Rows that the kernels cannot read where they are (a width that is no multiple of a
// step, rows off 16-byte boundaries): copied, the width filled up with zeros.
template <typename E>
__global__ __launch_bounds__(256) void k_stage_rows(int64_t T, int K, int Kp, int64_t stride,
                                                    const E* __restrict__ src, E* __restrict__ dst) {
  const int64_t n = T * Kp;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / Kp;
    const int k = (int)(i - t * Kp);
    dst[i] = k < K ? src[t * stride + k] : (E)0;
  }
}

// ---------------------------------------------------------------------------
// The tokens of a step by adapter: a stable counting sort over L + 1 buckets (the
// last: no adapter). Blocks of 512 tokens count themselves (k_lora_count, not needed for one
// block); then every block adds up the counts and ranks its own tokens: inside a wave
// by matching the buckets' bits, the waves by their counts in LDS.
// ---------------------------------------------------------------------------
namespace {

__device__ __forceinline__ int lora_bucket(const int32_t* __restrict__ adapter, int64_t t, int64_t T, int L) {
  if (t >= T) return -1;
  const int a = adapter[t];
  return a >= 0 && a < L ? a : L;
}

}  // namespace

__global__ __launch_bounds__(kLoraSortBlock) void k_lora_count(int T, int L, const int32_t* __restrict__ adapter,
                                                               int32_t* __restrict__ hist) {
  __shared__ int cnt[kLoraMaxAdapters + 1];
  for (int i = threadIdx.x; i <= L; i += kLoraSortBlock) cnt[i] = 0;
  __syncthreads();
  const int b = lora_bucket(adapter, (int64_t)blockIdx.x * kLoraSortBlock + threadIdx.x, T, L);
  if (b >= 0) atomicAdd(&cnt[b], 1);
  __syncthreads();
  for (int i = threadIdx.x; i <= L; i += kLoraSortBlock) hist[(int64_t)blockIdx.x * (L + 1) + i] = cnt[i];
}

__global__ __launch_bounds__(kLoraSortBlock) void k_lora_sort(int T, int L, const int32_t* __restrict__ adapter,
                                                              const int32_t* __restrict__ hist, int blocks,
                                                              int32_t* __restrict__ row_adapter,
                                                              int32_t* __restrict__ order,
                                                              int32_t* __restrict__ sorted,
                                                              int32_t* __restrict__ offsets) {
  constexpr int kWaves = kLoraSortBlock / 64;
  __shared__ int cnt[kWaves][kLoraMaxAdapters + 1];  // a wave's tokens of a bucket; then where its first goes
  __shared__ int total[kLoraMaxAdapters + 1];        // tokens of a bucket; then its start
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  for (int i = tid; i < kWaves * (kLoraMaxAdapters + 1); i += kLoraSortBlock) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * kLoraSortBlock + tid;
  const int b = lora_bucket(adapter, t, T, L);
  // the lanes with the same bucket (11 bits; those past the batch match each other)
  uint64_t same = ~0ull;
  for (int bit = 0; bit < 11; ++bit) {
    const uint64_t m = __ballot((b >> bit) & 1);
    same &= ((b >> bit) & 1) ? m : ~m;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1));
  if (b >= 0 && rank == 0) cnt[wv][b] = __popcll(same);
  __syncthreads();
  // per bucket: the tokens of the blocks before this one, of all blocks, and of this one's waves
  for (int i = tid; i <= L; i += kLoraSortBlock) {
    int before = 0, all = 0;
    if (blocks > 1) {
      for (int k = 0; k < blocks; ++k) {
        const int h = hist[(int64_t)k * (L + 1) + i];
        if (k < (int)blockIdx.x) before += h;
        all += h;
      }
    }
    int run = before;
    for (int w = 0; w < kWaves; ++w) {
      const int h = cnt[w][i];
      cnt[w][i] = run;
      run += h;
    }
    total[i] = blocks > 1 ? all : run;
  }
  __syncthreads();
  // the buckets' starts: one wave, 64 buckets at a time
  if (wv == 0) {
    int base = 0;
    for (int i0 = 0; i0 <= L; i0 += 64) {
      const int i = i0 + lane;
      const int v = i <= L ? total[i] : 0;
      int incl = v;
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
      }
      if (i <= L) total[i] = base + incl - v;
      base += __shfl(incl, 63, 64);
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = tid; i <= L; i += kLoraSortBlock) offsets[i] = total[i];
  if (b < 0) return;
  const int at = total[b] + cnt[wv][b] + rank;
  const int a = b < L ? b : -1;
  row_adapter[t] = a;
  order[at] = (int32_t)t;
  sorted[at] = a;
}

// ---------------------------------------------------------------------------
// u = factor x A for few tokens, a block's share: 16 ranks (group g) of token t, NW waves
// over the chunks.
// ---------------------------------------------------------------------------
template <int KIND, int NW>
__device__ __forceinline__ void shrink_row(const LinearArgs& p, int t, int g, float (*red)[16]) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, q = lane >> 4;
  const int ad = p.adapter[t];
  if (ad < 0) return;  // the whole block
  const float f = p.factor[ad] * (KIND == kII ? p.xs[t] : 1.0f);
  const char* xr = p.x + (size_t)t * p.row_bytes + q * (KIND == kII ? 16 : 32);
  const char* ar = p.a + (size_t)ad * p.rp * p.kcp * 128 + (size_t)g * p.kcp * 2048 + lane * 16;
  float acc = 0.0f;
#pragma unroll 4
  for (int kc = wv; kc < p.kc; kc += NW) {
    float fa[16], fx[16];
    unpack8(*reinterpret_cast<const uint4*>(ar + (size_t)kc * 2048), fa);
    unpack8(*reinterpret_cast<const uint4*>(ar + (size_t)kc * 2048 + 1024), fa + 8);
    if constexpr (KIND == kII) {
      const uint4 v = *reinterpret_cast<const uint4*>(xr + kc * 64);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 16; ++j) fx[j] = (float)(int8_t)((w[j >> 2] >> (8 * (j & 3))) & 0xffu);
    } else {
      unpack8(*reinterpret_cast<const uint4*>(xr + kc * 128), fx);
      unpack8(*reinterpret_cast<const uint4*>(xr + kc * 128 + 16), fx + 8);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) acc = __builtin_fmaf(fx[j], fa[j], acc);
  }
  acc += __shfl_xor(acc, 16, 64);
  acc += __shfl_xor(acc, 32, 64);
  if (lane < 16) red[wv][lane] = acc;
  __syncthreads();
  if (threadIdx.x < 16) {
    float s = 0.0f;
    for (int w = 0; w < NW; ++w) s += red[w][threadIdx.x];
    reinterpret_cast<float*>(p.u)[(size_t)t * p.rp + g * 16 + threadIdx.x] = s * f;
  }
}

// ---------------------------------------------------------------------------
// u for many tokens, 16 sorted rows per tile: MFMA, sixteen waves over the chunks, one
// pass per adapter of the tile and NG groups of 16 ranks; u as bf16 hi + lo. The passes are
// shared out over the blocks of the tile (y: the adapters, z: the groups). Bound by
// latency: the tile's adapters come with its rows, and all chunks of 4096 elements are in
// flight together. 128 rows of 64 adapters and rank 64, 2048 -> 5120: the call took 69.6 us with
// one block per tile (32.5 of them here), 40.4 with the passes shared out.
// ---------------------------------------------------------------------------
template <int KIND, int NG>
__global__ __launch_bounds__(1024) void k_lora_shrink(LinearArgs p) {
  constexpr int NW = 16;
  constexpr int CB = NG == 1 ? 4 : 2;  // chunks whose loads are in flight together (128 registers)
  constexpr int XL = KIND == kII ? 1 : 2;
  __shared__ floatx4 red[NW][NG][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, q = lane >> 4;
  const int r0 = blockIdx.x * 16, at = min(r0 + c, p.T - 1);
  const int row = p.order[at];
  const int mine = r0 + c < p.T ? p.sorted[at] : -1;
  uint64_t left = __ballot(mine >= 0);  // the tile's rows whose adapter is still to come
  auto first = [&] { return __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)left) - 1); };
  // to the block's next adapter, gridDim.y further on
  auto skip = [&](int k) {
    for (; k > 0 && left; --k) left &= ~__ballot(mine == first());
  };
  skip(blockIdx.y);
  if (!left) return;
  const char* const xr = p.x + (size_t)row * p.row_bytes + q * (16 * XL);
  const float xs = KIND == kII ? p.xs[row] : 1.0f;
  const int groups = (p.rank + 15) >> 4;
  uint4 x[CB][XL];
  auto load_x = [&](int kb) {
#pragma unroll
    for (int i = 0; i < CB; ++i) {
      if (kb + NW * i < p.kc) {
#pragma unroll
        for (int l = 0; l < XL; ++l) x[i][l] = *reinterpret_cast<const uint4*>(xr + (kb + NW * i) * (64 * XL) + l * 16);
      }
    }
  };
  // up to NW * CB chunks the rows stay in registers for every adapter and group
  const bool once = p.kc <= NW * CB;
  load_x(wv);
  for (; left; skip(gridDim.y)) {
    const int ad = first();
    const float f = p.factor[ad] * xs;
    uint16_t* const u = reinterpret_cast<uint16_t*>(p.u) + (size_t)(r0 + c) * p.rp * 2;
    // ranks r .. r + 3 of this lane's row
    auto put = [&](int r, const floatx4 v) {
      uint16_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split_bf16(v[j], hi[j], lo[j]);
      uint16_t* d = u + (r >> 5) * 64 + (r & 31);
      *reinterpret_cast<uint2*>(d) = uint2{hi[0] | (uint32_t)hi[1] << 16, hi[2] | (uint32_t)hi[3] << 16};
      *reinterpret_cast<uint2*>(d + 32) = uint2{lo[0] | (uint32_t)lo[1] << 16, lo[2] | (uint32_t)lo[3] << 16};
    };
    for (int g0 = blockIdx.z * NG; g0 < groups; g0 += gridDim.z * NG) {
      const char* ar = p.a + (size_t)ad * p.rp * p.kcp * 128 + (size_t)g0 * p.kcp * 2048 + lane * 16;
      floatx4 acc[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) acc[g] = floatx4{0.f, 0.f, 0.f, 0.f};
      for (int kb = wv; kb < p.kc; kb += NW * CB) {
        uint4 a[CB][NG][2];
        if (!once) load_x(kb);
#pragma unroll
        for (int i = 0; i < CB; ++i) {
          const int kc = kb + NW * i;
          if (kc < p.kc) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              // (a group past the last reads the last again; its sum is not used)
              const char* src = ar + ((size_t)min(g, groups - 1 - g0) * p.kcp + kc) * 2048;
              a[i][g][0] = *reinterpret_cast<const uint4*>(src);
              a[i][g][1] = *reinterpret_cast<const uint4*>(src + 1024);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < CB; ++i) {
          if (kb + NW * i < p.kc) {
            bf16x8 x0, x1;
            if constexpr (KIND == kII) {
              cvt16(x[i][0], x0, x1);
            } else {
              x0 = as_bf16x8(x[i][0]);
              x1 = as_bf16x8(x[i][XL - 1]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
              acc[g] = mfma16(as_bf16x8(a[i][g][1]), x1, mfma16(as_bf16x8(a[i][g][0]), x0, acc[g]));
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) red[wv][g][lane] = acc[g];
      __syncthreads();
      if (wv < NG && g0 + wv < groups && mine == ad) {
        floatx4 s = red[0][wv][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) s += red[w][wv][lane];
        put((g0 + wv) * 16 + 4 * q, s * f);
      }
      __syncthreads();
    }
    // the padding's ranks meet zeros of B, so they have to be finite
    if ((groups & 1) && blockIdx.z == 0 && wv == NW - 1 && mine == ad) put(groups * 16 + 4 * q, floatx4{0.f, 0.f, 0.f, 0.f});
  }
}

// ---------------------------------------------------------------------------
// Few tokens without adapters (LinearForm::kOne): the weights stream through registers once. A block takes 16 CG
// columns for all rows, its eight waves an eighth of the chunks each; the partial sums meet
// in LDS in wave order. Bound by latency: a wave requests NB chunks at once (the whole of its
// share up to 2048 inputs).
// ---------------------------------------------------------------------------
template <int KIND, int RB, int CG>
__global__ __launch_bounds__(512) void k_linear_decode(LinearArgs p) {
  constexpr int WL = KIND == kBB ? 2 : 1;   // 16-byte weight loads per chunk and group
  constexpr int XL = KIND == kII ? 1 : 2;   // and row loads per chunk and row block
  constexpr int kFit = 40 / (CG * WL + RB * XL);  // chunks in flight: at most 160 registers
  constexpr int NB = kFit > 4 ? 4 : kFit;
  __shared__ floatx4 red[8][CG][RB][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4;
  const char* wb[CG];
#pragma unroll
  for (int g = 0; g < CG; ++g)
    wb[g] = p.w + (size_t)min((int)blockIdx.x * CG + g, p.cgs - 1) * p.cg_bytes + lane * 16;
  const char* xr[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b)
    xr[b] = p.x + (size_t)min(b * 16 + c, p.T - 1) * p.row_bytes + q * (16 * XL);
  floatx4 acc[CG][RB];
  int32x4 iacc[CG][RB];
#pragma unroll
  for (int g = 0; g < CG; ++g)
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      acc[g][b] = floatx4{0.f, 0.f, 0.f, 0.f};
      iacc[g][b] = int32x4{0, 0, 0, 0};
    }
  const int c0 = p.kc * wv / 8, c1 = p.kc * (wv + 1) / 8;
  for (int cb = c0; cb < c1; cb += NB) {
    uint4 w[NB][CG][WL], x[NB][RB][XL];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (cb + i < c1) {
#pragma unroll
        for (int g = 0; g < CG; ++g)
#pragma unroll
          for (int l = 0; l < WL; ++l)
            w[i][g][l] = load_stream16(reinterpret_cast<const int8_t*>(wb[g]) + (size_t)(cb + i) * (1024 * WL) + l * 1024);
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int l = 0; l < XL; ++l)
            x[i][b][l] = *reinterpret_cast<const uint4*>(xr[b] + (cb + i) * (64 * XL) + l * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (cb + i < c1) {
#pragma unroll
        for (int g = 0; g < CG; ++g) {
          if constexpr (KIND == kII) {
#pragma unroll
            for (int b = 0; b < RB; ++b)
              iacc[g][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(as_i32x4(w[i][g][0]), as_i32x4(x[i][b][0]), iacc[g][b],
                                                                 0, 0, 0);
          } else {
            bf16x8 lo, hi;
            if constexpr (KIND == kBI) {
              cvt16(w[i][g][0], lo, hi);
            } else {
              lo = as_bf16x8(w[i][g][0]);
              hi = as_bf16x8(w[i][g][WL - 1]);
            }
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              acc[g][b] = mfma16(lo, as_bf16x8(x[i][b][0]), acc[g][b]);
              acc[g][b] = mfma16(hi, as_bf16x8(x[i][b][XL - 1]), acc[g][b]);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < CG; ++g)
#pragma unroll
    for (int b = 0; b < RB; ++b)
      red[wv][g][b][lane] = KIND == kII ? __builtin_bit_cast(floatx4, iacc[g][b]) : acc[g][b];
  __syncthreads();
  if (wv >= CG * RB) return;
  const int g = wv / RB, b = wv % RB;
  const int row = b * 16 + c, cg = blockIdx.x * CG + g, col = cg * 16 + 4 * q;
  if (row >= p.T || cg >= p.cgs) return;
  float v[4];
  const floatx4 sc = *reinterpret_cast<const floatx4*>(p.ws + col);
  if constexpr (KIND == kII) {
    int32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += __builtin_bit_cast(int32x4, red[k][g][b][lane]);
    const float xs = p.xs[row];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)sum[j] * xs * sc[j];
  } else {
    floatx4 sum = red[0][g][b][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += red[k][g][b][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = sum[j] * sc[j];
  }
  store4(p.out + (size_t)row * p.N, col, p.N, (p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0, v);
}

// ---------------------------------------------------------------------------
// Few tokens in two launches (LinearForm::kSplit). The first: blocks of 128 columns, above 32 rows 64,
// and eight steps (128 bytes of each row), every load of a block in flight at once - the rows through
// LDS, shared by NW waves of 16 CG columns, the weights in registers - whose partial sums go to the workspace;
// and beside them the blocks of the adapters' u, which thus costs no launch of its own. The
// second adds the partial sums in order and the adapters' part, and rounds.
// 64 rows with 32 adapters of rank 16, 2048 -> 5120, int8 weights: 14.0 us, the first kernel 10.0 and
// the second 4.7; the weights, adapters and rows alone would take 3.5 us of HBM. With u in a launch of
// its own and the adapters' part in the single launch above it took 19.7.
// ---------------------------------------------------------------------------
template <int KIND, int RB, int NW, int CG>
__global__ __launch_bounds__(64 * NW) void k_linear_split(LinearArgs p, int splits, int shrink_blocks) {
  constexpr int ST = kSplitSteps;
  constexpr int WL = KIND == kBI ? 1 : 2;        // 16-byte weight loads per step and group
  constexpr int SA = RB * 16 * 128;              // a step's rows
  constexpr int AJ = RB * 2;                     // loads of a step: 8 rows each
  constexpr int kOrder = KIND == kII ? 0 : 1;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[ST * SA];
  // u first: its blocks take longest
  if ((int)blockIdx.x < shrink_blocks) {
    const int groups = (p.rank + 15) >> 4;
    shrink_row<KIND, NW>(p, blockIdx.x / groups, blockIdx.x % groups, reinterpret_cast<float(*)[16]>(smem));
    return;
  }
  const int block = blockIdx.x - shrink_blocks;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int split = block % splits, cg0 = (block / splits) * (NW * CG) + wv * CG;
  const int steps = KIND == kII ? (p.kc + 1) >> 1 : p.kc;
  const int s0 = split * ST, n = min(ST, steps - s0);
  const uint32_t lds0 = lds_addr(smem);
  uint4 w[ST][CG][WL];
#pragma unroll
  for (int i = 0; i < ST; ++i) {
    if (i < n) {
#pragma unroll
      for (int g = 0; g < CG; ++g)
#pragma unroll
        for (int l = 0; l < WL; ++l)
          w[i][g][l] = load_stream16(reinterpret_cast<const int8_t*>(p.w) +
                                     (size_t)min(cg0 + g, p.cgs - 1) * p.cg_bytes + (size_t)(s0 + i) * (1024 * WL) +
                                     l * 1024 + lane * 16);
    }
  }
  // the loads of all steps' rows, shared out over the waves
#pragma unroll
  for (int j = 0; j < (ST * AJ + NW - 1) / NW; ++j) {
    const int i = (wv + NW * j) / AJ, r8 = (wv + NW * j) % AJ;
    if (i < n) {
      const int r = 8 * r8 + (lane >> 3);
      const uint32_t off = (uint32_t)min(r, p.T - 1) * p.row_bytes + (uint32_t)(a_piece_at<kOrder>(r, lane & 7) * 16);
      dma16(off, p.x + (size_t)(s0 + i) * 128, __builtin_amdgcn_readfirstlane(lds0 + i * SA + r8 * 1024));
    }
  }
  floatx4 acc[CG][RB];
  int32x4 iacc[CG][RB];
#pragma unroll
  for (int g = 0; g < CG; ++g)
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      acc[g][b] = floatx4{0.f, 0.f, 0.f, 0.f};
      iacc[g][b] = int32x4{0, 0, 0, 0};
    }
  vm_barrier<0>();
#pragma unroll
  for (int i = 0; i < ST; ++i) {
    if (i < n) {
      const uint16_t* As = reinterpret_cast<const uint16_t*>(smem + i * SA);
      bf16x8 f[CG][2];
#pragma unroll
      for (int g = 0; g < CG; ++g) {
        if constexpr (KIND == kBI) {
          cvt16(w[i][g][0], f[g][0], f[g][1]);
        } else {
          f[g][0] = as_bf16x8(w[i][g][0]);
          f[g][1] = as_bf16x8(w[i][g][WL - 1]);
        }
      }
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const bf16x8 a =
              *reinterpret_cast<const bf16x8*>(As + a_at<kOrder>(b * 16 + c, KIND == kII ? 4 * st + q : 2 * q + st));
#pragma unroll
          for (int g = 0; g < CG; ++g) {
            if constexpr (KIND == kII)
              iacc[g][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int32x4, f[g][st]),
                                                                 __builtin_bit_cast(int32x4, a), iacc[g][b], 0, 0, 0);
            else
              acc[g][b] = mfma16(f[g][st], a, acc[g][b]);
          }
        }
    }
  }
#pragma unroll
  for (int g = 0; g < CG; ++g) {
    if (cg0 + g >= p.cgs) continue;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int row = b * 16 + c;
      if (row < p.T)
        p.part[((size_t)split * p.T + row) * (p.cgs * 4) + (cg0 + g) * 4 + q] =
            KIND == kII ? __builtin_bit_cast(floatx4, iacc[g][b]) : acc[g][b];
    }
  }
}

// One wave: 256 columns of a row, four per lane, so that the adapter's B is read in whole
// lines (a wave on 16 columns of 16 rows, which its sums would come to more easily, took
// 23 us instead of 19.6 for 24 rows of rank 64, 4096 -> 9216).
template <int KIND>
__global__ __launch_bounds__(64) void k_linear_finish(LinearArgs p, int splits) {
  const int quad = blockIdx.x * 64 + threadIdx.x, row = blockIdx.y, cg = quad >> 2, q = quad & 3;
  if (cg >= p.cgs) return;
  const int ad = p.adapter ? p.adapter[row] : -1;
  const floatx4* part = p.part + (size_t)row * (p.cgs * 4) + quad;
  const size_t pitch = (size_t)p.T * (p.cgs * 4);
  const floatx4 sc = *reinterpret_cast<const floatx4*>(p.ws + quad * 4);
  float v[4];
  if constexpr (KIND == kII) {
    int32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
    for (int k = 0; k < splits; ++k) sum += __builtin_bit_cast(int32x4, part[k * pitch]);
    const float xs = p.xs[row];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)sum[j] * xs * sc[j];
  } else {
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < splits; ++k) sum += part[k * pitch];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = sum[j] * sc[j];
  }
  if (ad >= 0) {
    const float* const u = reinterpret_cast<const float*>(p.u) + (size_t)row * p.rp;
    const char* const bb = p.b + ((size_t)ad * p.cgs + cg) * (p.rp * 32) + q * 64;
    floatx4 extra = {0.f, 0.f, 0.f, 0.f};
    const int r8 = (p.rank + 7) >> 3;
#pragma unroll 4
    for (int s = 0; s < r8; ++s) {
      const floatx4 u0 = *reinterpret_cast<const floatx4*>(u + s * 8), u1 = *reinterpret_cast<const floatx4*>(u + s * 8 + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[8];
        unpack8(*reinterpret_cast<const uint4*>(bb + s * 256 + j * 16), f);
#pragma unroll
        for (int k = 0; k < 4; ++k) extra[j] = __builtin_fmaf(u0[k], f[k], extra[j]);
#pragma unroll
        for (int k = 0; k < 4; ++k) extra[j] = __builtin_fmaf(u1[k], f[4 + k], extra[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += extra[j];
  }
  store4(p.out + (size_t)row * p.N, quad * 4, p.N, (p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0, v);
}

// ---------------------------------------------------------------------------
// Many tokens or columns (LinearForm::kTiles): a GEMM over tiles of BM rows and BN columns. Steps of 128 bytes of
// every row (64 bf16, 128 int8) and the columns' weights of the same depth reach LDS by direct
// loads, a ring of NS stages. Rows as [row][8 x 16 B] with the pieces swizzled by row
// (a_piece_at), the weights in the packed order, which is the order their lanes read. The
// weights are the MFMA's first operand: a lane ends with four consecutive columns.
// A step is two halves, and each half's fragments are read while the MFMAs of the half before
// run (the order is held by scheduling groups); the one barrier of a step stands between
// them, where the stage has been read and the next one has landed.
//
// With adapters the rows are the sorted ones, so a tile meets few adapters. After the
// base sum, scaled to f32, each adapter of the tile adds steps of 32 ranks in the same
// ring: the tile's rows of u (hi and lo, 128 bytes) times the adapter's B. The product of a
// 16-row group is computed apart and added to the adapter's own rows by selection, so that
// nothing of another adapter (an infinity times zero) reaches a row, and a row's sums are the
// same whatever its neighbours take (adding in place where a group is of one adapter was no
// faster).
// ---------------------------------------------------------------------------
template <int KIND, int WM, int WN, int MI, int NI, int NS, bool LORA>
struct GemmShape {
  static constexpr int kThreads = 64 * WM * WN, kRows = 16 * WM * MI, kCols = 16 * WN * NI;
  static constexpr int kStage = kRows * 128 + kCols / 16 * (KIND == kBI ? 1024 : 2048);
  static constexpr int kLds = NS * kStage, kSeg = LORA ? 3 * kRows : 3;
};

// One tile: rows from r0 on and column groups from cg0 on, with smem of kLds bytes and seg of
// kSeg ints (per tile row: token, adapter, where the adapter's rows end). Every thread of the
// block calls it, once.
template <int KIND, int WM, int WN, int MI, int NI, int NS, bool LORA>
__device__ __forceinline__ void gemm_tile(const LinearArgs& p, uint8_t* smem, int* segs, int r0, int cg0) {
  constexpr int NW = WM * WN, BM = 16 * WM * MI, BN = 16 * WN * NI;
  constexpr int BB = KIND == kBI ? 1024 : 2048;  // weight bytes of a column group per step
  constexpr int SA = BM * 128, SB = BN / 16 * BB, SS = SA + SB;
  constexpr int AJ = BM / 8 / NW, BJ = SB / 1024 / NW, PER = AJ + BJ;
  constexpr int LJ = BN / 16 / NW, LPER = AJ + LJ;  // of an adapters' step; LJ <= BJ
  static_assert(BM % (8 * NW) == 0 && SB % (1024 * NW) == 0 && BN / 16 % NW == 0, "whole loads per wave");
  constexpr int kOrder = KIND == kII ? 0 : 1;
  int (*const seg)[LORA ? BM : 1] = reinterpret_cast<int(*)[LORA ? BM : 1]>(segs);
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int wm = wv / WN, wn = wv % WN;
  const int rows = min(BM, p.T - r0);
  const uint32_t lds0 = lds_addr(smem);
  auto stage_at = [&](int s, int off) { return __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)((s % NS) * SS + off)); };

  if constexpr (LORA) {
    for (int r = tid; r < BM; r += 64 * NW) {
      const int pos = min(r0 + r, p.T - 1);
      const int ad = r < rows ? p.sorted[pos] : -1;
      seg[0][r] = p.order[pos];
      seg[1][r] = ad;
      seg[2][r] = ad < 0 ? rows : min(max(p.offsets[ad + 1] - r0, r + 1), rows);
    }
  }
  const char* bsrc[BJ];
#pragma unroll
  for (int j = 0; j < BJ; ++j) {
    const int at = (wv + NW * j) * 1024;
    bsrc[j] = p.w + (size_t)min(cg0 + at / BB, p.cgs - 1) * p.cg_bytes + at % BB;
  }
  if constexpr (LORA) __syncthreads();
  uint32_t aoff[AJ];
#pragma unroll
  for (int j = 0; j < AJ; ++j) {
    const int r = 8 * (wv + NW * j) + (lane >> 3);
    int row = min(r0 + r, p.T - 1);
    if constexpr (LORA) row = seg[0][r];
    aoff[j] = (uint32_t)row * p.row_bytes + (uint32_t)(a_piece_at<kOrder>(r, lane & 7) * 16);
  }
  auto issue = [&](int s) {
#pragma unroll
    for (int j = 0; j < BJ; ++j)
      dma16(lane * 16, bsrc[j] + (size_t)s * BB, stage_at(s, SA + (wv + NW * j) * 1024));
#pragma unroll
    for (int j = 0; j < AJ; ++j) dma16(aoff[j], p.x + (size_t)s * 128, stage_at(s, (wv + NW * j) * 1024));
  };
  // the adapters' steps: `at` is the tile row where the adapter starts (rows: none left)
  struct Cursor {
    int at, ad, end, s;
  };
  const int rb = LORA ? p.rp >> 5 : 0;
  auto enter = [&](Cursor& k, int at) {
    k.at = at;
    k.s = 0;
    if (at < rows) {
      k.ad = __builtin_amdgcn_readfirstlane(seg[LORA ? 1 : 0][LORA ? at : 0]);
      k.end = __builtin_amdgcn_readfirstlane(seg[LORA ? 2 : 0][LORA ? at : 0]);
      if (k.ad < 0) k.at = rows;
    }
  };
  auto advance = [&](Cursor& k) {
    if (++k.s == rb) enter(k, k.end);
  };
  const char* const ubase = reinterpret_cast<const char*>(p.u) + (size_t)r0 * rb * 128;
  auto issue_lora = [&](const Cursor& k, int s) {
#pragma unroll
    for (int j = 0; j < LJ; ++j) {
      const int cg = min(cg0 + wv + NW * j, p.cgs - 1);
      dma16(lane * 16, p.b + (((size_t)k.ad * p.cgs + cg) * rb + k.s) * 1024, stage_at(s, SA + (wv + NW * j) * 1024));
    }
#pragma unroll
    for (int j = 0; j < AJ; ++j) {
      const int r = 8 * (wv + NW * j) + (lane >> 3);
      dma16((uint32_t)min(r, rows - 1) * (uint32_t)(rb * 128) + (uint32_t)(a_piece_at<1>(r, lane & 7) * 16),
            ubase + k.s * 128, stage_at(s, (wv + NW * j) * 1024));
    }
  };
  // the adapters' steps take the ring's stages after the base steps
  Cursor next{rows, -1, rows, 0}, cur{rows, -1, rows, 0};
  const int steps = KIND == kII ? (p.kc + 1) >> 1 : p.kc;
  int issued = steps;  // the first step whose loads are not under way (while base steps are left: that of the adapters')
  auto issue_next = [&] {
    if (next.at >= rows) return;
    issue_lora(next, issued++);
    advance(next);
  };
  // step s has landed, every wave is done with the stages before it, and of the steps behind
  // it the last NS - 2 may be under way, if there are as many
  auto lora_barrier = [&](int s) {
    if (NS > 2 && issued - s > NS - 2)
      vm_barrier<(NS - 2) * LPER>();
    else
      vm_barrier<0>();
  };
  if constexpr (LORA) {
    enter(next, 0);
    cur = next;
  }

  floatx4 acc[MI][NI];  // kII: the bits of i32 sums until they are scaled
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = floatx4{0.f, 0.f, 0.f, 0.f};
  // fragments of half a step (int8 weights with bf16 rows: the raw bytes of the whole step
  // are read with its first half)
  struct Half {
    bf16x8 a[MI];
    bf16x8 w[NI];
  };
  auto read_a = [&](int s, int st, Half& f) {
    const uint16_t* As = reinterpret_cast<const uint16_t*>(smem + (s % NS) * SS) + wm * MI * 16 * 64;
#pragma unroll
    for (int m = 0; m < MI; ++m)
      f.a[m] = *reinterpret_cast<const bf16x8*>(As + a_at<kOrder>(m * 16 + c, KIND == kII ? 4 * st + q : 2 * q + st));
  };
  auto weights = [&](int s) { return smem + (s % NS) * SS + SA + wn * NI * BB + lane * 16; };
  auto read_w = [&](int s, int st, Half& f) {
    const uint8_t* Bs = weights(s) + st * 1024;
#pragma unroll
    for (int n = 0; n < NI; ++n) f.w[n] = *reinterpret_cast<const bf16x8*>(Bs + n * BB);
  };
  auto multiply = [&](const Half& f) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if constexpr (KIND == kII)
          acc[m][n] = __builtin_bit_cast(
              floatx4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int32x4, f.w[n]),
                                                             __builtin_bit_cast(int32x4, f.a[m]),
                                                             __builtin_bit_cast(int32x4, acc[m][n]), 0, 0, 0));
        else
          acc[m][n] = mfma16(f.w[n], f.a[m], acc[m][n]);
      }
  };
  // one read, then its share of the MFMAs, ...
  auto interleave = [&] {
    constexpr int R = MI + NI, M = MI * NI, each = M / R < 1 ? 1 : M / R;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, each, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, M, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    if (s < steps)
      issue(s);
    else if constexpr (LORA)
      issue_next();
  }
  if (steps >= NS)
    vm_barrier<(NS - 1) * PER>();
  else
    vm_barrier<0>();
  Half f0, f1;
  uint4 raw[KIND == kBI ? NI : 1];
  auto read_first = [&](int s) {
    read_a(s, 0, f0);
    if constexpr (KIND == kBI) {
#pragma unroll
      for (int n = 0; n < NI; ++n) raw[n] = *reinterpret_cast<const uint4*>(weights(s) + n * BB);
    } else {
      read_w(s, 0, f0);
    }
  };
  auto step = [&](int s, auto tail) {
    read_a(s, 1, f1);
    if constexpr (KIND == kBI) {
#pragma unroll
      for (int n = 0; n < NI; ++n) cvt16(raw[n], f0.w[n], f1.w[n]);
    } else {
      read_w(s, 1, f1);
    }
    multiply(f0);
    interleave();
    if constexpr (decltype(tail)::value) {
      if constexpr (LORA) {
        lora_barrier(s + 1);
        issue_next();  // the adapters' first steps, while the last base steps run
      } else {
        vm_barrier<0>();
      }
    } else {
      vm_barrier<(NS - 2) * PER>();
      issue(s + NS);
    }
    __builtin_amdgcn_sched_barrier(0);
    read_first(s + 1);  // past the last step: what the stage holds, not used
    multiply(f1);
    interleave();
  };
  read_first(0);
  int s = 0;
  for (; s + NS < steps; ++s) step(s, std::false_type{});
  for (; s < steps; ++s) step(s, std::true_type{});

  // scaled to f32, row by row of the accumulators (all at once took 60 registers more)
  if constexpr (KIND != kBB) {
    floatx4 sc[NI];
#pragma unroll
    for (int n = 0; n < NI; ++n)
      sc[n] = *reinterpret_cast<const floatx4*>(p.ws + min(cg0 + wn * NI + n, p.cgs - 1) * 16 + 4 * q);
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      float xs = 1.0f;
      if constexpr (KIND == kII) {
        const int r = (wm * MI + m) * 16 + c;
        int row = min(r0 + r, p.T - 1);
        if constexpr (LORA) row = seg[0][r];
        xs = p.xs[row];
      }
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if constexpr (KIND == kII)
          acc[m][n] = __builtin_convertvector(__builtin_bit_cast(int32x4, acc[m][n]), floatx4) * xs * sc[n];
        else
          acc[m][n] *= sc[n];
      }
    }
  }
  if constexpr (LORA) {
    const int w0 = wm * MI * 16;  // the wave's rows in the tile
    for (; cur.at < rows; advance(cur), ++s) {
      lora_barrier(s);
      if (s > steps) issue_next();  // (the last base step's stage has its loads)
      const uint16_t* As = reinterpret_cast<const uint16_t*>(smem + (s % NS) * SS) + w0 * 64;
      const uint8_t* Bs = smem + (s % NS) * SS + SA + wn * NI * 1024 + c * 16;
      bf16x8 wf[2][NI];
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int n = 0; n < NI; ++n)
          wf[st][n] = *reinterpret_cast<const bf16x8*>(Bs + n * 1024 + (2 * (q & 1) + st) * 256);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int g0 = w0 + m * 16;
        if (g0 + 16 <= cur.at || g0 >= cur.end) continue;
        const bf16x8 a0 = *reinterpret_cast<const bf16x8*>(As + a_at<1>(m * 16 + c, 2 * q));
        const bf16x8 a1 = *reinterpret_cast<const bf16x8*>(As + a_at<1>(m * 16 + c, 2 * q + 1));
        const bool mine = g0 + c >= cur.at && g0 + c < cur.end;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          const floatx4 t = mfma16(wf[1][n], a1, mfma16(wf[0][n], a0, floatx4{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[m][n][j] = mine ? acc[m][n][j] + t[j] : acc[m][n][j];
        }
      }
    }
  }
  const bool vec = (p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0;
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int r = (wm * MI + m) * 16 + c;
    if (r >= rows) continue;
    int row = r0 + r;
    if constexpr (LORA) row = seg[0][r];
    uint16_t* o = p.out + (size_t)row * p.N;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int cg = cg0 + wn * NI + n;
      if (cg >= p.cgs) continue;
      const float v[4] = {acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]};
      store4(o, cg * 16 + 4 * q, p.N, vec, v);
    }
  }
}

// Tile L of tm x tn: groups of eight row tiles, row tiles fastest, so that the tiles that run
// together on an XCD share rows and columns in its L2.
__device__ __forceinline__ void tile_at(int L, int tm, int tn, int& mt, int& nt) {
  constexpr int GM = 8;
  const int grp = L / (GM * tn), in = L - grp * GM * tn, gsz = min(tm - grp * GM, GM);
  mt = grp * GM + in % gsz;
  nt = in / gsz;
}

// block i of n (a multiple of 8) as an index whose neighbours share an XCD
__device__ __forceinline__ int xcd_order(int i, int n) { return (i & 7) * (n >> 3) + (i >> 3); }

// Tiles of one size.
template <int KIND, int WM, int WN, int MI, int NI, int NS, bool LORA>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_linear_gemm(LinearArgs p, int tm, int tn) {
  using Sh = GemmShape<KIND, WM, WN, MI, NI, NS, LORA>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[Sh::kLds];
  __shared__ int seg[Sh::kSeg];
  const int L = xcd_order(blockIdx.x, gridDim.x);
  if (L >= tm * tn) return;
  int mt, nt;
  tile_at(L, tm, tn, mt, nt);
  gemm_tile<KIND, WM, WN, MI, NI, NS, LORA>(p, smem, seg, mt * Sh::kRows, nt * (Sh::kCols / 16));
}

// Many tiles: the first `whole` of 256 x 256, one per CU and round; the rest as quarters of
// 128 x 128, so that the last round is a short one.
template <int KIND, bool LORA>
__global__ __launch_bounds__(512, 2) void k_linear_gemm_mixed(LinearArgs p, int tm, int tn, int whole) {
  using Big = GemmShape<KIND, 2, 4, 8, 4, 2, LORA>;
  using Small = GemmShape<KIND, 2, 4, 4, 2, 4, LORA>;
  static_assert(Big::kThreads == Small::kThreads && Small::kLds <= Big::kLds && Small::kSeg <= Big::kSeg, "one block");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[Big::kLds];
  __shared__ int seg[Big::kSeg];
  int mt, nt;
  if ((int)blockIdx.x < whole) {
    const int L = xcd_order(blockIdx.x, whole);
    if (L >= tm * tn) return;
    tile_at(L, tm, tn, mt, nt);
    gemm_tile<KIND, 2, 4, 8, 4, 2, LORA>(p, smem, seg, mt * 256, nt * 16);
    return;
  }
  const int i = xcd_order(blockIdx.x - whole, gridDim.x - whole), L = whole + (i >> 2);
  if (L >= tm * tn) return;
  tile_at(L, tm, tn, mt, nt);
  const int r0 = mt * 256 + (i & 1) * 128, cg0 = nt * 16 + (i >> 1 & 1) * 8;
  if (r0 >= p.T || cg0 >= p.cgs) return;
  gemm_tile<KIND, 2, 4, 4, 2, 4, LORA>(p, smem, seg, r0, cg0);
}

}  // namespace kmoe

namespace kmoe_host {

using namespace kmoe;

namespace {

dim3 grid_for(int64_t items) {
  const int64_t blocks = (items + 255) / 256;
  return dim3((unsigned)(blocks < 1 ? 1 : (blocks > 65536 ? 65536 : blocks)));
}

template <int KIND, int RB>
void decode_of(const LinearArgs& p, bool split, hipStream_t st) {
  if (split) {
    // Up to 32 rows bf16 rows take eight waves of 16 columns, int8 rows, whose blocks cover twice the
    // inputs in the same LDS and convert nothing, four of 32; above, where a block's rows fill more of
    // the LDS, both take four of 16, so that more blocks run. us, 24 rows of rank 64, 4096 -> 9216: int8
    // weights 23.1 (four of 16 28.9), int8 rows 19.6 (28.2); 64 rows of rank 16, 4096 -> 2048, bf16
    // weights 16.3 with eight, 13.9 with four of 16, int8 rows 12.5 with four of 32, 11.0; 48 rows
    // 15.3, 13.1 and 11.5, 10.3.
    constexpr int NW = RB > 2 || KIND == kII ? 4 : 8, CG = RB < 3 && KIND == kII ? 2 : 1, ST = kSplitSteps;
    const int steps = KIND == kII ? (p.kc + 1) / 2 : p.kc, splits = (steps + ST - 1) / ST;
    const int blocks = (p.cgs + NW * CG - 1) / (NW * CG) * splits, shrink = p.adapter ? p.T * ((p.rank + 15) / 16) : 0;
    hipLaunchKernelGGL((k_linear_split<KIND, RB, NW, CG>), dim3(shrink + blocks), dim3(64 * NW), 0, st, p, splits,
                       shrink);
    hipLaunchKernelGGL((k_linear_finish<KIND>), dim3((p.cgs * 4 + 63) / 64, p.T), dim3(64), 0, st, p, splits);
  } else if (RB == 4 || decode_groups(p.cgs) == 1) {  // (four row groups never take two: linear_form)
    hipLaunchKernelGGL((k_linear_decode<KIND, RB, 1>), dim3(p.cgs), dim3(512), 0, st, p);
  } else if constexpr (RB < 4) {
    hipLaunchKernelGGL((k_linear_decode<KIND, RB, 2>), dim3((p.cgs + 1) / 2), dim3(512), 0, st, p);
  }
}

template <int KIND>
void decode(const LinearArgs& p, bool split, hipStream_t st) {
  switch ((p.T + 15) / 16) {
    case 1:
      return decode_of<KIND, 1>(p, split, st);
    case 2:
      return decode_of<KIND, 2>(p, split, st);
    case 3:
      return decode_of<KIND, 3>(p, split, st);
    default:
      return decode_of<KIND, 4>(p, split, st);
  }
}

template <int KIND, int WM, int WN, int MI, int NI, int NS>
void gemm_of(const LinearArgs& p, hipStream_t st) {
  constexpr int BM = 16 * WM * MI, BN = 16 * WN * NI;
  const int tm = (p.T + BM - 1) / BM, tn = (p.cgs * 16 + BN - 1) / BN;
  const dim3 grid((unsigned)((((int64_t)tm * tn + 7) >> 3) * 8));
  if (p.adapter)
    hipLaunchKernelGGL((k_linear_gemm<KIND, WM, WN, MI, NI, NS, true>), grid, dim3(64 * WM * WN), 0, st, p, tm, tn);
  else
    hipLaunchKernelGGL((k_linear_gemm<KIND, WM, WN, MI, NI, NS, false>), grid, dim3(64 * WM * WN), 0, st, p, tm, tn);
}

template <int KIND>
void gemm(const LinearArgs& p, hipStream_t st) {
  // The smaller tiles are bound by LDS reads, so their four waves stand 2 x 2; int8 weights with
  // bf16 rows, which each wave converts for itself, want them 1 x 4 (64 x 64: 2048 -> 5120, 512
  // rows 19.0 against 21.3, bf16 weights 22.8 against 22.0).
  switch (linear_tile(p.T, p.cgs, KIND == kBI, p.adapter != nullptr)) {
    case LinearTile::k256x256: {
      const int tm = (p.T + 255) / 256, tn = (p.cgs + 15) / 16;
      const LinearRounds r = linear_rounds((int64_t)tm * tn);
      if (p.adapter)
        hipLaunchKernelGGL((k_linear_gemm_mixed<KIND, true>), dim3((unsigned)r.blocks), dim3(512), 0, st, p, tm, tn,
                           (int)r.whole);
      else
        hipLaunchKernelGGL((k_linear_gemm_mixed<KIND, false>), dim3((unsigned)r.blocks), dim3(512), 0, st, p, tm, tn,
                           (int)r.whole);
      return;
    }
    case LinearTile::k128x128:
      return gemm_of<KIND, 2, 2, 4, 4, 2>(p, st);
    case LinearTile::k64x128:
      if constexpr (KIND == kBI)
        return gemm_of<KIND, 1, 4, 4, 2, 3>(p, st);
      else
        return gemm_of<KIND, 2, 2, 2, 4, 2>(p, st);
    case LinearTile::k64x64:
      if constexpr (KIND == kBI)
        return gemm_of<KIND, 1, 4, 4, 1, 4>(p, st);
      else
        return gemm_of<KIND, 2, 2, 2, 2, 4>(p, st);
    case LinearTile::k32x64:
      return gemm_of<KIND, 1, 4, 2, 1, 4>(p, st);
  }
}

template <int KIND>
void shrink(const LinearArgs& p, int adapters, hipStream_t st) {
  const LoraShrink s = lora_shrink(p.T, p.rank, adapters);
  const dim3 grid((p.T + 15) / 16, s.y, s.z);
  if (s.groups == 1)
    hipLaunchKernelGGL((k_lora_shrink<KIND, 1>), grid, dim3(1024), 0, st, p);
  else if (s.groups == 2)
    hipLaunchKernelGGL((k_lora_shrink<KIND, 2>), grid, dim3(1024), 0, st, p);
  else
    hipLaunchKernelGGL((k_lora_shrink<KIND, 4>), grid, dim3(1024), 0, st, p);
}

template <int KIND>
void linear_kind(const LinearArgs& p, LinearForm form, int adapters, hipStream_t st) {
  if (form != LinearForm::kTiles) return decode<KIND>(p, form == LinearForm::kSplit, st);
  if (p.adapter) shrink<KIND>(p, adapters, st);
  gemm<KIND>(p, st);
}

}  // namespace

hipError_t launch_linear_pack(const kmoe_weight& w, const kmoe_linear_weight& packed, hipStream_t st) {
  const int K = (int)packed.in_features, N = (int)packed.out_features;
  const int Kp = (int)padded_in(K), Np = (int)padded_out(N);
  if (packed.dtype == KMOE_DTYPE_BF16)
    hipLaunchKernelGGL(k_pack_bf16, grid_for((int64_t)Kp * Np / 8), dim3(256), 0, st, (int64_t)1, K, N, Kp, Np,
                       reinterpret_cast<const uint16_t*>(w.values), reinterpret_cast<uint16_t*>(packed.values));
  else
    hipLaunchKernelGGL(k_pack_i8, grid_for((int64_t)Kp * Np / 16), dim3(256), 0, st, K, N, Kp, Np,
                       reinterpret_cast<const uint8_t*>(w.values), reinterpret_cast<uint8_t*>(packed.values));
  hipLaunchKernelGGL(k_pack_scale, dim3((Np + 255) / 256), dim3(256), 0, st, N, Np, (int)w.scale_kind,
                     w.scale_dtype == KMOE_DTYPE_BF16 ? 1 : 0, w.scale, packed.scale);
  return hipGetLastError();
}

hipError_t launch_lora_pack(const kmoe_lora& l, int64_t first, int64_t count, int64_t rank, const void* a,
                            const void* b, const float* factor, hipStream_t st) {
  const int K = (int)l.in_features, N = (int)l.out_features, rp = (int)padded_rank(l.rank);
  const int Kp = (int)padded_in(K), Np = (int)padded_out(N);
  hipLaunchKernelGGL(k_pack_bf16, grid_for(count * rp * Kp / 8), dim3(256), 0, st, count, K, (int)rank, Kp, rp,
                     reinterpret_cast<const uint16_t*>(a), reinterpret_cast<uint16_t*>(l.a) + (size_t)first * rp * Kp);
  hipLaunchKernelGGL(k_pack_lora_b, grid_for(count * rp * Np / 8), dim3(256), 0, st, count, (int)rank, N, rp, Np,
                     reinterpret_cast<const uint16_t*>(b), reinterpret_cast<uint16_t*>(l.b) + (size_t)first * rp * Np);
  hipLaunchKernelGGL(k_copy_f32, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, st, count, factor,
                     l.factor + first);
  return hipGetLastError();
}

hipError_t launch_lora_sort(const int32_t* adapter, const kmoe_lora_batch& b, void* scratch, hipStream_t st) {
  const int T = (int)b.tokens, L = (int)b.num_adapters, blocks = (T + kLoraSortBlock - 1) / kLoraSortBlock;
  int32_t* hist = reinterpret_cast<int32_t*>(scratch);
  if (blocks > 1)
    hipLaunchKernelGGL(k_lora_count, dim3(blocks), dim3(kLoraSortBlock), 0, st, T, L, adapter, hist);
  hipLaunchKernelGGL(k_lora_sort, dim3(blocks), dim3(kLoraSortBlock), 0, st, T, L, adapter, hist, blocks, b.adapter,
                     b.order, b.sorted, b.offsets);
  return hipGetLastError();
}

hipError_t launch_linear(const kmoe_linear_weight& w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                         int64_t x_stride, const float* x_scale, const kmoe_lora* lora, const kmoe_lora_batch* batch,
                         void* out, void* workspace, const LinearSpace& space, hipStream_t st) {
  const int K = (int)w.in_features, Kp = (int)padded_in(K);
  const size_t size = dtype_size(x_dtype);
  char* const ws = reinterpret_cast<char*>(workspace);
  LinearArgs p{};
  p.x = reinterpret_cast<const char*>(x);
  p.row_bytes = (uint32_t)(x_stride * (int64_t)size);
  if (!linear_rows_fit(w, x, x_dtype, x_stride)) {
    const dim3 grid = grid_for(tokens * Kp);
    if (x_dtype == KMOE_DTYPE_I8)
      hipLaunchKernelGGL((k_stage_rows<uint8_t>), grid, dim3(256), 0, st, tokens, K, Kp, x_stride,
                         reinterpret_cast<const uint8_t*>(x), reinterpret_cast<uint8_t*>(ws));
    else
      hipLaunchKernelGGL((k_stage_rows<uint16_t>), grid, dim3(256), 0, st, tokens, K, Kp, x_stride,
                         reinterpret_cast<const uint16_t*>(x), reinterpret_cast<uint16_t*>(ws));
    p.x = ws;
    p.row_bytes = (uint32_t)(Kp * size);
  }
  p.xs = x_scale;
  p.w = reinterpret_cast<const char*>(w.values);
  p.ws = w.scale;
  p.out = reinterpret_cast<uint16_t*>(out);
  p.T = (int)tokens;
  p.N = (int)w.out_features;
  p.kc = (K + 63) / 64;
  p.cgs = (int)(padded_out(w.out_features) / 16);
  p.cg_bytes = (size_t)Kp * 16 * dtype_size(w.dtype);
  if (lora) {
    p.adapter = batch->adapter;
    p.order = batch->order;
    p.sorted = batch->sorted;
    p.offsets = batch->offsets;
    p.a = reinterpret_cast<const char*>(lora->a);
    p.b = reinterpret_cast<const char*>(lora->b);
    p.factor = lora->factor;
    p.rank = (int)lora->rank;
    p.rp = (int)padded_rank(lora->rank);
    p.kcp = Kp / 64;
    p.u = ws + space.u;
  }
  p.part = reinterpret_cast<floatx4*>(ws + space.part);
  const LinearForm form = linear_form(w, tokens, x_dtype, lora != nullptr);
  const int adapters = lora ? (int)lora->num_adapters : 0;
  if (x_dtype == KMOE_DTYPE_I8)
    linear_kind<kII>(p, form, adapters, st);
  else if (w.dtype == KMOE_DTYPE_I8)
    linear_kind<kBI>(p, form, adapters, st);
  else
    linear_kind<kBB>(p, form, adapters, st);
  return hipGetLastError();
}

}  // namespace kmoe_host
