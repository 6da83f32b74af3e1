// The steps on either side of the MoE block in a Qwen3 MoE layer
// (kappa/qwen3/block.py:196-207): the pre-FFN RMSNorm that produces the
// block's input, and (in the combine kernels of expert.hip) the residual add
// of its output.
//
// rms_norm (kappa/qwen3/norms.py:10-16) in a canonical order shared with the
// oracle: the squares f32(h)*f32(h), each rounded to float, are summed per
// 64-wide slice in a sequential chain from +0.0f, and the slice sums are
// combined by the same zero-padded pairwise tree as the router logits;
// var = S / D, r = 1 / sqrt(var + eps) with IEEE division and square root, and
// h2 = round_act((f32(h) * r) * f32(scale)).
#include <float.h>

#include <algorithm>

#include "common.h"
#include "expert_dev.h"
#include "launch.h"
#include "norm.h"

namespace kmoe {

constexpr int kNormWaves = 4;  // tokens per block, one wave each
constexpr int kNormNarrow = 128;    // 16-byte pieces of a row that one wave takes in add_rms_norm
constexpr int kNormManyRows = 1000;  // above this many rows

// 16 bytes (or the run of 16-byte loads) of the scale that go with a piece of the row
template <typename A, typename S>
__device__ __forceinline__ void scale_piece(const S* __restrict__ scale, int piece, float* f) {
  constexpr int n = NormRow<A>::kPiece;
  if constexpr (sizeof(S) == 2 && n == 4) {
    const uint2 v = reinterpret_cast<const uint2*>(scale)[piece];
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
  } else {
    constexpr int per = NormRow<S>::kPiece;
#pragma unroll
    for (int i = 0; i < n / per; ++i)
      NormRow<S>::unpack(reinterpret_cast<const uint4*>(scale)[piece * (n / per) + i], f + i * per);
  }
}

// One wave per token: wave_rms_factor stages the row in LDS and reduces it,
// then the wave writes round_act((x * r) * scale) from the pieces it still holds.
// Latency: one row's round trip, its 64-step chain and the store (33 MB at 30B-A3B
// T = 4096: 11.7 us; element by element, with the row in LDS as floats, 17 us).
template <typename A, typename S>
__global__ __launch_bounds__(256) void k_rms_norm(int T, int D, float eps, const A* __restrict__ h,
                                                   const S* __restrict__ scale, A* __restrict__ out) {
  using R = NormRow<A>;
  extern __shared__ __attribute__((aligned(16))) uint8_t rows[];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int t = blockIdx.x * kNormWaves + w;
  if (t >= T) return;  // per wave: this kernel has no block-wide barrier
  A* row = reinterpret_cast<A*>(rows + (size_t)w * R::bytes(D));
  const A* src = h + (int64_t)t * D;
  A* dst = out + (int64_t)t * D;
  uint4 v[R::kPieces];
  const float r = wave_rms_factor(src, D, eps, row, v);
  if (R::pieces(src, D) && ((reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(scale)) & 15) == 0) {
    const int n = D / R::kPiece;
#pragma unroll
    for (int i = 0; i < R::kPieces; ++i) {
      const int p = lane + 64 * i;
      if (p < n) {
        float f[R::kPiece], sc[R::kPiece];
        R::unpack(v[i], f);
        scale_piece<A, S>(scale, p, sc);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < R::kPiece; ++j) f[j] = rms_apply<A>(f[j], r, sc[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(A) == 2)
            o[j] = (uint32_t)f32_to_bf16_bits(f[2 * j]) | ((uint32_t)f32_to_bf16_bits(f[2 * j + 1]) << 16);
          else
            o[j] = __float_as_uint(f[j]);
        }
        reinterpret_cast<uint4*>(dst)[p] = uint4{o[0], o[1], o[2], o[3]};
      }
    }
    return;
  }
  if constexpr (sizeof(A) == 2) {
    for (int d = lane; d < D; d += 64)
      Act<A>::store(dst, d, rms_apply<A>(Act<A>::load(row, R::at(d)), r, Act<S>::load(scale, d)));
    return;
  }
  for (int base = 0; base < D; base += 64 * R::kBatch) {
    float sc[R::kBatch];
#pragma unroll
    for (int j = 0; j < R::kBatch; ++j) sc[j] = Act<S>::load(scale, min(base + 64 * j + lane, D - 1));
#pragma unroll
    for (int j = 0; j < R::kBatch; ++j) {
      const int d = base + 64 * j + lane;
      if (d < D) Act<A>::store(dst, d, rms_apply<A>(Act<A>::load(row, R::at(d)), r, sc[j]));
    }
  }
}

namespace {

// 16, 8 and 4 bytes at any element's address (the hardware takes dwords off their boundary)
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));

__device__ __forceinline__ uint4 load16(const void* p) {
  const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p);
  return uint4{v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ void store16(void* p, const uint4 v) {
  *reinterpret_cast<u32x4_any*>(p) = u32x4_any{v.x, v.y, v.z, v.w};
}

// the scales that go with 16 bytes of a row of A, from element d on
template <typename A, typename S>
__device__ __forceinline__ void scale_at(const S* __restrict__ scale, int d, float* f) {
  if constexpr (sizeof(S) == 2 && sizeof(A) == 4) {
    const u32x2_any v = *reinterpret_cast<const u32x2_any*>(scale + d);
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < NormRow<A>::kPiece; i += NormRow<S>::kPiece) NormRow<S>::unpack(load16(scale + d + i), f + i);
  }
}

}  // namespace

// The residual's addition and the norm of the sum: h = round_act(x + res), written to
// hout, then rms_norm's arithmetic on h. Q8 = false: out = round_act((h * r) * scale), the
// bits of k_rms_norm on h. Q8 = true: the same products in f32 to int8, with the row's
// scale s = max(m / 127, FLT_MIN), m the largest magnitude (as an integer maximum of the f32
// bits, which an infinity or a NaN tops: such a row gets s = NaN and zeros), and
// q = rint(v / s). hout may be x or res itself: a thread reads its elements of both
// before it writes them. res NULL: h is x, and hout is not written.
// Rows move in 16-byte pieces, of any alignment; the elements behind a row's last whole piece
// one by one, by the row's first threads.
// Bound by HBM for many rows, else by one row's round trip and its 64-step chain. W = 4 waves
// share a row, W = 1 (narrow rows, many of them: add_rms_norm) leaves each to one wave:
// bf16 16384 x 2048 47 us (5.7 TB/s) with four and 53 with one, one row 3.2 and 4.3; rows of
// 512, 65536 of them, 84 with four and 48 with one (1000 of them 3.7 each).
template <typename A, typename S, bool Q8, int W>
__global__ __launch_bounds__(64 * kNormWaves) void k_add_rms_norm(int T, int D, float eps, const A* x, const A* res,
                                                                   const S* __restrict__ scale, A* hout,
                                                                   A* __restrict__ out, int8_t* __restrict__ qout,
                                                                   float* __restrict__ qscale) {
#pragma clang fp contract(off)
  using R = NormRow<A>;
  constexpr int PT = W == 1 ? kNormNarrow / 64 : R::kPieces / W;  // pieces per thread of the widest row
  constexpr int NT = 64 * W;          // threads of a row
  constexpr int P = R::kPiece;
  extern __shared__ __attribute__((aligned(16))) uint8_t rows[];
  __shared__ uint32_t factor[kNormWaves], largest[kNormWaves];  // W > 1: per row, per wave
  const int wv = threadIdx.x >> 6, sub = wv / W, me = threadIdx.x - sub * NT;
  const int t = blockIdx.x * (kNormWaves / W) + sub;
  // rows past the last repeat it and store nothing (the waves of a block meet at barriers)
  const bool live = t < T;
  const size_t at = (size_t)(live ? t : T - 1) * D;
  A* row = reinterpret_cast<A*>(rows + (size_t)sub * R::bytes(D));
  const int n = D / P, end = n * P + me;  // this thread's element behind the pieces
  const bool one = end < D;
  uint4 v[PT], o[PT];
  float sc[PT][P], h1 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int p = me + NT * i;
    if (p < n) {
      v[i] = load16(x + at + p * P);
      if (res) o[i] = load16(res + at + p * P);
      scale_at<A, S>(scale, p * P, sc[i]);
    }
  }
  if (one) {
    h1 = Act<A>::load(x, at + end);
    if (res) h1 = Act<A>::round(h1 + Act<A>::load(res, at + end));
    s1 = Act<S>::load(scale, end);
  }
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int p = me + NT * i;
    if (p < n) {
      if (res) {
        float a[P], b[P];
        R::unpack(v[i], a);
        R::unpack(o[i], b);
#pragma unroll
        for (int j = 0; j < P; ++j) a[j] = a[j] + b[j];
        v[i] = R::pack(a);
        if (live) store16(hout + at + p * P, v[i]);
      }
      *reinterpret_cast<uint4*>(row + R::at(p * P)) = v[i];
    }
  }
  if (one) {
    if (res && live) Act<A>::store(hout, at + end, h1);
    Act<A>::store(row, R::at(end), h1);
  }
  // the last slice is filled up with zeros, whose squares leave its chain as it is
  const int fill = (D - 1) / kRouterSlice * kRouterSlice + me;
  if (me < kRouterSlice && fill >= D) row[R::at(fill)] = 0;
  float r;
  if constexpr (W == 1) {
    r = wave_rms_reduce(row, D, eps);
  } else {
    __syncthreads();
    if (me < 64) factor[sub] = __float_as_uint(wave_rms_reduce(row, D, eps));
    __syncthreads();
    r = __uint_as_float(factor[sub]);
  }
  if constexpr (!Q8) {
    if (!live) return;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int p = me + NT * i;
      if (p < n) {
        float f[P];
        R::unpack(v[i], f);
#pragma unroll
        for (int j = 0; j < P; ++j) f[j] = rms_apply<A>(f[j], r, sc[i][j]);
        store16(out + at + p * P, R::pack(f));
      }
    }
    if (one) Act<A>::store(out, at + end, rms_apply<A>(h1, r, s1));
  } else {
    uint32_t m = 0;
    float f[PT][P];
    auto note = [&](float y) { m = max(m, __float_as_uint(y) & 0x7fffffffu); };
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      if (me + NT * i < n) {
        R::unpack(v[i], f[i]);
#pragma unroll
        for (int j = 0; j < P; ++j) note(f[i][j] = rms_apply<float>(f[i][j], r, sc[i][j]));
      }
    }
    float f1 = rms_apply<float>(h1, r, s1);
    if (one) note(f1);
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, k, 64));
    if constexpr (W > 1) {
      if ((threadIdx.x & 63) == 0) largest[wv] = m;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < W; ++k) m = max(m, largest[sub * W + k]);
    }
    if (!live) return;
    const bool bad = m > 0x7f7fffffu;
    const float s = fmaxf(__uint_as_float(m) / 127.0f, FLT_MIN);
    // rint(y / s) from the row's reciprocal: a product and one of Markstein's corrections. With
    // 1 / s correctly rounded, which the division here is, that gave the division's own quotient
    // for every divisor and the floats around every half integer times it (run through on the
    // CPU; elsewhere an ulp does not matter). The residual must be exact, which it is while s >=
    // 2^-100; smaller rows are scaled up, exactly. The product alone put 3 of 4 million values on
    // the other side of a half. 8192 x 4096 bf16, with and without residual: the product 45.6 and
    // 27.7 us, corrected 45.6 and 28.5, a division for every value 46.7 and 32.5.
    float by = s;
    if (s < 0x1p-100f) {
      by *= 0x1p64f;
      f1 *= 0x1p64f;
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        if (me + NT * i < n) {
#pragma unroll
          for (int j = 0; j < P; ++j) f[i][j] *= 0x1p64f;
        }
      }
    }
    const float inv = 1.0f / by;
    // a bad row: (int)NaN would be the compiler's choice, so it is set apart
    auto quant = [&](float y) {
      float z = y * inv;
      z = __builtin_fmaf(__builtin_fmaf(-z, by, y), inv, z);
      z = fminf(fmaxf(rintf(z), -127.0f), 127.0f);
      return bad ? 0u : (uint32_t)(int)z & 0xffu;
    };
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int p = me + NT * i;
      if (p < n) {
        uint32_t q[P / 4];
#pragma unroll
        for (int j = 0; j < P / 4; ++j) {
          q[j] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) q[j] |= quant(f[i][4 * j + k]) << (8 * k);
        }
        if constexpr (P == 8)
          *reinterpret_cast<u32x2_any*>(qout + at + p * P) = u32x2_any{q[0], q[1]};
        else
          *reinterpret_cast<u32_any*>(qout + at + p * P) = q[0];
      }
    }
    if (one) qout[at + end] = (int8_t)quant(f1);
    if (me == 0) qscale[t] = bad ? __builtin_nanf("") : s;
  }
}

}  // namespace kmoe

namespace kmoe_host {

using namespace kmoe;

namespace {

// Rows of one launch, `per` to a block: its threads are counted in 32 bits, and a launch of more
// leaves the rows behind them out without an error.
int64_t launch_rows(int per) { return (((int64_t)1 << 32) / (64 * kNormWaves) - 1) * per; }

template <typename A, typename S, int W>
void add_rms_norm_of(const kmoe_desc& d, const void* x, const void* res, const void* scale, float eps, void* hout,
                     void* out, int8_t* q, float* qscale, hipStream_t st) {
  const int D = (int)d.hidden, per = kNormWaves / W;
  const size_t lds = per * NormRow<A>::bytes(D);
  const int64_t most = launch_rows(per);
  for (int64_t t = 0; t < d.tokens; t += most) {
    const int T = (int)std::min(d.tokens - t, most);
    const dim3 grid((T + per - 1) / per), block(64 * kNormWaves);
    auto rows = [&](auto* p) { return p ? p + t * D : nullptr; };
    const A* const xt = rows(reinterpret_cast<const A*>(x));
    const A* const rt = rows(reinterpret_cast<const A*>(res));
    A* const ht = rows(reinterpret_cast<A*>(hout));
    A* const ot = rows(reinterpret_cast<A*>(out));
    if (q)
      hipLaunchKernelGGL((k_add_rms_norm<A, S, true, W>), grid, block, lds, st, T, D, eps, xt, rt,
                         reinterpret_cast<const S*>(scale), ht, ot, rows(q), qscale + t);
    else
      hipLaunchKernelGGL((k_add_rms_norm<A, S, false, W>), grid, block, lds, st, T, D, eps, xt, rt,
                         reinterpret_cast<const S*>(scale), ht, ot, q, qscale);
  }
}

template <typename A, typename S>
void add_rms_norm(const kmoe_desc& d, const void* x, const void* res, const void* scale, float eps, void* hout,
                  void* out, int8_t* q, float* qscale, hipStream_t st) {
  // four waves per row spread a row's latency (64 rows of 4096: 3.9 us, one wave each 6.2),
  // but of narrow rows they leave most threads idle (see the kernel's figures)
  if (d.tokens > kNormManyRows && d.hidden <= kNormNarrow * NormRow<A>::kPiece)
    add_rms_norm_of<A, S, 1>(d, x, res, scale, eps, hout, out, q, qscale, st);
  else
    add_rms_norm_of<A, S, kNormWaves>(d, x, res, scale, eps, hout, out, q, qscale, st);
}

}  // namespace

hipError_t launch_add_rms_norm(const kmoe_desc& d, const void* x, const void* res, const void* scale,
                               kmoe_dtype scale_dtype, float eps, void* hout, void* out, int8_t* q, float* qscale,
                               hipStream_t st) {
  const bool s_bf16 = scale_dtype == KMOE_DTYPE_BF16;
  if (d.act_dtype == KMOE_DTYPE_BF16) {
    if (s_bf16)
      add_rms_norm<uint16_t, uint16_t>(d, x, res, scale, eps, hout, out, q, qscale, st);
    else
      add_rms_norm<uint16_t, float>(d, x, res, scale, eps, hout, out, q, qscale, st);
  } else {
    if (s_bf16)
      add_rms_norm<float, uint16_t>(d, x, res, scale, eps, hout, out, q, qscale, st);
    else
      add_rms_norm<float, float>(d, x, res, scale, eps, hout, out, q, qscale, st);
  }
  return hipGetLastError();
}

namespace {

template <typename A, typename S>
void rms_norm_of(const kmoe_desc& d, const void* h, const void* scale, float eps, void* out, hipStream_t st) {
  const int D = (int)d.hidden;
  const int64_t most = launch_rows(kNormWaves);
  for (int64_t t = 0; t < d.tokens; t += most) {
    const int T = (int)std::min(d.tokens - t, most);
    hipLaunchKernelGGL((k_rms_norm<A, S>), dim3((T + kNormWaves - 1) / kNormWaves), dim3(64 * kNormWaves),
                       kNormWaves * NormRow<A>::bytes(D), st, T, D, eps, reinterpret_cast<const A*>(h) + t * D,
                       reinterpret_cast<const S*>(scale), reinterpret_cast<A*>(out) + t * D);
  }
}

}  // namespace

hipError_t launch_rms_norm(const kmoe_desc& d, const void* h, const void* scale, kmoe_dtype scale_dtype, float eps,
                           void* out, hipStream_t st) {
  const bool s_bf16 = scale_dtype == KMOE_DTYPE_BF16;
  if (d.act_dtype == KMOE_DTYPE_BF16) {
    if (s_bf16)
      rms_norm_of<uint16_t, uint16_t>(d, h, scale, eps, out, st);
    else
      rms_norm_of<uint16_t, float>(d, h, scale, eps, out, st);
  } else {
    if (s_bf16)
      rms_norm_of<float, uint16_t>(d, h, scale, eps, out, st);
    else
      rms_norm_of<float, float>(d, h, scale, eps, out, st);
  }
  return hipGetLastError();
}

}  // namespace kmoe_host
