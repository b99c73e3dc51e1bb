// The gated block's forward for a few rows (decoding): y = (act(x Wg^T + bg) *
// (x Wu^T + bu)) Wd^T + bd with at most 16 rows of x.  Memory bound by the
// weights, each read once, as they lie (no packing), straight from memory to
// the matrix instructions: a workgroup takes 16 rows of a weight, its waves
// take the k axis in turn, and an LDS pass joins them.  The weight's rows are
// the instruction's first operand, x's its second; which k a lane group holds
// is free as long as both agree, so a lane reads 16 bytes of its row.
// bfloat16 on v_mfma_f32_16x16x32_bf16, float32 on v_mfma_f32_16x16x4_f32.
//
// With bfloat16 tensors and at most eight rows h = act(g) u goes to the down product
// as two bfloat16 parts, to 2^-16 of it: one part alone would be off by up to 2^-8, the
// largest error of the call.  The second parts are the matrix instruction's other
// eight rows, where they cost nothing: one row of 2048 x 5632 takes 20.4 us either way,
// four of 4096 x 11008 53 to 54.  More rows have one part, as a batch has: there h's
// bytes bound the down product, and two parts take 16 rows from 26.3 us to 31.0, of
// 4096 x 11008 from 61 to 73.
#pragma once

#include "mm.hpp"

namespace d3a {
namespace thin {

using mm::bf16x4;
using mm::bf16x8;
using mm::f32x4;

constexpr int kRows = 16;

template <class T>
struct Piece;  // what a lane holds of one row: 16 bytes
template <>
struct Piece<__bf16> {
  static constexpr int N = 8, K = 32;  // values a lane, ks an instruction group
  bf16x8 v;
};
template <>
struct Piece<float> {
  static constexpr int N = 4, K = 16;
  f32x4 v;
};

__device__ __forceinline__ f32x4 product(const Piece<__bf16>& w, const Piece<__bf16>& x, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v, x.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product(const Piece<float>& w, const Piece<float>& x, f32x4 c) {
#pragma unroll
  for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w.v[t], x.v[t], c, 0, 0, 0);
  return c;
}

// ks k .. k + N - 1 of the row at p, zero from K on; VEC: whole aligned pieces
template <class T, bool VEC>
__device__ __forceinline__ Piece<T> load(const T* p, int k, int K, bool on) {
  Piece<T> o;
#pragma unroll
  for (int i = 0; i < Piece<T>::N; ++i) o.v[i] = (T)0.f;
  if constexpr (VEC) {
    if (on && k < K) o.v = *reinterpret_cast<const decltype(o.v)*>(p + k);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (on && k + i < K) o.v[i] = p[k + i];
  }
  return o;
}

// the waves' accumulators, added in order by the first wave
template <int NACC, int WAVES>
__device__ __forceinline__ void join(f32x4 (&acc)[NACC], f32x4* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < NACC; ++i) red[(w * NACC + i) * 64 + lane] = acc[i];
  __syncthreads();
  if (w != 0) return;
  for (int v = 1; v < WAVES; ++v)
#pragma unroll
    for (int i = 0; i < NACC; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] += red[(v * NACC + i) * 64 + lane][e];
}

template <class T>
struct GateArgs {
  const T *x, *Wg, *Wu, *bg, *bu;
  int64_t ldx, sx, ldg, sg, ldu, su;
  float *g, *u;           // kept, or null
  T *h, *lo;              // [members][R] rows of ld, zero past F; lo: the second part, or null
  int64_t ld;
  int32_t R, D, F, act;
};

// grid (16 hidden units, members), 8 waves
template <class T, bool VEC, class Act>
__global__ __launch_bounds__(512) void gate_kernel(const GateArgs<T> A, Act activation) {
  constexpr int WAVES = 8, N = Piece<T>::N, KP = Piece<T>::K;
  __shared__ f32x4 red[WAVES * 2 * 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = blockIdx.y;
  const int n0 = blockIdx.x * 16, row = lane & 15, k0 = (lane >> 4) * N;
  const int n = min(n0 + row, A.F - 1);  // (a row past the last is read twice and not written)
  const T* x = A.x + c * A.sx + row * A.ldx;
  const T* wg = A.Wg + c * A.sg + n * A.ldg;
  const T* wu = A.Wu + c * A.su + n * A.ldu;
  f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int k = w * KP; k < A.D; k += WAVES * KP) {
    const Piece<T> a = load<T, VEC>(wg, k + k0, A.D, true), b = load<T, VEC>(wu, k + k0, A.D, true);
    const Piece<T> v = load<T, VEC>(x, k + k0, A.D, row < A.R);
    acc[0] = product(a, v, acc[0]);
    acc[1] = product(b, v, acc[1]);
  }
  join<2, WAVES>(acc, red);
  // the lane has row `lane & 15` of x, four hidden units
  const int m = n0 + 4 * (lane >> 4);
  if (w != 0 || row >= A.R || m >= A.ld) return;
  float h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = min(m + i, A.F - 1);
    if (A.bg) acc[0][i] += (float)A.bg[c * A.F + at];
    if (A.bu) acc[1][i] += (float)A.bu[c * A.F + at];
    float a, da;
    activation(A.act, acc[0][i], a, da);
    h[i] = m + i < A.F ? a * acc[1][i] : 0.f;
  }
  const int64_t at = (c * A.R + row) * A.ld + m;
  if (A.g) {
    *reinterpret_cast<f32x4*>(A.g + at) = acc[0];
    *reinterpret_cast<f32x4*>(A.u + at) = acc[1];
  }
  if constexpr (sizeof(T) == 4) {
    mm::store4(A.h + at, h);
  } else {
    bf16x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = (__bf16)h[i];
      lo[i] = (__bf16)mm::left_of(h[i]);
    }
    *reinterpret_cast<bf16x4*>(A.h + at) = hi;
    if (A.lo) *reinterpret_cast<bf16x4*>(A.lo + at) = lo;
  }
}

template <class T>
struct DownArgs {
  const T *h, *lo, *W, *b;
  T* y;  // [members][R][O]
  int64_t ld, ldw, sw;
  int32_t R, F, O;
};

// grid (16 outputs, members), 16 waves; PARTS: h's, two of at most eight rows
template <class T, bool VEC, int PARTS>
__global__ __launch_bounds__(1024) void down_kernel(const DownArgs<T> A) {
  constexpr int WAVES = 16, N = Piece<T>::N, KP = Piece<T>::K;
  __shared__ f32x4 red[WAVES * 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = blockIdx.y;
  const int n0 = blockIdx.x * 16, row = lane & 15, k0 = (lane >> 4) * N;
  const T* wd = A.W + c * A.sw + (int64_t)min(n0 + row, A.O - 1) * A.ldw;
  const int hrow = PARTS == 2 ? row & 7 : row;
  const bool on = hrow < A.R;
  const int64_t at = (c * A.R + hrow) * A.ld;
  const T* h = (PARTS == 2 && row >= 8 ? A.lo : A.h) + at;
  f32x4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int k = w * KP; k < A.F; k += WAVES * KP) {
    const Piece<T> a = load<T, VEC>(wd, k + k0, A.F, true);
    const Piece<T> v = load<T, true>(h, k + k0, (int)A.ld, on);
    acc[0] = product(a, v, acc[0]);
  }
  join<1, WAVES>(acc, red);
  if (w != 0) return;
  if constexpr (PARTS == 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[0][i] += __shfl_xor(acc[0][i], 8);
  if (row >= A.R) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + 4 * (lane >> 4) + i;
    if (n < A.O) A.y[(c * A.R + row) * A.O + n] = (T)(acc[0][i] + (A.b ? (float)A.b[c * A.O + n] : 0.f));
  }
}

}  // namespace thin
}  // namespace d3a
