// Products of a minibatch's size, straight from the tensors: D(m, n) = sum over
// segments and k of A(m, k) B(n, k) as in mm.hpp, for work so small that the
// tiles' packing pass, their k loop's load latencies and the passes after it
// (partial sums, column sums) are most of the time.
//
// A workgroup makes one 32 x 32 tile; its eight waves take the 16-deep k steps
// in turn, so that all of a tile's loads are in flight together, read their
// operands from memory into registers (float32 split there into the three
// bfloat16 parts of mm.hpp's six products), and add up in LDS.  The sums of A's
// rows, which are a layer's bias gradient where A is its output gradient
// transposed, come with the first tile column.  Bound by latency: two members'
// 256 x 512 x 256 dual product takes 10 to 12 us in float32 (24 TFLOP/s); against
// the tiles, see small().
#pragma once

#include "mm.hpp"

namespace d3a {
namespace direct {

using mm::bf16x4;
using mm::bf16x8;
using mm::f32x16;
using mm::f32x4;

template <class T>
struct Operand {
  const T* p;
  int64_t ld, s_batch, s_outer, s_inner;  // (s_inner: A alone)
  int32_t vec;  // k-contiguous: rows are whole aligned pieces of eight
};

template <class T>
struct Problem {
  Operand<T> a, b, b2;  // b2: the second B of dual products, or of the second inner segment
  T* rowsum;        // [batch][M]: the sums of A's rows, or null
  mm::Factor sum_factor;
  int32_t M, N, K, batch, n_outer, n_inner;
  int32_t fold;     // 0, or up to 16: A has twice as many rows, D is the sum of both halves
  int32_t tiles_m, tiles_n, first;
};

constexpr int kMaxProblems = 3;
template <class T, class Epi>
struct Launch {
  Problem<T> p[kMaxProblems];
  Epi e[kMaxProblems];
  int32_t n, total;
};

constexpr int kWaves = 8, kLine = 36;  // a tile's row in LDS, in floats (32 and padding)

// ks k .. k + 7 of row `row` (clamped by the caller), zero from K on.  TR:
// row-contiguous operand (32 lanes read 32 neighbours of one k).
template <class T, bool TR>
__device__ __forceinline__ void load8(const Operand<T>& o, const T* p, int row, int k, int K, float v[8]) {
  if (TR || !o.vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kk = min(k + j, K - 1);
      const float x = (float)(TR ? p[kk * o.ld + row] : p[row * o.ld + kk]);
      v[j] = k + j < K ? x : 0.f;
    }
  } else {
    const T* q = p + row * o.ld + (k < K ? k : 0);
    if constexpr (sizeof(T) == 4) {
      mm::load8(q, v);
    } else {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)x[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k < K ? v[j] : 0.f;
  }
}

template <int NP>
__device__ __forceinline__ void split(const float v[8], bf16x8 (&o)[NP]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (NP == 1) {
      o[0][j] = (__bf16)v[j];
    } else {
      __bf16 a, b, c;
      mm::split3(v[j], a, b, c);
      o[0][j] = a;
      o[1][j] = b;
      o[2][j] = c;
    }
  }
}

template <int NP>
__device__ __forceinline__ f32x16 products(const bf16x8 (&b)[NP], const bf16x8 (&a)[NP], f32x16 acc) {
  if constexpr (NP == 3) {
    acc = mm::mma(b[0], a[2], acc);
    acc = mm::mma(b[1], a[1], acc);
    acc = mm::mma(b[2], a[0], acc);
    acc = mm::mma(b[0], a[1], acc);
    acc = mm::mma(b[1], a[0], acc);
  }
  return mm::mma(b[0], a[0], acc);
}

template <class T, bool AT, bool BT, bool DUAL, class Epi>
__global__ __launch_bounds__(64 * kWaves, 2) void direct_kernel(const Launch<T, Epi> L) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1, NACC = DUAL ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float red[NACC][kWaves][32 * kLine];
  __shared__ float sums[kWaves][32];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x, pi = 0;
  while (pi + 1 < L.n && id >= L.p[pi + 1].first) ++pi;
  const Problem<T>& P = L.p[pi];
  id -= P.first;
  const int per = P.tiles_m * P.tiles_n, batch = id / per;
  id -= batch * per;
  const int tn = id / P.tiles_m, m0 = (id - tn * P.tiles_m) * 32, n0 = tn * 32;
  const int ra = min(m0 + (lane & 31), P.M - 1), rb = min(n0 + (lane & 31), P.N - 1);
  const bool want_sum = P.rowsum && n0 == 0;

  f32x16 acc[NACC];
#pragma unroll
  for (int i = 0; i < NACC; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float sum = 0.f;
  const int steps = (P.K + 15) / 16;
  for (int seg = 0; seg < P.n_outer * P.n_inner; ++seg) {
    const int o = seg / P.n_inner, i = seg - o * P.n_inner;
    const T* pa = P.a.p + batch * P.a.s_batch + o * P.a.s_outer + i * P.a.s_inner;
    const Operand<T>& B = i ? P.b2 : P.b;
    const T* pb = B.p + batch * B.s_batch + o * B.s_outer;
    const T* pb2 = DUAL ? P.b2.p + batch * P.b2.s_batch : nullptr;
    // (steps in pairs: one past K is zeros)
    for (int s = w; s < steps; s += 2 * kWaves) {
      float a[2][8], b[2][NACC][8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = 16 * (s + j * kWaves) + 8 * (lane >> 5);
        load8<T, AT>(P.a, pa, ra, k, P.K, a[j]);
        load8<T, BT>(B, pb, rb, k, P.K, b[j][0]);
        if constexpr (DUAL) load8<T, BT>(P.b2, pb2, rb, k, P.K, b[j][1]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        bf16x8 fa[NP], fb[NP];
        split<NP>(a[j], fa);
#pragma unroll
        for (int q = 0; q < NACC; ++q) {
          split<NP>(b[j][q], fb);
          acc[q] = products<NP>(fb, fa, acc[q]);
        }
        if (want_sum)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += a[j][e];
      }
    }
  }

  // a lane holds row `lane & 31`, runs of four columns
#pragma unroll
  for (int i = 0; i < NACC; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(&red[i][w][(lane & 31) * kLine + 8 * q + 4 * (lane >> 5)]) =
          f32x4{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
  if (want_sum) {
    sum += __shfl_xor(sum, 32);
    if (lane < 32) sums[w][lane] = sum;
  }
  __syncthreads();
  if (want_sum && threadIdx.x < 32 && m0 + (int)threadIdx.x < P.M) {
    float s = 0.f;
    for (int v = 0; v < kWaves; ++v) s += sums[v][threadIdx.x];
    P.rowsum[(int64_t)batch * P.M + m0 + threadIdx.x] = (T)(s * P.sum_factor.get());
  }
  // two neighbouring columns a thread, sixteen threads a row
  const int r = threadIdx.x >> 4, c = 2 * (threadIdx.x & 15);
  float v[NACC][2];
#pragma unroll
  for (int i = 0; i < NACC; ++i) {
    v[i][0] = v[i][1] = 0.f;
    for (int u = 0; u < kWaves; ++u) {
      const float2 x = *reinterpret_cast<const float2*>(&red[i][u][r * kLine + c]);
      v[i][0] += x.x;
      v[i][1] += x.y;
    }
    if (P.fold)
      for (int u = 0; u < kWaves; ++u) {
        const float2 x = *reinterpret_cast<const float2*>(&red[i][u][((r + P.fold) & 31) * kLine + c]);
        v[i][0] += x.x;
        v[i][1] += x.y;
      }
  }
  L.e[pi].run(batch, m0 + r, n0 + c, P.fold ? P.fold : P.M, P.N, v[0], v[NACC - 1]);
}

// D (+ bias) in T
template <class T>
struct StoreEpi {
  T* out;           // null: nothing is written
  int64_t ld, s_batch;
  const T* bias;
  int64_t s_bias;
  mm::Factor factor;
  __device__ __forceinline__ void run(int batch, int m, int n, int M, int N, const float v[2], const float*) const {
    if (m >= M || !out) return;
    T* o = out + batch * s_batch + m * ld;
    const float by = factor.get();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (n + i < N) o[n + i] = (T)(v[i] * by + (bias ? (float)bias[batch * s_bias + n + i] : 0.f));
  }
};

// ---- host -------------------------------------------------------------------
template <class T>
Operand<T> operand(const void* p, int64_t ld, int64_t s_batch, int64_t K) {
  Operand<T> o{};
  o.p = static_cast<const T*>(p);
  o.ld = ld;
  o.s_batch = s_batch;
  o.vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && s_batch % 8 == 0 && K % 8 == 0;
  return o;
}

template <class T>
Problem<T> problem(const Operand<T>& a, const Operand<T>& b, int64_t M, int64_t N, int64_t K, int64_t batch) {
  Problem<T> p{};
  p.a = a;
  p.b = b;
  p.M = (int32_t)M;
  p.N = (int32_t)N;
  p.K = (int32_t)K;
  p.batch = (int32_t)batch;
  p.n_outer = p.n_inner = 1;
  return p;
}

template <bool AT, bool BT, bool DUAL, class T, class Epi>
int launch(Launch<T, Epi>& L, hipStream_t stream, const char* what) {
  int64_t total = 0;
  for (int i = 0; i < L.n; ++i) {
    Problem<T>& p = L.p[i];
    p.tiles_m = (p.M + 31) / 32;
    p.tiles_n = (p.N + 31) / 32;
    p.first = (int32_t)total;
    total += (int64_t)p.tiles_m * p.tiles_n * p.batch;
  }
  if (total == 0) return 0;
  if (total >= (1 << 30)) {
    set_error("product has too many tiles");
    return -1;
  }
  L.total = (int32_t)total;
  direct_kernel<T, AT, BT, DUAL, Epi><<<L.total, 64 * kWaves, 0, stream>>>(L);
  D3A_LAUNCH_CHECK(what);
  return 0;
}

// Whether an operator whose products each have `work` multiply-adds and k axes
// up to `axis` runs here.  Trained in float32 / bfloat16, us here against the
// tiles: 512 x 256 x 1024 82 / 55 against 100 / 63, 1024 x 512 x 256 69 / 44
// against 113 / 49 (both 2^27); with a k of 2048, 128 x 512 x 2048, 122 / 90
// against 111 / 64, since a wave then has sixteen k steps one after another.
inline bool small(double work, int64_t axis) { return work <= (double)(1 << 27) && axis <= 1024; }

}  // namespace direct
}  // namespace d3a
