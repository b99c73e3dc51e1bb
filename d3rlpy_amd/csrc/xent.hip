// Softmax cross entropy of a linear head over a large vocabulary, forward and
// backward, without the logits in memory:
//
//   z = x W^T + b,  lse_r = log sum_v exp z_rv,  loss_r = lse_r - z_r,target
//   dz_rv = (exp(z_rv - lse_r) - [v = target_r]) dloss_r  (dloss_r: a row's own;
//     one for all rows multiplies the products' results instead, see loss_factor)
// lse_r = m + log s (m the row's largest logit, s its sum of exp(z - m)) rounds to
// steps of 2^-24 |m|, which is all of log s where a row's logits share a large value.
// So the loss is (m - z_target) + log s, and the backward goes by lse and by what its
// rounding left, low_r = (m - lse_r) + log s.
//   dx = dz W,  dW = dz^T x,  db_v = sum_r dz_rv
//
// Forward: the tiles of mm.hpp over (rows, vocabulary); a tile's epilogue
// reduces each of its rows to (max, sum of exp(z - max)) and picks the
// target's logit, and a second pass joins the tiles of a row.  Backward: the
// logits again, a piece of the vocabulary at a time, whose epilogue writes dz
// of the piece in the operand layout of the two products that follow.  Neither grows
// with rows x vocabulary: the forward's parts and dz stay within kPieceBytes each, by
// cutting first the vocabulary (backward) and then the rows.  What does grow: the
// operands' packed copies, with x and W; a float32 sum of dx, with x, where there are
// several pieces.  All products are bound by
// the matrix cores, and their epilogues by the exponentials: 8192 x 1024 -> 32768 in
// bfloat16 takes 510 to 650 us for the logits' sums, 635 to 730 for dz, 475 to 530 for dx and
// 460 to 505 for dW, of 550 GFLOP each; 1500 x 777 -> 10007 in float32 146, 152, 141, 176.
//
// A row whose target is ignore_index has loss 0 and no gradient, whatever its
// logits are; a row whose target is outside the vocabulary has loss NaN and a
// NaN gradient.
#include "direct.hpp"
#include "mm_host.hpp"
#include "../../include/d3rlpy_amd.h"

namespace d3a {
namespace {

using namespace mm;

constexpr int64_t kPieceBytes = 512LL << 20;

// The size of equal parts of `all`, at most `most` each: a multiple of the widest tile's
// 256 where that leaves any.
int64_t equal_parts(int64_t all, int64_t most) {
  if (all <= most) return all;
  const int64_t step = most >= 256 ? 256 : 1;
  most = std::max<int64_t>(most / step, 1) * step;
  const int64_t n = (all + most - 1) / most;
  return ((all + n - 1) / n + step - 1) / step * step;
}

// exp(z - ref), of the forward's sums.  (With bfloat16 tensors the hardware's
// exponential: within 2 ulp and a product's rounding of its argument it is no more than
// the float32 sum's own, and in the backward far below dz's rounding.)
template <int NP>
__device__ __forceinline__ float exp_to(float z, float ref) {
  return NP == 1 ? __expf(z - ref) : expf(z - ref);
}

// exp(z - (lse + low)); `low` as low_factor gives it: with bfloat16 tensors it goes
// into the product by log2 e that the hardware's exponential takes anyway.
constexpr float kLog2e = 1.44269504088896341f;
template <int NP>
__device__ __forceinline__ float low_factor(float low) {
  return NP == 1 ? -low * kLog2e : low;
}
template <int NP>
__device__ __forceinline__ float probability(float z, float lse, float low) {
  return NP == 1 ? __builtin_amdgcn_exp2f(fmaf(z - lse, kLog2e, low)) : expf((z - lse) - low);
}

// What a row's maximum m and sum s of exp(z - m) give; z: the target's logit.
struct RowLoss {
  float lse, low, loss;
};
__device__ __forceinline__ RowLoss row_loss(float m, float s, float z, int64_t target, int64_t vocab,
                                            int64_t ignore) {
  const float log_s = logf(s), lse = m + log_s;
  const float loss = target == ignore ? 0.f : target >= 0 && target < vocab ? (m - z) + log_s : NAN;
  return {lse, (m - lse) + log_s, loss};
}

// (max, sum of exp(z - max)) of a + b; an empty side has max -inf, sum 0
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float a = m == top ? s : s * expf(m - top);
  const float b = m2 == top ? s2 : s2 * expf(m2 - top);
  m = top;
  s = a + b;
}

// One (max, sum) a row and wave column; z of the target.
template <class T, int NP>
struct LsePartEpi {
  static constexpr bool kStaged = false;
  static constexpr int kRowBytes = 0;
  const T* bias;
  const int64_t* target;
  float2* part;     // [columns of waves][M]
  float* ztarget;   // [M]
  int32_t v0;       // vocabulary index of column 0
  int32_t wave_cols;  // columns a wave covers

  template <class C>
  __device__ __forceinline__ void run(f32x16 (&acc)[C::MT][C::NT], const Tile& t) const {
    // (bounds and the target's column cost a pass of their own only in tiles that
    // have a border or a target in them: the exponentials' 65536 of a 256 x 256
    // tile are already a tenth of its products' time)
    const bool border = t.n0 + C::TN > t.N;
    int want[C::MT];  // the target's column of the wave's, or -1
#pragma unroll
    for (int i = 0; i < C::MT; ++i) {
      const int m = t.m0 + 32 * i + (t.lane & 31);
      const int64_t y = m < t.M ? target[m] - v0 - t.n0 : -1;
      want[i] = y >= 0 && y < min(C::TN, t.N - t.n0) ? (int)y : -1;
    }
    wait_loads();
#pragma unroll
    for (int i = 0; i < C::MT; ++i) {
      const int m = t.m0 + 32 * i + (t.lane & 31);
      const int n0 = t.n0 + 4 * (t.lane >> 5);
      if (bias || border) {
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int n = n0 + 32 * j + 8 * (r / 4) + r % 4;
            const float v = acc[i][j][r] + (bias ? (float)bias[min(n, t.N - 1)] : 0.f);
            acc[i][j][r] = n < t.N ? v : -INFINITY;
          }
      }
      if (__ballot(want[i] >= 0)) {
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (4 * (t.lane >> 5) + 32 * j + 8 * (r / 4) + r % 4 == want[i]) ztarget[m] = acc[i][j][r];
      }
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
      // a row of -inf alone: any finite reference gives its sum of 0
      const float ref = top == -INFINITY ? 0.f : top;
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += exp_to<NP>(acc[i][j][r], ref);
      const float m2 = __shfl_xor(top, 32), s2 = __shfl_xor(s, 32);
      join(top, s, m2, s2);
      // (a wave past the last column has no part)
      if (t.lane < 32 && m < t.M && t.n0 < t.N)
        part[(int64_t)(t.n0 / wave_cols) * t.M + m] = make_float2(top, s);
    }
  }
};

// ---- a minibatch and a small vocabulary: direct.hpp -------------------------------
// One (max, sum) a row and 32 columns: a row's columns lie with 16 threads.
template <class T>
struct DirectLseEpi {
  const T* bias;
  const int64_t* target;
  float2* part;
  float* ztarget;
  __device__ __forceinline__ void run(int, int m, int n, int M, int N, const float v[2], const float*) const {
    const int64_t y = m < M ? target[m] : -1;
    float z[2], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      z[i] = n + i < N ? v[i] + (bias ? (float)bias[n + i] : 0.f) : -INFINITY;
      if (n + i < N && n + i == y) ztarget[m] = z[i];
      top = fmaxf(top, z[i]);
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float s = exp_to<3>(z[0], ref) + exp_to<3>(z[1], ref);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float m2 = __shfl_xor(top, o), s2 = __shfl_xor(s, o);
      join(top, s, m2, s2);
    }
    if ((threadIdx.x & 15) == 0 && m < M) part[(int64_t)(n / 32) * M + m] = make_float2(top, s);
  }
};

template <class T>
struct DirectDzEpi {
  const T* bias;
  const int64_t* target;
  const float *lse, *low, *gloss;  // low: or null (0)
  int64_t ignore, vocab;
  T *dz, *second;  // second: dz's second part, or null
  int64_t ld;
  __device__ __forceinline__ void run(int, int m, int n, int M, int N, const float v[2], const float*) const {
    if (m >= M) return;
    const int64_t y = target[m];
    const float l = lse[m], g = y >= 0 && y < vocab ? (gloss ? gloss[m] : 1.f) : NAN;
    const float lo = low_factor<3>(low ? low[m] : 0.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (n + i >= N) continue;
      const float z = v[i] + (bias ? (float)bias[n + i] : 0.f);
      const float d = (probability<3>(z, l, lo) - (n + i == y ? 1.f : 0.f)) * g;
      const float kept = y == ignore ? 0.f : d;
      dz[m * ld + n + i] = (T)kept;
      if (second) second[m * ld + n + i] = (T)left_of(kept);
    }
  }
};

// What every row's gradient has in common multiplies the products' results and
// not dz: near a target dz is -1 times it, so that its rounding to bfloat16, up
// to 2^-8, would be every gradient's.
Factor loss_factor(const d3a_linear_xent_desc& d) {
  return d.reduction == 0 ? Factor{} : Factor{d.gloss, d.reduction == 1 ? d.scale : nullptr};
}

// A few bfloat16 rows keep dz in two parts, to 2^-16: with one row the rounding of its
// target's dz, up to 2^-8, is an error that every gradient shares (1.8 times the plain
// gradient's own rounding in W's; of many rows these average to 1.2 times).  The second
// parts cost no product: dx takes them as rows that its tile has free and adds both
// halves up, dW as a second k segment, of the tile's pair.  Their bytes do: forward and
// backward of 1 x 112 -> 39680 take 52.1 us, of 47.6 with one part, 16 x 256 -> 1024
// 27.5 of 26.6, 8 x 1024 -> 65536 151 of 145.
constexpr int64_t kTwoPartsDirect = 16, kTwoPartsTiles = 32;

bool is_direct(const d3a_linear_xent_desc& d) {
  // (the vocabulary is a k axis of one product of four: 256 x 256 x 2048 in
  // float32 takes 61 us here, 70 with tiles)
  return direct::small((double)d.rows * d.n_in * d.vocab, std::max({d.rows, d.n_in, d.vocab / 2}));
}

// Joins the rows' parts: 8 rows x 32 threads a workgroup, first their largest
// maximum, then the sums that refer to it (the parts again, from the cache).
__global__ __launch_bounds__(256) void lse_join_kernel(const float2* part, int32_t parts, int32_t rows,
                                                       const float* ztarget, const int64_t* target,
                                                       int64_t vocab, int64_t ignore, float* lse,
                                                       float* low, float* loss, int32_t r0) {
  __shared__ float red[256];
  const int q = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int r = r0 + blockIdx.x * 8 + q;
  float m = -INFINITY, s = 0.f;
  if (r < rows)
#pragma unroll 4
    for (int p = g; p < parts; p += 32) m = fmaxf(m, part[(int64_t)p * rows + r].x);
  red[threadIdx.x] = m;
  __syncthreads();
  for (int k = 0; k < 32; ++k) m = fmaxf(m, red[8 * k + q]);
  __syncthreads();
  if (r < rows)
#pragma unroll 4
    for (int p = g; p < parts; p += 32) {
      const float2 v = part[(int64_t)p * rows + r];
      s += v.x == m ? v.y : v.y * expf(v.x - m);
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (g != 0 || r >= rows) return;
  for (int k = 1; k < 32; ++k) s += red[8 * k + q];
  const RowLoss o = row_loss(m, s, ztarget[r], target[r], vocab, ignore);
  lse[r] = o.lse;
  if (low) low[r] = o.low;
  loss[r] = o.loss;
}

// The same with a workgroup a row, for few rows of many parts: us, 1024 parts
// 8 / 64 / 256 / 1024 rows 3.9 / 4.6 / 6.1 / 21.6,
// the other 6.6 / 8.0 / 7.6 / 8.1; with 256 parts both take 3 to 4.
__global__ __launch_bounds__(256) void lse_join_wide_kernel(const float2* part, int32_t parts, int32_t rows,
                                                            const float* ztarget, const int64_t* target,
                                                            int64_t vocab, int64_t ignore, float* lse,
                                                            float* low, float* loss) {
  __shared__ float red[8];
  const int r = blockIdx.x, w = threadIdx.x >> 6;
  float m = -INFINITY, s = 0.f;
#pragma unroll 4
  for (int p = threadIdx.x; p < parts; p += 256) m = fmaxf(m, part[(int64_t)p * rows + r].x);
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((threadIdx.x & 63) == 0) red[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
#pragma unroll 4
  for (int p = threadIdx.x; p < parts; p += 256) {
    const float2 v = part[(int64_t)p * rows + r];
    s += v.x == m ? v.y : v.y * expf(v.x - m);
  }
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[4 + w] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  const RowLoss o = row_loss(m, (red[4] + red[5]) + (red[6] + red[7]), ztarget[r], target[r], vocab, ignore);
  lse[r] = o.lse;
  if (low) low[r] = o.low;
  loss[r] = o.loss;
}

// The sum of the rows' losses (mean: over the counted rows, at least one), and
// the factor of each row's gradient.  One workgroup of 1024: fixed order,
// float64.
__device__ __forceinline__ void reduce_loss(double s, int n, int32_t mean, float* out, float* scale) {
  __shared__ double ps[16];
  __shared__ int pn[16];
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o);
    n += __shfl_xor(n, o);
  }
  if ((threadIdx.x & 63) == 0) {
    ps[threadIdx.x >> 6] = s;
    pn[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.0;
  n = 0;
  for (int k = 0; k < 16; ++k) {
    s += ps[k];
    n += pn[k];
  }
  const double by = mean ? (double)max(n, 1) : 1.0;
  out[0] = (float)(s / by);
  scale[0] = (float)(1.0 / by);
}

__global__ __launch_bounds__(1024) void loss_reduce_kernel(const float* loss, const int64_t* target,
                                                           int64_t ignore, int32_t rows, int32_t mean,
                                                           float* out, float* scale) {
  double s = 0.0;
  int n = 0;
  for (int r = threadIdx.x; r < rows; r += 1024) {
    s += (double)loss[r];
    n += target[r] != ignore;
  }
  reduce_loss(s, n, mean, out, scale);
}

// Both passes in one workgroup, a thread a row, for few rows and parts (1024 x
// 16: two launches' 9 us are one of 5).
constexpr int64_t kJoinSmall = 16384;

__global__ __launch_bounds__(1024) void lse_join_small_kernel(const float2* part, int32_t parts, int32_t rows,
                                                              const float* ztarget, const int64_t* target,
                                                              int64_t vocab, int64_t ignore, int32_t mean,
                                                              float* lse, float* low, float* loss,
                                                              float* out, float* scale) {
  double sum = 0.0;
  int n = 0;
  for (int r = threadIdx.x; r < rows; r += 1024) {
    float m = -INFINITY, s = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) m = fmaxf(m, part[(int64_t)p * rows + r].x);
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float2 v = part[(int64_t)p * rows + r];
      s += v.x == m ? v.y : v.y * expf(v.x - m);
    }
    const int64_t t = target[r];
    const RowLoss o = row_loss(m, s, ztarget[r], t, vocab, ignore);
    lse[r] = o.lse;
    if (low) low[r] = o.low;
    loss[r] = o.loss;
    sum += (double)o.loss;
    n += t != ignore;
  }
  reduce_loss(sum, n, mean, out, scale);
}

// dz of a piece of the vocabulary, as operand planes
template <class T, int NP>
struct DzEpi {
  static constexpr bool kStaged = true;
  static constexpr int kRowBytes = 16;
  const T* bias;
  const int64_t* target;
  const float *lse, *low;  // low: or null (0)
  const float* gloss;      // the rows' own, or null (one for all: a factor of the products)
  int64_t ignore, vocab;
  __bf16 *dz, *second;               // planes, rows of ld; one plane's second part, or null
  int64_t ld, s_part;
  int32_t v0;
  float* db;                         // the waves' sums of their rows, [M / C::TM][quads of N][4], or null

  template <class C>
  __device__ __forceinline__ void run(f32x16 (&acc)[C::MT][C::NT], const Tile& t) const {
    // the wave's rows, two a lane: their lse, gradient factor, target column (-1: in
    // no column here; -2: the row is ignored) and lse's low part
    float4* rows = reinterpret_cast<float4*>(t.rows);
#pragma unroll
    for (int k = 0; k < (C::TM + 63) / 64; ++k) {
      const int i = 64 * k + t.lane, m = min(t.m0 + i, t.M - 1);
      const int64_t y = target[m];
      const float l = lse[m], g = y >= 0 && y < vocab ? (gloss ? gloss[m] : 1.f) : NAN;
      const int64_t want = y - v0;
      const int col = y == ignore ? -2 : want >= 0 && want < t.N ? (int)want : -1;
      if (i < C::TM) rows[i] = make_float4(l, g, __int_as_float(col), low_factor<NP>(low ? low[m] : 0.f));
    }
    float b[8];
    load_bias(bias, first_column<false>(t), t.N, b);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto none = [](int, int) { return Nothing{}; };
    each8<C, false>(acc, t, none, [&](int m, int n, float* v, float*, Nothing) {
      if (n >= ld) return;
      const float4 row = rows[m - t.m0];
      const int col = __float_as_int(row.z), want = col - n;
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = probability<NP>(v[r] + b[r], row.x, row.w);
      if (want >= 0 && want < 8) {
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] -= r == want ? 1.f : 0.f;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] *= row.y;
      if (col == -2 || n + 8 > t.N) {
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = col != -2 && n + r < t.N ? v[r] : 0.f;
      }
      if (db) {
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] += v[r];
      }
      store_planes<NP>(dz + (int64_t)m * ld + n, s_part, v);
      if constexpr (NP == 1)
        if (second) {
          float left[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) left[r] = left_of(v[r]);
          store8(second + (int64_t)m * ld + n, left);
        }
    });
    if (!db) return;
    // eight lanes have the same columns
#pragma unroll
    for (int o = 8; o < 64; o <<= 1)
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] += __shfl_xor(s[r], o);
    const int n = first_column<false>(t);
    if (t.lane >= 8 || t.m0 >= t.M) return;
    float* at = db + (int64_t)(t.m0 / C::TM) * ((t.N + 3) / 4 * 4) + n;
    if (n < t.N) store4(at, s);
    if (n + 4 < t.N) store4(at + 4, s + 4);
  }
};

int check(const d3a_linear_xent_desc* d, bool bwd) {
  D3A_CHECK_ARG(d, "linear_cross_entropy: null descriptor");
  D3A_CHECK_ARG(d->dtype == D3A_F32 || d->dtype == D3A_BF16,
                "linear_cross_entropy: dtype must be float32 or bfloat16");
  D3A_CHECK_ARG(d->reduction >= 0 && d->reduction <= 2, "linear_cross_entropy: unknown reduction");
  D3A_CHECK_ARG(d->rows >= 0 && d->n_in >= 1 && d->vocab >= 1, "linear_cross_entropy: sizes must be positive");
  D3A_CHECK_ARG(d->rows <= kMaxRows && d->n_in <= kMaxWidth && d->vocab <= kMaxRows,
                "linear_cross_entropy: size too large");
  D3A_CHECK_ARG(d->ldx >= d->n_in && d->ldW >= d->n_in, "linear_cross_entropy: row stride smaller than the row");
  D3A_CHECK_ARG(d->W, "linear_cross_entropy: null weight");
  if (d->rows > 0)
    D3A_CHECK_ARG(d->x && d->target && d->lse && d->loss, "linear_cross_entropy: null operand");
  D3A_CHECK_ARG(d->reduction == 0 || (d->out && d->scale), "linear_cross_entropy: a reduction needs out and scale");
  if (bwd) D3A_CHECK_ARG(d->gloss || d->rows == 0, "linear_cross_entropy: null gradient");
  return 0;
}

template <int NP>
int wave_columns(TileSize s) {
  typedef Tiles<NP> X;
  return s == kLarge ? X::Large::TN : s == kMid ? X::Mid::TN : X::Small::TN;
}
template <int NP>
int wave_rows(TileSize s) {
  typedef Tiles<NP> X;
  return s == kLarge ? X::Large::TM : s == kMid ? X::Mid::TM : X::Small::TM;
}

// lse and loss of n rows from r0 on, from their parts
// (of kJoinRows at a time: a launch holds less than 2^32 threads)
constexpr int64_t kJoinRows = 1 << 26;
int join(const d3a_linear_xent_desc& d, int64_t r0, int64_t n, const float2* part, int64_t parts,
         const float* ztarget, hipStream_t stream) {
  const int64_t* target = d.target + r0;
  float *lse = d.lse + r0, *low = d.low ? d.low + r0 : nullptr, *loss = d.loss + r0;
  if (n <= 256 && parts >= 512)
    lse_join_wide_kernel<<<(unsigned)n, 256, 0, stream>>>(part, (int32_t)parts, (int32_t)n, ztarget, target, d.vocab,
                                                          d.ignore_index, lse, low, loss);
  else
    for (int64_t at = 0; at < n; at += kJoinRows)
      lse_join_kernel<<<(unsigned)((std::min(n - at, kJoinRows) + 7) / 8), 256, 0, stream>>>(
          part, (int32_t)parts, (int32_t)n, ztarget, target, d.vocab, d.ignore_index, lse, low, loss, (int32_t)at);
  D3A_LAUNCH_CHECK("linear_cross_entropy");
  return 0;
}

int reduce(const d3a_linear_xent_desc& d, hipStream_t stream) {
  if (d.reduction == 0) return 0;
  loss_reduce_kernel<<<1, 1024, 0, stream>>>(d.loss, d.target, d.ignore_index, (int32_t)d.rows, d.reduction == 1,
                                             d.out, d.scale);
  D3A_LAUNCH_CHECK("linear_cross_entropy");
  return 0;
}

// both, of all rows
int finish(const d3a_linear_xent_desc& d, const float2* part, int64_t parts, const float* ztarget,
           hipStream_t stream) {
  const int64_t R = d.rows;
  if (d.reduction != 0 && R >= 64 && R * parts <= kJoinSmall) {
    lse_join_small_kernel<<<1, 1024, 0, stream>>>(part, (int32_t)parts, (int32_t)R, ztarget, d.target, d.vocab,
                                                  d.ignore_index, d.reduction == 1, d.lse, d.low, d.loss, d.out, d.scale);
    D3A_LAUNCH_CHECK("linear_cross_entropy");
    return 0;
  }
  if (R > 0 && join(d, 0, R, part, parts, ztarget, stream) != 0) return -1;
  return reduce(d, stream);
}

template <class T>
int forward_direct(const d3a_linear_xent_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  const int64_t R = d.rows, D = d.n_in, V = d.vocab, parts = (V + 31) / 32;
  direct::Launch<T, DirectLseEpi<T>> L{};
  L.n = 1;
  L.p[0] = direct::problem(direct::operand<T>(d.x, d.ldx, 0, D), direct::operand<T>(d.W, d.ldW, 0, D), R, V, D, 1);
  L.e[0] = DirectLseEpi<T>{static_cast<const T*>(d.b), d.target, ws.take<float2>(parts * R), ws.take<float>(R)};
  *bytes = ws.used;
  if (dry) return 0;
  if (R > 0 && direct::launch<false, false, false>(L, stream, "linear_cross_entropy") != 0) return -1;
  return finish(d, L.e[0].part, parts, L.e[0].ztarget, stream);
}

template <class T>
int backward_direct(const d3a_linear_xent_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  const int64_t R = d.rows, D = d.n_in, V = d.vocab, ld = round8(V);
  const bool two = sizeof(T) == 2 && R <= kTwoPartsDirect;
  T* dz = ws.take<T>((two ? 2 : 1) * R * ld);
  *bytes = ws.used;
  if (dry) return 0;
  if (R > 0) {
    direct::Launch<T, DirectDzEpi<T>> L{};
    L.n = 1;
    L.p[0] = direct::problem(direct::operand<T>(d.x, d.ldx, 0, D), direct::operand<T>(d.W, d.ldW, 0, D), R, V, D, 1);
    L.e[0] = DirectDzEpi<T>{static_cast<const T*>(d.b), d.target, d.lse, d.low,
                            d.reduction == 0 ? d.gloss : nullptr, d.ignore_index, V, dz,
                            two ? dz + R * ld : nullptr, ld};
    if (direct::launch<false, false, false>(L, stream, "linear_cross_entropy_bwd") != 0) return -1;
    if (d.dx) {
      direct::Launch<T, direct::StoreEpi<T>> X{};
      X.n = 1;
      X.p[0] = direct::problem(direct::operand<T>(dz, ld, 0, V), direct::operand<T>(d.W, d.ldW, 0, V),
                               two ? 2 * R : R, D, V, 1);
      X.p[0].fold = two ? (int32_t)R : 0;
      X.e[0] = direct::StoreEpi<T>{static_cast<T*>(d.dx), D, 0, nullptr, 0, loss_factor(d)};
      if (direct::launch<false, true, false>(X, stream, "linear_cross_entropy_bwd") != 0) return -1;
    }
  }
  if (!d.dW && !d.db) return 0;
  direct::Launch<T, direct::StoreEpi<T>> W{};
  W.n = 1;
  W.p[0] = direct::problem(direct::operand<T>(dz, ld, 0, R), direct::operand<T>(d.x, d.ldx, 0, R), V, d.dW ? D : 1, R, 1);
  if (two) {
    W.p[0].n_inner = 2;
    W.p[0].a.s_inner = R * ld;
    W.p[0].b2 = W.p[0].b;
  }
  W.p[0].rowsum = static_cast<T*>(d.db);
  W.p[0].sum_factor = loss_factor(d);
  W.e[0] = direct::StoreEpi<T>{static_cast<T*>(d.dW), D, 0, nullptr, 0, loss_factor(d)};
  return direct::launch<true, true, false>(W, stream, "linear_cross_entropy_bwd");
}

template <class T, int NP>
int forward(const d3a_linear_xent_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  if (is_direct(d)) return forward_direct<T>(d, ws, dry, stream, bytes);
  const int64_t R = d.rows, D = d.n_in, V = d.vocab;
  Packer<T, NP> pack(ws);
  Launch<LsePartEpi<T, NP>> L{};
  L.n = 1;
  Problem& p = L.p[0];
  const Operand x = pack.operand(d.x, d.ldx, 0, 1, R, D);
  p.b = pack.operand(d.W, d.ldW, 0, 1, V, D);
  p.M = (int32_t)R;
  p.N = (int32_t)V;
  p.K = (int32_t)D;
  p.batch = p.n_outer = p.n_inner = p.splits = 1;
  const TileSize size = choose<NP>(L, false).size;
  const int cols = wave_columns<NP>(size);
  const int64_t parts = (V + cols - 1) / cols;
  // (a wave's 64 columns are 8 bytes: rows are cut from 2^32 logits on)
  const int64_t block = equal_parts(R, kPieceBytes / (parts * (int64_t)sizeof(float2)));
  LsePartEpi<T, NP>& e = L.e[0];
  e.bias = static_cast<const T*>(d.b);
  e.part = ws.take<float2>(parts * block);
  e.ztarget = ws.take<float>(block);
  e.wave_cols = cols;
  *bytes = ws.used;
  if (dry) return 0;
  if (R > 0 && pack.launch(stream) != 0) return -1;
  for (int64_t r0 = 0; r0 < R; r0 += block) {
    // (the blocks reuse one workspace: a stream runs them in order)
    p.a = x;
    p.a.p += r0 * x.ld;
    p.M = (int32_t)std::min(block, R - r0);
    e.target = d.target + r0;
    if (run<NP, false, false, false>(L, size, stream, "linear_cross_entropy") != 0) return -1;
    if (block < R && join(d, r0, p.M, e.part, parts, e.ztarget, stream) != 0) return -1;
  }
  return block < R ? reduce(d, stream) : finish(d, e.part, parts, e.ztarget, stream);
}

template <class T, int NP>
int backward(const d3a_linear_xent_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  const int64_t R = d.rows, D = d.n_in, V = d.vocab;
  if (!d.dx && !d.dW && !d.db) {
    *bytes = 0;
    return 0;
  }
  if (is_direct(d)) return backward_direct<T>(d, ws, dry, stream, bytes);
  const Factor by = loss_factor(d);
  Packer<T, NP> pack(ws);
  const Operand x = pack.operand(d.x, d.ldx, 0, 1, R, D);
  const Operand w = pack.operand(d.W, d.ldW, 0, 1, V, D);
  // pieces of the vocabulary; where all rows of 256 columns are too much, blocks of rows
  const int64_t most = kPieceBytes / (2 * NP * std::max<int64_t>(R, 1)) / 256 * 256;
  const int64_t piece = equal_parts(V, std::min(std::max<int64_t>(most, 256), kMaxWidth));
  const int64_t ld = round8(piece), block = equal_parts(R, kPieceBytes / (2 * NP * ld));
  const int64_t n_pieces = (V + piece - 1) / piece, n_blocks = R > 0 ? (R + block - 1) / block : 1;
  const bool two = NP == 1 && R <= kTwoPartsTiles && n_pieces == 1;
  Operand dz{};
  dz.p = ws.take<__bf16>((two ? 2 : NP) * block * ld);
  dz.ld = ld;
  dz.s_part = block * ld;
  float* sum = n_pieces > 1 && d.dx ? ws.take<float>(R * round8(D)) : nullptr;
  float* sum_w = n_blocks > 1 && d.dW ? ws.take<float>(piece * round8(D)) : nullptr;
  const int64_t keep = ws.used;
  if (!dry && R > 0 && pack.launch(stream) != 0) return -1;
  for (int64_t v0 = 0, k = 0; v0 < V; v0 += piece, ++k) {
    const int64_t n = std::min(piece, V - v0);
    Colsum<T, NP> cs;
    int64_t columns = keep;  // what the piece's column sums hold of the workspace
    for (int64_t b = 0; b < n_blocks; ++b) {
      // (pieces and blocks reuse one workspace: a stream runs them in order)
      ws.used = columns;
      const int64_t r0 = b * block, m = std::min(block, R - r0);
      Launch<DzEpi<T, NP>> L{};
      L.n = 1;
      Problem& p = L.p[0];
      p.a = x;
      p.a.p += r0 * x.ld;
      p.b = w;
      p.b.p += v0 * w.ld;
      p.M = (int32_t)m;
      p.N = (int32_t)n;
      p.K = (int32_t)D;
      p.batch = p.n_outer = p.n_inner = p.splits = 1;
      DzEpi<T, NP>& e = L.e[0];
      e.bias = d.b ? static_cast<const T*>(d.b) + v0 : nullptr;
      e.target = d.target + r0;
      e.lse = d.lse + r0;
      e.low = d.low ? d.low + r0 : nullptr;
      e.gloss = d.reduction == 0 ? d.gloss + r0 : nullptr;
      e.ignore = d.ignore_index;
      e.vocab = V;
      e.dz = const_cast<__bf16*>(dz.p);
      e.second = two ? e.dz + block * ld : nullptr;
      e.ld = ld;
      e.s_part = dz.s_part;
      e.v0 = (int32_t)v0;

      // db: the waves' sums from the epilogue, up to 256 of a column; of more rows a
      // pass over dz, whose second part would be the long one.  8192 x 1024 -> 32768 in
      // bfloat16, both directions: 2195 us, of 2322 with the pass; 1500 x 777 -> 10007
      // in float32 651, of 673.
      const TileSize size = choose<NP>(L, false).size;
      if (b == 0 && d.db) {
        const int64_t chunks = (m + wave_rows<NP>(size) - 1) / wave_rows<NP>(size);
        T* db = static_cast<T*>(d.db) + v0;
        cs.blocks = n_blocks;
        if (n_blocks == 1 && chunks <= 256) e.db = cs.given(n, (int32_t)chunks, db, by, ws);
        else cs.add(dz, m, n, 1, db, by);
        cs.reserve(ws);
        columns = ws.used;
      }
      if (d.db) cs.set_rows(m);
      Products<T, NP> dx, dw;
      if (d.dx) {
        T* out = static_cast<T*>(d.dx) + r0 * D;
        dx.add(dz, p.b, two ? 2 * m : m, D, n, 1, 1, 1, out, D, 0, nullptr, 0, by);
        if (n_pieces > 1) {
          dx.L.e[0].sum = sum + r0 * round8(D);
          dx.L.e[0].mode = v0 + n == V ? 4 : k == 0 ? 2 : 3;
        }
        dx.reserve(ws, n_pieces == 1, two ? 2 : 1);
      }
      if (d.dW) {
        Operand xb = x;
        xb.p += r0 * x.ld;
        Operand dzb = dz;
        if (two) dzb.s_inner = block * ld;
        dw.add(dzb, xb, n, D, m, 1, 1, two ? 2 : 1, static_cast<T*>(d.dW) + v0 * D, D, 0, nullptr, 0, by);
        if (n_blocks > 1) {
          dw.L.e[0].sum = sum_w;
          dw.L.e[0].mode = b + 1 == n_blocks ? 4 : b == 0 ? 2 : 3;
        }
        dw.reserve(ws, n_blocks == 1);
      }
      *bytes = std::max(*bytes, ws.used);
      if (dry) continue;
      if (R > 0) {
        if (run<NP, false, false, false>(L, size, stream, "linear_cross_entropy_bwd") != 0) return -1;
        if (dx.template launch<false, true>(stream, "linear_cross_entropy_bwd") != 0) return -1;
      }
      if (dw.template launch<true, true>(stream, "linear_cross_entropy_bwd") != 0) return -1;
      if (cs.launch(stream, b) != 0) return -1;
    }
  }
  return 0;
}

int call(const d3a_linear_xent_desc* d, bool bwd, bool dry, hipStream_t stream, int64_t* bytes) {
  Arena ws{dry ? nullptr : static_cast<char*>(d->ws)};
  *bytes = 0;
  if (d->dtype == D3A_F32)
    return bwd ? backward<float, 3>(*d, ws, dry, stream, bytes) : forward<float, 3>(*d, ws, dry, stream, bytes);
  return bwd ? backward<__bf16, 1>(*d, ws, dry, stream, bytes) : forward<__bf16, 1>(*d, ws, dry, stream, bytes);
}

int entry(const d3a_linear_xent_desc* d, bool bwd, void* stream) {
  if (check(d, bwd) != 0) return -1;
  int64_t need = 0;
  if (call(d, bwd, true, nullptr, &need) != 0) return -1;
  D3A_CHECK_ARG(need == 0 || (d->ws && d->ws_bytes >= need && (reinterpret_cast<uintptr_t>(d->ws) & 255) == 0),
                "linear_cross_entropy: workspace of %lld bytes (256-byte aligned) needed", (long long)need);
  return call(d, bwd, false, static_cast<hipStream_t>(stream), &need);
}

}  // namespace
}  // namespace d3a

extern "C" {

int d3a_linear_xent_workspace(const d3a_linear_xent_desc* d, int32_t backward, int64_t* bytes) {
  if (d3a::check(d, backward != 0) != 0) return -1;
  D3A_CHECK_ARG(bytes, "linear_cross_entropy: null size");
  return d3a::call(d, backward != 0, true, nullptr, bytes);
}

int d3a_linear_xent(const d3a_linear_xent_desc* d, void* stream) { return d3a::entry(d, false, stream); }

int d3a_linear_xent_bwd(const d3a_linear_xent_desc* d, void* stream) { return d3a::entry(d, true, stream); }

}  // extern "C"
