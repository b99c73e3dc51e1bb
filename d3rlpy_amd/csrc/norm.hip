// Layer norm, forward and backward, of rows of n values:
//
//   xh = (x - mean) rstd,  y = xh w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   t = dy w,  dx = rstd (t - mean(t) - xh mean(t xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Memory bound: forward reads x and writes y, backward reads x and dy and
// writes dx.  A row is held in registers (by a wave, or by four where it is
// long), so each value is read once and the variance is that of the centred
// values; the backward's waves walk the rows and keep the columns' sums of dw
// and db in registers, one partial a workgroup, which a second pass adds in
// order.  Statistics and sums are float32.
#include <algorithm>

#include "mm_host.hpp"
#include "../../include/d3rlpy_amd.h"

namespace d3a {
namespace {

using mm::Arena;
using mm::bf16x8;
using mm::f32x4;

// VEC values at p as float; VEC 1, or 16 bytes of T (and as many of another type)
template <int VEC, class T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = (float)p[0];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) mm::load4(p + k, v + k);
  } else {
    static_assert(VEC == 8, "16 bytes");
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)x[k];
  }
}

// the same as it lies in memory, to be converted when it is used
template <int VEC, class T>
struct Raw {
  typedef std::conditional_t<VEC == 1, T, std::conditional_t<sizeof(T) == 4, f32x4, bf16x8>> V;
  V v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const V*>(p); }
  __device__ __forceinline__ void get(float* o) const {
    if constexpr (VEC == 1) {
      o[0] = (float)v;
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) o[k] = (float)v[k];
    }
  }
};

template <int VEC, class T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  if constexpr (VEC == 1) {
    p[0] = (T)v[0];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) mm::store4(p + k, v + k);
  } else {
    bf16x8 x;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (__bf16)v[k];
    *reinterpret_cast<bf16x8*>(p) = x;
  }
}

struct Args {
  const void *x, *w, *b, *dy;
  void *y, *dx, *dw, *db;
  float *mean, *rstd, *part;
  int64_t rows, members, ldx, sx, lddy, sdy;
  int32_t n;
  float eps;
};

// the sum over the WPR waves that hold a row
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  if constexpr (WPR == 1) return wave_sum(v);
  return block_sum(v, scratch);
}

// NCH pieces of VEC values a lane; WPR waves a row (1: four rows a workgroup).
// Grid (workgroups, members): workgroup g of a member takes rows g, g + grid, ..
// (times the rows it holds at once).  Single values (VEC 1) are bound by the
// loads' number, so w and b stay in registers over 2048 workgroups' rows and the
// next row is loaded ahead; pieces take a workgroup for every row (up to 2^22, of the
// 2^24 that a launch holds) and load w and b when they need them: 8192 x 2048 in
// bfloat16 takes 14 to 15 us, 18 the other way, and 8192 x 2047 22, of 38.
template <class T, class W, int VEC, int NCH, int WPR>
__global__ __launch_bounds__(256) void norm_kernel(const Args A) {
  constexpr bool kWalk = VEC == 1, kAhead = kWalk && NCH <= 16;
  __shared__ float scratch[4];
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int l = (wid % WPR) * 64 + lane;
  const int64_t c = blockIdx.y;
  Raw<VEC, T> rx[NCH];
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
    const T* x = static_cast<const T*>(A.x) + c * A.sx + r * A.ldx;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * WPR * 64 + l) * VEC;
      if (col < A.n) rx[j].load(x + col);
    }
  };
  const int64_t step = (int64_t)gridDim.x * (4 / WPR);
  const int64_t r0 = (int64_t)blockIdx.x * (4 / WPR) + wid / WPR;
  if (r0 >= A.rows) return;  // (WPR 4: the whole workgroup or none of it)
  fetch(r0);
  const W* w = static_cast<const W*>(A.w) + c * A.n;
  const W* b = static_cast<const W*>(A.b) + c * A.n;
  float wv[NCH][VEC], bv[NCH][VEC];
  auto affine = [&](int j) __attribute__((always_inline)) {
    const int col = (j * WPR * 64 + l) * VEC;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      wv[j][k] = 1.f;
      bv[j][k] = 0.f;
    }
    if (A.w && col < A.n) load_vec<VEC>(w + col, wv[j]);
    if (A.b && col < A.n) load_vec<VEC>(b + col, bv[j]);
  };
  if (kWalk)
#pragma unroll
    for (int j = 0; j < NCH; ++j) affine(j);
  for (int64_t r = r0; r < A.rows; r += step) {
    const int64_t row = c * A.rows + r;
    float v[NCH][VEC], s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if ((j * WPR * 64 + l) * VEC < A.n) {
        rx[j].get(v[j]);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j][k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) s += v[j][k];
    }
    if (kAhead && r + step < A.rows) fetch(r + step);
    const float mean = row_sum<WPR>(s, scratch) / (float)A.n;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * WPR * 64 + l) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[j][k] = col < A.n ? v[j][k] - mean : 0.f;
        s = fmaf(v[j][k], v[j][k], s);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<WPR>(s, scratch) / (float)A.n + A.eps);
    if (A.mean && l == 0) {
      A.mean[row] = mean;
      A.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(A.y) + row * A.n;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * WPR * 64 + l) * VEC;
      if (col >= A.n) continue;
      if (!kWalk) affine(j);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[j][k] = fmaf(v[j][k] * rstd, wv[j][k], bv[j][k]);
      store_vec<VEC>(y + col, v[j]);
    }
    if (!kAhead && r + step < A.rows) fetch(r + step);
  }
}

// Grid and rows as the forward's; a row that leaves registers free is loaded one
// ahead.  Four waves a row from 1025 values on, since a wave that holds 2048 of x, dy,
// w, dw and db has two neighbours a SIMD at most: 8192 x 2048 in bfloat16 takes 23.5 us
// (117 MB with the partials, 5 TB/s), of 36; 3001 x 1537 in float32 13.6, of 23.5.
template <class T, class W, int VEC, int NCH, int WPR>
__global__ __launch_bounds__(256) void norm_bwd_kernel(const Args A) {
  constexpr bool kAhead = NCH * VEC <= 16;
  __shared__ float scratch[8];
  __shared__ float cols[WPR == 1 ? 2 * NCH * VEC * 64 : 1];
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int l = (wid % WPR) * 64 + lane;
  const int64_t c = blockIdx.y;
  const W* w = static_cast<const W*>(A.w) + c * A.n;
  float wv[NCH][VEC], dw[NCH][VEC], db[NCH][VEC];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * WPR * 64 + l) * VEC;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      wv[j][k] = 1.f;
      dw[j][k] = db[j][k] = 0.f;
    }
    if (A.w && col < A.n) load_vec<VEC>(w + col, wv[j]);
  }
  const int64_t step = (int64_t)gridDim.x * (4 / WPR);
  Raw<VEC, T> rx[NCH], ry[NCH];
  float mean, rstd, next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
    const T* x = static_cast<const T*>(A.x) + c * A.sx + r * A.ldx;
    const T* dy = static_cast<const T*>(A.dy) + c * A.sdy + r * A.lddy;
    next_mean = A.mean[c * A.rows + r];
    next_rstd = A.rstd[c * A.rows + r];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * WPR * 64 + l) * VEC;
      if (col < A.n) {
        rx[j].load(x + col);
        ry[j].load(dy + col);
      }
    }
  };
  const int64_t r0 = (int64_t)blockIdx.x * (4 / WPR) + wid / WPR;
  if (kAhead && r0 < A.rows) fetch(r0);
  for (int64_t r = r0; r < A.rows; r += step) {
    const int64_t row = c * A.rows + r;
    if (!kAhead) fetch(r);
    mean = next_mean;
    rstd = next_rstd;
    float xh[NCH][VEC], t[NCH][VEC], s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      if ((j * WPR * 64 + l) * VEC < A.n) {
        rx[j].get(xh[j]);
        ry[j].get(t[j]);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          xh[j][k] = mean;
          t[j][k] = 0.f;
        }
      }
    }
    if (kAhead && r + step < A.rows) fetch(r + step);
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        xh[j][k] = (xh[j][k] - mean) * rstd;
        dw[j][k] = fmaf(t[j][k], xh[j][k], dw[j][k]);
        db[j][k] += t[j][k];
        t[j][k] *= wv[j][k];
        s[0] += t[j][k];
        s[1] = fmaf(t[j][k], xh[j][k], s[1]);
      }
    if (!A.dx) continue;
    if constexpr (WPR == 1) {
      s[0] = wave_sum(s[0]);
      s[1] = wave_sum(s[1]);
    } else {
      block_sum_k<2>(s, scratch);
    }
    const float m0 = s[0] / (float)A.n, m1 = s[1] / (float)A.n;
    T* dx = static_cast<T*>(A.dx) + row * A.n;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * WPR * 64 + l) * VEC;
      if (col >= A.n) continue;
#pragma unroll
      for (int k = 0; k < VEC; ++k) t[j][k] = rstd * (t[j][k] - m0 - xh[j][k] * m1);
      store_vec<VEC>(dx + col, t[j]);
    }
  }
  if (!A.part) return;
  if constexpr (WPR == 1) {
    // the four waves' sums, added in order
    for (int q = 0; q < 4; ++q) {
      if (wid == q) {
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const int at = (j * VEC + k) * 64 + lane;
            cols[at] = q ? cols[at] + dw[j][k] : dw[j][k];
            cols[NCH * VEC * 64 + at] = q ? cols[NCH * VEC * 64 + at] + db[j][k] : db[j][k];
          }
      }
      __syncthreads();
    }
    if (wid != 0) return;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        dw[j][k] = cols[(j * VEC + k) * 64 + lane];
        db[j][k] = cols[(NCH * VEC + j * VEC + k) * 64 + lane];
      }
  }
  float* part = A.part + (c * gridDim.x + blockIdx.x) * 2 * A.n;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * WPR * 64 + l) * VEC;
    if (col >= A.n) continue;
    store_vec<VEC == 1 ? 1 : 4>(part + col, dw[j]);
    store_vec<VEC == 1 ? 1 : 4>(part + A.n + col, db[j]);
    if constexpr (VEC == 8) {
      store_vec<4>(part + col + 4, dw[j] + 4);
      store_vec<4>(part + A.n + col + 4, db[j] + 4);
    }
  }
}

// dw, db of a member: 64 of its 2 n columns a workgroup, the parts over sixteen
// waves
template <class W>
__global__ __launch_bounds__(1024) void norm_finish_kernel(const Args A, int32_t parts, int64_t first) {
  __shared__ float red[1024];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t col = (first + blockIdx.x) * 64 + lane, c = blockIdx.y;
  const int64_t n = A.n;
  float s = 0.f;
  if (col < 2 * n) {
    const float* p = A.part + c * parts * 2 * n + col;
#pragma unroll 8
    for (int k = wid; k < parts; k += 16) s += p[k * 2 * n];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (wid != 0 || col >= 2 * n) return;
  for (int k = 1; k < 16; ++k) s += red[64 * k + lane];
  if (col < n) {
    if (A.dw) static_cast<W*>(A.dw)[c * n + col] = (W)s;
  } else {
    if (A.db) static_cast<W*>(A.db)[c * n + col - n] = (W)s;
  }
}

// rows too long for four waves' registers: a workgroup a row, in passes
template <class T, class W>
__global__ __launch_bounds__(256) void norm_long_kernel(const Args A, int64_t first) {
  __shared__ float scratch[4];
  const int64_t row = first + blockIdx.x, c = row / A.rows, r = row - c * A.rows;
  const T* x = static_cast<const T*>(A.x) + c * A.sx + r * A.ldx;
  const W* w = static_cast<const W*>(A.w) + c * A.n;
  const W* b = static_cast<const W*>(A.b) + c * A.n;
  float s = 0.f;
  for (int i = threadIdx.x; i < A.n; i += 256) s += (float)x[i];
  const float mean = block_sum(s, scratch) / (float)A.n;
  s = 0.f;
  for (int i = threadIdx.x; i < A.n; i += 256) {
    const float v = (float)x[i] - mean;
    s = fmaf(v, v, s);
  }
  const float rstd = 1.f / sqrtf(block_sum(s, scratch) / (float)A.n + A.eps);
  if (A.mean && threadIdx.x == 0) {
    A.mean[row] = mean;
    A.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(A.y) + row * A.n;
  for (int i = threadIdx.x; i < A.n; i += 256)
    y[i] = (T)fmaf(((float)x[i] - mean) * rstd, A.w ? (float)w[i] : 1.f, A.b ? (float)b[i] : 0.f);
}

template <class T, class W>
__global__ __launch_bounds__(256) void norm_long_dx_kernel(const Args A, int64_t first) {
  __shared__ float scratch[8];
  const int64_t row = first + blockIdx.x, c = row / A.rows, r = row - c * A.rows;
  const T* x = static_cast<const T*>(A.x) + c * A.sx + r * A.ldx;
  const T* dy = static_cast<const T*>(A.dy) + c * A.sdy + r * A.lddy;
  const W* w = static_cast<const W*>(A.w) + c * A.n;
  const float mean = A.mean[row], rstd = A.rstd[row];
  float s[2] = {0.f, 0.f};
  for (int i = threadIdx.x; i < A.n; i += 256) {
    const float t = (float)dy[i] * (A.w ? (float)w[i] : 1.f);
    s[0] += t;
    s[1] = fmaf(t, ((float)x[i] - mean) * rstd, s[1]);
  }
  block_sum_k<2>(s, scratch);
  const float m0 = s[0] / (float)A.n, m1 = s[1] / (float)A.n;
  T* dx = static_cast<T*>(A.dx) + row * A.n;
  for (int i = threadIdx.x; i < A.n; i += 256) {
    const float t = (float)dy[i] * (A.w ? (float)w[i] : 1.f);
    dx[i] = (T)(rstd * (t - m0 - ((float)x[i] - mean) * rstd * m1));
  }
}

// partials of dw, db: 64 columns x a chunk of rows (grid x: columns, y: chunks, z: members)
template <class T>
__global__ __launch_bounds__(256) void norm_long_cols_kernel(const Args A, int64_t first) {
  __shared__ float red[2][256];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int64_t col = (first + blockIdx.x) * 64 + lane, c = blockIdx.z;
  const int64_t per = (A.rows + gridDim.y - 1) / gridDim.y, r0 = per * blockIdx.y;
  const int64_t r1 = min(r0 + per, A.rows);
  float dw = 0.f, db = 0.f;
  if (col < A.n)
    for (int64_t r = r0 + wid; r < r1; r += 4) {
      const int64_t row = c * A.rows + r;
      const float x = (float)static_cast<const T*>(A.x)[c * A.sx + r * A.ldx + col];
      const float t = (float)static_cast<const T*>(A.dy)[c * A.sdy + r * A.lddy + col];
      dw = fmaf(t, (x - A.mean[row]) * A.rstd[row], dw);
      db += t;
    }
  red[0][threadIdx.x] = dw;
  red[1][threadIdx.x] = db;
  __syncthreads();
  if (wid != 0 || col >= A.n) return;
  float* part = A.part + (c * gridDim.y + blockIdx.y) * 2 * A.n + col;
#pragma unroll
  for (int q = 0; q < 2; ++q)
    part[q * A.n] = ((red[q][lane] + red[q][64 + lane]) + red[q][128 + lane]) + red[q][192 + lane];
}

// ---- host -------------------------------------------------------------------
constexpr int kWave = 1024;  // values that a wave holds
constexpr int kLong = 8192;  // values that four waves hold

int check(const d3a_layer_norm_desc* d, bool bwd) {
  D3A_CHECK_ARG(d, "layer_norm: null descriptor");
  D3A_CHECK_ARG(d->dtype == D3A_F32 || d->dtype == D3A_BF16, "layer_norm: dtype must be float32 or bfloat16");
  D3A_CHECK_ARG(d->wtype == d->dtype || d->wtype == D3A_F32,
                "layer_norm: weight and bias must have x's dtype or be float32");
  D3A_CHECK_ARG(d->rows >= 0 && d->members >= 1 && d->members <= 65535 && d->n >= 1,
                "layer_norm: sizes must be positive");
  D3A_CHECK_ARG(d->n < (1LL << 30) && d->rows < (1LL << 31) && d->rows * d->members < (1LL << 31),
                "layer_norm: size too large");
  D3A_CHECK_ARG(d->ldx >= d->n && (!bwd || d->lddy >= d->n), "layer_norm: row stride smaller than the row");
  D3A_CHECK_ARG((d->mean == nullptr) == (d->rstd == nullptr), "layer_norm: mean and rstd go together");
  if (d->rows > 0) {
    D3A_CHECK_ARG(d->x && (bwd ? d->dy != nullptr : d->y != nullptr), "layer_norm: null operand");
    D3A_CHECK_ARG(!bwd || d->mean, "layer_norm: the backward needs the forward's mean and rstd");
  }
  return 0;
}

Args args_of(const d3a_layer_norm_desc& d) {
  Args a{};
  a.x = d.x;
  a.w = d.w;
  a.b = d.b;
  a.dy = d.dy;
  a.y = d.y;
  a.dx = d.dx;
  a.dw = d.dw;
  a.db = d.db;
  a.mean = d.mean;
  a.rstd = d.rstd;
  a.rows = d.rows;
  a.members = d.members;
  a.ldx = d.ldx;
  a.sx = d.sx;
  a.lddy = d.lddy;
  a.sdy = d.sdy;
  a.n = (int32_t)d.n;
  a.eps = (float)d.eps;
  return a;
}

// every row of every array starts on 16 bytes and is whole 16-byte pieces
bool aligned(const d3a_layer_norm_desc& d, bool bwd) {
  const int64_t vec = d.dtype == D3A_F32 ? 4 : 8;
  uintptr_t p = reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.w) |
                reinterpret_cast<uintptr_t>(bwd ? d.dx : d.y) |
                reinterpret_cast<uintptr_t>(bwd ? d.dy : d.b);
  int64_t s = d.n | d.ldx | d.sx;
  if (bwd) s |= d.lddy | d.sdy;
  return (p & 15) == 0 && s % vec == 0;
}

// workgroups a member of a kernel whose waves walk over rows: enough to fill the
// chip (`all` over the members), each wave at least one row
int64_t blocks_of(const d3a_layer_norm_desc& d, int64_t at_once, int64_t all) {
  return std::max<int64_t>(1, std::min((d.rows + at_once - 1) / at_once, std::max<int64_t>(1, all / d.members)));
}
// The backward's, each of which writes a partial: three to a CU.  With its second
// pass 8192 rows of 2048 / 1024 in bfloat16 take 30 / 17 us (two to a CU 33 / 17, four
// 30 / 21), of 2048 in float32 39 (38, 41).
int64_t bwd_blocks(const d3a_layer_norm_desc& d) { return blocks_of(d, d.n > kWave ? 1 : 4, 768); }

template <class T, class W, int VEC, int NCH, int WPR>
int launch(const d3a_layer_norm_desc& d, const Args& a, bool bwd, hipStream_t stream) {
  constexpr int at_once = 4 / WPR;
  if (bwd) {
    norm_bwd_kernel<T, W, VEC, NCH, WPR><<<dim3((unsigned)bwd_blocks(d), (unsigned)d.members), 256, 0, stream>>>(a);
  } else {
    const int64_t blocks = blocks_of(d, at_once, VEC == 1 ? 2048 : 1 << 22);
    norm_kernel<T, W, VEC, NCH, WPR><<<dim3((unsigned)blocks, (unsigned)d.members), 256, 0, stream>>>(a);
  }
  D3A_LAUNCH_CHECK("layer_norm");
  return 0;
}

// pieces of 16 bytes where every row allows them, else single values
template <class T, class W>
int dispatch(const d3a_layer_norm_desc& d, const Args& a, bool bwd, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int64_t n = d.n;
  if (aligned(d, bwd)) {
    if (n > 4096) return launch<T, W, V, 8192 / (256 * V), 4>(d, a, bwd, s);
    if (n > 2048) return launch<T, W, V, 4096 / (256 * V), 4>(d, a, bwd, s);
    if (n > kWave && !bwd) return launch<T, W, V, 2048 / (64 * V), 1>(d, a, bwd, s);
    if (n > kWave) return launch<T, W, V, 2048 / (256 * V), 4>(d, a, bwd, s);
    if (n > 512) return launch<T, W, V, 1024 / (64 * V), 1>(d, a, bwd, s);
    // (one piece a lane: 512 values of bfloat16, 256 of float32)
    if constexpr (V < 8)
      if (n > 256) return launch<T, W, V, 512 / (64 * V), 1>(d, a, bwd, s);
    return launch<T, W, V, 1, 1>(d, a, bwd, s);
  }
  if (n > 4096) return launch<T, W, 1, 32, 4>(d, a, bwd, s);
  if (n > 2048) return launch<T, W, 1, 16, 4>(d, a, bwd, s);
  if (n > kWave) return launch<T, W, 1, 8, 4>(d, a, bwd, s);
  if (n > 512) return launch<T, W, 1, 16, 1>(d, a, bwd, s);
  return launch<T, W, 1, 8, 1>(d, a, bwd, s);
}

// f(first, workgroups) over `all` workgroups of `threads`: a launch holds less than
// 2^32 threads an axis
template <class F>
int in_launches(int64_t all, int64_t threads, const char* what, const F& f) {
  const int64_t most = (1LL << 31) / threads;
  for (int64_t first = 0; first < all; first += most) {
    f(first, (unsigned)std::min(all - first, most));
    D3A_LAUNCH_CHECK(what);
  }
  return 0;
}

template <class T, class W>
int forward(const d3a_layer_norm_desc& d, hipStream_t stream) {
  const Args a = args_of(d);
  if (d.rows == 0) return 0;
  if (d.n <= kLong) return dispatch<T, W>(d, a, false, stream);
  return in_launches(d.rows * d.members, 256, "layer_norm", [&](int64_t first, unsigned n) {
    norm_long_kernel<T, W><<<n, 256, 0, stream>>>(a, first);
  });
}

int64_t long_chunks(const d3a_layer_norm_desc& d) {
  const int64_t blocks = (d.n + 63) / 64 * d.members;
  return std::max<int64_t>(1, std::min<int64_t>((d.rows + 31) / 32, 2048 / blocks));
}

template <class T, class W>
int backward(const d3a_layer_norm_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  Args a = args_of(d);
  const bool cols = d.dw || d.db, is_long = d.n > kLong;
  const int64_t parts = is_long ? long_chunks(d) : bwd_blocks(d);
  if (cols) a.part = ws.take<float>(d.members * parts * 2 * d.n);
  *bytes = ws.used;
  if (dry || (!cols && (!d.dx || d.rows == 0))) return 0;
  if (is_long) {
    if (d.dx && in_launches(d.rows * d.members, 256, "layer_norm_bwd", [&](int64_t first, unsigned n) {
          norm_long_dx_kernel<T, W><<<n, 256, 0, stream>>>(a, first);
        }) != 0)
      return -1;
    if (cols && in_launches((d.n + 63) / 64, 256, "layer_norm_bwd", [&](int64_t first, unsigned n) {
          norm_long_cols_kernel<T><<<dim3(n, (unsigned)parts, (unsigned)d.members), 256, 0, stream>>>(a, first);
        }) != 0)
      return -1;
  } else {
    if (dispatch<T, W>(d, a, true, stream) != 0) return -1;
  }
  if (!cols) return 0;
  return in_launches((2 * d.n + 63) / 64, 1024, "layer_norm_bwd", [&](int64_t first, unsigned n) {
    norm_finish_kernel<W><<<dim3(n, (unsigned)d.members), 1024, 0, stream>>>(a, (int32_t)parts, first);
  });
}

int call_bwd(const d3a_layer_norm_desc* d, bool dry, hipStream_t stream, int64_t* bytes) {
  Arena ws{dry ? nullptr : static_cast<char*>(d->ws)};
  if (d->dtype == D3A_F32) return backward<float, float>(*d, ws, dry, stream, bytes);
  if (d->wtype == D3A_F32) return backward<__bf16, float>(*d, ws, dry, stream, bytes);
  return backward<__bf16, __bf16>(*d, ws, dry, stream, bytes);
}

}  // namespace
}  // namespace d3a

extern "C" {

int d3a_layer_norm_workspace(const d3a_layer_norm_desc* d, int32_t backward, int64_t* bytes) {
  if (d3a::check(d, backward != 0) != 0) return -1;
  D3A_CHECK_ARG(bytes, "layer_norm: null size");
  *bytes = 0;
  return backward ? d3a::call_bwd(d, true, nullptr, bytes) : 0;
}

int d3a_layer_norm(const d3a_layer_norm_desc* d, void* stream) {
  if (d3a::check(d, false) != 0) return -1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == D3A_F32) return d3a::forward<float, float>(*d, s);
  if (d->wtype == D3A_F32) return d3a::forward<__bf16, float>(*d, s);
  return d3a::forward<__bf16, __bf16>(*d, s);
}

int d3a_layer_norm_bwd(const d3a_layer_norm_desc* d, void* stream) {
  if (d3a::check(d, true) != 0) return -1;
  int64_t need = 0;
  if (d3a::call_bwd(d, true, nullptr, &need) != 0) return -1;
  D3A_CHECK_ARG(need == 0 || (d->ws && d->ws_bytes >= need && (reinterpret_cast<uintptr_t>(d->ws) & 255) == 0),
                "layer_norm: workspace of %lld bytes (256-byte aligned) needed", (long long)need);
  return d3a::call_bwd(d, false, static_cast<hipStream_t>(stream), &need);
}

}  // extern "C"
