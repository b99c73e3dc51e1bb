// Host side of the products of mm.hpp, and the small passes around them:
// packing an operand (float32: its exact three-way bf16 split; bfloat16: an
// aligned copy of one that the tiles cannot read in place), column sums (bias
// gradients) and the sum of split-k partials.
#pragma once

#include <algorithm>
#include <cmath>

#include "mm.hpp"

namespace d3a {
namespace mm {

// The longest axes: a tile's rows are addressed within 2 GiB of its first (256
// rows of kMaxWidth bfloat16 values are 1 GiB), and a row's number is an int.
constexpr int64_t kMaxWidth = 1LL << 21, kMaxRows = (1LL << 31) - 4096;

inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// Bump allocation over the caller's workspace; with a null base it measures.
struct Arena {
  char* base;
  int64_t used = 0;
  template <class T>
  T* take(int64_t n) {
    used = (used + 255) / 256 * 256;
    T* p = reinterpret_cast<T*>(base ? base + used : nullptr);
    used += n * (int64_t)sizeof(T);
    return p;
  }
};

// ---- packing ------------------------------------------------------------------
struct PackJob {
  const void* src;
  __bf16* dst;             // [planes][batch][rows][round8(cols)], the tail zero
  int64_t ld, s_batch;     // of src, elements
  int64_t rows, cols, batch;
};
constexpr int kMaxPack = 6;
struct PackJobs {
  PackJob j[kMaxPack];
  int64_t end[kMaxPack];  // running count of 8-wide pieces
  int32_t n;
};

// One 8-wide piece a thread: 32 bytes (16) in, 48 (16) out; memory bound.
template <class T, int NP>
__global__ __launch_bounds__(256) void pack_kernel(const PackJobs J, int64_t p0) {
  int64_t p = p0 + (int64_t)blockIdx.x * 256 + threadIdx.x;
  int i = 0;
  while (i < J.n && p >= J.end[i]) ++i;
  if (i == J.n) return;
  if (i > 0) p -= J.end[i - 1];
  const PackJob& j = J.j[i];
  const int64_t blocks = (j.cols + 7) / 8;
  const int64_t row = p / blocks;  // batch * rows + r
  const int c = (int)(p - row * blocks) * 8;
  const int64_t b = row / j.rows, r = row - b * j.rows;
  const T* s = static_cast<const T*>(j.src) + b * j.s_batch + r * j.ld + c;
  float v[8];
  if (c + 8 <= j.cols && (reinterpret_cast<uintptr_t>(s) & 15) == 0) {
    if constexpr (sizeof(T) == 4) {
      load4(s, v);
      load4(s + 4, v + 4);
    } else {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(s);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (float)x[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? (float)s[k] : 0.f;
  }
  const int64_t s_part = j.batch * j.rows * blocks * 8;
  __bf16* d = j.dst + row * blocks * 8 + c;
  bf16x8 o[NP];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (NP == 1) {
      o[0][k] = (__bf16)v[k];
    } else {
      __bf16 x, y, z;
      split3(v[k], x, y, z);
      o[0][k] = x;
      o[1][k] = y;
      o[2][k] = z;
    }
  }
#pragma unroll
  for (int q = 0; q < NP; ++q) *reinterpret_cast<bf16x8*>(d + q * s_part) = o[q];
}

// Collects what one call has to pack and launches it once.
template <class T, int NP>
struct Packer {
  PackJobs jobs{};
  Arena& ws;
  explicit Packer(Arena& a) : ws(a) {}

  // The operand planes of a [batch][rows][cols] array (s_batch 0: one shared
  // batch), in place where the tiles can read it: one plane, 16-byte rows, and
  // offsets within a tile that fit the resource.
  Operand operand(const void* p, int64_t ld, int64_t s_batch, int64_t batch, int64_t rows,
                  int64_t cols, bool force = false) {
    Operand o{};
    const int64_t c8 = round8(cols);
    const int64_t nb = s_batch == 0 ? 1 : batch;
    const bool in_place = NP == 1 && !force && cols % 8 == 0 && ld % 8 == 0 && s_batch % 8 == 0 &&
                          (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld <= kMaxWidth;
    if (in_place) {
      o.p = static_cast<const __bf16*>(p);
      o.ld = ld;
      o.s_batch = s_batch;
      return o;
    }
    __bf16* d = ws.take<__bf16>(NP * nb * rows * c8);
    o.p = d;
    o.ld = c8;
    o.s_batch = s_batch == 0 ? 0 : rows * c8;
    o.s_part = nb * rows * c8;
    PackJob& j = jobs.j[jobs.n];
    j = PackJob{p, d, ld, s_batch, rows, cols, nb};
    jobs.end[jobs.n] = (jobs.n ? jobs.end[jobs.n - 1] : 0) + nb * rows * (c8 / 8);
    ++jobs.n;
    return o;
  }

  int launch(hipStream_t stream) {
    if (jobs.n == 0 || jobs.end[jobs.n - 1] == 0) return 0;
    // (a launch holds less than 2^32 threads)
    constexpr int64_t most = 1LL << 31;
    const int64_t pieces = jobs.end[jobs.n - 1];
    for (int64_t p0 = 0; p0 < pieces; p0 += most) {
      pack_kernel<T, NP><<<(unsigned)((std::min(pieces - p0, most) + 255) / 256), 256, 0, stream>>>(jobs, p0);
      D3A_LAUNCH_CHECK("pack");
    }
    return 0;
  }
};

// ---- column sums -----------------------------------------------------------------
// out[b][c] = sum over rows of the value at [b][r][c] of NP operand planes.
// Rows are cut into chunks whose float32 sums a second pass adds in order, so
// the result does not depend on timing; few rows are one chunk and one pass.
// Memory bound: four columns (8 bytes a plane) a lane.
struct ColsumJob {
  const __bf16* src;
  int64_t ld, s_batch, s_part;
  void* out;       // T [batch][cols]
  int32_t rows, cols, batch;
  Factor factor;
};
constexpr int kMaxColsum = 3;
struct ColsumJobs {
  ColsumJob j[kMaxColsum];
  float* part;                    // [chunks][quads][4]
  int64_t first[kMaxColsum + 1];  // running count of batch * quads of columns
  int32_t n, chunks;
  int32_t all;                    // chunks of all blocks of rows (chunks: of one)
};

// the job that quad q of all belongs to, its batch and its first column there
__device__ __forceinline__ const ColsumJob& colsum_job(const ColsumJobs& J, int64_t q, int64_t& b, int& col) {
  int i = 0;
  while (i + 1 < J.n && q >= J.first[i + 1]) ++i;
  const ColsumJob& j = J.j[i];
  const int64_t quads = (j.cols + 3) / 4, at = q - J.first[i];
  b = at / quads;
  col = (int)(at - b * quads) * 4;
  return j;
}

template <class T>
__device__ __forceinline__ void colsum_store(const ColsumJob& j, int64_t b, int col, const float s[4]) {
  T* o = static_cast<T*>(j.out) + b * j.cols + col;
  const float by = j.factor.get();
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (col + k < j.cols) o[k] = (T)(s[k] * by);
}

// a workgroup: 64 quads (one a lane) x its chunk of rows over sixteen waves
template <class T, int NP>
__global__ __launch_bounds__(1024) void colsum_kernel(const ColsumJobs J) {
  __shared__ f32x4 red[1024];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t quads = J.first[J.n], q = (int64_t)blockIdx.x * 64 + lane;
  const bool on = q < quads;
  int64_t b;
  int col;
  const ColsumJob& j = colsum_job(J, on ? q : 0, b, col);
  const __bf16* p = j.src + b * j.s_batch + col;
  const int64_t per = (j.rows + J.chunks - 1) / J.chunks;
  const int64_t r0 = per * blockIdx.y, r1 = min(r0 + per, (int64_t)j.rows);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (on)
#pragma unroll 4
    for (int64_t r = r0 + w; r < r1; r += 16) {
      bf16x4 x[NP];
#pragma unroll
      for (int k = 0; k < NP; ++k) x[k] = *reinterpret_cast<const bf16x4*>(p + k * j.s_part + r * j.ld);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = (float)x[NP - 1][e];
#pragma unroll
        for (int k = NP - 2; k >= 0; --k) v += (float)x[k][e];
        s[e] += v;
      }
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (w != 0 || !on) return;
  for (int k = 1; k < 16; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += red[64 * k + lane][e];
  const float v[4] = {s[0], s[1], s[2], s[3]};
  if (J.all == 1) colsum_store<T>(j, b, col, v);
  else store4(J.part + (blockIdx.y * quads + q) * 4, v);
}

// 64 quads x the chunks over sixteen waves
template <class T>
__global__ __launch_bounds__(1024) void colsum_finish(const ColsumJobs J) {
  __shared__ f32x4 red[1024];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t quads = J.first[J.n], q = (int64_t)blockIdx.x * 64 + lane;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (q < quads)
#pragma unroll 4
    for (int k = w; k < J.all; k += 16) {
      float v[4];
      load4(J.part + (k * quads + q) * 4, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (w != 0 || q >= quads) return;
  for (int k = 1; k < 16; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += red[64 * k + lane][e];
  int64_t b;
  int col;
  const ColsumJob& j = colsum_job(J, q, b, col);
  const float v[4] = {s[0], s[1], s[2], s[3]};
  colsum_store<T>(j, b, col, v);
}

// Rows that come in `blocks` of the same buffer: one add() and one reserve(), then a
// launch(stream, k) for each, the last of which adds them all up.
template <class T, int NP>
struct Colsum {
  ColsumJobs jobs{};
  bool from_epilogue = false;
  int64_t blocks = 1;
  void add(const Operand& o, int64_t rows, int64_t cols, int64_t batch, void* out, Factor factor = {}) {
    jobs.j[jobs.n] = ColsumJob{o.p, o.ld, o.s_batch, o.s_part, out, (int32_t)rows, (int32_t)cols, (int32_t)batch, factor};
    jobs.first[jobs.n + 1] = jobs.first[jobs.n] + batch * ((cols + 3) / 4);
    ++jobs.n;
    // about 768 workgroups, chunks of at least 64 rows (four a wave)
    const int64_t wide = (jobs.first[jobs.n] + 63) / 64;
    jobs.chunks = rows <= 512 ? 1
                              : (int32_t)std::max<int64_t>(
                                    1, std::min<int64_t>({768 / std::max<int64_t>(wide, 1), rows / 64, 256}));
    jobs.all = (int32_t)(jobs.chunks * blocks);
  }
  // instead of add(): the chunks' sums come from an epilogue, [chunks][quads][4]
  float* given(int64_t cols, int32_t chunks, void* out, Factor factor, Arena& ws) {
    jobs.j[0] = ColsumJob{nullptr, 0, 0, 0, out, 0, (int32_t)cols, 1, factor};
    jobs.first[1] = (cols + 3) / 4;
    jobs.n = 1;
    jobs.chunks = jobs.all = chunks;
    from_epilogue = true;
    return jobs.part = ws.take<float>(chunks * jobs.first[1] * 4);
  }
  void reserve(Arena& ws) {
    if (jobs.n && !from_epilogue && jobs.all > 1) jobs.part = ws.take<float>(jobs.all * jobs.first[jobs.n] * 4);
  }
  // the rows of job 0 in this block
  void set_rows(int64_t rows) { jobs.j[0].rows = (int32_t)rows; }
  int launch(hipStream_t stream, int64_t k = 0) {
    const int64_t quads = jobs.first[jobs.n];
    if (jobs.n == 0 || quads == 0) return 0;
    const unsigned wide = (unsigned)((quads + 63) / 64);
    if (!from_epilogue) {
      ColsumJobs block = jobs;
      if (jobs.all > 1) block.part += k * jobs.chunks * quads * 4;
      colsum_kernel<T, NP><<<dim3(wide, jobs.chunks), 1024, 0, stream>>>(block);
      D3A_LAUNCH_CHECK("column sums");
      if (jobs.all == 1 || k + 1 < blocks) return 0;
    }
    colsum_finish<T><<<wide, 1024, 0, stream>>>(jobs);
    D3A_LAUNCH_CHECK("column sums");
    return 0;
  }
};

// ---- split-k partials -------------------------------------------------------------
template <class T>
struct SumJob {
  const float* part;  // [splits][batch][M] rows of round8(N)
  T* out;
  const T* bias;      // [batch][N] or null
  int64_t ld, s_batch, s_bias;
  int64_t n;          // batch * M * round8(N)
  int32_t M, N, splits, vec;  // vec: out takes eight values at a time
  Factor factor;
};
template <class T>
struct SumJobs {
  SumJob<T> j[kMaxProblems];
  int64_t end[kMaxProblems];  // running count of pieces: a row's eight columns
  int32_t n;
};

template <class T>
__global__ __launch_bounds__(256) void sum_kernel(const SumJobs<T> J) {
  int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int i = 0;
  while (i < J.n && e >= J.end[i]) ++i;
  if (i == J.n) return;
  if (i > 0) e -= J.end[i - 1];
  const SumJob<T>& j = J.j[i];
  const int64_t pieces = (j.N + 7) / 8, row = e / pieces, b = row / j.M;
  const int n = (int)(e - row * pieces) * 8, left = j.N - n;
  const float* p = j.part + (row * pieces) * 8 + n;
  T* o = j.out + b * j.s_batch + (row - b * j.M) * j.ld + n;
  float s[8], bias[8];
  load_bias(j.bias ? j.bias + b * j.s_bias : nullptr, n, j.N, bias);
  const float by = j.factor.get();
#pragma unroll
  for (int r = 0; r < 8; ++r) s[r] = 0.f;
#pragma unroll 2
  for (int k = 0; k < j.splits; ++k) {
    float v[8];
    load8(p + k * j.n, v);
#pragma unroll
    for (int r = 0; r < 8; ++r) s[r] += v[r];
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) s[r] = s[r] * by + bias[r];
  if (j.vec && left >= 8) {
    store8(o, s);
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < left) o[r] = (T)s[r];
  }
}

// ---- tile choice --------------------------------------------------------------------
// Three tiles: a large one uses each staged byte most, the small ones keep the
// chip busy on less.
enum TileSize { kLarge, kMid, kSmall };

template <int NP>
struct Tiles;
template <>
struct Tiles<1> {
  typedef Config<256, 256, 64, 2, 4, 1> Large;
  typedef Config<128, 128, 64, 2, 2, 1> Mid;
  typedef Config<64, 64, 64, 2, 1, 1> Small;
};
template <>
struct Tiles<3> {
  typedef Config<256, 128, 32, 4, 2, 3> Large;
  typedef Config<128, 128, 32, 4, 2, 3> Mid;
  typedef Config<64, 64, 32, 2, 1, 3> Small;
};

// What a tile costs: `busy` us a k tile that a CU spends on one where several
// share it, `alone` us a k tile that one takes by itself (its loads' latency),
// `ends` us of prologue and epilogue, `resident` workgroups a CU.  Fitted to
// measured products, of which (us by large / mid / small tiles, * the best cut
// of k)  bfloat16: 8192 x 1024 x 4096 82 / 58 / 84, 8192 x 1024 x 32768 415* /
// 516 / 853, 32768 x 1024 x 8192 373 / 471 / 994, 1024 x 2048 x 1024 28 / 15 /
// 12;  float32: 1500 x 777 x 10007 134* / 150* / 205*, 1500 x 10007 x 777 152 /
// 186 / 223, 1999 x 513 x 1366 40* / 39* / 43*, 256 x 512 x 256 19 / 12 / 9.  (Timed
// alone: inside a block, whose operands come from other kernels, a product can take a
// fifth longer, as the gated block's dx of 8192 x 1024 x 8192, 154 to 173 us of 134.)
struct Cost {
  int bm, bn, bk, resident;
  double busy, alone, ends;
};

template <int NP>
Cost cost_of(TileSize s) {
  typedef Tiles<NP> X;
  if (NP == 1) {
    if (s == kLarge) return {X::Large::BM, X::Large::BN, X::Large::BK, 1, 1.6, 1.4, 6.0};
    if (s == kMid) return {X::Mid::BM, X::Mid::BN, X::Mid::BK, 2, 0.5, 0.58, 5.5};
    return {X::Small::BM, X::Small::BN, X::Small::BK, 5, 0.22, 0.27, 5.5};
  }
  if (s == kLarge) return {X::Large::BM, X::Large::BN, X::Large::BK, 1, 2.1, 1.9, 6.0};
  if (s == kMid) return {X::Mid::BM, X::Mid::BN, X::Mid::BK, 1, 1.25, 1.15, 5.5};
  return {X::Small::BM, X::Small::BN, X::Small::BK, 3, 0.47, 0.6, 5.5};
}

struct Choice {
  TileSize size;
  int splits;
};

// The tile and, where `may_split`, the cuts of the k axis that the model gives
// the least time: the fullest CU's tiles, and the partial sums' way out and
// back in at 4 TB/s plus 12 us for their pass (5 of them on the host).
template <int NP, class Epi>
Choice choose(const Launch<Epi>& L, bool dual, bool may_split = false) {
  Choice best{kSmall, 1};
  double least = 1e30;
  for (TileSize s : {kLarge, kMid, kSmall}) {
    const Cost c = cost_of<NP>(s);
    double tiles = 0, steps = 1, partial = 0;
    for (int i = 0; i < L.n; ++i) {
      const Problem& p = L.p[i];
      const int bn = dual ? c.bn / 2 : c.bn;
      tiles += (double)((p.M + c.bm - 1) / c.bm) * ((p.N + bn - 1) / bn) * p.batch;
      steps = std::max(steps, (double)((p.K + c.bk - 1) / c.bk) * p.n_outer * p.n_inner);
      partial += (double)p.M * p.N * p.batch;
    }
    for (int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (splits > 1 && (!may_split || steps < 4 * splits || tiles * splits > 1280)) break;
      const int each = (int)std::ceil(tiles * splits / 256), full = each / c.resident, over = each % c.resident;
      double t = full * std::max(c.resident * c.busy, c.alone) + (over ? std::max(over * c.busy, c.alone) : 0.0);
      t = t * std::ceil(steps / splits) + (full + (over > 0)) * c.ends;
      if (splits > 1) t += partial * 4 * (2 * splits) / 4e6 + 12;
      if (t < least) {
        least = t;
        best = Choice{s, splits};
      }
    }
  }
  return best;
}

template <int NP, bool AT, bool BT, bool DUAL, class Epi>
int run(Launch<Epi>& L, TileSize s, hipStream_t stream, const char* what) {
  typedef Tiles<NP> X;
  if (s == kLarge) return launch<typename X::Large, AT, BT, DUAL>(L, stream, what);
  if (s == kMid) return launch<typename X::Mid, AT, BT, DUAL>(L, stream, what);
  return launch<typename X::Small, AT, BT, DUAL>(L, stream, what);
}

// A launch of plain products D -> T (StoreEpi), with the k axis cut where that
// is the quicker way.
template <class T, int NP>
struct Products {
  Launch<StoreEpi<T>> L{};
  SumJobs<T> sums{};
  TileSize size = kSmall;

  void add(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t K, int64_t batch,
           int64_t n_outer, int64_t n_inner, void* out, int64_t ld, int64_t s_batch,
           const void* bias, int64_t s_bias, Factor factor = {}) {
    Problem& p = L.p[L.n];
    p = Problem{};
    p.a = a;
    p.b = b;
    p.M = (int32_t)M;
    p.N = (int32_t)N;
    p.K = (int32_t)K;
    p.batch = (int32_t)batch;
    p.n_outer = (int32_t)n_outer;
    p.n_inner = (int32_t)n_inner;
    p.splits = 1;
    StoreEpi<T>& e = L.e[L.n];
    e = StoreEpi<T>{};
    e.out = static_cast<T*>(out);
    e.ld = ld;
    e.s_batch = s_batch;
    e.bias = static_cast<const T*>(bias);
    e.s_bias = s_bias;
    e.n_batch = (int32_t)batch;
    e.factor = factor;
    e.vec = ld * sizeof(T) % 16 == 0 && s_batch * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    ++L.n;
  }

  // after every add(): the tile, the splits and their partials.  fold: A's rows are this
  // many times the result's, which is their sum (row m, M / fold + m, ..): in the
  // partials' layout each split is then `fold` of them
  void reserve(Arena& ws, bool may_split, int fold = 1) {
    if (L.n == 0) return;
    const Choice c = choose<NP>(L, false, may_split);
    size = c.size;
    if (c.splits == 1 && fold == 1) return;
    for (int i = 0; i < L.n; ++i) {
      Problem& p = L.p[i];
      p.splits = c.splits;
      StoreEpi<T>& e = L.e[i];
      const int64_t n = (int64_t)p.batch * p.M * round8(p.N);
      e.sum = ws.take<float>(c.splits * n);
      e.mode = 1;
      sums.j[sums.n] = SumJob<T>{e.sum, e.out, e.bias, e.ld, e.s_batch, e.s_bias, n / fold, p.M / fold, p.N,
                                 p.splits * fold, e.vec, e.factor};
      sums.end[sums.n] = (sums.n ? sums.end[sums.n - 1] : 0) + (int64_t)p.batch * (p.M / fold) * ((p.N + 7) / 8);
      ++sums.n;
    }
  }

  template <bool AT, bool BT>
  int launch(hipStream_t stream, const char* what) {
    if (L.n == 0) return 0;
    if (run<NP, AT, BT, false>(L, size, stream, what) != 0) return -1;
    if (sums.n == 0) return 0;
    sum_kernel<T><<<(unsigned)((sums.end[sums.n - 1] + 255) / 256), 256, 0, stream>>>(sums);
    D3A_LAUNCH_CHECK(what);
    return 0;
  }
};

}  // namespace mm
}  // namespace d3a
