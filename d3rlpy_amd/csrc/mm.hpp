// Tiled matrix products on the bf16 matrix cores with the epilogue fused, the
// core of the gated block (gated.hip) and of the linear cross entropy
// (xent.hip).
//
//   D(m, n) = sum over segments and k of A(m, k) B(n, k)
//
// An operand is either k-contiguous (element (r, k) at p + r * ld + k) or
// row-contiguous (p + k * ld + r); the tile of either goes from memory to LDS
// without passing registers (16 bytes a lane), and a row-contiguous tile is
// transposed by the LDS reads.  A bfloat16 operand has one plane; a float32
// operand is given as its exact three-way bf16 split (three planes, see pack_kernel),
// and a k step then takes the six part products that matter, smallest first: fp32
// accuracy at six bf16 products a term.  (An infinity has NaN parts: its row's or
// column's results are NaN.  The third part of a value under 2^-110 falls under
// bfloat16's smallest, 2^-133, and so does what is lost of it.)
//
// Bound by the matrix cores: 32768 x 1024 x 8192 in bfloat16 takes 373 us (1.47
// PFLOP/s), 8192 x 1024 x 4096 58 (1.19), 4096 cubed in float32 539 (255 TFLOP/s of
// terms, 1.53 PFLOP/s of part products).
//
// 16-byte pieces outside the operand (rows past its end, ks past K) read as
// zero through the buffer resource's range check, so M, N and K are free; the
// contiguous axis of an operand is a multiple of 8 elements long and 16-byte
// aligned (the caller packs one that is not).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.hpp"

namespace d3a {
namespace mm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

struct Operand {
  const __bf16* p;
  int64_t ld;
  int64_t s_batch, s_outer, s_inner, s_part;  // elements
};

// One product of a launch.  K is one segment's length; the sum runs over
// n_outer * n_inner segments at offsets o * s_outer + i * s_inner of both
// operands.  splits > 1: workgroup split s sums its share of the k tiles
// (the epilogue writes a partial).
struct Problem {
  Operand a, b;
  const __bf16* b2;  // dual products: the second B (b's strides), else null
  int32_t M, N, K;
  int32_t batch, n_outer, n_inner, splits;
  int32_t tiles_m, tiles_n, first;  // set by plan()
};

constexpr int kMaxProblems = 3;

template <class Epi>
struct Launch {
  Problem p[kMaxProblems];
  Epi e[kMaxProblems];
  int32_t n, total;
};

constexpr int kSlab = 32 * 64 * 4;  // 32 rows of a wave's 64 columns in float32

// BM x BN output tile, BK deep k tiles, WM x WN waves, NP planes an operand
template <int BM_, int BN_, int BK_, int WM_, int WN_, int NP_>
struct Config {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_, NP = NP_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int TM = BM / WM, TN = BN / WN;  // a wave's tile
  static constexpr int MT = TM / 32, NT = TN / 32;
  static constexpr int A = NP * BM * BK * 2, B = NP * BN * BK * 2;  // bytes of a buffer
  // the waves' slabs lie in the second buffers, and what is over in an array of its own
  static constexpr int SLABS_A = A / kSlab, SLABS_B = B / kSlab;
  static constexpr int MORE = NW > SLABS_A + SLABS_B ? (NW - SLABS_A - SLABS_B) * kSlab : 0;
};

// LDS of a workgroup: the buffers, and what the epilogue keeps of a wave's rows
template <class C, class Epi>
constexpr int lds_bytes() {
  return 2 * (C::A + C::B) + (Epi::kStaged ? C::MORE : 0) + C::NW * C::TM * Epi::kRowBytes;
}

struct Tile {
  int m0, n0;            // first row / column of this wave's part
  int batch, split, lane;
  int M, N;
  char *slab, *rows;     // the wave's own LDS: kSlab bytes of a staged epilogue, kRowBytes a row
};


constexpr unsigned kOutside = 0x80000000u;  // = the resource's extent

// Rows x BK tile of one operand: where each lane's pieces come from and go to.
// T: row-contiguous operand.  ROWS: tile rows; NW: waves that load it.
template <int ROWS, int BK, int NP, int NW, bool T>
struct Loader {
  static constexpr int PER_PART = ROWS * BK / 512;  // wave instructions a plane
  static constexpr int NJ = NP * PER_PART / NW;     // of each wave
  static_assert(NP * PER_PART % NW == 0 && ROWS * BK % 512 == 0, "tile split");
  static constexpr int LANES = T ? ROWS / 8 : BK / 8;  // lanes a line of the tile
  static constexpr int LINES = 64 / LANES;             // lines an instruction
  static_assert(LANES <= 64, "line length");

  unsigned off[NJ];  // byte offset from the tile's base, or kOutside
  int kk;            // k-contiguous: the first k of the lane's piece
  int sel;           // dual: bit j set = instruction j reads the second matrix

  // LDS serves 256 bytes a cycle.  k-contiguous lines are rows of BK: piece c
  // (16 bytes) of row r sits at c ^ swz(r), so that sixteen rows' pieces of one
  // k cover all banks.  Row-contiguous lines are ks of ROWS: unit u (32 bytes) of
  // k sits at u ^ unit_swz(k), so that the four ks x two units of half a
  // transposed read do.
  static __device__ __forceinline__ int swz(int r) {
    static_assert(BK == 64 || BK == 32, "depth");
    return BK == 64 ? ((r >> 1) & 7) : ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int unit_swz(int k) {
    return ROWS >= 128 ? (k & 3) << 1 : ((k >> 1) & 1) << 1;
  }

  template <bool DUAL>
  __device__ __forceinline__ void init(int w, int lane, int row0, int rows, int64_t ld) {
    sel = 0;
    const int line0 = lane / LANES, c = lane % LANES;
    // (one k for all the lane's pieces: its lines are whole periods of swz apart)
    static_assert(T || NW * LINES % 16 == 0, "period of swz");
    kk = T ? 0 : 8 * (c ^ swz(w % PER_PART * LINES + line0));
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int q = (j * NW + w) % PER_PART, line = q * LINES + line0;
      if constexpr (T) {
        const int cc = c ^ (unit_swz(line) << 1);
        off[j] = row0 + 8 * cc < rows ? (unsigned)(line * ld * 2) + 16u * cc : kOutside;
      } else {
        int row = line;
        if constexpr (DUAL) {
          sel |= ((q * LINES / 32) & 1) << j;
          row = (line / 64) * 32 + line % 32;
        }
        off[j] = row0 + row < rows ? (unsigned)(row * ld * 2) + 2u * kk : kOutside;
      }
    }
  }

  // p: the tile's first element (plane 0); k_left: ks of the segment from the
  // tile's first on
  template <bool DUAL>
  __device__ __forceinline__ void load(char* lds, int w, int lane, const __bf16* p, const __bf16* p2,
                                       int64_t s_part, int k_left) const {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int part = NP == 1 ? 0 : (j * NW + w) / PER_PART;
      const __bf16* base = DUAL && ((sel >> j) & 1) ? p2 : p;
      base += part * s_part;
      const int k = T ? ((j * NW + w) % PER_PART) * LINES + lane / LANES : kk;
      const unsigned o = k < k_left ? off[j] : kOutside;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<__bf16*>(base), (short)0, (int)kOutside, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + (j * NW + w) * 1024), 16, o, 0, 0, 0);
    }
  }
};

// Fragments of a tile in LDS: 32 rows x 16 ks for v_mfma_f32_32x32x16_bf16,
// lane l holding row l % 32, ks 8 (l / 32) .. + 7 of the step.
template <int ROWS, int BK, bool T>
struct Frag {
  // byte offset of plane `part`, rows rb .. rb + 31 (rb a multiple of 32), step s
  static __device__ __forceinline__ bf16x8 get(const char* lds, int part, int rb, int s, int lane) {
    const char* base = lds + part * (ROWS * BK * 2);
    if constexpr (!T) {
      const int r = lane & 31, c = 2 * s + (lane >> 5);
      const int x = Loader<ROWS, BK, 1, 1, false>::swz(r);
      return *reinterpret_cast<const bf16x8*>(base + (rb + r) * (BK * 2) + ((c ^ x) << 4));
    } else {
      // a 16-lane group reads a 4 (k) x 16 (row) block: lane 4 q + p of it
      // addresses k q, rows 4 p .. 4 p + 3, and receives row `lane & 15`'s ks
      const int G = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
      const int k = 16 * s + 8 * (G >> 1) + q;
      const int unit = (rb / 16 + (G & 1)) ^ Loader<ROWS, BK, 1, 1, true>::unit_swz(q);
      const char* a = base + k * (ROWS * 2) + unit * 32 + p * 8;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(a));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) i16x4*)(a + 4 * (ROWS * 2)));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A wave's operands of one 16-deep step, and their products.  The B rows are
// the MFMA's first operand, so a lane ends with one output row m (lane % 32)
// and runs of four consecutive columns n.
template <class C, bool AT, bool BT>
struct Step {
  bf16x8 a[C::MT][C::NP], b[C::NT][C::NP];

  __device__ __forceinline__ void read(const char* sa, const char* sb, int s, int wm, int wn, int lane) {
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int p = 0; p < C::NP; ++p)
        b[j][p] = Frag<C::BN, C::BK, BT>::get(sb, p, wn * C::TN + 32 * j, s, lane);
#pragma unroll
    for (int i = 0; i < C::MT; ++i)
#pragma unroll
      for (int p = 0; p < C::NP; ++p)
        a[i][p] = Frag<C::BM, C::BK, AT>::get(sa, p, wm * C::TM + 32 * i, s, lane);
  }

  __device__ __forceinline__ void products(f32x16 (&acc)[C::MT][C::NT]) const {
    // (2,0) (1,1) (0,2) (1,0) (0,1) (0,0): the six products of the split
    // above 2^-24 of the leading one, smallest first
    constexpr int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
    for (int t = C::NP == 1 ? 5 : 0; t < 6; ++t)
#pragma unroll
      for (int i = 0; i < C::MT; ++i)
#pragma unroll
        for (int j = 0; j < C::NT; ++j) acc[i][j] = mma(b[j][pb[t]], a[i][pa[t]], acc[i][j]);
  }
};

template <class F, int... I>
__device__ __forceinline__ void each_of(const F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// f(0), f(1), .. f(N - 1) with the number as a type
template <int N, class F>
__device__ __forceinline__ void static_for(const F& f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

template <class V>
__device__ __forceinline__ V pick(bool c, V a, V b) {
  return c ? a : b;
}

// all but the wave's last `N` loads have arrived, its reads are done, and every
// wave says so
template <int N>
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <class C, bool AT, bool BT, bool DUAL, class Epi>
__global__ __launch_bounds__(C::THREADS, 2) void mm_kernel(const Launch<Epi> L) {
  static_assert(!DUAL || (C::TN == 64 && !BT), "dual: a wave's columns are 32 of each matrix");
  // (arrays of their own, each named where it is used: so the compiler sees that
  // the loads in flight go to other arrays than the reads, and waits for none;
  // with one array for both operands it waited for all in the transposed reads)
  __shared__ __attribute__((aligned(1024))) char a0[C::A], a1[C::A], b0[C::B], b1[C::B];

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / C::WN, wn = w % C::WN;

  // The tile being loaded: its operands' pieces, the next k tile's first
  // elements, the ks its segment has left, its place among the inner segments,
  // and the k tiles to go.  The loads have no branches: their address work runs
  // between the matrix instructions of one block.
  Loader<C::BM, C::BK, C::NP, C::NW, AT> la;
  Loader<C::BN, C::BK, C::NP, C::NW, BT> lb;
  const __bf16 *pa, *pb;
  int64_t a_k, b_k, a_in, b_in, a_out, b_out, a_part, b_part, b_up;
  int K, n_inner, inner, left, to_load;
  auto load = [&](char* sa, char* sb) __attribute__((always_inline)) {
    const int k_left = to_load > 0 ? left : 0;  // past the last tile: zeros, which the waits count
    la.template load<false>(sa, w, lane, pa, nullptr, a_part, k_left);
    lb.template load<DUAL>(sb, w, lane, pb, pb + b_up, b_part, k_left);
    const bool end = left <= C::BK, last = inner + 1 == n_inner;
    // (by value: a choice between variables would be one between addresses)
    pa += pick(end, pick(last, a_out, a_in), a_k);
    pb += pick(end, pick(last, b_out, b_in), b_k);
    left = pick(end, K, left - C::BK);
    inner = pick(end, pick(last, 0, inner + 1), inner);
    --to_load;
  };

  // tile `id` of the launch -> the loads' state, and where it lies
  int pi;
  auto enter = [&](int id) __attribute__((always_inline)) {
    // workgroups go to the eight XCDs in turn: give each XCD a run of
    // neighbouring tiles, whose operand rows then meet in its L2
    {
      const int q = L.total / 8, r = L.total % 8, x = id % 8;
      id = id / 8 + x * q + (x < r ? x : r);
    }
    pi = 0;
    while (pi + 1 < L.n && id >= L.p[pi + 1].first) ++pi;
    const Problem& P = L.p[pi];
    id -= P.first;
    const int per = P.tiles_m * P.tiles_n;
    int batch = 0, split = 0;
    if (id >= per) {
      const int bs = id / per;
      id -= bs * per;
      split = bs / P.batch;
      batch = bs - split * P.batch;
    }
    constexpr int GM = 8;  // and the run is a block of GM tile rows
    const int group = id / (GM * P.tiles_n), in = id - group * (GM * P.tiles_n);
    const int gm = min(P.tiles_m - group * GM, GM), col = in / gm;
    const int m0 = (group * GM + in - col * gm) * C::BM, n0 = col * (DUAL ? C::BN / 2 : C::BN);
    la.template init<false>(w, lane, m0, P.M, P.a.ld);
    lb.template init<DUAL>(w, lane, n0, P.N, P.b.ld);

    K = P.K;
    n_inner = P.n_inner;
    const int kt_seg = max((K + C::BK - 1) / C::BK, 1);  // K = 0: one empty tile
    int t = 0, seg = 0, kt = 0;
    to_load = K > 0 ? kt_seg * P.n_outer * n_inner : 0;
    inner = 0;
    if (P.splits > 1) {
      const int share = to_load / P.splits, over = to_load - share * P.splits;
      t = share * split + min(split, over);
      to_load = share + (split < over ? 1 : 0);
      seg = t / kt_seg;
      kt = t - seg * kt_seg;
      inner = seg % n_inner;
    }
    left = K - kt * C::BK;
    a_k = AT ? P.a.ld * C::BK : (int64_t)C::BK;
    b_k = BT ? P.b.ld * C::BK : (int64_t)C::BK;
    pa = P.a.p + batch * P.a.s_batch + kt * a_k + (AT ? (int64_t)m0 : (int64_t)m0 * P.a.ld);
    pb = P.b.p + batch * P.b.s_batch + kt * b_k + (BT ? (int64_t)n0 : (int64_t)n0 * P.b.ld);
    if (seg > 0) {
      pa += (seg - inner) / n_inner * P.a.s_outer + inner * P.a.s_inner;
      pb += (seg - inner) / n_inner * P.b.s_outer + inner * P.b.s_inner;
    }
    // from a segment's last tile to the next segment's first
    a_in = P.a.s_inner - (kt_seg - 1) * a_k;
    b_in = P.b.s_inner - (kt_seg - 1) * b_k;
    a_out = a_in + P.a.s_outer - n_inner * P.a.s_inner;
    b_out = b_in + P.b.s_outer - n_inner * P.b.s_inner;
    a_part = P.a.s_part;
    b_part = P.b.s_part;
    b_up = DUAL ? P.b2 - P.b.p : 0;
    return Tile{m0 + wm * C::TM, n0 + wn * (DUAL ? 32 : C::TN), batch, split, lane, P.M, P.N, nullptr, nullptr};
  };

  // Two buffers.  Each step's operands are read while the step before it is in
  // the matrix cores, also across the tiles' border: the barrier stands before
  // a tile's last step, where the wave has read that step's operands.  It says
  // that the next tile is there and that the present one is read, so behind it
  // the next tile's first step is read and the loads of the tile after that
  // start, into the present buffer: they have all of a tile's products to arrive.
  constexpr int LPT = Loader<C::BM, C::BK, C::NP, C::NW, AT>::NJ + Loader<C::BN, C::BK, C::NP, C::NW, BT>::NJ;
  constexpr int STEPS = C::BK / 16;
  static_assert(STEPS % 2 == 0, "the operand registers alternate");
  Step<C, AT, BT> f0, f1;
  auto iteration = [&](f32x16 (&acc)[C::MT][C::NT], char* ca, char* cb, const char* na, const char* nb) __attribute__((always_inline)) {
    static_for<STEPS>([&](auto step) __attribute__((always_inline)) {
      constexpr int S = decltype(step)::value;
      constexpr bool last = S + 1 == STEPS;
      Step<C, AT, BT>&now = S & 1 ? f1 : f0, &next = S & 1 ? f0 : f1;
      if constexpr (last) arrive<0>();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (last) {
        load(ca, cb);
        next.read(na, nb, 0, wm, wn, lane);
      } else {
        next.read(ca, cb, S + 1, wm, wn, lane);
      }
      now.products(acc);
      // the step's products, with the reads, the loads and the loads' address
      // work spread between them
      constexpr int MF = C::MT * C::NT * (C::NP == 1 ? 1 : 6);
      constexpr int DS = (C::MT * (AT ? 2 : 1) + C::NT * (BT ? 2 : 1)) * C::NP;
      static_for<MF>([&](auto mf) __attribute__((always_inline)) {
        constexpr int k = decltype(mf)::value;
        constexpr int ds = (k + 1) * DS / MF - k * DS / MF, vm = (k + 1) * LPT / MF - k * LPT / MF;
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (ds > 0) __builtin_amdgcn_sched_group_barrier(0x100, ds, 0);
        if constexpr (last) __builtin_amdgcn_sched_group_barrier(0x006, 6, 0);
        if constexpr (last && vm > 0) __builtin_amdgcn_sched_group_barrier(0x010, vm, 0);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // A workgroup takes tiles gridDim apart; the next one's first loads start
  // before the epilogue, which has the second buffers to itself.
  int id = blockIdx.x;
  Tile tile = enter(id);
  load(a0, b0);
  for (bool first = true;; first = false) {
    f32x16 acc[C::MT][C::NT];
#pragma unroll
    for (int i = 0; i < C::MT; ++i)
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    int n = to_load + 1;  // k tiles
    load(a1, b1);
    // (a later tile's first loads arrived before the epilogue's first store, see
    // wait_loads: waiting for them here would be waiting for its stores)
    if (first) arrive<LPT>();
    f0.read(a0, b0, 0, wm, wn, lane);
    // (in pairs: a tile past the last is zeros)
    do {
      iteration(acc, a0, b0, a1, b1);
      iteration(acc, a1, b1, a0, b0);
      n -= 2;
    } while (n > 0);
    arrive<0>();  // nothing more arrives in LDS, and nobody reads it

    const Epi& epi = L.e[pi];
    const Tile now = tile;
    id += gridDim.x;
    const bool more = id < L.total;
    if (more) {
      tile = enter(id);
      load(a0, b0);
    }
    Tile out = now;
    if constexpr (Epi::kStaged) {
      const int in_b = w - C::SLABS_A;
      out.slab = in_b < 0 ? a1 + w * kSlab : b1 + in_b * kSlab;
      if constexpr (C::MORE > 0) {
        __shared__ __attribute__((aligned(16))) char more[C::MORE];
        if (in_b >= C::SLABS_B) out.slab = more + (in_b - C::SLABS_B) * kSlab;
      }
    }
    if constexpr (Epi::kRowBytes > 0) {
      __shared__ __attribute__((aligned(16))) char rows[C::NW * C::TM * Epi::kRowBytes];
      out.rows = rows + w * C::TM * Epi::kRowBytes;
    }
    epi.template run<C>(acc, out);
    if (!more) break;
    // every wave is through with its slab
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
}

// ---- host -------------------------------------------------------------------
template <class C, bool DUAL, class Epi>
int plan(Launch<Epi>& L) {
  int64_t total = 0;
  for (int i = 0; i < L.n; ++i) {
    Problem& p = L.p[i];
    const int bn = DUAL ? C::BN / 2 : C::BN;
    p.tiles_m = (p.M + C::BM - 1) / C::BM;
    p.tiles_n = (p.N + bn - 1) / bn;
    p.first = (int32_t)total;
    total += (int64_t)p.tiles_m * p.tiles_n * p.batch * p.splits;
    if (total >= (1 << 30)) {
      set_error("product has too many tiles");
      return -1;
    }
  }
  L.total = (int32_t)total;
  return 0;
}

template <class C, bool AT, bool BT, bool DUAL, class Epi>
int launch(Launch<Epi>& L, hipStream_t stream, const char* what) {
  if (plan<C, DUAL>(L) != 0) return -1;
  if (L.total == 0) return 0;
  // as many workgroups as the chip holds (a multiple of the XCDs), or fewer
  constexpr int resident = 256 * (160 * 1024 / lds_bytes<C, Epi>());
  mm_kernel<C, AT, BT, DUAL, Epi><<<std::min(L.total, resident), C::THREADS, 0, stream>>>(L);
  D3A_LAUNCH_CHECK(what);
  return 0;
}

// The split of a float32 value in three bfloat16 parts, exact from 2^-110 up.  (Values
// above the largest bfloat16 would round to an infinity: their first part is the
// largest.  NaN and infinities have NaN among their parts.)
__device__ __forceinline__ void split3(float x, __bf16& p0, __bf16& p1, __bf16& p2) {
  constexpr float kLargest = 3.38953139e38f;  // 2^128 - 2^120
  p0 = (__bf16)__builtin_amdgcn_fmed3f(x, -kLargest, kLargest);
  const float r = x - (float)p0;
  p1 = (__bf16)r;
  p2 = (__bf16)(r - (float)p1);
}

// v[0..7] to NP planes at p (16-byte aligned)
template <int NP>
__device__ __forceinline__ void store_planes(__bf16* p, int64_t s_part, const float v[8]) {
  bf16x8 o[NP];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (NP == 1) {
      o[0][i] = (__bf16)v[i];
    } else {
      __bf16 a, b, c;
      split3(v[i], a, b, c);
      o[0][i] = a;
      o[1][i] = b;
      o[2][i] = c;
    }
  }
#pragma unroll
  for (int q = 0; q < NP; ++q) *reinterpret_cast<bf16x8*>(p + q * s_part) = o[q];
}

__device__ __forceinline__ void store4(float* p, const float v[4]) {
  *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void load4(const float* p, float v[4]) {
  const f32x4 x = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = x[i];
}
__device__ __forceinline__ void store8(float* p, const float v[8]) {
  store4(p, v);
  store4(p + 4, v + 4);
}
__device__ __forceinline__ void store8(__bf16* p, const float v[8]) { store_planes<1>(p, 0, v); }
__device__ __forceinline__ void load8(const float* p, float v[8]) {
  load4(p, v);
  load4(p + 4, v + 4);
}

// what v's rounding to bfloat16 left (nothing of an infinity or NaN)
__device__ __forceinline__ float left_of(float v) {
  const float left = v - (float)(__bf16)v;
  return fabsf(left) < INFINITY ? left : 0.f;
}

// ---- staged epilogues ---------------------------------------------------------
// A wave's tile, 32 rows at a time, is turned in LDS from the matrix
// instructions' layout (a lane holds one row's runs of four columns, 64 rows
// apart in memory) to rows of eight consecutive columns a lane, so that the
// epilogue's loads and stores are 16 bytes a lane and contiguous.  Writing
// straight from the layout cost the 8192 x 32768 x 1024 logits' gradient 1220
// us, of 620 without its stores.  16-byte piece c of row r sits at c ^ (r & 15).
//
// Loads and stores finish in order, so a load issued after a store waits for
// it: what an epilogue loads, it loads before its first store (columns' biases,
// rows' statistics by way of LDS) or a pass ahead of the stores (load(), below).
template <class C>
__device__ __forceinline__ void turn(const f32x16 (&acc)[C::MT][C::NT], const Tile& t, int i) {
  static_assert(C::TN == 64, "slab");
  const int row = t.lane & 31, half = t.lane >> 5;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 8 * j + 2 * q + half;
      const f32x16& a = acc[i][j];
      *reinterpret_cast<f32x4*>(t.slab + row * 256 + ((c ^ (row & 15)) << 4)) =
          f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// eight columns from piece c on, of row r
__device__ __forceinline__ void slab8(const Tile& t, int r, int c, float v[8]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(t.slab + r * 256 + (((c + k) ^ (r & 15)) << 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * k + e] = x[e];
  }
}

// the first of a lane's eight columns (the same in every pass)
template <bool DUAL>
__device__ __forceinline__ int first_column(const Tile& t) {
  return t.n0 + 8 * (t.lane % (DUAL ? 4 : 8));
}

struct Nothing {};

// Every epilogue's, before its first store: the next tile's first loads have
// arrived, and the main loop need not wait for the stores behind them.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// load(m, n) -> L, a pass ahead; f(m, n, v[8], up[8], L) for m < M.  DUAL: the
// wave's 32 columns of both matrices, v and up.
template <class C, bool DUAL, class G, class F>
__device__ __forceinline__ void each8(const f32x16 (&acc)[C::MT][C::NT], const Tile& t, G load, F f) {
  constexpr int LANES = DUAL ? 4 : 8, PASSES = 32 * LANES / 64;  // lanes a row; passes a slab
  const int n = first_column<DUAL>(t), c = 2 * (t.lane % LANES), r0 = t.lane / LANES;
  auto row = [&](int pass) __attribute__((always_inline)) {
    return t.m0 + pass / PASSES * 32 + pass % PASSES * (64 / LANES) + r0;
  };
  auto next = load(min(row(0), t.M - 1), n);
#pragma unroll
  for (int i = 0; i < C::MT; ++i) {
    turn<C>(acc, t, i);
    if (i == 0) wait_loads();
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int pass = i * PASSES + p, r = p * (64 / LANES) + r0, m = row(pass);
      const auto now = next;
      if (pass + 1 < C::MT * PASSES) next = load(min(row(pass + 1), t.M - 1), n);
      float v[8], up[8];
      slab8(t, r, c, v);
      if constexpr (DUAL) slab8(t, r, c + 8, up);
      if (m < t.M) f(m, n, v, up, now);
    }
  }
}

// f(m, n, v) of one column a lane, whole rows of 64: for outputs whose rows are
// not 16-byte aligned
template <class C, class F>
__device__ __forceinline__ void each1(const f32x16 (&acc)[C::MT][C::NT], const Tile& t, F f) {
  const int n = t.n0 + t.lane;
#pragma unroll
  for (int i = 0; i < C::MT; ++i) {
    turn<C>(acc, t, i);
    if (i == 0) wait_loads();
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      const float v = *reinterpret_cast<const float*>(t.slab + r * 256 + (((t.lane >> 2) ^ (r & 15)) << 4) +
                                                      4 * (t.lane & 3));
      const int m = t.m0 + 32 * i + r;
      if (m < t.M && n < t.N) f(m, n, v);
    }
  }
}

// a lane's eight columns of a bias (zero past N, or without one)
template <class T>
__device__ __forceinline__ void load_bias(const T* bias, int n, int N, float b[8]) {
#pragma unroll
  for (int r = 0; r < 8; ++r) b[r] = bias && n + r < N ? (float)bias[n + r] : 0.f;
}

// A factor of a result that is only known on the device: a[0] * b[0] (null: 1).
struct Factor {
  const float *a, *b;
  __device__ __forceinline__ float get() const { return (a ? a[0] : 1.f) * (b ? b[0] : 1.f); }
};

// D (+ bias) in T, or a float32 partial of a split / running sum over launches
template <class T>
struct StoreEpi {
  static constexpr bool kStaged = true;
  static constexpr int kRowBytes = 0;
  T* out;           // [batch][M] rows of ld
  int64_t ld, s_batch;
  const T* bias;    // [batch][N] or null
  int64_t s_bias;
  float* sum;       // splits: [split][batch][M], running sum: [M] rows of round8(N)
  int32_t mode;     // 0 out = D, 1 partial, 2 sum = D, 3 sum += D, 4 out = sum + D
  int32_t vec;      // out's rows are 16-byte aligned
  int32_t n_batch;
  Factor factor;    // of D, in what goes to out

  template <class C>
  __device__ __forceinline__ void run(f32x16 (&acc)[C::MT][C::NT], const Tile& t) const {
    const int64_t lds = (t.N + 7) / 8 * 8;
    const T* bias_b = bias ? bias + t.batch * s_bias : nullptr;
    const float by = mode == 0 || mode == 4 ? factor.get() : 1.f;
    if (mode == 0 && !vec) {
      const int n = t.n0 + t.lane;
      const float b = bias_b && n < t.N ? (float)bias_b[n] : 0.f;
      T* o = out + t.batch * s_batch;
      each1<C>(acc, t, [&](int m, int n, float v) { o[m * ld + n] = (T)(v * by + b); });
      return;
    }
    float b[8];
    load_bias(bias_b, first_column<false>(t), t.N, b);
    struct Sum {
      float v[8];
    };
    auto load = [&](int m, int n) {
      Sum o;
      if (mode >= 3 && n < t.N) {
        load8(sum + m * lds + n, o.v);
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) o.v[r] = 0.f;
      }
      return o;
    };
    each8<C, false>(acc, t, load, [&](int m, int n, float* v, float*, const Sum& o) {
      if (n >= t.N) return;
      const int left = t.N - n;
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = mode == 0 ? v[r] * by + b[r] : (v[r] + o.v[r]) * by;
      if (mode != 0 && mode <= 3) {
        store8(sum + ((mode == 1 ? ((int64_t)t.split * n_batch + t.batch) * t.M : 0) + m) * lds + n, v);
        return;
      }
      T* p = out + t.batch * s_batch + (int64_t)m * ld + n;
      if (vec && left >= 8) {
        store8(p, v);
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < left) p[r] = (T)v[r];
      }
    });
  }
};

}  // namespace mm
}  // namespace d3a
