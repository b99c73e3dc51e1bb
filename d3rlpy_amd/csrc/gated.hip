// The gated feed-forward block, forward and backward, of every ensemble member:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u,  y = h Wd^T + bd
//   dh = dy Wd,  dg = dh * u * act'(g),  du = dh * act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// All products are tiles of mm.hpp for many rows, bound by the matrix cores and the
// float32 g and u: 8192 x 1024 x 4096 in bfloat16 takes 174 to 203 us for g, u and h (137
// GFLOP, 335 MB out), 81 to 83 for y, 170 for dg and du, 154 to 173 for dx, 207 to 250 for
// the three weight gradients (206 GFLOP, 192 tiles for 256 CUs).  The first forward launch
// stages gate and up weights as one B tile whose waves hold the same 32 columns of both,
// so activation and product happen on the accumulators; the backward's first launch forms
// dh and, from the kept g and u, dg and du in its epilogue.  Kept between the two: h as
// the down product's operand, and g and u in float32.  In bfloat16 they would halve 270 MB
// of traffic at 8192 x 4096 hidden values, but a second rounding on the way to each
// gradient takes its error from 1.4 to 2 times that of the result's own rounding.
// h, dg and du are rounded to bfloat16 where the tensors are, as the operands of one
// matrix instruction a term; second parts would double the work of y, of dx and of the
// weights' gradients, six of the nine products.  So those and the biases' gradients, sums
// of dg and du as they lie, are off by about 1.4 times their own rounding.
#include "direct.hpp"
#include "mm_host.hpp"
#include "thin.hpp"
#include "../../include/d3rlpy_amd.h"

namespace d3a {
namespace {

using namespace mm;

// act(g) and act'(g).  FAST (bfloat16 tensors): the hardware's exponential and
// reciprocal, good to a few 2^-24, where h is rounded by 2^-8 next.
template <bool FAST>
__device__ __forceinline__ void activation(int act, float g, float& a, float& da) {
  if (act == D3A_ACT_RELU) {
    a = fmaxf(g, 0.f);
    if (g != g) a = g;
    da = g > 0.f ? 1.f : 0.f;
  } else if (act == D3A_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    da = cdf + g * (FAST ? __expf(-0.5f * g * g) : expf(-0.5f * g * g)) * 0.3989422804014327f;
  } else {
    const float e = FAST ? __expf(-g) : expf(-g);
    const float s = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  }
}

template <class T, int NP>
struct GatedEpi {
  static constexpr bool kStaged = true;
  static constexpr int kRowBytes = 0;
  float *g, *u;    // kept pre-activations, [batch][M] rows of ld, or null
  __bf16* h;       // planes [NP][batch][M] rows of ld
  int64_t ld, s_part;
  const T *bg, *bu;
  int64_t s_bias;
  int32_t act;

  template <class C>
  __device__ __forceinline__ void run(f32x16 (&acc)[C::MT][C::NT], const Tile& t) const {
    float b[8], c[8];
    load_bias(bg ? bg + t.batch * s_bias : nullptr, first_column<true>(t), t.N, b);
    load_bias(bu ? bu + t.batch * s_bias : nullptr, first_column<true>(t), t.N, c);
    auto none = [](int, int) { return Nothing{}; };
    each8<C, true>(acc, t, none, [&](int m, int n, float* v, float* up, Nothing) {
      if (n >= ld) return;
      float h8[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        v[r] += b[r];
        up[r] += c[r];
        float a, da;
        activation<NP == 1>(act, v[r], a, da);
        h8[r] = n + r < t.N ? a * up[r] : 0.f;
      }
      const int64_t at = ((int64_t)t.batch * t.M + m) * ld + n;
      if (g) {
        store8(g + at, v);
        store8(u + at, up);
      }
      store_planes<NP>(h + at, s_part, h8);
    });
  }
};

template <int NP>
struct GatedBwdEpi {
  static constexpr bool kStaged = true;
  static constexpr int kRowBytes = 0;
  const float *g, *u;
  __bf16 *dg, *du;  // planes, rows of ld
  int64_t ld, s_part;
  int32_t act;

  template <class C>
  __device__ __forceinline__ void run(f32x16 (&acc)[C::MT][C::NT], const Tile& t) const {
    struct Both {
      float g[8], u[8];
    };
    auto load = [&](int m, int n) {
      Both k;
      const int64_t at = ((int64_t)t.batch * t.M + m) * ld + min((int64_t)n, ld - 8);
      load8(g + at, k.g);
      load8(u + at, k.u);
      return k;
    };
    each8<C, false>(acc, t, load, [&](int m, int n, float* v, float*, const Both& k) {
      if (n >= ld) return;
      const int64_t at = ((int64_t)t.batch * t.M + m) * ld + n;
      float g8[8], u8[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float a, da;
        activation<NP == 1>(act, k.g[r], a, da);
        const bool on = n + r < t.N;
        g8[r] = on ? v[r] * k.u[r] * da : 0.f;
        u8[r] = on ? v[r] * a : 0.f;
      }
      store_planes<NP>(dg + at, s_part, g8);
      store_planes<NP>(du + at, s_part, u8);
    });
  }
};

int check(const d3a_gated_mlp_desc* d, bool bwd) {
  D3A_CHECK_ARG(d, "gated_mlp: null descriptor");
  D3A_CHECK_ARG(d->dtype == D3A_F32 || d->dtype == D3A_BF16, "gated_mlp: dtype must be float32 or bfloat16");
  D3A_CHECK_ARG(d->act >= D3A_ACT_SILU && d->act <= D3A_ACT_RELU, "gated_mlp: unknown activation");
  D3A_CHECK_ARG(d->rows >= 0 && d->members >= 1 && d->n_in >= 1 && d->n_hidden >= 1 && d->n_out >= 1,
                "gated_mlp: sizes must be positive");
  D3A_CHECK_ARG(d->rows <= kMaxRows && d->n_in <= kMaxWidth && d->n_hidden <= kMaxWidth &&
                    d->n_out <= kMaxWidth && d->members <= 65535,
                "gated_mlp: size too large");
  D3A_CHECK_ARG(d->ldx >= d->n_in && d->ldWg >= d->n_in && d->ldWu >= d->n_in && d->ldWd >= d->n_hidden,
                "gated_mlp: row stride smaller than the row");
  D3A_CHECK_ARG(d->Wg && d->Wu && d->Wd, "gated_mlp: null weight");
  if (d->rows > 0) D3A_CHECK_ARG(d->x && (bwd ? d->dy != nullptr : d->y != nullptr), "gated_mlp: null operand");
  D3A_CHECK_ARG((reinterpret_cast<uintptr_t>(d->kept) & 15) == 0, "gated_mlp: kept must be 16-byte aligned");
  if (bwd) {
    D3A_CHECK_ARG(d->kept || d->rows == 0, "gated_mlp: the backward needs what the forward kept");
    D3A_CHECK_ARG(d->lddy >= d->n_out, "gated_mlp: row stride smaller than the row");
  }
  return 0;
}

// What the forward keeps: g and u, then h, rows of F8 each; h as the operand
// planes of the tiles, or (is_plain) as an array of T in their place.
template <int NP>
struct Kept {
  float *g = nullptr, *u = nullptr;
  Operand h{};
  explicit Kept(const d3a_gated_mlp_desc& d) {
    const int64_t F8 = round8(d.n_hidden), n = d.members * d.rows * F8;
    h.ld = F8;
    h.s_batch = d.rows * F8;
    h.s_part = n;
    if (!d.kept) return;
    g = static_cast<float*>(d.kept);
    u = g + n;
    h.p = reinterpret_cast<const __bf16*>(u + n);
  }
  static int64_t bytes(const d3a_gated_mlp_desc& d) {
    return d.members * d.rows * round8(d.n_hidden) * (2 * 4 + NP * 2);
  }
};

// ---- a minibatch of a small block: direct.hpp ------------------------------------
// (dg, du and h are plain arrays of T here; h lies where its planes would)
template <class T>
struct DirectGateEpi {
  float *g, *u;
  T* h;
  int64_t ld;
  const T *bg, *bu;
  int32_t act;
  __device__ __forceinline__ void run(int batch, int m, int n, int M, int N, const float v[2], const float up[2]) const {
    if (m >= M) return;
    const int64_t at = ((int64_t)batch * M + m) * ld;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (n + i >= N) continue;
      const float x = v[i] + (bg ? (float)bg[(int64_t)batch * N + n + i] : 0.f);
      const float y = up[i] + (bu ? (float)bu[(int64_t)batch * N + n + i] : 0.f);
      float a, da;
      activation<sizeof(T) == 2>(act, x, a, da);
      if (g) {
        g[at + n + i] = x;
        u[at + n + i] = y;
      }
      h[at + n + i] = (T)(a * y);
    }
  }
};

template <class T>
struct DirectGateBwdEpi {
  const float *g, *u;
  T *dg, *du;
  int64_t ld;
  int32_t act;
  __device__ __forceinline__ void run(int batch, int m, int n, int M, int N, const float v[2], const float*) const {
    if (m >= M) return;
    const int64_t at = ((int64_t)batch * M + m) * ld;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (n + i >= N) continue;
      float a, da;
      activation<sizeof(T) == 2>(act, g[at + n + i], a, da);
      dg[at + n + i] = (T)(v[i] * u[at + n + i] * da);
      du[at + n + i] = (T)(v[i] * a);
    }
  }
};

bool is_direct(const d3a_gated_mlp_desc& d) {
  return direct::small((double)d.members * d.rows * d.n_hidden * std::max(d.n_in, d.n_out),
                       std::max({d.rows, d.n_in, d.n_hidden, d.n_out}));
}

bool is_plain(const d3a_gated_mlp_desc& d) { return d.rows <= thin::kRows || is_direct(d); }

struct Activation {
  __device__ __forceinline__ void operator()(int act, float g, float& a, float& da) const {
    activation<false>(act, g, a, da);
  }
};

// a weight or x whose rows are whole aligned 16-byte pieces
template <class T>
bool whole(const void* p, int64_t ld, int64_t s, int64_t n) {
  constexpr int64_t N = 16 / sizeof(T);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % N == 0 && s % N == 0 && n % N == 0;
}

template <class T, int NP>
int forward_direct(const d3a_gated_mlp_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  const int64_t C = d.members, R = d.rows, D = d.n_in, F = d.n_hidden, O = d.n_out, F8 = round8(F);
  const Kept<NP> k(d);
  T* h = d.kept ? reinterpret_cast<T*>(const_cast<__bf16*>(k.h.p)) : ws.take<T>(C * R * F8);
  *bytes = ws.used;
  if (dry || R == 0) return 0;
  direct::Launch<T, DirectGateEpi<T>> L{};
  L.n = 1;
  L.p[0] = direct::problem(direct::operand<T>(d.x, d.ldx, C > 1 ? d.sx : 0, D),
                           direct::operand<T>(d.Wg, d.ldWg, C > 1 ? d.sWg : 0, D), R, F, D, C);
  L.p[0].b2 = direct::operand<T>(d.Wu, d.ldWu, C > 1 ? d.sWu : 0, D);
  L.e[0] = DirectGateEpi<T>{k.g, k.u, h, F8, static_cast<const T*>(d.bg), static_cast<const T*>(d.bu), d.act};
  if (direct::launch<false, false, true>(L, stream, "gated_mlp") != 0) return -1;
  direct::Launch<T, direct::StoreEpi<T>> Y{};
  Y.n = 1;
  Y.p[0] = direct::problem(direct::operand<T>(h, F8, R * F8, F), direct::operand<T>(d.Wd, d.ldWd, C > 1 ? d.sWd : 0, F),
                           R, O, F, C);
  Y.e[0] = direct::StoreEpi<T>{static_cast<T*>(d.y), O, R * O, static_cast<const T*>(d.bd), O, {}};
  return direct::launch<false, false, false>(Y, stream, "gated_mlp");
}

template <class T, int NP>
int backward_direct(const d3a_gated_mlp_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  const int64_t C = d.members, R = d.rows, D = d.n_in, F = d.n_hidden, O = d.n_out, F8 = round8(F);
  const bool hidden = d.dx || d.dWg || d.dWu || d.dbg || d.dbu;
  const int64_t plane = C * R * F8;
  T* dg = hidden ? ws.take<T>(2 * plane) : nullptr;
  *bytes = ws.used;
  if (dry) return 0;
  T* du = dg + plane;
  const Kept<NP> k(d);
  const int64_t sdy = C > 1 ? d.sdy : 0, sx = C > 1 ? d.sx : 0, sWd = C > 1 ? d.sWd : 0;
  if (hidden && R > 0) {
    direct::Launch<T, DirectGateBwdEpi<T>> L{};
    L.n = 1;
    L.p[0] = direct::problem(direct::operand<T>(d.dy, d.lddy, sdy, O), direct::operand<T>(d.Wd, d.ldWd, sWd, O), R, F,
                             O, C);
    L.e[0] = DirectGateBwdEpi<T>{k.g, k.u, dg, du, F8, d.act};
    if (direct::launch<false, true, false>(L, stream, "gated_mlp_bwd") != 0) return -1;
  }
  if (d.dx && R > 0) {
    const bool shared = C > 1 && d.sx == 0;
    direct::Launch<T, direct::StoreEpi<T>> L{};
    L.n = 1;
    direct::Operand<T> a = direct::operand<T>(dg, F8, R * F8, F);
    direct::Operand<T> b = direct::operand<T>(d.Wg, d.ldWg, C > 1 ? d.sWg : 0, F);
    direct::Operand<T> b2 = direct::operand<T>(d.Wu, d.ldWu, C > 1 ? d.sWu : 0, F);
    a.s_inner = plane;
    if (shared) {
      for (direct::Operand<T>* o : {&a, &b, &b2}) {
        o->s_outer = o->s_batch;
        o->s_batch = 0;
      }
    }
    L.p[0] = direct::problem(a, b, R, D, F, shared ? 1 : C);
    L.p[0].b2 = b2;
    L.p[0].n_inner = 2;
    L.p[0].n_outer = shared ? (int32_t)C : 1;
    L.e[0] = direct::StoreEpi<T>{static_cast<T*>(d.dx), D, R * D, nullptr, 0, {}};
    if (direct::launch<false, true, false>(L, stream, "gated_mlp_bwd") != 0) return -1;
  }
  // the weights' gradients, with the biases' as the sums of their A's rows
  direct::Launch<T, direct::StoreEpi<T>> W{};
  auto weight = [&](const direct::Operand<T>& a, const direct::Operand<T>& b, int64_t M, int64_t N, void* dW,
                    void* db) {
    // (a bias gradient alone: the product of its first column, written nowhere)
    if (!dW && !db) return;
    direct::Problem<T>& p = W.p[W.n];
    p = direct::problem(a, b, M, dW ? N : 1, R, C);
    p.rowsum = static_cast<T*>(db);
    W.e[W.n] = direct::StoreEpi<T>{static_cast<T*>(dW), N, M * N, nullptr, 0, {}};
    ++W.n;
  };
  const direct::Operand<T> x = direct::operand<T>(d.x, d.ldx, sx, R);
  weight(direct::operand<T>(dg, F8, R * F8, R), x, F, D, d.dWg, d.dbg);
  weight(direct::operand<T>(du, F8, R * F8, R), x, F, D, d.dWu, d.dbu);
  weight(direct::operand<T>(d.dy, d.lddy, sdy, R),
         direct::operand<T>(reinterpret_cast<const T*>(k.h.p), F8, R * F8, R), O, F, d.dWd, d.dbd);
  return W.n ? direct::launch<true, true, false>(W, stream, "gated_mlp_bwd") : 0;
}

// At most 16 rows: the weights read once.  One row of 2048 x 5632 bfloat16: 13.7
// to 15 us and 8.2 (3.1 to 3.4 and 2.8 TB/s; four rows of 4096 x 11008 35 and 18.5, 5
// TB/s), where the tiles take 20.6 and 14.6.  The short ones do not fill the chip: 352
// and 128 workgroups, one and a half rounds of 256 CUs and half of one.
template <class T, int NP>
int forward_thin(const d3a_gated_mlp_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  const int64_t C = d.members, R = d.rows, D = d.n_in, F = d.n_hidden, O = d.n_out, F8 = round8(F);
  const Kept<NP> k(d);
  T* h = d.kept ? reinterpret_cast<T*>(const_cast<__bf16*>(k.h.p)) : ws.take<T>(C * R * F8);
  const bool two = NP == 1 && R <= 8;
  T* lo = two ? ws.take<T>(C * R * F8) : nullptr;
  *bytes = ws.used;
  if (dry || R == 0) return 0;
  thin::GateArgs<T> a{};
  a.x = static_cast<const T*>(d.x);
  a.Wg = static_cast<const T*>(d.Wg);
  a.Wu = static_cast<const T*>(d.Wu);
  a.bg = static_cast<const T*>(d.bg);
  a.bu = static_cast<const T*>(d.bu);
  a.ldx = d.ldx;
  a.sx = C > 1 ? d.sx : 0;
  a.ldg = d.ldWg;
  a.sg = C > 1 ? d.sWg : 0;
  a.ldu = d.ldWu;
  a.su = C > 1 ? d.sWu : 0;
  a.g = k.g;
  a.u = k.u;
  a.h = h;
  a.lo = lo;
  a.ld = F8;
  a.R = (int32_t)R;
  a.D = (int32_t)D;
  a.F = (int32_t)F;
  a.act = d.act;
  const dim3 gate((unsigned)((F + 15) / 16), (unsigned)C), down((unsigned)((O + 15) / 16), (unsigned)C);
  if (whole<T>(d.x, a.ldx, a.sx, D) && whole<T>(d.Wg, a.ldg, a.sg, D) && whole<T>(d.Wu, a.ldu, a.su, D))
    thin::gate_kernel<T, true><<<gate, 512, 0, stream>>>(a, Activation{});
  else
    thin::gate_kernel<T, false><<<gate, 512, 0, stream>>>(a, Activation{});
  D3A_LAUNCH_CHECK("gated_mlp");
  thin::DownArgs<T> b{};
  b.h = h;
  b.lo = lo;
  b.W = static_cast<const T*>(d.Wd);
  b.b = static_cast<const T*>(d.bd);
  b.y = static_cast<T*>(d.y);
  b.ld = F8;
  b.ldw = d.ldWd;
  b.sw = C > 1 ? d.sWd : 0;
  b.R = (int32_t)R;
  b.F = (int32_t)F;
  b.O = (int32_t)O;
  const bool vec = whole<T>(d.Wd, b.ldw, b.sw, F);
  if (!two) {
    if (vec) thin::down_kernel<T, true, 1><<<down, 1024, 0, stream>>>(b);
    else thin::down_kernel<T, false, 1><<<down, 1024, 0, stream>>>(b);
  } else if constexpr (NP == 1) {
    if (vec) thin::down_kernel<T, true, 2><<<down, 1024, 0, stream>>>(b);
    else thin::down_kernel<T, false, 2><<<down, 1024, 0, stream>>>(b);
  }
  D3A_LAUNCH_CHECK("gated_mlp");
  return 0;
}

// run (stream given) or measure (ws null): the same walk over the workspace
template <class T, int NP>
int forward(const d3a_gated_mlp_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  if (d.rows <= thin::kRows) return forward_thin<T, NP>(d, ws, dry, stream, bytes);
  if (is_direct(d)) return forward_direct<T, NP>(d, ws, dry, stream, bytes);
  const int64_t C = d.members, R = d.rows, D = d.n_in, F = d.n_hidden, O = d.n_out, F8 = round8(F);
  Packer<T, NP> pack(ws);
  const Operand x = pack.operand(d.x, d.ldx, C > 1 ? d.sx : 0, C, R, D);
  const bool apart = d.ldWg != d.ldWu || (C > 1 && d.sWg != d.sWu) ||
                     (reinterpret_cast<uintptr_t>(d.Wg) & 15) || (reinterpret_cast<uintptr_t>(d.Wu) & 15);
  const Operand wg = pack.operand(d.Wg, d.ldWg, C > 1 ? d.sWg : 0, C, F, D, apart);
  const Operand wu = pack.operand(d.Wu, d.ldWu, C > 1 ? d.sWu : 0, C, F, D, apart);
  const Operand wd = pack.operand(d.Wd, d.ldWd, C > 1 ? d.sWd : 0, C, O, F);
  const Kept<NP> k(d);
  Operand h = k.h;
  if (!d.kept) h.p = ws.take<__bf16>(NP * C * R * F8);

  Launch<GatedEpi<T, NP>> L{};
  L.n = 1;
  Problem& p = L.p[0];
  p.a = x;
  p.b = wg;
  p.b2 = wu.p;
  p.M = (int32_t)R;
  p.N = (int32_t)F;
  p.K = (int32_t)D;
  p.batch = (int32_t)C;
  p.n_outer = p.n_inner = p.splits = 1;
  GatedEpi<T, NP>& e = L.e[0];
  e.g = k.g;
  e.u = k.u;
  e.h = const_cast<__bf16*>(h.p);
  e.ld = F8;
  e.s_part = h.s_part;
  e.bg = static_cast<const T*>(d.bg);
  e.bu = static_cast<const T*>(d.bu);
  e.s_bias = F;
  e.act = d.act;

  Products<T, NP> down;
  down.add(h, wd, R, O, F, C, 1, 1, d.y, O, R * O, d.bd, O);
  down.reserve(ws, true);
  *bytes = ws.used;
  if (dry) return 0;
  if (pack.launch(stream) != 0) return -1;
  if (run<NP, false, false, true>(L, choose<NP>(L, true).size, stream, "gated_mlp") != 0) return -1;
  return down.template launch<false, false>(stream, "gated_mlp");
}

template <class T, int NP>
int backward(const d3a_gated_mlp_desc& d, Arena ws, bool dry, hipStream_t stream, int64_t* bytes) {
  if (is_direct(d)) return backward_direct<T, NP>(d, ws, dry, stream, bytes);
  const int64_t C = d.members, R = d.rows, D = d.n_in, F = d.n_hidden, O = d.n_out, F8 = round8(F);
  const bool hidden = d.dx || d.dWg || d.dWu || d.dbg || d.dbu;  // dg and du are needed
  Packer<T, NP> pack(ws);
  Operand dy{}, x{}, wd{}, wg{}, wu{};
  if (hidden || d.dWd || d.dbd) dy = pack.operand(d.dy, d.lddy, C > 1 ? d.sdy : 0, C, R, O);
  if (hidden) {
    wd = pack.operand(d.Wd, d.ldWd, C > 1 ? d.sWd : 0, C, O, F);
  }
  if (d.dWg || d.dWu) x = pack.operand(d.x, d.ldx, C > 1 ? d.sx : 0, C, R, D);
  if (d.dx) {
    const bool apart = d.ldWg != d.ldWu || (C > 1 && d.sWg != d.sWu) ||
                       (reinterpret_cast<uintptr_t>(d.Wg) & 15) || (reinterpret_cast<uintptr_t>(d.Wu) & 15);
    wg = pack.operand(d.Wg, d.ldWg, C > 1 ? d.sWg : 0, C, F, D, apart);
    wu = pack.operand(d.Wu, d.ldWu, C > 1 ? d.sWu : 0, C, F, D, apart);
  }
  const int64_t plane = C * R * F8;
  Operand dg{};
  dg.p = hidden ? ws.take<__bf16>(2 * NP * plane) : nullptr;  // dg, du
  dg.ld = F8;
  dg.s_batch = R * F8;
  dg.s_part = plane;
  Operand du = dg;
  du.p += NP * plane;
  const Kept<NP> k(d);

  Launch<GatedBwdEpi<NP>> L{};
  L.n = 1;
  Problem& p = L.p[0];
  p.a = dy;
  p.b = wd;
  p.M = (int32_t)R;
  p.N = (int32_t)F;
  p.K = (int32_t)O;
  p.batch = (int32_t)C;
  p.n_outer = p.n_inner = p.splits = 1;
  GatedBwdEpi<NP>& e = L.e[0];
  e.g = k.g;
  e.u = k.u;
  e.dg = const_cast<__bf16*>(dg.p);
  e.du = const_cast<__bf16*>(du.p);
  e.ld = F8;
  e.s_part = plane;
  e.act = d.act;

  Operand h = k.h;
  if (NP > 1 && is_plain(d) && d.dWd) h = pack.operand(k.h.p, F8, C > 1 ? R * F8 : 0, C, R, F);
  Products<T, NP> dx, dw;
  if (d.dx) {
    // K runs over the gate's and the up's hidden units (and, for an x that the
    // members share, over the members)
    Operand a = dg, b = wg;
    a.s_inner = du.p - dg.p;
    b.s_inner = reinterpret_cast<const __bf16*>(wu.p) - wg.p;
    const bool shared = C > 1 && d.sx == 0;
    if (shared) {
      a.s_outer = a.s_batch;
      b.s_outer = b.s_batch;
      a.s_batch = b.s_batch = 0;
    }
    dx.add(a, b, R, D, F, shared ? 1 : C, shared ? C : 1, 2, d.dx, D, shared ? 0 : R * D, nullptr, 0);
    dx.reserve(ws, true);
  }
  if (d.dWg) dw.add(dg, x, F, D, R, C, 1, 1, d.dWg, D, F * D, nullptr, 0);
  if (d.dWu) dw.add(du, x, F, D, R, C, 1, 1, d.dWu, D, F * D, nullptr, 0);
  if (d.dWd) dw.add(dy, h, O, F, R, C, 1, 1, d.dWd, F, O * F, nullptr, 0);
  dw.reserve(ws, true);
  Colsum<T, NP> cs;
  if (d.dbg) cs.add(dg, R, F, C, d.dbg);
  if (d.dbu) cs.add(du, R, F, C, d.dbu);
  if (d.dbd) cs.add(dy, R, O, C, d.dbd);
  cs.reserve(ws);
  *bytes = ws.used;
  if (dry) return 0;
  if (R > 0 && pack.launch(stream) != 0) return -1;
  if (hidden && R > 0) {
    if (run<NP, false, true, false>(L, choose<NP>(L, false).size, stream, "gated_mlp_bwd") != 0) return -1;
    if (dx.template launch<false, true>(stream, "gated_mlp_bwd") != 0) return -1;
  }
  if (dw.template launch<true, true>(stream, "gated_mlp_bwd") != 0) return -1;
  return cs.launch(stream);
}

int call(const d3a_gated_mlp_desc* d, bool bwd, bool dry, hipStream_t stream, int64_t* bytes) {
  Arena ws{dry ? nullptr : static_cast<char*>(d->ws)};
  if (d->dtype == D3A_F32)
    return bwd ? backward<float, 3>(*d, ws, dry, stream, bytes) : forward<float, 3>(*d, ws, dry, stream, bytes);
  return bwd ? backward<__bf16, 1>(*d, ws, dry, stream, bytes) : forward<__bf16, 1>(*d, ws, dry, stream, bytes);
}

int entry(const d3a_gated_mlp_desc* d, bool bwd, void* stream) {
  if (check(d, bwd) != 0) return -1;
  int64_t need = 0;
  if (call(d, bwd, true, nullptr, &need) != 0) return -1;
  D3A_CHECK_ARG(need == 0 || (d->ws && d->ws_bytes >= need && (reinterpret_cast<uintptr_t>(d->ws) & 255) == 0),
                "gated_mlp: workspace of %lld bytes (256-byte aligned) needed", (long long)need);
  return call(d, bwd, false, static_cast<hipStream_t>(stream), &need);
}

}  // namespace
}  // namespace d3a

extern "C" {

int d3a_gated_mlp_workspace(const d3a_gated_mlp_desc* d, int32_t backward, int64_t* bytes) {
  if (d3a::check(d, backward != 0) != 0) return -1;
  D3A_CHECK_ARG(bytes, "gated_mlp: null size");
  return d3a::call(d, backward != 0, true, nullptr, bytes);
}

int d3a_gated_mlp_kept(const d3a_gated_mlp_desc* d, int64_t* bytes) {
  D3A_CHECK_ARG(d && bytes, "gated_mlp: null descriptor or size");
  *bytes = d->dtype == D3A_F32 ? d3a::Kept<3>::bytes(*d) : d3a::Kept<1>::bytes(*d);
  return 0;
}

int d3a_gated_mlp(const d3a_gated_mlp_desc* d, void* stream) { return d3a::entry(d, false, stream); }

int d3a_gated_mlp_bwd(const d3a_gated_mlp_desc* d, void* stream) { return d3a::entry(d, true, stream); }

}  // extern "C"
