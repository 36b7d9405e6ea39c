// The gated feed-forward block up to its down projection, and its backward pass:
//
//   g = x Wg^T, u = x Wu^T, h = silu(g) u                               x [M, C], Wg, Wu [I, C], h [M, I]
//   dg = dh u s (1 + g (1 - s)), du = dh g s, s = 1 / (1 + exp(-g))
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Forward: one product whose column tiles interleave 16 rows of Wg with 16 of Wu, so that a lane holds g and
// u of the same elements and only h is written.
//
// Backward: the forward keeps nothing but x.  The first launch makes g and u again (4 M C I operations, which
// cost about what writing and reading the two would at C <= 1000 or so) and its epilogue turns them with dh
// into [dg | du], rounded once to 16 bits as an operand of the next products: kept in fp32 to here, so the
// gradients carry that one rounding and their own.  The second launch is dx over k = [dg | du]'s columns with
// both weights read along their columns, the third [dWg; dWu] = [dg | du]^T x, summed over token ranges into
// fp32 partials that a last launch adds in order (the same bits every time).
//
// In fp16 [dg | du] is held times a power of two, from the bounds |dg|, |du| <= 1.1 |dh| max(|g|, |u|) and
// |g|, |u| <= |x| |w|, norms of rows: two launches before the first (Magnitudes).
#include <algorithm>

#include "ffn_common.h"
#include "ffn_skinny.h"

namespace maba {
namespace ffn {

// A wave's 32 columns of a tile are 16 of g and the same 16 of u; the epilogues take four such blocks at once.
struct EpiGated {
  static constexpr bool LONG = false, GROUPS = false;
  struct Args { Rows h; int M, I; };
  static __device__ __forceinline__ f32x4 gated(f32x4 g, f32x4 u) {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = g[r] * sigmoid(g[r]) * u[r];
    return v;
  }
  template <class T>
  static __device__ __forceinline__ void quad(const Args& e, int64_t m, int n, f32x4 g, f32x4 u) {
    store4<T>(e.h, m, n, e.I, gated(g, u));
  }
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + 16 * i + c;
      if constexpr (NI % 4 == 0) {
#pragma unroll
        for (int j = 0; j < NI; j += 4)
          store8(e.h, m, n0 / 2 + 8 * j + 8 * q, e.M, e.I,
                 eight_of({down4<T>(gated(acc[i][j], acc[i][j + 1])), down4<T>(gated(acc[i][j + 2], acc[i][j + 3]))}));
      } else {
#pragma unroll
        for (int j = 0; j < NI; j += 2) {
          const int n = n0 / 2 + 8 * j + 4 * q;
          if (m < e.M && n < e.I) quad<T>(e, m, n, acc[i][j], acc[i][j + 1]);
        }
      }
    }
  }
};

// d [M, 2 Iw], Iw = I rounded up to 16: dg at column 0, du at column Iw, zeros behind each.
struct EpiGatedBack {
  static constexpr bool LONG = false, GROUPS = false;
  struct Args { Rows dh, d; int M, I, Iw; const int* exponent; };
  static __device__ __forceinline__ void grads(f32x4 g, f32x4 u, f32x4 dh, f32x4& dg, f32x4& du) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float s = sigmoid(g[r]), a = dh[r] * s;
      du[r] = a * g[r];
      dg[r] = a * u[r] * (1.f + g[r] * (1.f - s));
    }
  }
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
    const float scale = power_of<T>(e.exponent, 1);
    if constexpr (NI % 4 == 0) {
      u32x4 dh[MI][NI / 4];      // all of dh first: the loads are in flight together
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI / 4; ++j) dh[i][j] = load8(e.dh, m0 + 16 * i + c, n0 / 2 + 32 * j + 8 * q, e.M, e.I);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = m0 + 16 * i + c;
#pragma unroll
        for (int j = 0; j < NI / 4; ++j) {
          const int n = n0 / 2 + 32 * j + 8 * q;
          const Quads d = quads_of(dh[i][j]);
          f32x4 dg[2], du[2];
          grads(acc[i][4 * j], acc[i][4 * j + 1], up4<T>(d.a) * scale, dg[0], du[0]);
          grads(acc[i][4 * j + 2], acc[i][4 * j + 3], up4<T>(d.b) * scale, dg[1], du[1]);
          store8(e.d, m, n, e.M, e.Iw, eight_of({down4<T>(dg[0]), down4<T>(dg[1])}));
          // columns behind Iw would be du's neighbours: none is stored there
          const u32x4 u = eight_of({down4<T>(du[0]), down4<T>(du[1])});
          if (n < e.Iw) store8(e.d, m, e.Iw + n, e.M, 2 * e.Iw, u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = m0 + 16 * i + c;
#pragma unroll
        for (int j = 0; j < NI; j += 2) {
          const int n = n0 / 2 + 8 * j + 4 * q;
          if (m >= e.M || n >= e.Iw) continue;
          f32x4 dg, du;
          grads(acc[i][j], acc[i][j + 1], up4<T>(load4(e.dh, m, n, e.I)) * scale, dg, du);
          store4<T>(e.d, m, n, e.Iw, dg);
          store4<T>(e.d, m, e.Iw + n, 2 * e.Iw, du);
        }
      }
    }
  }
};

// The forward's sum split over few rows' long k: h from the partial products' sums [splits][M][2 Iw], in split order.
template <class T>
__global__ __launch_bounds__(256) void reduce_gated_forward(const float* p, int splits, int64_t plane, int Iw, EpiGated::Args e) {
  const int quads = Iw / 4;
  const int64_t total = (int64_t)e.M * quads;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    if (n >= e.I) continue;
    const float* at = p + (int64_t)m * 2 * Iw + 2 * (n & ~15) + (n & 15);
    f32x4 g = {0.f, 0.f, 0.f, 0.f}, u = g;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      g += *(const f32x4*)(at + s * plane);
      u += *(const f32x4*)(at + s * plane + 16);
    }
    EpiGated::quad<T>(e, m, n, g, u);
  }
}

// Where everything of a call lies: operands in place or copied into the workspace.
struct GatedPlan {
  int64_t M, C, I, Cp, Iw;       // widths padded to 8 (C) and to 16 (I, a half of [dg | du])
  bool copy_x, copy_w[2];
  uint16_t *x, *w[2], *d;
  float* part;             // fp32 partials, of dx and then of the weights
  float* magnitudes;       // and the power of two of d, in fp16
  int* exponent;
  GemmPlan gu, dx, dw;     // the products with both weights, for dx and for the weights' gradients
  size_t bytes;
};

static GatedPlan gated_plan(const maba_tensor* x, const maba_tensor* scales, const maba_tensor* wg, const maba_tensor* wu,
                            bool back, bool dx, bool dw, void* ws) {
  GatedPlan p = {};
  p.M = x->shape[0];
  p.C = x->shape[1];
  p.I = wg->shape[0];
  p.Cp = pad8(p.C);
  p.Iw = ceil_div(p.I, 16) * 16;
  const bool few = !back && few_rows(p.M, p.C);       // that kernel reads any rows
  const auto in_place = back ? aligned_columns : aligned_rows;
  p.copy_x = !few && (scales || !in_place(x));
  p.copy_w[0] = !few && !in_place(wg);
  p.copy_w[1] = !few && !in_place(wu);
  // dx reads both weights with one stride: each in place at the same stride, or both copied
  if (back && (p.copy_w[0] || p.copy_w[1] || wg->stride[0] != wu->stride[0])) p.copy_w[0] = p.copy_w[1] = true;
  Carve c = {(char*)ws, 0};
  if (p.copy_x) p.x = c.take<uint16_t>(p.M * p.Cp);
  for (int i = 0; i < 2; ++i)
    if (p.copy_w[i]) p.w[i] = c.take<uint16_t>(p.I * p.Cp);
  if (back) {
    p.d = c.take<uint16_t>(p.M * 2 * p.Iw);
    int64_t part = 0;
    if (dx) {
      p.dx = gemm_plan(p.M, p.Cp, gemm_stages(p.Iw, 2), PLAN_COLUMNS | PLAN_SPLIT | PLAN_GROUPS);
      if (p.dx.splits > 1) part = (int64_t)p.dx.splits * p.M * p.Cp;
    }
    if (dw) {
      p.dw = gemm_plan(2 * p.Iw, p.Cp, gemm_stages(p.M, 1), PLAN_COLUMNS | PLAN_SPLIT);
      part = std::max(part, (int64_t)p.dw.splits * 2 * p.Iw * p.Cp);
    }
    p.part = c.take<float>(part);
    if (wg->dtype == MABA_F16) {
      p.magnitudes = c.take<float>(MAX_FACTORS * MAGNITUDE_GROUPS);
      p.exponent = c.take<int>(1);
    }
  }
  p.gu = gemm_plan(p.M, 2 * p.Iw, gemm_stages(p.Cp, 1), PLAN_PAIRS | (back || few ? 0 : PLAN_SPLIT));
  if (p.gu.splits > 1) p.part = c.take<float>((int64_t)p.gu.splits * p.M * 2 * p.Iw);
  p.bytes = c.used;
  return p;
}

// The operands of x W^T with both weights, after any copies.
static int gated_operands(GatedPlan& p, const maba_tensor* x, const maba_tensor* scales, const maba_tensor* wg,
                          const maba_tensor* wu, hipStream_t s, Operand& ox, Operand& ow) {
  const maba_tensor* w[2] = {wg, wu};
  Copies copies;
  if (p.copy_x) copies.add(x, scales, p.x);
  ox = p.copy_x ? rows_operand(p.x, p.Cp, p.M) : rows_operand((const uint16_t*)x->data, x->stride[0], p.M);
  ow = {};
  ow.rows = (int)p.I;
  for (int i = 0; i < 2; ++i) {
    if (p.copy_w[i]) copies.add(w[i], nullptr, p.w[i]);
    ow.p[i] = p.copy_w[i] ? p.w[i] : (const uint16_t*)w[i]->data;
    ow.ld[i] = p.copy_w[i] ? p.Cp : w[i]->stride[0];
  }
  return copies.launch(wg->dtype, s);
}

template <class T>
static int gated_forward(GatedPlan& p, const maba_tensor* x, const maba_tensor* wg, const maba_tensor* wu, maba_tensor* out,
                         hipStream_t s, const char* who) {
  const EpiGated::Args e = {rows_of(out), (int)p.M, (int)p.I};
  if (few_rows(p.M, p.C)) {
    SkinnyArgs a = {(const uint16_t*)x->data, x->stride[0], {(const uint16_t*)wg->data, (const uint16_t*)wu->data},
                    {wg->stride[0], wu->stride[0]}, (int)p.M, (int)p.I, (int)p.C, aligned_rows(x),
                    aligned_rows(wg) && aligned_rows(wu)};
    return skinny<T, true, EpiGated>(a, e, s, who);
  }
  GemmArgs g = {};
  if (int rc = gated_operands(p, x, nullptr, wg, wu, s, g.a, g.b)) return rc;
  g.K = p.Cp;
  if (p.gu.splits == 1) return gemm<T, K_ROWS, K_ROWS_PAIR, EpiGated>(g, e, p.M, 2 * p.Iw, p.gu, s, who);
  const EpiPartial::Args ep = {p.part, (int)p.M, (int)(2 * p.Iw)};
  if (int rc = gemm<T, K_ROWS, K_ROWS_PAIR, EpiPartial>(g, ep, p.M, 2 * p.Iw, p.gu, s, who)) return rc;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(p.M * (p.Iw / 4), 256), 16384));
  hipLaunchKernelGGL(reduce_gated_forward<T>, grid, dim3(256), 0, s, p.part, p.gu.splits, p.M * 2 * p.Iw, (int)p.Iw, e);
  return check_launch(who);
}

template <class T>
static int gated_backward(GatedPlan& p, const maba_tensor* dh, const maba_tensor* x, const maba_tensor* scales,
                          const maba_tensor* wg, const maba_tensor* wu, maba_tensor* dx, maba_tensor* dwg, maba_tensor* dwu,
                          hipStream_t s, const char* who) {
  Operand ox, ow;
  if (int rc = gated_operands(p, x, scales, wg, wu, s, ox, ow)) return rc;
  const Operand d = rows_operand(p.d, 2 * p.Iw, p.M);
  if (p.M > 0) {
    if (T::SCALED) {
      Magnitudes m;
      m.add(0, dh->data, dh->stride[0], p.M, p.I, false);
      m.add(1, ox.p[0], ox.ld[0], p.M, p.C, true);
      for (int i = 0; i < 2; ++i) m.add(2, ow.p[i], ow.ld[i], p.I, p.C, true);
      if (int rc = m.launch(1.1f, p.magnitudes, p.exponent, s)) return rc;
    }
    GemmArgs g = {};
    g.a = ox;
    g.b = ow;
    g.K = p.Cp;
    const Rows rd = {p.d, 2 * p.Iw};
    const EpiGatedBack::Args e = {rows_of(dh), rd, (int)p.M, (int)p.I, (int)p.Iw, p.exponent};
    if (int rc = gemm<T, K_ROWS, K_ROWS_PAIR, EpiGatedBack>(g, e, p.M, 2 * p.Iw, p.gu, s, who)) return rc;
  }
  if (dx && p.M > 0) {
    GemmArgs g = {};
    g.a = d;
    g.b = cols_operand(ow, p.Cp);
    g.K = p.Iw;
    g.segments = 2;
    const Outputs o = {{rows_of(dx), rows_of(nullptr)}, INT32_MAX, (int)p.M, (int)p.C, p.exponent};
    if (int rc = product_to<T, K_ROWS, K_COLS>(g, o, p.M, p.Cp, p.dx, p.part, s, who)) return rc;
  }
  if (dwg || dwu) {
    const Outputs o = {{rows_of(dwg), rows_of(dwu)}, (int)p.Iw, (int)p.I, (int)p.C, p.exponent};
    if (p.M == 0) return zeros_to<T>(o, 2 * p.Iw, p.Cp, s);
    GemmArgs g = {};
    g.a = cols_operand(d, 2 * p.Iw);
    g.b = cols_operand(ox, p.Cp);
    g.K = p.M;
    if (int rc = product_to<T, K_COLS, K_COLS>(g, o, 2 * p.Iw, p.Cp, p.dw, p.part, s, who)) return rc;
  }
  return MABA_OK;
}

static int gated_check(const maba_tensor* x, const maba_tensor* scales, const maba_tensor* wg, const maba_tensor* wu,
                       const char* who) {
  if (!x || !wg || !wu) return fail(MABA_ERR_INVALID, "%s: x, w_gate and w_up required", who);
  if (wg->dtype != MABA_BF16 && wg->dtype != MABA_F16)
    return fail(wg->dtype == MABA_F32 ? MABA_ERR_UNSUPPORTED : MABA_ERR_DTYPE, "%s: 16-bit weights only, got dtype code %d", who, wg->dtype);
  if (x->ndim != 2 || wg->ndim != 2) return fail(MABA_ERR_INVALID, "%s: x and the weights must be 2D", who);
  int rc = check_sizes(who, x->shape[0], wg->shape[0], x->shape[1]);
  if (!rc) rc = check_kept(x, scales, who, wg->dtype, -1, x->shape[1]);
  if (!rc) rc = check_rows(wg, who, "w_gate", wg->dtype, -1, x->shape[1]);
  if (!rc) rc = check_rows(wu, who, "w_up", wg->dtype, wg->shape[0], x->shape[1]);
  if (!rc && scales && scales->shape[0] != x->shape[0]) rc = fail(MABA_ERR_INVALID, "%s: scales do not match the codes", who);
  return rc;
}

}  // namespace ffn
}  // namespace maba

using namespace maba;
using namespace maba::ffn;

extern "C" size_t maba_hip_gated_ffn_workspace_size(const maba_tensor* x, const maba_tensor* w_gate, const maba_tensor* w_up) {
  if (gated_check(x, nullptr, w_gate, w_up, "gated_ffn")) return 0;
  return gated_plan(x, nullptr, w_gate, w_up, false, false, false, nullptr).bytes;
}

extern "C" int maba_hip_gated_ffn(const maba_tensor* x, const maba_tensor* w_gate, const maba_tensor* w_up, maba_tensor* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "gated_ffn";
  int rc = gated_check(x, nullptr, w_gate, w_up, who);
  if (!rc) rc = check_out(out, who, "out", w_gate->dtype, x->shape[0], w_gate->shape[0]);
  if (rc) return rc;
  if (overlap(out, x) || overlap(out, w_gate) || overlap(out, w_up)) return fail(MABA_ERR_INVALID, "%s: out overlaps an input", who);
  GatedPlan p = gated_plan(x, nullptr, w_gate, w_up, false, false, false, workspace);
  if ((rc = check_workspace(who, workspace, workspace_bytes, p.bytes))) return rc;
  if (p.M == 0) return MABA_OK;
  return w_gate->dtype == MABA_BF16 ? gated_forward<Bf16>(p, x, w_gate, w_up, out, (hipStream_t)stream, who)
                                    : gated_forward<Fp16>(p, x, w_gate, w_up, out, (hipStream_t)stream, who);
}

extern "C" size_t maba_hip_gated_ffn_backward_workspace_size(const maba_tensor* x, const maba_tensor* x_scales,
                                                             const maba_tensor* w_gate, const maba_tensor* w_up, int needs) {
  if (gated_check(x, x_scales, w_gate, w_up, "gated_ffn_backward")) return 0;
  return gated_plan(x, x_scales, w_gate, w_up, true, needs & 1, needs & 2, nullptr).bytes;
}

extern "C" int maba_hip_gated_ffn_backward(const maba_tensor* dh, const maba_tensor* x, const maba_tensor* x_scales,
                                           const maba_tensor* w_gate, const maba_tensor* w_up, maba_tensor* dx,
                                           maba_tensor* dw_gate, maba_tensor* dw_up, void* workspace, size_t workspace_bytes,
                                           void* stream) {
  const char* who = "gated_ffn_backward";
  int rc = gated_check(x, x_scales, w_gate, w_up, who);
  if (rc) return rc;
  const int dt = w_gate->dtype;
  const int64_t M = x->shape[0], C = x->shape[1], I = w_gate->shape[0];
  rc = check_rows(dh, who, "dh", dt, M, I);
  if (!rc && dx) rc = check_out(dx, who, "dx", dt, M, C);
  if (!rc && dw_gate) rc = check_out(dw_gate, who, "dw_gate", dt, I, C);
  if (!rc && dw_up) rc = check_out(dw_up, who, "dw_up", dt, I, C);
  if (rc) return rc;
  const maba_tensor *outs[3] = {dx, dw_gate, dw_up}, *ins[5] = {dh, x, x_scales, w_gate, w_up};
  for (int i = 0; i < 3; ++i) {
    for (int j = 0; j < 5; ++j)
      if (overlap(outs[i], ins[j])) return fail(MABA_ERR_INVALID, "%s: a gradient overlaps an input", who);
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return fail(MABA_ERR_INVALID, "%s: two gradients overlap", who);
  }
  GatedPlan p = gated_plan(x, x_scales, w_gate, w_up, true, dx != nullptr, dw_gate || dw_up, workspace);
  if ((rc = check_workspace(who, workspace, workspace_bytes, p.bytes))) return rc;
  return dt == MABA_BF16 ? gated_backward<Bf16>(p, dh, x, x_scales, w_gate, w_up, dx, dw_gate, dw_up, (hipStream_t)stream, who)
                         : gated_backward<Fp16>(p, dh, x, x_scales, w_gate, w_up, dx, dw_gate, dw_up, (hipStream_t)stream, who);
}
