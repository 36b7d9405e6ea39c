// A linear layer with its epilogue, and its backward pass:
//
//   z = x W^T + b,  y = r + gate * act(z)           x [M, K], W [N, K], b, gate [N], r, y [M, N]
//   dz = dy * gate * act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz,  dgate = sum_m dy * act(z),  dr = dy
//
// act is none, relu, silu or gelu (with the error function); b, r and gate are each optional.  The epilogue works
// on the fp32 accumulators and y is rounded once.
//
// Backward with an activation: one launch makes z again from x and its epilogue writes dz, rounded
// once to 16 bits as the next products' operand, and the column sums of a tile's rows (fp32, before that
// rounding) for db and dgate, which a later launch adds in order.  Then dx = dz W reads W along its columns, and
// dW = dz^T x both operands, summed over token ranges into fp32 partials added in order.
//
// Without an activation z is not needed.  dz = dy * gate, so with G = dy^T x (the fp32 partials)
//   dx = dy (diag(gate) W),  dW = diag(gate) G,  dgate = rowdot(W, G) + b * colsum(dy),  db = gate * colsum(dy):
// the gate goes onto the N x K weight (one rounding, as dz would have) and into the reduction, not onto the M x N
// gradient (the down projection of 16,384 tokens: 48 us of 205).
//
// In fp16 dz and gate * W are held times a power of two, from the bounds |dz| <= 1.13 |dy| |gate| and |gate| |W| (two
// launches; Magnitudes).
#include <algorithm>

#include "ffn_common.h"
#include "ffn_skinny.h"

namespace maba {
namespace ffn {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// The normal distribution function: for z < 0, Phi(z) = e^(-z^2/2) t P(t) with t = 1 / (1 + 0.35 |z|), where P is the
// least-error fit of degree six to erfcx(|z| / sqrt 2) / 2t made for this (a linear program over 500 points): within
// 2.0e-7 of Phi in fp32 everywhere, and but for the exponential's own rounding within 1e-5 of Phi relative to it for
// z >= -13 (below, e^(-z^2/2) leaves fp32's normal range and only the first bound holds).  Both signs take one path, and the
// exponential is the density's too: 16 operations where the library's erff alone has both its branches (16,384 x 2,496
// gelus, forward: 129 us with it, of which 45 were erff).
__device__ __forceinline__ float normal(float z, float& e) {
  const float a = fabsf(z), t = fast_rcp(fmaf(0.35f, a, 1.f));
  e = fast_exp(-0.5f * z * z);
  float p = 0.043667048f;
  p = fmaf(p, t, -0.18067843f);
  p = fmaf(p, t, 0.20517235f);
  p = fmaf(p, t, 0.013616925f);
  p = fmaf(p, t, 0.14121465f);
  p = fmaf(p, t, 0.13726018f);
  p = fmaf(p, t, 0.13974728f);
  p *= t * e;
  return z < 0.f ? p : 1.f - p;
}

template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? z : z != z ? z : 0.f;
  else if constexpr (ACT == ACT_SILU) return z * sigmoid(z);
  else if constexpr (ACT == ACT_GELU) {
    float e;
    return z * normal(z, e);
  }
  else return z;
}
template <int ACT>
__device__ __forceinline__ float dact_of(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return s * (1.f + z * (1.f - s));
  } else if constexpr (ACT == ACT_GELU) {
    float e;
    const float phi = normal(z, e);
    return phi + z * 0.39894228f * e;
  } else return 1.f;
}

// The quads at n of a vector [N], or of a constant in its place.
template <class T>
__device__ __forceinline__ f32x4 vec4(const uint16_t* p, float other, int n, int nend) {
  if (!p) return f32x4{other, other, other, other};
  return up4<T>(load4(Rows{(uint16_t*)p, 0}, 0, n, nend));
}

// What an epilogue reads for 32 columns of a wave: a row tensor's eights (zeros without one) and the quads of bias and
// gate.
template <int MI>
struct Reads {
  u32x4 rows[MI];
  u32x2 bias[2], gate[2];
  template <class Args>
  __device__ __forceinline__ void load(const Rows& r, const Args& e, int m0, int n, int c, int q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bias[h] = e.bias ? load4(Rows{(uint16_t*)e.bias, 0}, 0, n + 16 * h + 4 * q, e.N) : u32x2{0, 0};
      gate[h] = e.gate ? load4(Rows{(uint16_t*)e.gate, 0}, 0, n + 16 * h + 4 * q, e.N) : u32x2{0, 0};
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) rows[i] = r.p ? load8(r, m0 + 16 * i + c, n + 8 * q, e.M, e.N) : u32x4{0, 0, 0, 0};
  }
  template <class T, class Args>
  __device__ __forceinline__ void vectors(const Args& e, f32x4 (&b)[2], f32x4 (&g)[2]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      b[h] = up4<T>(bias[h]);
      g[h] = e.gate ? up4<T>(gate[h]) : f32x4{1.f, 1.f, 1.f, 1.f};
    }
  }
};

template <int ACT>
struct EpiLinear {
  static constexpr bool LONG = false, GROUPS = true;
  struct Args { Rows y, res; const uint16_t *bias, *gate; int M, N; };
  static __device__ __forceinline__ f32x4 value(f32x4 z, f32x4 bias, f32x4 gate, f32x4 res) {
    z += bias;
#pragma unroll
    for (int r = 0; r < 4; ++r) z[r] = act_of<ACT>(z[r]);
    return z * gate + res;
  }
  template <class T>
  static __device__ __forceinline__ void quad(const Args& e, int64_t m, int n, f32x4 z, f32x4) {
    const u32x2 res = e.res.p ? load4(e.res, m, n, e.N) : u32x2{0, 0};
    store4<T>(e.y, m, n, e.N, value(z, vec4<T>(e.bias, 0.f, n, e.N), vec4<T>(e.gate, 1.f, n, e.N), up4<T>(res)));
  }
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
    // 32 columns at a time, what the next ones read in flight meanwhile
    Reads<MI> cur, next;
    cur.load(e.res, e, m0, n0, c, q);
#pragma unroll
    for (int j = 0; j < NI / 2; ++j) {
      if (j + 1 < NI / 2) next.load(e.res, e, m0, n0 + 32 * (j + 1), c, q);
      f32x4 bias[2], gate[2];
      cur.template vectors<T>(e, bias, gate);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const Quads r = quads_of(cur.rows[i]);
        const f32x4 a = value(acc[i][2 * j], bias[0], gate[0], up4<T>(r.a));
        const f32x4 b = value(acc[i][2 * j + 1], bias[1], gate[1], up4<T>(r.b));
        store8(e.y, m0 + 16 * i + c, n0 + 32 * j + 8 * q, e.M, e.N, eight_of({down4<T>(a), down4<T>(b)}));
      }
      cur = next;
    }
  }
};

// dz [M, Np] (Np = N rounded up to 8, zeros behind N) and, with sums, the tile's column sums [tiles_m][2][N]: of dz
// for the bias, of dy * act(z) for the gate.
template <int ACT>
struct EpiLinearBack {
  // beside a 256 x 256 tile's sums its values do not fit into the registers (16,384 x 640 to 2,496: relu 150 us and gelu
  // 202, with 192 x 128 92 and 121)
  static constexpr bool LONG = true, GROUPS = false;
  struct Args { Rows dy, dz; const uint16_t *bias, *gate; float* sums; int M, N, Np; const int* exponent; };
  // dz, and its terms and those of dy * act(z) added to the column sums.  dy is zero behind the last row.
  static __device__ __forceinline__ f32x4 value(f32x4 z, f32x4 dy, f32x4 bias, f32x4 gate, f32x4& sb, f32x4& sg, bool in) {
    f32x4 dz;
    z += bias;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      dz[r] = dy[r] * gate[r] * dact_of<ACT>(z[r]);
      sg[r] += in ? dy[r] * act_of<ACT>(z[r]) : 0.f;
      sb[r] += in ? dz[r] : 0.f;
    }
    return dz;
  }
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
    float* part = (float*)lds;                    // [WM][2][BN]
    const float scale = power_of<T>(e.exponent, 1);
    if (e.sums) __syncthreads();                  // the last stage has been read
    // 32 columns at a time, what the next ones read in flight meanwhile where that fits into the registers too
    constexpr bool AHEAD = MI < 6;
    Reads<MI> cur, next;
    cur.load(e.dy, e, m0, n0, c, q);
#pragma unroll
    for (int j = 0; j < NI / 2; ++j) {
      if (AHEAD && j + 1 < NI / 2) next.load(e.dy, e, m0, n0 + 32 * (j + 1), c, q);
      f32x4 bias[2], gate[2], sb[2], sg[2];
      cur.template vectors<T>(e, bias, gate);
      sb[0] = sb[1] = sg[0] = sg[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = m0 + 16 * i + c;
        const Quads d = quads_of(cur.rows[i]);
        const f32x4 a = value(acc[i][2 * j], up4<T>(d.a), bias[0], gate[0], sb[0], sg[0], m < e.M);
        const f32x4 b = value(acc[i][2 * j + 1], up4<T>(d.b), bias[1], gate[1], sb[1], sg[1], m < e.M);
        store8(e.dz, m, n0 + 32 * j + 8 * q, e.M, e.Np, eight_of({down4<T>(a * scale), down4<T>(b * scale)}));
      }
      if (e.sums) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {           // over the 16 rows that the lanes of a quarter hold
            sb[h][r] = sum16(sb[h][r]);
            sg[h][r] = sum16(sg[h][r]);
          }
          if (c == 0) {
            const int col = (wave % WN) * (BN / WN) + 32 * j + 16 * h + 4 * q;
            *(f32x4*)(part + ((wave / WN) * 2 + 0) * BN + col) = sb[h];
            *(f32x4*)(part + ((wave / WN) * 2 + 1) * BN + col) = sg[h];
          }
        }
      }
      if (AHEAD) cur = next;
      else if (j + 1 < NI / 2) cur.load(e.dy, e, m0, n0 + 32 * (j + 1), c, q);
    }
    if (e.sums) {
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * BN; i += 64 * WM * WN) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WM; ++w) v += part[(w * 2 + i / BN) * BN + i % BN];
        const int n = t.n * BN + i % BN;
        if (n < e.N) e.sums[((int64_t)t.m * 2 + i / BN) * e.N + n] = v;
      }
    }
  }
};

// The forward's sum split over few rows' long k: y from the partial products' sums [splits][M][Np], in split order.
template <class T, int ACT>
__global__ __launch_bounds__(256) void reduce_linear_forward(const float* p, int splits, int64_t plane, int Np,
                                                             typename EpiLinear<ACT>::Args e) {
  const int quads = Np / 4;
  const int64_t total = (int64_t)e.M * quads;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    if (n >= e.N) continue;
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) z += *(const f32x4*)(p + s * plane + (int64_t)m * Np + n);
    EpiLinear<ACT>::template quad<T>(e, m, n, z, z);
  }
}

struct LinearPlan {
  int64_t M, N, K, Kp, Np, sum_rows;
  bool copy_x, copy_w, copy_dy, z;      // z: dz is made from z, otherwise the products take dy
  bool g, cols;                         // G is made; column sums are
  uint16_t *x, *w, *dz;
  float *part, *sums, *colsum, *magnitudes;
  int* exponent;                        // of dz, or of gate * W, in fp16
  GemmPlan xw, dx, dw;                  // the products x W^T, dz W and dz^T x
  size_t bytes;
};

struct LinearNeeds { bool dx, dw, dbias, dgate; };

static LinearPlan linear_plan(const maba_tensor* x, const maba_tensor* scales, const maba_tensor* w, int act, bool gate, bool bias,
                              const maba_tensor* dy, const LinearNeeds* need, void* ws) {
  LinearPlan p = {};
  p.M = x->shape[0];
  p.K = x->shape[1];
  p.N = w->shape[0];
  p.Kp = pad8(p.K);
  p.Np = pad8(p.N);
  const bool few = !need && few_rows(p.M, p.K);
  p.z = need && act != ACT_NONE;
  // the sum over tokens that dW and, without z, dgate come from
  p.g = need && (need->dw || (!p.z && need->dgate));
  // which products read x and W: forward both; backward x for z and G, W for z and dx
  const bool use_x = !need || p.z || p.g, use_w = !need || p.z || need->dx;
  const auto in_place = need ? aligned_columns : aligned_rows;
  p.copy_x = !few && use_x && (scales || !in_place(x));
  p.copy_w = !few && use_w && (!in_place(w) || (need && !p.z && gate));          // gate * W
  p.copy_dy = need && !p.z && (need->dx || p.g) && !in_place(dy);
  Carve c = {(char*)ws, 0};
  if (p.copy_x) p.x = c.take<uint16_t>(p.M * p.Kp);
  if (p.copy_w) p.w = c.take<uint16_t>(p.N * p.Kp);
  if (need) {
    if (p.z || p.copy_dy) p.dz = c.take<uint16_t>(p.M * p.Np);
    int64_t part = 0;
    if (need->dx) {
      p.dx = gemm_plan(p.M, p.Kp, gemm_stages(p.Np, 1), PLAN_COLUMNS | PLAN_SPLIT | PLAN_GROUPS);
      if (p.dx.splits > 1) part = (int64_t)p.dx.splits * p.M * p.Kp;
    }
    if (p.g) {
      p.dw = gemm_plan(p.Np, p.Kp, gemm_stages(p.M, 1), PLAN_COLUMNS | PLAN_SPLIT);
      part = std::max(part, (int64_t)p.dw.splits * p.Np * p.Kp);
    }
    p.part = c.take<float>(part);
    if (w->dtype == MABA_F16 && (p.z || (gate && need->dx))) {
      p.magnitudes = c.take<float>(MAX_FACTORS * MAGNITUDE_GROUPS);
      p.exponent = c.take<int>(1);
    }
  }
  p.xw = gemm_plan(p.M, p.Np, gemm_stages(p.Kp, 1), need ? PLAN_LONG : few ? 0 : PLAN_SPLIT | PLAN_GROUPS);
  if (p.xw.splits > 1) p.part = c.take<float>((int64_t)p.xw.splits * p.M * p.Np);
  p.cols = need && (need->dbias || (need->dgate && (p.z || bias)));
  if (p.cols) {
    p.colsum = c.take<float>(p.N);
    p.sum_rows = p.z ? p.xw.tiles_m : ceil_div(p.M, 128);     // a tile's rows, or those of column_partials
    p.sums = c.take<float>(p.sum_rows * 2 * p.N);
  }
  p.bytes = c.used;
  return p;
}

static int linear_operands(LinearPlan& p, const maba_tensor* x, const maba_tensor* scales, const maba_tensor* w,
                           const maba_tensor* gate, const maba_tensor* dy, hipStream_t s, Operand& ox, Operand& ow) {
  Copies copies;
  if (p.copy_x) copies.add(x, scales, p.x);
  if (p.copy_w) copies.add(w, nullptr, p.w, p.z ? nullptr : gate, p.exponent);
  if (p.copy_dy) copies.add(dy, nullptr, p.dz);
  if (int rc = copies.launch(w->dtype, s)) return rc;
  ox = p.copy_x ? rows_operand(p.x, p.Kp, p.M) : rows_operand((const uint16_t*)x->data, x->stride[0], p.M);
  ow = p.copy_w ? rows_operand(p.w, p.Kp, p.N) : rows_operand((const uint16_t*)w->data, w->stride[0], p.N);
  return MABA_OK;
}

static const uint16_t* vec_of(const maba_tensor* t) { return t ? (const uint16_t*)t->data : nullptr; }

template <class T, int ACT>
static int linear_forward(LinearPlan& p, const maba_tensor* x, const maba_tensor* w, const maba_tensor* bias,
                          const maba_tensor* res, const maba_tensor* gate, maba_tensor* y, hipStream_t s, const char* who) {
  typedef EpiLinear<ACT> E;
  const typename E::Args e = {rows_of(y), rows_of(res), vec_of(bias), vec_of(gate), (int)p.M, (int)p.N};
  if (few_rows(p.M, p.K)) {
    const uint16_t* wp = (const uint16_t*)w->data;
    SkinnyArgs a = {(const uint16_t*)x->data, x->stride[0], {wp, wp}, {w->stride[0], w->stride[0]}, (int)p.M, (int)p.N,
                    (int)p.K, aligned_rows(x), aligned_rows(w)};
    return skinny<T, false, E>(a, e, s, who);
  }
  GemmArgs g = {};
  if (int rc = linear_operands(p, x, nullptr, w, nullptr, nullptr, s, g.a, g.b)) return rc;
  g.K = p.Kp;
  if (p.xw.splits == 1) return gemm<T, K_ROWS, K_ROWS, E>(g, e, p.M, p.Np, p.xw, s, who);
  const EpiPartial::Args ep = {p.part, (int)p.M, (int)p.Np};
  if (int rc = gemm<T, K_ROWS, K_ROWS, EpiPartial>(g, ep, p.M, p.Np, p.xw, s, who)) return rc;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(p.M * (p.Np / 4), 256), 16384));
  hipLaunchKernelGGL((reduce_linear_forward<T, ACT>), grid, dim3(256), 0, s, p.part, p.xw.splits, p.M * p.Np, (int)p.Np, e);
  return check_launch(who);
}

template <class T, int ACT>
static int make_dz(const LinearPlan& p, const Operand& ox, const Operand& ow, const maba_tensor* dy, const maba_tensor* bias,
                   const maba_tensor* gate, hipStream_t s, const char* who) {
  typedef EpiLinearBack<ACT> E;
  GemmArgs g = {};
  g.a = ox;
  g.b = ow;
  g.K = p.Kp;
  const Rows dz = {p.dz, p.Np};
  const typename E::Args e = {rows_of(dy), dz, vec_of(bias), vec_of(gate), p.sums, (int)p.M, (int)p.N, (int)p.Np, p.exponent};
  return gemm<T, K_ROWS, K_ROWS, E>(g, e, p.M, p.Np, p.xw, s, who);
}

template <class T>
static int linear_backward(LinearPlan& p, const maba_tensor* dy, const maba_tensor* x, const maba_tensor* scales,
                           const maba_tensor* w, const maba_tensor* bias, int act, const maba_tensor* gate, maba_tensor* dx,
                           maba_tensor* dw, maba_tensor* dbias, maba_tensor* dgate, hipStream_t s, const char* who) {
  Operand ox, ow;
  if (p.exponent && p.M > 0) {
    Magnitudes m;
    if (p.z) m.add(0, dy->data, dy->stride[0], p.M, p.N, false);
    else m.add(0, w->data, w->stride[0], p.N, p.K, false);
    if (gate) m.add(1, gate->data, 0, 1, p.N, false);
    if (int rc = m.launch(p.z ? 1.13f : 1.f, p.magnitudes, p.exponent, s)) return rc;
  }
  if (int rc = linear_operands(p, x, scales, w, gate, dy, s, ox, ow)) return rc;
  Operand dz = rows_operand((const uint16_t*)dy->data, dy->stride[0], p.M);
  if (p.z || p.copy_dy) dz = rows_operand(p.dz, p.Np, p.M);
  if (p.M > 0) {
    int rc = MABA_OK;
    if (p.z)
      rc = act == ACT_RELU   ? make_dz<T, ACT_RELU>(p, ox, ow, dy, bias, gate, s, who)
           : act == ACT_SILU ? make_dz<T, ACT_SILU>(p, ox, ow, dy, bias, gate, s, who)
                             : make_dz<T, ACT_GELU>(p, ox, ow, dy, bias, gate, s, who);
    else if (p.cols) rc = column_partials(dy, p.sums, s);
    if (rc) return rc;
  }
  if (p.cols)
    if (int rc = reduce_columns(p.sums, p.sum_rows, (int)p.N, dbias ? dbias->data : nullptr,
                                p.z && dgate ? dgate->data : nullptr, !p.z && gate ? gate->data : nullptr,
                                p.z ? nullptr : p.colsum, w->dtype, s))
      return rc;
  if (dx && p.M > 0) {
    GemmArgs g = {};
    g.a = dz;
    g.b = cols_operand(ow, p.Kp);
    g.K = p.Np;                 // dz is N wide where N is a whole number of chunks, padded with zeros otherwise
    const Outputs o = {{rows_of(dx), rows_of(nullptr)}, INT32_MAX, (int)p.M, (int)p.K, p.exponent};
    if (int rc = product_to<T, K_ROWS, K_COLS>(g, o, p.M, p.Kp, p.dx, p.part, s, who)) return rc;
  }
  if (p.g) {
    GemmArgs g = {};
    g.a = cols_operand(dz, p.Np);
    g.b = cols_operand(ox, p.Kp);
    g.K = p.M;
    if (!p.z && gate) {
      if (p.M > 0) {
        const EpiPartial::Args e = {p.part, (int)p.Np, (int)p.Kp};
        if (int rc = gemm<T, K_COLS, K_COLS, EpiPartial>(g, e, p.Np, p.Kp, p.dw, s, who)) return rc;
      }
      const GatedReduceArgs a = {p.part, p.M > 0 ? p.dw.splits : 0, (int)p.Np, (int)p.Kp, (int)p.K, rows_of(dw), rows_of(w),
                                 vec_of(gate), vec_of(bias), p.colsum, dgate ? (uint16_t*)dgate->data : nullptr};
      return reduce_gated(a, (int)p.N, w->dtype, s);
    }
    const Outputs o = {{rows_of(dw), rows_of(nullptr)}, INT32_MAX, (int)p.N, (int)p.K, p.z ? p.exponent : nullptr};
    if (p.M == 0) return zeros_to<T>(o, p.Np, p.Kp, s);
    if (int rc = product_to<T, K_COLS, K_COLS>(g, o, p.Np, p.Kp, p.dw, p.part, s, who)) return rc;
  }
  return MABA_OK;
}

static int linear_check(const maba_tensor* x, const maba_tensor* scales, const maba_tensor* w, const maba_tensor* bias, int act,
                        const maba_tensor* gate, const char* who) {
  if (!x || !w) return fail(MABA_ERR_INVALID, "%s: x and weight required", who);
  if (w->dtype != MABA_BF16 && w->dtype != MABA_F16)
    return fail(w->dtype == MABA_F32 ? MABA_ERR_UNSUPPORTED : MABA_ERR_DTYPE, "%s: 16-bit weights only, got dtype code %d", who, w->dtype);
  if (x->ndim != 2 || w->ndim != 2) return fail(MABA_ERR_INVALID, "%s: x and weight must be 2D", who);
  if (act < ACT_NONE || act > ACT_GELU) return fail(MABA_ERR_INVALID, "%s: activation code %d is not in [0, 3]", who, act);
  int rc = check_sizes(who, x->shape[0], w->shape[0], x->shape[1]);
  if (!rc) rc = check_kept(x, scales, who, w->dtype, -1, x->shape[1]);
  if (!rc && scales && scales->shape[0] != x->shape[0]) rc = fail(MABA_ERR_INVALID, "%s: scales do not match the codes", who);
  if (!rc) rc = check_rows(w, who, "weight", w->dtype, -1, x->shape[1]);
  if (!rc && bias) rc = check_vec(bias, who, "bias", w->dtype, w->shape[0]);
  if (!rc && gate) rc = check_vec(gate, who, "gate", w->dtype, w->shape[0]);
  return rc;
}

}  // namespace ffn
}  // namespace maba

using namespace maba;
using namespace maba::ffn;

extern "C" size_t maba_hip_linear_epilogue_workspace_size(const maba_tensor* x, const maba_tensor* weight) {
  if (linear_check(x, nullptr, weight, nullptr, 0, nullptr, "linear_epilogue")) return 0;
  return linear_plan(x, nullptr, weight, 0, false, false, nullptr, nullptr, nullptr).bytes;
}

extern "C" int maba_hip_linear_epilogue(const maba_tensor* x, const maba_tensor* weight, const maba_tensor* bias, int act,
                                        const maba_tensor* residual, const maba_tensor* gate, maba_tensor* out, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  const char* who = "linear_epilogue";
  int rc = linear_check(x, nullptr, weight, bias, act, gate, who);
  if (rc) return rc;
  const int dt = weight->dtype;
  const int64_t M = x->shape[0], N = weight->shape[0];
  if (residual) rc = check_rows(residual, who, "residual", dt, M, N);
  if (!rc) rc = check_out(out, who, "out", dt, M, N);
  if (rc) return rc;
  if (overlap(out, x) || overlap(out, weight) || overlap(out, bias) || overlap(out, gate))
    return fail(MABA_ERR_INVALID, "%s: out overlaps an input", who);
  // each element of the residual is read by the lane that then writes its sum: the very same rows may be out
  if (residual && overlap(out, residual) && (out->data != residual->data || out->stride[0] != residual->stride[0]))
    return fail(MABA_ERR_INVALID, "%s: out overlaps the residual at another place", who);
  LinearPlan p = linear_plan(x, nullptr, weight, act, gate != nullptr, bias != nullptr, nullptr, nullptr, workspace);
  if ((rc = check_workspace(who, workspace, workspace_bytes, p.bytes))) return rc;
  if (p.M == 0) return MABA_OK;
  const hipStream_t s = (hipStream_t)stream;
#define LINEAR_FORWARD(T)                                                                                  \
  (act == ACT_RELU   ? linear_forward<T, ACT_RELU>(p, x, weight, bias, residual, gate, out, s, who)        \
   : act == ACT_SILU ? linear_forward<T, ACT_SILU>(p, x, weight, bias, residual, gate, out, s, who)        \
   : act == ACT_GELU ? linear_forward<T, ACT_GELU>(p, x, weight, bias, residual, gate, out, s, who)        \
                     : linear_forward<T, ACT_NONE>(p, x, weight, bias, residual, gate, out, s, who))
  return dt == MABA_BF16 ? LINEAR_FORWARD(Bf16) : LINEAR_FORWARD(Fp16);
#undef LINEAR_FORWARD
}

extern "C" size_t maba_hip_linear_epilogue_backward_workspace_size(const maba_tensor* dy, const maba_tensor* x,
                                                                   const maba_tensor* x_scales, const maba_tensor* weight, int act,
                                                                   int with_bias, int with_gate, int needs) {
  if (linear_check(x, x_scales, weight, nullptr, act, nullptr, "linear_epilogue_backward")) return 0;
  if (check_rows(dy, "linear_epilogue_backward", "dy", weight->dtype, x->shape[0], weight->shape[0])) return 0;
  const LinearNeeds n = {(needs & 1) != 0, (needs & 2) != 0, (needs & 4) != 0, (needs & 8) != 0};
  return linear_plan(x, x_scales, weight, act, with_gate != 0, with_bias != 0, dy, &n, nullptr).bytes;
}

extern "C" int maba_hip_linear_epilogue_backward(const maba_tensor* dy, const maba_tensor* x, const maba_tensor* x_scales,
                                                 const maba_tensor* weight, const maba_tensor* bias, int act,
                                                 const maba_tensor* gate, maba_tensor* dx, maba_tensor* dw, maba_tensor* dbias,
                                                 maba_tensor* dgate, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "linear_epilogue_backward";
  int rc = linear_check(x, x_scales, weight, bias, act, gate, who);
  if (rc) return rc;
  const int dt = weight->dtype;
  const int64_t M = x->shape[0], K = x->shape[1], N = weight->shape[0];
  rc = check_rows(dy, who, "dy", dt, M, N);
  if (!rc && dx) rc = check_out(dx, who, "dx", dt, M, K);
  if (!rc && dw) rc = check_out(dw, who, "dw", dt, N, K);
  if (!rc && dbias) rc = check_vec(dbias, who, "dbias", dt, N);
  if (!rc && dgate) rc = check_vec(dgate, who, "dgate", dt, N);
  if (!rc && dgate && !gate) rc = fail(MABA_ERR_INVALID, "%s: dgate without a gate", who);
  if (rc) return rc;
  const maba_tensor *outs[4] = {dx, dw, dbias, dgate}, *ins[6] = {dy, x, x_scales, weight, bias, gate};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 6; ++j)
      if (overlap(outs[i], ins[j])) return fail(MABA_ERR_INVALID, "%s: a gradient overlaps an input", who);
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return fail(MABA_ERR_INVALID, "%s: two gradients overlap", who);
  }
  const LinearNeeds need = {dx != nullptr, dw != nullptr, dbias != nullptr, dgate != nullptr};
  LinearPlan p = linear_plan(x, x_scales, weight, act, gate != nullptr, bias != nullptr, dy, &need, workspace);
  if ((rc = check_workspace(who, workspace, workspace_bytes, p.bytes))) return rc;
  return dt == MABA_BF16
             ? linear_backward<Bf16>(p, dy, x, x_scales, weight, bias, act, gate, dx, dw, dbias, dgate, (hipStream_t)stream, who)
             : linear_backward<Fp16>(p, dy, x, x_scales, weight, bias, act, gate, dx, dw, dbias, dgate, (hipStream_t)stream, who);
}
