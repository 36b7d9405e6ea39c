// The boundary between two sub-layers and dropout by itself, forward and backward:
//   z  = RMSNorm(y) * w_post  (or y)             the norm after the sub-layer that made y
//   x' = x + scale * gate * dropout(z)           the residual stream
//   h  = RMSNorm(x') * w                         the norm before the next sub-layer
// (reference model.py:11-22, 92-128 has the gated residual and the norm before, composed of torch modules.)
//
// Backward, for the gradients d' of x' and dh of h, with x^ = x' r, y^ = y rp the normalised rows and x' as the forward had it
// before it was rounded, made again from x and y:
//   dX = d' + r (dh w - x^ mean(dh w x^))        the gradient of x, and of x' behind its norm
//   dz = scale gate dropout(dX)                  the same mask, made again
//   dy = rp (dz w_post - y^ mean(dz w_post y^))
//   dw = sum dh x^,  dgate = sum scale dX dropout(z),  dw_post = sum dz y^     over the rows
// Nothing but x and y is kept from the forward pass.  (From the rounded x' instead, h would be another function's by a rounding of
// its argument: a gradient of weight over a few rows 1.4 times as far off as its own rounding leaves it.)
//
// Bound: HBM.  Forward reads x and y and writes x' and h; backward reads d', dh, x, y and writes dx and dy, once each.
// Times below are of single kernels on cold tensors; a copy of 1 GiB reaches 5.1 TB/s, and tensors that the 256 MB cache in
// front of HBM holds in part go faster.
#include "row_vec.h"

namespace maba {
namespace rowvec {

struct BoundaryArgs {
  const void *x, *y, *w, *wp, *g;
  void *xo, *h;
  int64_t xs, ys, xos, hs, R;
  int C, lg;
  float scale, eps;
  Drop d;
};

// A row stays in the registers of its lanes from the load to both stores: the sums of y^2 and of x'^2 cost two exchanges, no
// second read.  16,384 x 640 bf16 with dropout 18.4 us, 4.6 TB/s, and 16.6 without (5.0); 32,768 x 640 30 us, 5.5 TB/s; 8,192 x
// 4,096 with both norms and dropout 45 us, 5.9 TB/s.  A single row of 640 takes 3.1 us, most of it the launch.
// CUT: rows end inside a chunk (CutRows): their accesses are 2- or 4-byte aligned, and the memory path splits most of them in
// two (8,191 x 4,095 bf16 65 us, 4.1 TB/s).
template <class T, int NCH, bool CUT>
__global__ __launch_bounds__(1 << MAX_LG) void boundary_kernel(BoundaryArgs a) {
  constexpr int V = Traits<T>::VEC;
  __shared__ float red[2 * (1 << MAX_LG) / 64];
  int turn = 0;
  const int lg = a.lg, l = threadIdx.x & ((1 << lg) - 1), slots = blockDim.x >> lg;
  // the wave's first row of the workgroup's, and which of the wave's this lane is in
  const int first = __builtin_amdgcn_readfirstlane(threadIdx.x >> lg), sub = lg < 6 ? (threadIdx.x & 63) >> lg : 0;
  const Walk<T> wx(a.x, a.xs, l, sub), wy(a.y, a.ys, l, sub), wxo(a.xo, a.xos, l, sub), wh(a.h, a.hs, l, sub);
  const Walk<T> vw(a.w, 0, l, 0), vp(a.wp, 0, l, 0), vg(a.g, 0, l, 0);
  const uint64_t key = a.d.mode == 1 ? *a.d.seed : 0;
  const float inv_c = 1.f / (float)a.C;
  const CutRows<T, CUT ? NCH : 1> rows(a.R, a.C, l, lg);
  u32x4 w[NCH] = {}, wp[NCH] = {}, g[NCH] = {};
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int at = (l + (i << lg)) * V;
    if (a.w) w[i] = load_chunk<T>(vw.at(0, i << lg), vw.off, a.C - at);
    if (a.wp) wp[i] = load_chunk<T>(vp.at(0, i << lg), vp.off, a.C - at);
    if (a.g) g[i] = load_chunk<T>(vg.at(0, i << lg), vg.off, a.C - at);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * slots; r0 < a.R; r0 += (int64_t)gridDim.x * slots) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(w[i]), "+v"(wp[i]), "+v"(g[i]));     // held packed, not unpacked ahead of the loop
    const int64_t ru = r0 + first, r = ru + sub;
    const int C = r < a.R ? a.C : 0;               // a row past the last one has no elements
    u32x4 x[NCH], y[NCH];
    if constexpr (CUT) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        x[i] = rows.load(wx, ru, r < a.R, i);
        if (a.y) y[i] = rows.load(wy, ru, r < a.R, i);
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int left = C - (l + (i << lg)) * V;
        x[i] = ended<T>(x[i], left);
        if (a.y) y[i] = ended<T>(y[i], left);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int at = (l + (i << lg)) * V;
        x[i] = load_chunk<T>(wx.at(ru, i << lg), wx.off, C - at);
        if (a.y) y[i] = load_chunk<T>(wy.at(ru, i << lg), wy.off, C - at);
      }
    }
    float rp = 1.f;
    if (a.wp) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float v[V];
        unpack<T>(y[i], v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] = fmaf(v[e], v[e], s[0]);
      }
      row_sums<1>(s, lg, red, turn);
      rp = rsqrtf(s[0] * inv_c + a.eps);
    }
    float xn[NCH][V], ss[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int at = (l + (i << lg)) * V;
      unpack<T>(x[i], xn[i]);
      if (a.y) {
        float z[V], p[V];
        unpack<T>(y[i], z);
        if (a.wp) {
          unpack<T>(wp[i], p);
#pragma unroll
          for (int e = 0; e < V; ++e) z[e] *= rp * p[e];
        }
        drop_chunk<V>(z, a.d, key, r, at);
        if (a.g) {
          unpack<T>(g[i], p);
#pragma unroll
          for (int e = 0; e < V; ++e) z[e] *= p[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) xn[i][e] = fmaf(a.scale, z[e], xn[i][e]);
        if (a.xo) store_chunk<T>(wxo.at(ru, i << lg), wxo.off, C - at, pack<T>(xn[i]));
      }
#pragma unroll
      for (int e = 0; e < V; ++e) ss[0] = fmaf(xn[i][e], xn[i][e], ss[0]);
      __builtin_amdgcn_sched_barrier(0);           // chunk after chunk: side by side their masks cost 50 registers more
    }
    if (a.w) {
      row_sums<1>(ss, lg, red, turn);
      const float rx = rsqrtf(ss[0] * inv_c + a.eps);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int at = (l + (i << lg)) * V;
        float p[V];
        unpack<T>(w[i], p);
#pragma unroll
        for (int e = 0; e < V; ++e) p[e] *= xn[i][e] * rx;
        store_chunk<T>(wh.at(ru, i << lg), wh.off, C - at, pack<T>(p));
      }
    }
  }
}

// The parameters' gradients: a lane sums its columns over its rows in registers, a workgroup its rows' lanes in LDS, and
// columns_kernel the workgroups' partials [groups][n][C] in their order.
enum { GRAD_W = 1, GRAD_GATE = 2, GRAD_POST = 4 };
struct BoundaryBackArgs {
  const void *dxo, *dh, *x, *y, *w, *wp, *g;
  void *dx, *dy;
  float* partial;
  int64_t dxos, dhs, xs, ys, dxs, dys, R;
  int C, lg, grads;
  bool cut;
  float scale, eps;
  Drop d;
};

// A row's sums are exchanged twice: those of dh w x' and x'^2 (the mean of dh w x^ is r times that of dh w x'), and with POST that
// for dy together with the next row's of y^2.  The chunks stay packed in registers between their uses, the mask as bits.  HBM, and
// arithmetic that its waits do not hide: 16,384 x 640 bf16 with dropout 36 us with the sums over the partials, 3.5 TB/s (three
// lanes of four have one chunk of two), 8,192 x 4,096 85 us, 4.7 TB/s, and with both norms 98, 4.1 TB/s, the vector units 65 %
// busy; 8,191 x 4,095 106 us, 3.8 TB/s, and 123.
// WHOLE: rows of whole 16-byte chunks (WholeWalk).  The next rows' chunks are loaded ahead of the present ones' arithmetic.
// back_size() says how many threads a workgroup has.  Registers: of fp32 rows of more than 6,144 a lane has four chunks, which
// with POST or without WHOLE spill 52 to 212 bytes a lane (4,096 x 8,192 169 us, 4.8 TB/s, and with both norms 239; x 6,144, whose
// three chunks fit, 127 and 133), and 16-bit rows of one chunk with POST and without WHOLE 16.
constexpr int back_threads(int nch) { return nch == 1 ? 1024 : 512; }
template <class T, int NCH, bool POST, bool WHOLE>
__global__ __launch_bounds__(back_threads(NCH)) void boundary_back_kernel(BoundaryBackArgs a) {
  constexpr int V = Traits<T>::VEC, NG = POST ? 3 : 2;
  __shared__ float red[2 * 2 * back_threads(NCH) / 64];
  extern __shared__ float sums[];                  // [NG][threads * V]; before that, the parameters' chunks
  const int threads = blockDim.x;
  int turn = 0;
  const int lg = a.lg, l = threadIdx.x & ((1 << lg) - 1), slots = threads >> lg;
  const int first = __builtin_amdgcn_readfirstlane(threadIdx.x >> lg), sub = lg < 6 ? (threadIdx.x & 63) >> lg : 0;
  typedef std::conditional_t<WHOLE, WholeWalk<T>, Walk<T>> Rows;
  const Rows wd(a.dxo, a.dxos, l, sub), wh(a.dh, a.dhs, l, sub), wx(a.x, a.xs, l, sub), wy(a.y, a.ys, l, sub);
  const Rows wdx(a.dx, a.dxs, l, sub), wdy(a.dy, a.dys, l, sub);
  const uint64_t key = a.d.mode == 1 ? *a.d.seed : 0;
  const float inv_c = 1.f / (float)a.C, scale = a.scale * a.d.keep;      // of what is kept
  // chunk c of the parameters: weight's, gate's, post_weight's
  const int chunks = (a.C + V - 1) / V;
  u32x4* par = (u32x4*)sums;
  for (int c = threadIdx.x; c < chunks; c += threads) {
    if (a.dh) par[c] = load_chunk<T>(a.w, c * 16, a.C - c * V);
    if (a.g) par[chunks + c] = load_chunk<T>(a.g, c * 16, a.C - c * V);
    if constexpr (POST) par[2 * chunks + c] = load_chunk<T>(a.wp, c * 16, a.C - c * V);
  }
  __syncthreads();
  uint32_t where[NCH];                             // of chunk i behind chunk 0
  int pc[NCH];                                     // its parameters; a lane without a chunk reads the last one's
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = l + (i << lg);
    where[i] = c < chunks ? (uint32_t)(16 * (i << lg)) : NOWHERE;
    pc[i] = min(c, chunks - 1);
  }
  const CutRows<T, WHOLE ? 1 : NCH> cut(a.R, a.C, l, lg);
  struct Raw { u32x4 d[NCH], h[NCH], x[NCH], y[NCH]; };
  const auto fetch = [&](int64_t r0, Raw& u) {
    const int64_t ru = r0 + first;
    const bool live = ru + sub < a.R;
    if constexpr (WHOLE) {
      const uint32_t dead = live ? 0u : NOWHERE;
      const auto rd = wd.rows(ru), rh = wh.rows(ru), rx = wx.rows(ru), ry = wy.rows(ru);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const uint32_t at = where[i] | dead;
        u.h[i] = wh.load(rh, at);
        u.x[i] = wx.load(rx, at);
        u.d[i] = wd.load(rd, at);
        u.y[i] = wy.load(ry, at);
      }
    } else {
      const auto one = [&](const Rows& w, int i) {
        if (a.cut) return cut.load(w, ru, live, i);
        return load_chunk<T>(w.at(ru, i << lg), w.off, live ? a.C - (l + (i << lg)) * V : 0);
      };
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        u.h[i] = u.x[i] = u.d[i] = u.y[i] = u32x4{0, 0, 0, 0};
        if (a.dh) {
          u.h[i] = one(wh, i);
          u.x[i] = one(wx, i);
        }
        if (a.dxo) u.d[i] = one(wd, i);
        if (a.y) u.y[i] = one(wy, i);
      }
    }
  };
  float acc[NG][NCH][V] = {};
  const int64_t step = (int64_t)gridDim.x * slots;
  int64_t r0 = (int64_t)blockIdx.x * slots;
  // the row's own part of sum y^2, of chunks as they are then used
  const auto squares = [&](int64_t row, Raw& u) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if constexpr (!WHOLE)
        if (a.cut) u.y[i] = ended<T>(u.y[i], row < a.R ? a.C - (l + (i << lg)) * V : 0);
      float y[V];
      unpack<T>(u.y[i], y);
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf(y[e], y[e], s);
    }
    return s;
  };
  Raw next;
  float yy[1] = {0.f};
  if (r0 < a.R) {
    fetch(r0, next);
    if constexpr (POST) {
      yy[0] = squares(r0 + first + sub, next);
      row_sums<1, 2>(yy, lg, red, turn);
    }
  }
  for (; r0 < a.R; r0 += step) {
    const int64_t ru = r0 + first, r = ru + sub;
    Raw u = next;
    fetch(r0 + step, next);
    if constexpr (!WHOLE) {
      if (a.cut)
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const int left = r < a.R ? a.C - (l + (i << lg)) * V : 0;
          u.h[i] = ended<T>(u.h[i], left);
          u.x[i] = ended<T>(u.x[i], left);
          u.d[i] = ended<T>(u.d[i], left);
          if constexpr (!POST) u.y[i] = ended<T>(u.y[i], left);
        }
    }
    const auto put = [&](const Rows& w, int i, const float (&v)[V]) {
      if constexpr (WHOLE) w.store(w.rows(ru), where[i] | (r < a.R ? 0u : NOWHERE), pack<T>(v));
      else store_chunk<T>(w.at(ru, i << lg), w.off, r < a.R ? a.C - (l + (i << lg)) * V : 0, pack<T>(v));
    };
    // (a row past the last one has no part in the sums over rows, whatever eps is)
    const float rp = !POST ? 1.f : r < a.R ? rsqrtf(yy[0] * inv_c + a.eps) : 0.f;
    uint32_t bits[NCH];
    float xn[NCH][V], s[2] = {0.f, 0.f};     // x', and the sums of dh w x' and x'^2
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      bits[i] = kept_bits<V>(a.d, key, r, (l + (i << lg)) * V);
      if constexpr (!POST) u.y[i] = drop_packed<T>(u.y[i], a.d, bits[i]);      // all that y is used for is dropped with it
      if (a.dh) {
        float h[V], p[V];
        unpack<T>(u.x[i], xn[i]);
        if (a.y) {                           // as the forward does, but for the order of its factors
          float z[V];
          unpack<T>(u.y[i], z);
          if constexpr (POST) {
            unpack<T>(par[2 * chunks + pc[i]], p);
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] *= rp * p[e];
            drop_by<V>(z, a.d, bits[i]);
          }
          if (a.g) {
            unpack<T>(par[chunks + pc[i]], p);
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] *= p[e];
          }
#pragma unroll
          for (int e = 0; e < V; ++e) xn[i][e] = fmaf(scale, z[e], xn[i][e]);
        }
        unpack<T>(u.h[i], h);
        unpack<T>(par[pc[i]], p);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[0] = fmaf(h[e] * p[e], xn[i][e], s[0]);
          s[1] = fmaf(xn[i][e], xn[i][e], s[1]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);           // chunk after chunk: side by side their masks cost 50 registers more
    }
    if (a.dh) row_sums<2>(s, lg, red, turn);
    const float rx = r < a.R ? rsqrtf(s[1] * inv_c + a.eps) : 0.f, mean = s[0] * rx * inv_c;
    float dz[POST ? NCH : 1][V], t[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float d[V];
      unpack<T>(u.d[i], d);
      if (a.dh) {
        float h[V], p[V];
        unpack<T>(u.h[i], h);
        unpack<T>(par[pc[i]], p);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = xn[i][e] * rx;
          d[e] = fmaf(rx, fmaf(h[e], p[e], -xh * mean), d[e]);
          acc[0][i][e] = fmaf(h[e], xh, acc[0][i][e]);
        }
      }
      if (a.dx) put(wdx, i, d);
      if (a.dy || (a.grads & (GRAD_GATE | GRAD_POST))) {
        // dropout(z) = m z with m in {0, 1 / (1 - p)}, the factor being in scale; a dropped z is zero whatever it was, also for dgate
        float p[V], y[V];
        unpack<T>(u.y[i], y);
        if constexpr (POST) {
#pragma unroll
          for (int e = 0; e < V; ++e) y[e] *= rp;
          unpack<T>(par[2 * chunks + pc[i]], p);
        }
        if (a.grads & GRAD_GATE) {
          float z[V];
#pragma unroll
          for (int e = 0; e < V; ++e) z[e] = POST ? y[e] * p[e] : y[e];
          if constexpr (POST) drop_by<V>(z, a.d, bits[i]);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[1][i][e] = fmaf(d[e], z[e], acc[1][i][e]);
        }
        drop_by<V>(d, a.d, bits[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] *= scale;
        if (a.g) {
          float q[V];
          unpack<T>(par[chunks + pc[i]], q);
#pragma unroll
          for (int e = 0; e < V; ++e) d[e] *= q[e];
        }
        if constexpr (POST) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            acc[NG - 1][i][e] = fmaf(d[e], y[e], acc[NG - 1][i][e]);
            dz[i][e] = d[e] * p[e];
            t[0] = fmaf(dz[i][e], y[e], t[0]);
          }
        } else if (a.dy) {
          put(wdy, i, d);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (POST) {
      t[1] = squares(r + step, next);
      row_sums<2>(t, lg, red, turn);
      if (a.dy) {
        const float m = t[0] * inv_c * rp;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          float y[V];
          unpack<T>(u.y[i], y);
#pragma unroll
          for (int e = 0; e < V; ++e) dz[i][e] = rp * fmaf(-y[e], m, dz[i][e]);
          put(wdy, i, dz[i]);
        }
      }
      yy[0] = t[1];
    }
  }
  if (!a.grads) return;
  __syncthreads();                                 // the parameters are read no more
  // rows that share a wave first, then those of the workgroup's waves
  const int lanes = 1 << lg, wave = threadIdx.x >> 6;
  const int units = lg < 6 ? threads / 64 : slots;
  const int mine = lg < 6 ? wave * lanes + (threadIdx.x & 63) : threadIdx.x;
  const bool writes = lg >= 6 || (int)(threadIdx.x & 63) < lanes;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = acc[n][i][e];
        if (lg < 5) v += __shfl_xor(v, 16);
        if (lg < 6) v += __shfl_xor(v, 32);
        if (writes) sums[(n * threads + mine) * V + e] = v;
      }
    __syncthreads();
    int k = 0;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      if (!(a.grads >> n & 1)) continue;
      float* out = a.partial + ((int64_t)blockIdx.x * __builtin_popcount(a.grads) + k++) * a.C;
      for (int c = threadIdx.x; c < lanes * V; c += threads) {
        const int col = (i << lg) * V + c;
        if (col >= a.C) continue;
        float v = 0.f;
        for (int u = 0; u < units; ++u) v += sums[(n * threads + u * lanes) * V + c];
        out[col] = v;
      }
    }
    __syncthreads();
  }
}

// out[c] = factor * the sum over g of p[g][n][c]: 32 runs of g side by side, each in its order, then the runs in theirs.
// Bound by the latency of a run's loads: 256 partials of 2 x 640 columns 4.0 us, of 3 x 4,096 5.0 us.
struct ColumnsArgs {
  const float* p;
  void* out[3];
  float factor[3];
  int groups, n, C;
};
template <class T>
__global__ __launch_bounds__(1024) void columns_kernel(ColumnsArgs a) {
  constexpr int RUNS = 32;
  __shared__ float part[RUNS][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5, n = blockIdx.y;
  float s = 0.f;
  if (c < a.C) {
    const float* p = a.p + (int64_t)n * a.C + c;
#pragma unroll 8
    for (int g = run; g < a.groups; g += RUNS) s += p[(int64_t)g * a.n * a.C];
  }
  part[run][threadIdx.x & 31] = s;
  __syncthreads();
  if (run == 0 && c < a.C) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) v += part[i][threadIdx.x];
    v *= a.factor[n];
    if constexpr (T::CODE == MABA_F32) ((float*)a.out[n])[c] = v;
    else ((uint16_t*)a.out[n])[c] = (uint16_t)T::down(v);
  }
}

// ---------------------------------------------------------------- dropout

struct DropArgs {
  const void* x; void* y;
  int64_t xs, ys, R;
  int C, lg;
  Drop d;
};
// 2^lg lanes a row, four chunks a lane in flight.  Bound by the generator's 32-bit multiplications and HBM about alike: 32,768 x
// 1,024 bf16 26.6 us, 5.0 TB/s; 16,384 x 640 12.1 us.  A row is one workgroup's at most: few long ones leave the chip idle (16.8M
// elements as 16,384 rows 17 us, as 256 24, as 16 264, as one 4.0 ms).
template <class T>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
  constexpr int V = Traits<T>::VEC, N = 4;
  const int l = threadIdx.x & ((1 << a.lg) - 1), slots = 256 >> a.lg;
  const uint64_t key = a.d.mode == 1 ? *a.d.seed : 0;
  const int chunks = (a.C + V - 1) / V;
  for (int64_t r = (int64_t)blockIdx.x * slots + (threadIdx.x >> a.lg); r < a.R; r += (int64_t)gridDim.x * slots)
    for (int c0 = l; c0 < chunks; c0 += N << a.lg) {
      u32x4 u[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t at = ((int64_t)c0 + (i << a.lg)) * V;
        u[i] = load_chunk<T>((const typename Traits<T>::elem*)a.x + r * a.xs + at, 0, at < a.C ? (int)(a.C - at) : 0);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t at = ((int64_t)c0 + (i << a.lg)) * V;
        if (at >= a.C) continue;
        float v[V];
        unpack<T>(u[i], v);
        drop_chunk<V>(v, a.d, key, r, (int)at);
        store_chunk<T>((typename Traits<T>::elem*)a.y + r * a.ys + at, 0, (int)(a.C - at), pack<T>(v));
      }
    }
}

// ---------------------------------------------------------------- arguments

static int check_float_rows(const maba_tensor* t, const char* who) {
  if (!t) return fail(MABA_ERR_INVALID, "%s: x is missing", who);
  if (!is_float_dt(t->dtype)) return fail(MABA_ERR_DTYPE, "%s: f32, f16 or bf16 only, got dtype code %d", who, t->dtype);
  if (t->ndim != 2) return fail(MABA_ERR_INVALID, "%s: x must be 2D, got %dD", who, t->ndim);
  if (t->shape[1] < 1) return fail(MABA_ERR_INVALID, "%s: the width must be positive", who);
  if (t->shape[0] < 0) return fail(MABA_ERR_INVALID, "%s: x has a negative size", who);
  if (t->shape[1] > (1 << 30) || t->shape[0] > (int64_t)1 << 40) return fail(MABA_ERR_UNSUPPORTED, "%s: sizes out of range", who);
  return MABA_OK;
}
static int check_drop(const char* who, double p, const int64_t* seed) {
  if (!(p >= 0.0 && p <= 1.0)) return fail(MABA_ERR_INVALID, "%s: p=%g must be in [0, 1]", who, p);
  if (p > 0.0 && p < 1.0 && (!seed || (uintptr_t)seed % 8)) return fail(MABA_ERR_INVALID, "%s: dropout needs a seed", who);
  return MABA_OK;
}
static int chunk_elems(int dtype) { return dtype == MABA_F32 ? 4 : 8; }
// Whether rows end inside a chunk that is not their first.
static bool cut_rows(int64_t C, int dtype) { return C > chunk_elems(dtype) && C % chunk_elems(dtype); }
static bool same_place(const maba_tensor* a, const maba_tensor* b) {
  return a->data == b->data && (a->shape[0] <= 1 || a->stride[0] == b->stride[0]);
}

static int64_t row_stride(const maba_tensor* t) { return t ? walked(t->shape[0], t->stride[0]) : 0; }
static bool far_rows(std::initializer_list<const maba_tensor*> all) {
  for (const maba_tensor* t : all)
    if (t && far_apart(t->shape[0], t->stride[0])) return true;
  return false;
}
// Whether the rows of all of them are whole 16-byte chunks.
static bool whole_rows(std::initializer_list<const maba_tensor*> all) {
  for (const maba_tensor* t : all)
    if (t) {
      const int64_t size = t->dtype == MABA_F32 ? 4 : 2;
      if (t->shape[1] * size % 16 || (uintptr_t)t->data % 16 || (t->shape[0] > 1 && t->stride[0] * size % 16)) return false;
    }
  return true;
}
// Elements of a row a lane has.  Few give every row more lanes and the chip more waves; more leave fewer lanes without work
// (80 chunks of 640 16-bit elements fill 62 % of 128 lanes and 83 % of 32 with three each) and share out what a row costs
// besides its elements.  Forward, in us, 8 / 24 elements: 1 x 640 bf16 3.1 / 4.1, 2,048 x 640 5.5 / 5.8, 32,768 x 640
// 42.8 / 32.8, 8,192 x 4,096 50.5 / 47.3; fp32 8,192 x 1,000 22.9 / 24.6.
// Backward: two chunks a lane make one wave's of a row that would be two waves', so that its sums need no LDS and no barrier.
// That pays for many rows, and where all 128 lanes would have had work it costs more than it saves.  In us, 8 / 16 elements:
// 64 x 640 8.3 / 10.5, 2,048 x 640 12.3 / 13.0, 16,384 x 640 37.7 / 36.4, 65,536 x 640 113 / 107 and with post_weight 152 / 129,
// 24,576 x 767 69 / 71 and with post_weight 85 / 78, x 1,001 72 / 74; rows of one wave 24,576 x 512 37 / 40, and of more than a wave either
// way 24,576 x 1,345 117 / 148, 8,192 x 4,096 85 / 86, 2,048 x 4,096 33 / 35.
constexpr int MOST_ELEMS = 24, MOST_BACK = 16;
static int forward_elems(int64_t R, int64_t C, int dtype) { return C > 8 << MAX_LG ? 16 : dtype != MABA_F32 && R > 4096 ? MOST_ELEMS : 8; }
static int back_elems(int64_t R, int64_t C, int dtype) {
  if (C > 8 << MAX_LG) return MOST_BACK;
  const int64_t chunks = ceil_div(C, 8);
  int64_t lanes = 64;
  while (lanes < chunks) lanes *= 2;
  return dtype != MABA_F32 && R >= 16384 && lanes == 128 && chunks * 4 <= lanes * 3 ? MOST_BACK : 8;
}
// A backward pass's threads a workgroup, and so how many workgroups a compute unit has: together four waves a SIMD with one
// chunk a lane, two beyond, as registers allow.  Many rows: one workgroup, since the fewest partials are then written (in us, one /
// as many as there are of 256 threads or a row's: 2,048 x 640 bf16 12.3 / 14.4, 8,192 x 4,096 85 / 91, 8,191 x 4,095 106 / 115,
// fp32 8,192 x 2,048 83 / 86.5).  Two where rows end inside a chunk, whose accesses keep the waves apart, and a row does not need all
// threads (one / two: 24,576 x 1,345 128 / 117, x 1,001 78 / 72).  Until rows fill the chip the smallest (64 x 640 8.4, of 1,024
// threads 10.6).
static int back_size(int64_t R, const Geometry& geo, bool cut) {
  const int most = cut && geo.lg < MAX_LG ? std::min(back_threads(geo.nch), 512) : back_threads(geo.nch);
  return R >= (int64_t)device_cu_count() * (most >> geo.lg) ? most : std::max(256, 1 << geo.lg);
}
static int back_groups(int64_t R, const Geometry& geo, bool cut) {
  const int threads = back_size(R, geo, cut);
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(R, threads >> geo.lg), (int64_t)device_cu_count() * (back_threads(geo.nch) / threads)));
}
template <int N>
struct Num { static constexpr int value = N; };
// f(Num<nch>()), nch chunks of T being at most MOST elements.
template <class T, int MOST, int N = 1, class F>
static void with_chunks(int nch, F f) {
  if constexpr ((N + 1) * Traits<T>::VEC <= MOST) {
    if (nch > N) return with_chunks<T, MOST, N + 1>(nch, f);
  }
  f(Num<N>());
}
template <class F>
static void with_type(int dtype, F f) {
  if (dtype == MABA_F32) return f(F32());
  if (dtype == MABA_BF16) return f(Bf16());
  return f(Fp16());
}

}  // namespace rowvec
}  // namespace maba

using namespace maba;
using namespace maba::rowvec;
using ffn::check_out;
using ffn::check_rows;
using ffn::check_vec;
using ffn::overlap;

extern "C" int maba_hip_dropout(const maba_tensor* x, double p, const int64_t* seed, uint32_t stream_id, maba_tensor* out,
                                void* stream) {
  const char* who = "dropout";
  int rc = check_float_rows(x, who);
  if (!rc) rc = check_drop(who, p, seed);
  if (!rc) rc = check_rows(x, who, "x", x->dtype, -1, -1);
  if (!rc) rc = check_out(out, who, "out", x->dtype, x->shape[0], x->shape[1]);
  if (rc) return rc;
  if (overlap(x, out) && !same_place(x, out)) return fail(MABA_ERR_INVALID, "%s: x and out overlap", who);
  DropArgs a = {x->data, out->data, row_stride(x), row_stride(out), x->shape[0], (int)x->shape[1], 0, make_drop(p, seed, stream_id)};
  if (a.R == 0) return MABA_OK;
  const int64_t chunks = ceil_div(a.C, chunk_elems(x->dtype));
  while (a.lg < 8 && chunks > (int64_t)4 << a.lg) ++a.lg;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(a.R, 256 >> a.lg), 65536));
  auto k = x->dtype == MABA_F32 ? dropout_kernel<F32> : x->dtype == MABA_BF16 ? dropout_kernel<Bf16> : dropout_kernel<Fp16>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(who);
}

extern "C" int maba_hip_residual_norm(const maba_tensor* x, const maba_tensor* y, const maba_tensor* weight,
                                      const maba_tensor* post_weight, const maba_tensor* gate, float scale, double p,
                                      const int64_t* seed, uint32_t stream_id, float eps, maba_tensor* x_out, maba_tensor* h,
                                      void* stream) {
  const char* who = "residual_norm";
  int rc = check_float_rows(x, who);
  if (!rc) rc = check_drop(who, p, seed);
  if (!rc) rc = check_rows(x, who, "x", x->dtype, -1, -1);
  if (rc) return rc;
  const int64_t R = x->shape[0], C = x->shape[1];
  const int dt = x->dtype;
  if (!y && (post_weight || gate || x_out)) return fail(MABA_ERR_INVALID, "%s: post_weight, gate and x_out go with y", who);
  if (!weight != !h) return fail(MABA_ERR_INVALID, "%s: weight and h go together", who);
  if (!h && !x_out) return fail(MABA_ERR_INVALID, "%s: nothing to compute", who);
  if (y) rc = check_rows(y, who, "y", dt, R, C);
  if (!rc && weight) rc = check_vec(weight, who, "weight", dt, C);
  if (!rc && post_weight) rc = check_vec(post_weight, who, "post_weight", dt, C);
  if (!rc && gate) rc = check_vec(gate, who, "gate", dt, C);
  if (!rc && x_out) rc = check_out(x_out, who, "x_out", dt, R, C);
  if (!rc && h) rc = check_out(h, who, "h", dt, R, C);
  if (rc) return rc;
  // x_out may be x itself: a lane reads all it needs of a row before it writes
  if (overlap(h, x) || overlap(h, y) || overlap(h, x_out) || overlap(x_out, y) || (overlap(x_out, x) && !same_place(x_out, x)))
    return fail(MABA_ERR_INVALID, "%s: tensors overlap", who);
  if (C > MAX_WIDTH) return fail(MABA_ERR_UNSUPPORTED, "%s: at most %d channels", who, MAX_WIDTH);
  const Geometry geo = row_geometry(C, chunk_elems(dt), forward_elems(R, C, dt), far_rows({x, y, x_out, h}));
  BoundaryArgs a = {x->data, y ? y->data : nullptr, weight ? weight->data : nullptr, post_weight ? post_weight->data : nullptr,
                    gate ? gate->data : nullptr, x_out ? x_out->data : nullptr, h ? h->data : nullptr,
                    row_stride(x), row_stride(y), row_stride(x_out), row_stride(h), R, (int)C, geo.lg, scale, eps,
                    make_drop(p, seed, stream_id)};
  if (R == 0) return MABA_OK;
  const int threads = std::max(256, 1 << geo.lg);
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(R, threads >> geo.lg), (int64_t)device_cu_count() * 8));
  with_type(dt, [&](auto type) {
    typedef decltype(type) T;
    with_chunks<T, T::CODE == MABA_F32 ? MOST_BACK : MOST_ELEMS>(geo.nch, [&](auto n) {
      constexpr int N = decltype(n)::value;
      hipLaunchKernelGGL((cut_rows(C, dt) ? boundary_kernel<T, N, true> : boundary_kernel<T, N, false>), grid, dim3(threads), 0,
                         (hipStream_t)stream, a);
    });
  });
  return check_launch(who);
}

extern "C" size_t maba_hip_residual_norm_backward_workspace_size(const maba_tensor* x, int grads) {
  if (!x || x->ndim != 2 || x->shape[1] < 1 || !is_float_dt(x->dtype) || !(grads & 7)) return 0;
  if (x->shape[1] > MAX_WIDTH) return 0;
  const int64_t R = x->shape[0], C = x->shape[1];
  int groups = 0;
  for (const bool far : {false, true})               // which of them the call takes depends on all its tensors' strides
    groups = std::max(groups, back_groups(R, row_geometry(C, chunk_elems(x->dtype), back_elems(R, C, x->dtype), far), cut_rows(C, x->dtype)));
  return (size_t)groups * __builtin_popcount(grads & 7) * C * sizeof(float);
}

extern "C" int maba_hip_residual_norm_backward(const maba_tensor* dx_out, const maba_tensor* dh, const maba_tensor* x,
                                               const maba_tensor* y, const maba_tensor* weight, const maba_tensor* post_weight,
                                               const maba_tensor* gate, float scale, double p, const int64_t* seed,
                                               uint32_t stream_id, float eps, maba_tensor* dx, maba_tensor* dy,
                                               maba_tensor* dweight, maba_tensor* dpost_weight, maba_tensor* dgate,
                                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "residual_norm_backward";
  int rc = check_float_rows(x, who);
  if (!rc) rc = check_drop(who, p, seed);
  if (!rc && (dh || x->data)) rc = check_rows(x, who, "x", x->dtype, -1, -1);
  if (rc) return rc;
  const int64_t R = x->shape[0], C = x->shape[1];
  const int dt = x->dtype;
  if (!dx_out && !dh) return fail(MABA_ERR_INVALID, "%s: dx_out or dh is required", who);
  if (dh && !weight) return fail(MABA_ERR_INVALID, "%s: dh goes with weight", who);
  if (!y && (post_weight || dpost_weight || dgate)) return fail(MABA_ERR_INVALID, "%s: post_weight and its and gate's gradients go with y", who);
  if (dh && dy && !y) return fail(MABA_ERR_INVALID, "%s: with dh, dy goes with y", who);
  if ((dpost_weight && !post_weight) || (dgate && !gate) || (dweight && !weight))
    return fail(MABA_ERR_INVALID, "%s: a gradient of a missing parameter", who);
  for (const auto& t : {std::make_pair(dx_out, "dx_out"), std::make_pair(dh, "dh"), std::make_pair(y, "y")})
    if (!rc && t.first) rc = check_rows(t.first, who, t.second, dt, R, C);
  for (const auto& t : {std::make_pair(weight, "weight"), std::make_pair(post_weight, "post_weight"), std::make_pair(gate, "gate"),
                        std::make_pair((const maba_tensor*)dweight, "dweight"),
                        std::make_pair((const maba_tensor*)dpost_weight, "dpost_weight"),
                        std::make_pair((const maba_tensor*)dgate, "dgate")})
    if (!rc && t.first) rc = check_vec(t.first, who, t.second, dt, C);
  if (!rc && dx) rc = check_out(dx, who, "dx", dt, R, C);
  if (!rc && dy) rc = check_out(dy, who, "dy", dt, R, C);
  if (rc) return rc;
  maba_tensor* outs[] = {dx, dy, dweight, dpost_weight, dgate};
  const maba_tensor* rx = dh ? x : nullptr;                // x as it is read
  for (int i = 0; i < 5; ++i) {
    for (const maba_tensor* in : {dx_out, dh, rx, y, weight, post_weight, gate})
      if (overlap(outs[i], in)) return fail(MABA_ERR_INVALID, "%s: an output overlaps an input", who);
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return fail(MABA_ERR_INVALID, "%s: outputs overlap", who);
  }
  if (C > MAX_WIDTH) return fail(MABA_ERR_UNSUPPORTED, "%s: at most %d channels", who, MAX_WIDTH);
  const Geometry geo = row_geometry(C, chunk_elems(dt), back_elems(R, C, dt), far_rows({dx_out, dh, rx, y, dx, dy}));
  const int grads = (dweight ? GRAD_W : 0) | (dgate ? GRAD_GATE : 0) | (dpost_weight ? GRAD_POST : 0);
  if (!grads && !dx && !dy) return MABA_OK;
  const int groups = back_groups(R, geo, cut_rows(C, dt)), n = __builtin_popcount(grads);
  rc = ffn::check_workspace(who, workspace, workspace_bytes, (size_t)groups * n * C * sizeof(float));
  if (rc) return rc;
  const bool need_y = y && (dh || post_weight || dgate);
  BoundaryBackArgs a = {dx_out ? dx_out->data : nullptr, dh ? dh->data : nullptr, rx ? rx->data : nullptr, need_y ? y->data : nullptr,
                        weight ? weight->data : nullptr, post_weight ? post_weight->data : nullptr, gate ? gate->data : nullptr,
                        dx ? dx->data : nullptr, dy ? dy->data : nullptr, (float*)workspace,
                        row_stride(dx_out), row_stride(dh), row_stride(rx), row_stride(y), row_stride(dx), row_stride(dy), R, (int)C,
                        geo.lg, grads, cut_rows(C, dt), scale, eps, make_drop(p, seed, stream_id)};
  if (R > 0) {
    const int threads = back_size(R, geo, cut_rows(C, dt));
    const size_t params = (size_t)(post_weight ? 3 : 2) * ceil_div(C, chunk_elems(dt)) * 16;
    const size_t lds = std::max(params, grads ? (size_t)(post_weight ? 3 : 2) * threads * chunk_elems(dt) * sizeof(float) : 0);
    const bool whole = whole_rows({dx_out, dh, rx, y, dx, dy});
    with_type(dt, [&](auto type) {
      typedef decltype(type) T;
      auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(threads), lds, (hipStream_t)stream, a);
      };
      if (post_weight)
        with_chunks<T, MOST_BACK>(geo.nch, [&](auto n) {
          constexpr int N = decltype(n)::value;
          run(whole ? boundary_back_kernel<T, N, true, true> : boundary_back_kernel<T, N, true, false>);
        });
      else
        with_chunks<T, MOST_BACK>(geo.nch, [&](auto n) {
          constexpr int N = decltype(n)::value;
          run(whole ? boundary_back_kernel<T, N, false, true> : boundary_back_kernel<T, N, false, false>);
        });
    });
    rc = check_launch(who);
    if (rc) return rc;
  }
  if (grads) {
    ColumnsArgs c = {(const float*)workspace, {}, {}, R > 0 ? groups : 0, n, (int)C};
    int k = 0;
    if (dweight) { c.out[k] = dweight->data; c.factor[k++] = 1.f; }
    if (dgate) { c.out[k] = dgate->data; c.factor[k++] = scale * a.d.keep; }
    if (dpost_weight) { c.out[k] = dpost_weight->data; c.factor[k++] = 1.f; }
    auto f = dt == MABA_F32 ? columns_kernel<F32> : dt == MABA_BF16 ? columns_kernel<Bf16> : columns_kernel<Fp16>;
    hipLaunchKernelGGL(f, dim3((unsigned)ceil_div(C, 32), n), dim3(1024), 0, (hipStream_t)stream, c);
    return check_launch(who);
  }
  return MABA_OK;
}
