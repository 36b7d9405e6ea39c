// What the gated block and the linear layer share around the matrix-product core: launches with
// their tile, operand copies where the core cannot read a tensor in place, and reductions.
#pragma once

#include <algorithm>

#include "ffn_gemm.h"

namespace maba {
namespace ffn {

// ---------------------------------------------------------------- copies and reductions (ffn_common.hip)

// dst [rows, chunks * 8] (contiguous) = src [rows, cols] with zeros behind each row, of 16-bit elements at any
// alignment, times gate[row] and 2^*exponent where there are any; with scales: src holds the e4m3 codes of a packed activation,
// dst its values.
struct CopyJob {
  const void* src; int64_t ld;
  const uint8_t* scales; int64_t scale_ld;
  const uint16_t* gate;
  const int* exponent;
  int64_t rows;
  int cols, chunks;
  uint16_t* dst;
};
constexpr int MAX_COPIES = 3;
// A call's copies, made by one launch.
struct Copies {
  CopyJob job[MAX_COPIES];
  int count = 0;
  void add(const maba_tensor* src, const maba_tensor* scales, uint16_t* dst, const maba_tensor* gate = nullptr,
           const int* exponent = nullptr) {
    job[count++] = {src->data, src->stride[0], scales ? (const uint8_t*)scales->data : nullptr, scales ? scales->stride[0] : 0,
                    gate ? (const uint16_t*)gate->data : nullptr, exponent, src->shape[0], (int)src->shape[1],
                    (int)((src->shape[1] + 7) / 8), dst};
  }
  int launch(int dtype, hipStream_t s) const;
};

// out = the sum of `splits` fp32 partials [splits][M][N] in split order, times 2^-*exponent where there is one, rounded
// to 16 bits; row m goes to row m of out[0], or from `second` on to row m - second of out[1]; only `rows` rows of each
// are written, and nothing to a null one.
struct ReduceArgs {
  const float* p;
  int splits, M, N, second, rows, ncols;
  Rows out[2];
  const int* exponent;
};
int reduce_splits(const ReduceArgs& a, int dtype, hipStream_t s);

// out[t][n] = the sum over r of p[r][t][n] (fp32 partials [R][2][N], t = 0, 1; a null out is skipped), 16 bits; with a
// gate out[0] is multiplied by it; sum[n] is t = 0's in fp32.
int reduce_columns(const float* p, int64_t R, int N, void* out0, void* out1, const void* gate, float* sum, int dtype, hipStream_t s);

// For G = the sum of `splits` partials [splits][M][N]: dw = gate * G, dgate[m] = <w[m], G[m]> + bias[m] colsum[m]; a null
// dw or dgate is skipped.
struct GatedReduceArgs {
  const float* p;
  int splits, M, N, ncols;
  Rows dw, w;
  const uint16_t *gate, *bias;
  const float* colsum;
  uint16_t* dgate;
};
int reduce_gated(const GatedReduceArgs& a, int rows, int dtype, hipStream_t s);

// p[r][0][n] = the sum of rows [128 r, 128 r + 128) of src [M, N] (16-bit), [ceil(M / 128)][2][N].
int column_partials(const maba_tensor* src, float* p, hipStream_t s);

// What a backward pass makes as a 16-bit operand of its next products ([dg | du], dz, gate * W) is held in fp16 as its
// value times 2^e, and the products' results are multiplied by 2^-e: fp16's own range loses small gradients and gates
// below its smallest step and turns large ones into infinities, which fp32 does not.  e is the largest with
// bound * 2^e <= 2^15 for a bound of the operand's magnitudes made before it, as a product of up to three factors: each
// is the largest element of some tensors, or the largest norm of their rows.  So every operand is below 2^16, and
// one of 2^-28 of the bound still has all of fp16's bits.  bf16 has fp32's range and takes none of this.
//
// (Elements that are not finite do not count: their rows' results are not finite either.)
constexpr int MAX_FACTORS = 3, MAX_MAGNITUDES = 4, MAGNITUDE_GROUPS = 2048;
struct Magnitude {
  const uint16_t* p; int64_t ld, cols, segments;      // of a row, SEGMENT elements each
  int64_t units;                                       // segments of all rows
  int factor, norm;
};
struct Magnitudes {
  static constexpr int SEGMENT = 1024;
  Magnitude job[MAX_MAGNITUDES];
  int count = 0;
  void add(int factor, const void* p, int64_t ld, int64_t rows, int64_t cols, bool norm) {
    if (!norm && ld == cols) {                         // elements one after another
      cols *= rows;
      rows = 1;
    }
    const int64_t segments = ceil_div(cols, SEGMENT);
    job[count++] = {(const uint16_t*)p, ld, cols, segments, rows * segments, factor, norm};
  }
  // *exponent = e; partial: MAX_FACTORS * MAGNITUDE_GROUPS floats of workspace.
  int launch(float slope, float* partial, int* exponent, hipStream_t s) const;
};

// ---------------------------------------------------------------- launches

// The tiles: BM, BN, waves along m and n, stages in LDS, groups of waves.  Two stages leave room for other workgroups on
// the compute unit, which hide the loads better than more stages do; Tile64Deep is for rows whose few tiles are all
// resident at once (64 rows, 2,048 to 2 x 5,504, weights from HBM: 26.1 us with two stages, 16.7 with three, 14.3 with
// four; 2,048 rows, 1,248 to 640 with a residual, 320 tiles: 14.6 with two, 13.2 with four; 4,096 rows, 640 tiles: 15.4
// with two, 19.2 with four).
struct Tile256 { static constexpr int BM = 256, BN = 256, WM = 2, WN = 4, ST = 2, KG = 1; };
struct Tile192 { static constexpr int BM = 192, BN = 128, WM = 2, WN = 2, ST = 2, KG = 1; };
struct Tile160 { static constexpr int BM = 128, BN = 160, WM = 4, WN = 1, ST = 2, KG = 1; };
struct Tile128 { static constexpr int BM = 128, BN = 128, WM = 2, WN = 2, ST = 2, KG = 1; };
struct Tile64 { static constexpr int BM = 64, BN = 64, WM = 2, WN = 2, ST = 2, KG = 1; };
struct Tile160Two { static constexpr int BM = 128, BN = 160, WM = 4, WN = 1, ST = 2, KG = 2; };
struct Tile128Two { static constexpr int BM = 128, BN = 128, WM = 2, WN = 2, ST = 2, KG = 2; };
struct Tile64Two { static constexpr int BM = 64, BN = 64, WM = 2, WN = 2, ST = 2, KG = 2; };
struct Tile64Deep { static constexpr int BM = 64, BN = 64, WM = 2, WN = 2, ST = 4, KG = 1; };

// How a product runs: which tile, and into how many runs of stages its sum is split (more than one writes fp32
// partials that reduce_splits adds).
struct GemmPlan {
  int tile, splits, split_stages, tiles_m;
};
// An operand is read along its columns; the sum may be split; the columns are a gate's and an up's by turns; the
// epilogue takes long and many registers, and no tile that has a compute unit to itself is taken; the epilogue can do with
// half of a tile's rows, so that two groups of waves may share a tile (KG = 2).
enum { PLAN_COLUMNS = 1, PLAN_SPLIT = 2, PLAN_PAIRS = 4, PLAN_LONG = 8, PLAN_GROUPS = 16 };
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t stages, int what);

template <class T, class Tile, int AMODE, int BMODE, class Epi>
int gemm_tile(GemmArgs& g, const typename Epi::Args& e, int64_t M, int64_t N, int splits, hipStream_t s, const char* who) {
  g.tiles_m = (int)ceil_div(M, Tile::BM);
  g.tiles_n = (int)ceil_div(N, Tile::BN);
  const int64_t grid = (int64_t)g.tiles_m * g.tiles_n * splits;
  if (grid > INT32_MAX) return fail(MABA_ERR_UNSUPPORTED, "%s: too many tiles", who);
  hipLaunchKernelGGL((gemm_kernel<T, Tile::BM, Tile::BN, Tile::WM, Tile::WN, Tile::ST, AMODE, BMODE, Epi, Tile::KG>),
                     dim3((unsigned)grid), dim3(64 * Tile::WM * Tile::WN * Tile::KG), 0, s, g, e);
  return check_launch(who);
}

inline int64_t gemm_stages(int64_t K, int segments) { return ceil_div(K, GEMM_BK) * segments; }

template <class T, int AMODE, int BMODE, class Epi>
int gemm(GemmArgs g, const typename Epi::Args& e, int64_t M, int64_t N, const GemmPlan& p, hipStream_t s, const char* who) {
  g.segments = g.segments ? g.segments : 1;
  g.split_stages = p.split_stages;
  switch (p.tile) {
    case 0:
      if constexpr (!Epi::LONG) return gemm_tile<T, Tile256, AMODE, BMODE, Epi>(g, e, M, N, p.splits, s, who);
      else return fail(MABA_ERR_INVALID, "%s: no such tile", who);
    case 1: return gemm_tile<T, Tile192, AMODE, BMODE, Epi>(g, e, M, N, p.splits, s, who);
    case 2:
      if constexpr (BMODE != K_ROWS_PAIR) return gemm_tile<T, Tile160, AMODE, BMODE, Epi>(g, e, M, N, p.splits, s, who);
      else return fail(MABA_ERR_INVALID, "%s: no such tile", who);
    case 3: return gemm_tile<T, Tile128, AMODE, BMODE, Epi>(g, e, M, N, p.splits, s, who);
    case 5:
    case 6:
    case 7:
      if constexpr (Epi::GROUPS && AMODE == K_ROWS)
        return p.tile == 5   ? gemm_tile<T, Tile160Two, AMODE, BMODE, Epi>(g, e, M, N, 1, s, who)
               : p.tile == 6 ? gemm_tile<T, Tile128Two, AMODE, BMODE, Epi>(g, e, M, N, 1, s, who)
                             : gemm_tile<T, Tile64Two, AMODE, BMODE, Epi>(g, e, M, N, 1, s, who);
      else return fail(MABA_ERR_INVALID, "%s: no such tile", who);
    default:
      if constexpr (AMODE == K_ROWS && BMODE != K_COLS)
        if (ceil_div(M, 64) * ceil_div(N, 64) * p.splits <= 2 * device_cu_count())
          return gemm_tile<T, Tile64Deep, AMODE, BMODE, Epi>(g, e, M, N, p.splits, s, who);
      return gemm_tile<T, Tile64, AMODE, BMODE, Epi>(g, e, M, N, p.splits, s, who);
  }
}

// A product of M x Np in 16-bit outputs of N columns, through fp32 partials where its plan splits it: rows from
// `second` on (a multiple of 16, or M and more: none) are the second output's; either may be null, and has `rows` rows.
struct Outputs {
  Rows out[2];
  int second, rows, N;
  const int* exponent;       // the operands' power of two, taken out of the result
};
template <class T, int AMODE, int BMODE>
int product_to(const GemmArgs& g, const Outputs& o, int64_t M, int64_t Np, const GemmPlan& p, float* part, hipStream_t s,
               const char* who) {
  if (p.splits == 1) {
    const EpiStore::Args e = {{o.out[0], o.out[1]}, o.second, o.rows, o.N, o.exponent};
    return gemm<T, AMODE, BMODE, EpiStore>(g, e, M, Np, p, s, who);
  }
  const EpiPartial::Args e = {part, (int)M, (int)Np};
  if (int rc = gemm<T, AMODE, BMODE, EpiPartial>(g, e, M, Np, p, s, who)) return rc;
  const ReduceArgs r = {part, p.splits, (int)M, (int)Np, o.second, o.rows, o.N, {o.out[0], o.out[1]}, o.exponent};
  return reduce_splits(r, T::CODE, s);
}
// Zeros in the outputs, for a sum over no rows.
template <class T>
int zeros_to(const Outputs& o, int64_t M, int64_t Np, hipStream_t s) {
  const ReduceArgs r = {nullptr, 0, (int)M, (int)Np, o.second, o.rows, o.N, {o.out[0], o.out[1]}, nullptr};
  return reduce_splits(r, T::CODE, s);
}

// ---------------------------------------------------------------- argument checks

// A 2-D 16-bit tensor [rows, cols] (-1: any) with unit column stride.
inline int check_rows(const maba_tensor* t, const char* who, const char* name, int dtype, int64_t rows, int64_t cols) {
  if (!t) return fail(MABA_ERR_INVALID, "%s: %s is missing", who, name);
  if (t->ndim != 2) return fail(MABA_ERR_INVALID, "%s: %s must be 2D, got %dD", who, name, t->ndim);
  if ((rows >= 0 && t->shape[0] != rows) || (cols >= 0 && t->shape[1] != cols))
    return fail(MABA_ERR_INVALID, "%s: %s is [%lld, %lld], expected [%lld, %lld]", who, name, (long long)t->shape[0],
                (long long)t->shape[1], (long long)rows, (long long)cols);
  if (t->dtype != dtype) return fail(MABA_ERR_DTYPE, "%s: %s has dtype code %d, expected %d", who, name, t->dtype, dtype);
  if (t->shape[1] > 1 && t->stride[1] != 1) return fail(MABA_ERR_INVALID, "%s: %s needs unit column stride", who, name);
  if (t->stride[0] < 0) return fail(MABA_ERR_INVALID, "%s: %s has a negative stride", who, name);
  if (t->shape[0] > 0 && t->shape[1] > 0 && !t->data) return fail(MABA_ERR_INVALID, "%s: %s has no data", who, name);
  return MABA_OK;
}
// An output: like check_rows, and its rows must not overlap one another.
inline int check_out(const maba_tensor* t, const char* who, const char* name, int dtype, int64_t rows, int64_t cols) {
  const int rc = check_rows(t, who, name, dtype, rows, cols);
  if (rc) return rc;
  if (t->shape[0] > 1 && t->stride[0] < t->shape[1]) return fail(MABA_ERR_INVALID, "%s: rows of %s overlap", who, name);
  return MABA_OK;
}
inline int check_vec(const maba_tensor* t, const char* who, const char* name, int dtype, int64_t n) {
  if (t->ndim != 1 || t->shape[0] != n) return fail(MABA_ERR_INVALID, "%s: %s must be [%lld]", who, name, (long long)n);
  if (t->dtype != dtype) return fail(MABA_ERR_DTYPE, "%s: %s has dtype code %d, expected %d", who, name, t->dtype, dtype);
  if (n > 1 && t->stride[0] != 1) return fail(MABA_ERR_INVALID, "%s: %s needs unit stride", who, name);
  if (!t->data) return fail(MABA_ERR_INVALID, "%s: %s has no data", who, name);
  return MABA_OK;
}
// Widths and row counts the kernels index with 32 bits.
inline int check_sizes(const char* who, int64_t M, int64_t N, int64_t K) {
  if (N < 1 || K < 1) return fail(MABA_ERR_INVALID, "%s: widths must be positive, got %lld and %lld", who, (long long)N, (long long)K);
  if (M > (1 << 30) || N > (1 << 20) || K > (1 << 20)) return fail(MABA_ERR_UNSUPPORTED, "%s: sizes out of range", who);
  return MABA_OK;
}
// The bytes that a tensor's elements span, as [first, last); and whether two spans meet.
inline bool overlap(const maba_tensor* a, const maba_tensor* b) {
  if (!a || !b) return false;
  auto span = [](const maba_tensor* t, uintptr_t& lo, uintptr_t& hi) {
    const int64_t size = t->dtype == MABA_F32 ? 4 : t->dtype == MABA_E4M3 || t->dtype == MABA_U8 ? 1 : 2;
    int64_t last = 0;
    for (int i = 0; i < t->ndim; ++i) {
      if (t->shape[i] == 0) return false;
      last += (t->shape[i] - 1) * t->stride[i];
    }
    lo = (uintptr_t)t->data;
    hi = lo + (uintptr_t)((last + 1) * size);
    return true;
  };
  uintptr_t al, ah, bl, bh;
  return span(a, al, ah) && span(b, bl, bh) && al < bh && bl < ah;
}

// x of a backward pass: 16-bit rows, or the codes of a packed activation and their scales.
inline int check_kept(const maba_tensor* x, const maba_tensor* scales, const char* who, int dtype, int64_t M, int64_t K) {
  if (!scales) return check_rows(x, who, "x", dtype, M, K);
  int rc = check_rows(x, who, "the codes of x", MABA_E4M3, M, K);
  if (!rc) rc = check_rows(scales, who, "the scales of x", MABA_U8, M, ceil_div(K, 32));
  return rc;
}

// What a call needs of its workspace: the bytes, at an address that 16-byte accesses can take.
inline int check_workspace(const char* who, const void* p, size_t bytes, size_t need) {
  if (need == 0) return MABA_OK;
  if (!p || bytes < need) return fail(MABA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, p ? bytes : 0, need);
  if ((uintptr_t)p % 16) return fail(MABA_ERR_INVALID, "%s: the workspace must be 16-byte aligned", who);
  return MABA_OK;
}

// A workspace handed out front to back in 256-byte steps.
struct Carve {
  char* p;
  size_t used;
  template <class U>
  U* take(size_t n) {
    U* r = (U*)(p ? p + used : nullptr);
    used += up256(n * sizeof(U));
    return r;
  }
};

// p [rows][..] read along its rows; and the same [krows][cols] read along its columns.
inline Operand rows_operand(const uint16_t* p, int64_t ld, int64_t rows) {
  Operand o = {};
  o.p[0] = o.p[1] = p;
  o.ld[0] = o.ld[1] = ld;
  o.rows = (int)rows;
  return o;
}
inline Operand cols_operand(Operand o, int64_t cols) {
  o.krows = o.rows;
  o.rows = (int)cols;
  return o;
}

}  // namespace ffn
}  // namespace maba
