// Copies and reductions of the feed-forward operators.
#include <algorithm>

#include "ffn_common.h"

namespace maba {
namespace ffn {

// The plan is the least of a sum's estimated times over the tiles and splits.  A compute unit with n tiles takes for
// each its stages at `full` and `ends` for its first loads and its epilogue; with fewer than `slots`, which is what it
// holds at once, a stage's latency (`lone`) bounds it.  Measured on MI355X, us, with an operand read along its columns
// in brackets:
//              256 x 256      192 x 128      128 x 160      128 x 128      64 x 64
//   full       1.36 (1.38)    0.55 (0.63)    0.57 (0.64)    0.46 (0.50)    0.20 (0.25)
//   lone       1.36 (1.38)    0.80 (1.00)    0.75 (0.95)    0.60 (0.74)    0.36 (0.47)
//   ends       9              4              3              3              0.75
// Over 31 products of rows and columns, in up to twelve splits, each timed with every tile of one group
// (profiles/feed_forward_tiles.txt), the plan's choice of the timed ones takes 1.6 % more than the best of them on
// average, 20 % at most and but for that one 9 %.  (4,096 x 11,008 x 2,048, rows: 150, 169, -, 175 us with the first four; 16,384 x 640 x 2,496, columns: 70, 58,
// 56, 79, and 32,768 x 640 x 1,248, rows: 70, 64, 58, 63, where 160 columns leave no part of a tile over; 16,384 x 2,496 x 640,
// rows: 60, 54, -, 57, the smallest 81; 64 x 640 x 2,496 with the last, in 1, 4 and 8 splits: 19.9, 7.2 and 5.2.)  The smallest
// tile is priced with two stages; rows whose few tiles are all resident then run it with four (Tile64Deep).
//
// Two groups of waves on a tile (`groups`; a stage is then two) serve tiles too few to share a compute unit.  Its one
// group of four waves keeps the matrix units 26 % busy; a second workgroup's would do the same as a second group.
// 640 columns, k = 2 x 1,248, of 8,191, 6,000 and 2,048 rows: 41 us -> 35 (128 x 160), 36 -> 31 (128 x 128), 26 -> 20.5
// (64 x 64).  With more tiles than that they cost more (8,191 rows in 128 x 128: 58) and are not taken.
//              128 x 160      128 x 128      64 x 64
//   full       1.20 (1.45)    0.95 (1.27)    0.47 (0.46)
//   lone       1.20 (1.45)    0.95 (1.27)    0.60 (0.60)
//   ends       5              5              0.9
struct TileCost { int bm, bn, slots, groups; float full[2], lone[2], ends; };
constexpr int TILE_COUNT = 8;
static const TileCost TILES[TILE_COUNT] = {{256, 256, 1, 1, {1.36f, 1.38f}, {1.36f, 1.38f}, 9.f},
                                           {192, 128, 2, 1, {0.55f, 0.63f}, {0.80f, 1.00f}, 4.f},
                                           {128, 160, 2, 1, {0.57f, 0.64f}, {0.75f, 0.95f}, 3.f},
                                           {128, 128, 2, 1, {0.46f, 0.50f}, {0.60f, 0.74f}, 3.f},
                                           {64, 64, 5, 1, {0.20f, 0.25f}, {0.36f, 0.47f}, 0.75f},
                                           {128, 160, 1, 2, {1.20f, 1.45f}, {1.20f, 1.45f}, 5.f},
                                           {128, 128, 1, 2, {0.95f, 1.27f}, {0.95f, 1.27f}, 5.f},
                                           {64, 64, 2, 2, {0.47f, 0.46f}, {0.60f, 0.60f}, 0.9f}};

GemmPlan gemm_plan(int64_t M, int64_t N, int64_t stages, int what) {
  const bool columns = what & PLAN_COLUMNS, may_split = what & PLAN_SPLIT;
  const int64_t cus = device_cu_count();
  stages = std::max<int64_t>(stages, 1);      // no rows: nothing is launched
  GemmPlan best = {};
  float least = 0.f;
  for (int i = 0; i < TILE_COUNT; ++i) {
    const TileCost& t = TILES[i];
    if (t.bn % 64 && (what & PLAN_PAIRS)) continue;      // whose epilogue takes 64 columns at a time
    if (t.slots == 1 && (what & PLAN_LONG)) continue;
    if (t.groups > 1 && !(what & PLAN_GROUPS)) continue;
    const int64_t tiles = ceil_div(M, t.bm) * ceil_div(N, t.bn);
    const int most = may_split && t.groups == 1 ? (int)std::max<int64_t>(1, std::min<int64_t>({32, stages / 2, 8 * cus / std::max<int64_t>(tiles, 1)})) : 1;
    for (int want = 1; want <= most; ++want) {
      const int64_t per = ceil_div(stages, want), splits = ceil_div(stages, per);
      if (splits != want) continue;
      const int64_t n = ceil_div(tiles * splits, cus);
      if (t.groups > 1 && n > t.slots) continue;
      const int64_t turns = ceil_div(per, t.groups);
      float us = n * (turns * t.full[columns] + t.ends);
      if (n < t.slots) us = std::max(us, turns * t.lone[columns] + t.ends);
      if (splits > 1) us += 2.5f + (float)(M * N) * (8.f * splits + 2.f) / 5e6f;     // the partials, at 5 TB/s
      if (least == 0.f || us < least) {
        least = us;
        best = {i, (int)splits, (int)per, (int)ceil_div(M, t.bm)};
      }
    }
  }
  return best;
}

// A thread makes eight elements of a padded row of one of the launch's copies.  Bound by the launch or by HBM.  A
// workgroup's chunks belong to one copy, so that its description is read once, by scalar loads (unpacking 16,384 x
// 1,248 codes: 15.4 us; 18.4 with a thread's copy found by itself).
struct CopyArgs {
  CopyJob job[MAX_COPIES];
  int64_t end[MAX_COPIES];     // workgroups of 256 chunks up to and with each copy's
};

// The values of e4m3 codes: code * 2^e, exact in fp32, rounded once to T (a bf16 holds it exactly unless it is
// subnormal there).
template <class T>
__device__ __forceinline__ u32x4 unpack8(u32x2 w, int e) {
  u32x4 v;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
    v[2 * h] = T::down(scaled(a[0], e, T::MOST)) | (T::down(scaled(a[1], e, T::MOST)) << 16);
    v[2 * h + 1] = T::down(scaled(b[0], e, T::MOST)) | (T::down(scaled(b[1], e, T::MOST)) << 16);
  }
  return v;
}

template <class T>
__global__ __launch_bounds__(256) void copy_rows_kernel(CopyArgs a) {
  typedef u32x2 u32x2_byte __attribute__((aligned(1)));
  for (int64_t b = blockIdx.x; b < a.end[MAX_COPIES - 1]; b += gridDim.x) {
    const int t = b < a.end[0] ? 0 : b < a.end[1] ? 1 : 2;
    const CopyJob& c = a.job[t];
    const int64_t first = (b - (t ? a.end[t - 1] : 0)) * 256, at = first + threadIdx.x, r0 = first / c.chunks;
    if (at >= c.rows * c.chunks) continue;
    const uint32_t local = (uint32_t)(first - r0 * c.chunks) + threadIdx.x, dr = local / (uint32_t)c.chunks;
    const int64_t r = r0 + dr;
    const int k = (int)(local - dr * (uint32_t)c.chunks) * 8, n = c.cols - k;
    u32x4 v = {0, 0, 0, 0};
    if (c.scales) {
      const uint8_t* p = (const uint8_t*)c.src + r * c.ld + k;
      u32x2 w = {0, 0};
      if (n >= 8) w = *(const u32x2_byte*)p;
      else
#pragma unroll
        for (int j = 0; j < 7; ++j) w[j >> 2] |= (j < n ? (uint32_t)p[j] : 0u) << (8 * (j & 3));
      v = unpack8<T>(w, (int)c.scales[r * c.scale_ld + (k >> 5)] - 127);
    } else {
      const uint16_t* p = (const uint16_t*)c.src + r * c.ld + k;
      if (n >= 8) v = *(const u32x4_any*)p;
      else
#pragma unroll
        for (int j = 0; j < 7; ++j) v[j >> 1] |= (j < n ? (uint32_t)p[j] : 0u) << (16 * (j & 1));
      if (c.gate) {
        const float g = T::up(c.gate[r]) * power_of<T>(c.exponent, 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = T::down(T::up(v[j] & 0xffffu) * g) | (T::down(T::up(v[j] >> 16) * g) << 16);
      }
    }
    *(u32x4*)(c.dst + at * 8) = v;
  }
}

int Copies::launch(int dtype, hipStream_t s) const {
  CopyArgs a = {};
  int64_t total = 0;
  for (int i = 0; i < MAX_COPIES; ++i) {
    if (i < count) {
      a.job[i] = job[i];
      total += ceil_div(job[i].rows * job[i].chunks, 256);
    }
    a.end[i] = total;
  }
  if (total == 0) return MABA_OK;
  const dim3 grid((unsigned)std::min<int64_t>(total, 1 << 20));
  auto k = dtype == MABA_BF16 ? copy_rows_kernel<Bf16> : copy_rows_kernel<Fp16>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, s, a);
  return check_launch("copy_rows");
}

// Eight partials' loads are in flight at once, added in order (64 rows, 5,504 to 2,048, product and sum: 12.0 us; 13.1 one
// by one).
template <class T>
__global__ __launch_bounds__(256) void reduce_splits_kernel(ReduceArgs a) {
  const int quads = a.N / 4;
  const int64_t total = (int64_t)a.M * quads, plane = (int64_t)a.M * a.N;
  const float scale = power_of<T>(a.exponent, -1);
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) v += *(const f32x4*)(a.p + s * plane + (int64_t)m * a.N + n);
    const int t = m >= a.second, r = t ? m - a.second : m;
    if (r < a.rows && a.out[t].p) store4<T>(a.out[t], r, n, a.ncols, v * scale);
  }
}

int reduce_splits(const ReduceArgs& a, int dtype, hipStream_t s) {
  const int64_t total = (int64_t)a.M * (a.N / 4);
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(total, 256), 16384));
  auto k = dtype == MABA_BF16 ? reduce_splits_kernel<Bf16> : reduce_splits_kernel<Fp16>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, s, a);
  return check_launch("reduce_splits");
}

// Sixteen lanes take a segment of a row, 64 elements a lane loaded together, a wave four of one tensor.
// partial[f][b]: workgroup b's largest of factor f.  A norm is bounded by its largest segment's times the root of their
// number.  Bound by HBM: 34 MB (dh of 8,191 x 1,248, x of 8,191 x 640 and two weights) take 7.7 us, and 16 with a wave per
// row, where a wave waits for several rows one by one.
struct MagnitudeArgs {
  Magnitude job[MAX_MAGNITUDES];
  int64_t end[MAX_MAGNITUDES];      // fours of segments up to and with each job's
  float* partial;
};
// The finite ones of two fp16 numbers' magnitudes, zero for the others.
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  typedef __attribute__((ext_vector_type(2))) int16_t i16x2;
  const uint32_t m = v & 0x7fff7fffu;
  const i16x2 bad = __builtin_bit_cast(i16x2, m + 0x04000400u) >> 15;       // from 0x7c00 on
  return m & ~__builtin_bit_cast(uint32_t, bad);
}
__global__ __launch_bounds__(256) void magnitudes_kernel(MagnitudeArgs a) {
  constexpr int SEG = Magnitudes::SEGMENT, LOADS = SEG / 128;
  typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
  __shared__ uint32_t part[MAX_FACTORS];             // bits: they order as the magnitudes do
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  if (threadIdx.x < MAX_FACTORS) part[threadIdx.x] = 0;
  __syncthreads();
  for (int64_t u = blockIdx.x * (int64_t)4 + wave; u < a.end[MAX_MAGNITUDES - 1]; u += (int64_t)gridDim.x * 4) {
    int t = 0;
#pragma unroll
    for (int i = 0; i < MAX_MAGNITUDES - 1; ++i) t += u >= a.end[i];
    const Magnitude& j = a.job[t];
    const int64_t at = (u - (t ? a.end[t - 1] : 0)) * 4 + (lane >> 4);
    const bool in = at < j.units;
    int64_t row = 0, seg = 0;                        // both 0 past the end, where nothing is read
    if (j.segments == 1) row = at;
    else if (j.segments == j.units) seg = at;
    else row = at / j.segments, seg = at - row * j.segments;
    const Rows r = {(uint16_t*)j.p + (in ? row * j.ld + seg * SEG : 0), 0};
    const int n = in ? (int)min(j.cols - seg * SEG, (int64_t)SEG) : 0;
    u32x4 v[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) v[i] = load8(r, 0, 8 * (lane & 15) + 128 * i, n ? 1 : 0, n);
    float x = 0.f;
    if (j.norm) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float lo = Fp16::up(v[i][h] & 0xffffu), hi = Fp16::up(v[i][h] >> 16);
          x = fmaf(hi, hi, fmaf(lo, lo, x));
        }
      x = x < 3e38f ? x : 0.f;                       // not finite: nor are the products of this row
      x = sqrtf(sum16(x) * (float)j.segments);
    } else {
      u16x2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
#pragma unroll
        for (int h = 0; h < 4; ++h) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, finite2(v[i][h])));
      x = Fp16::up(max((uint32_t)m[0], (uint32_t)m[1]));
      x = max16(x);
    }
    if ((lane & 15) == 0) atomicMax(&part[j.factor], __float_as_uint(x));
  }
  __syncthreads();
  if (threadIdx.x < MAX_FACTORS) a.partial[threadIdx.x * MAGNITUDE_GROUPS + blockIdx.x] = __uint_as_float(part[threadIdx.x]);
}

// bound = 1.25 slope * the factors' product (the quarter covers the rounding of the sums that the operand is made of
// and of these); a wave reads a factor's partials.  2 us, most of it the launch.
__global__ __launch_bounds__(64 * MAX_FACTORS) void exponent_kernel(const float* partial, int groups, int factors, float slope,
                                                                    int* exponent) {
  __shared__ float part[MAX_FACTORS];
  const int f = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float x = 0.f;
#pragma unroll 8
  for (int i = lane; i < groups; i += 64) x = fmaxf(x, partial[f * MAGNITUDE_GROUPS + i]);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x = fmaxf(x, __shfl_xor(x, s));
  if (lane == 0) part[f] = f < factors ? x : 1.f;
  __syncthreads();
  if (threadIdx.x == 0) {
    float bound = 1.25f * slope;
#pragma unroll
    for (int i = 0; i < MAX_FACTORS; ++i) bound *= part[i];
    // bound < 2^(E + 1)
    const int e = 14 - ((int)(__float_as_uint(bound) >> 23) - 127);
    *exponent = bound > 0.f ? min(e, 100) : 0;
  }
}

int Magnitudes::launch(float slope, float* partial, int* exponent, hipStream_t s) const {
  MagnitudeArgs a = {};
  int64_t total = 0;
  int factors = 0;
  for (int i = 0; i < MAX_MAGNITUDES; ++i) {
    if (i < count) {
      a.job[i] = job[i];
      total += ceil_div(job[i].units, 4);
      factors = std::max(factors, job[i].factor + 1);
    }
    a.end[i] = total;
  }
  a.partial = partial;
  const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(total, 4), MAGNITUDE_GROUPS));
  hipLaunchKernelGGL(magnitudes_kernel, dim3(groups), dim3(256), 0, s, a);
  if (int rc = check_launch("magnitudes")) return rc;
  hipLaunchKernelGGL(exponent_kernel, dim3(1), dim3(64 * MAX_FACTORS), 0, s, partial, groups, factors, slope, exponent);
  return check_launch("exponent");
}

// A workgroup a row of G = sum of the partials: dw = gate * G, and dgate = <w, G> (+ bias * colsum, added by the caller's
// term), the lanes' parts added in a fixed order.
template <class T>
__global__ __launch_bounds__(256) void reduce_gated_kernel(GatedReduceArgs a) {
  __shared__ float part[4];
  const int m = blockIdx.x, wave = threadIdx.x >> 6;
  const int64_t plane = (int64_t)a.M * a.N;
  const float gate = T::up(a.gate[m]);
  float dot = 0.f;
  for (int n = threadIdx.x * 4; n < a.ncols; n += 1024) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) v += *(const f32x4*)(a.p + s * plane + (int64_t)m * a.N + n);
    if (a.dgate) {
      const f32x4 w = up4<T>(load4(a.w, m, n, a.ncols));
      dot += v[0] * w[0] + v[1] * w[1] + v[2] * w[2] + v[3] * w[3];
    }
    if (a.dw.p) store4<T>(a.dw, m, n, a.ncols, v * gate);
  }
  if (a.dgate) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) dot += __shfl_xor(dot, s);
    if ((threadIdx.x & 63) == 0) part[wave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
      float v = part[0] + part[1] + part[2] + part[3];
      if (a.bias) v += T::up(a.bias[m]) * a.colsum[m];
      a.dgate[m] = (uint16_t)T::down(v);
    }
  }
}

int reduce_gated(const GatedReduceArgs& a, int rows, int dtype, hipStream_t s) {
  auto k = dtype == MABA_BF16 ? reduce_gated_kernel<Bf16> : reduce_gated_kernel<Fp16>;
  hipLaunchKernelGGL(k, dim3((unsigned)rows), dim3(256), 0, s, a);
  return check_launch("reduce_gated");
}

// 32 columns of one output a workgroup, eight threads each, added through LDS in a fixed order.
template <class T>
__global__ __launch_bounds__(256) void reduce_columns_kernel(const float* p, int64_t R, int N, uint16_t* out0, uint16_t* out1,
                                                             const uint16_t* gate, float* sum) {
  __shared__ float part[8][32];
  uint16_t* out = blockIdx.y ? out1 : out0;
  if (!out && !sum) return;
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, n = blockIdx.x * 32 + col;
  float v = 0.f;
  if (n < N)
    for (int64_t r = lane; r < R; r += 8) v += p[(r * 2 + blockIdx.y) * N + n];
  part[lane][col] = v;
  __syncthreads();
  if (lane == 0 && n < N) {
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) w += part[i][col];
    if (sum) sum[n] = w;
    if (out) out[n] = (uint16_t)T::down(gate ? w * T::up(gate[n]) : w);
  }
}

int reduce_columns(const float* p, int64_t R, int N, void* out0, void* out1, const void* gate, float* sum, int dtype, hipStream_t s) {
  auto k = dtype == MABA_BF16 ? reduce_columns_kernel<Bf16> : reduce_columns_kernel<Fp16>;
  hipLaunchKernelGGL(k, dim3((unsigned)ceil_div(N, 32), out1 ? 2 : 1), dim3(256), 0, s, p, R, N, (uint16_t*)out0, (uint16_t*)out1,
                     (const uint16_t*)gate, sum);
  return check_launch("reduce_columns");
}

// A wave adds 64 columns of 32 rows, a workgroup of four its 128 rows through LDS.
template <class T>
__global__ __launch_bounds__(256) void column_partials_kernel(const uint16_t* src, int64_t ld, int64_t M, int N, float* p) {
  __shared__ float part[4][64];
  const int col = threadIdx.x & 63, w = threadIdx.x >> 6, n = blockIdx.y * 64 + col;
  float v = 0.f;
  if (n < N) {
    const int64_t r0 = blockIdx.x * (int64_t)128 + w * 32, r1 = min(r0 + 32, M);
    for (int64_t r = r0; r < r1; ++r) v += T::up(src[r * ld + n]);
  }
  part[w][col] = v;
  __syncthreads();
  if (w == 0 && n < N) p[blockIdx.x * (int64_t)2 * N + n] = part[0][col] + part[1][col] + part[2][col] + part[3][col];
}

int column_partials(const maba_tensor* src, float* p, hipStream_t s) {
  const int64_t M = src->shape[0], N = src->shape[1];
  auto k = src->dtype == MABA_BF16 ? column_partials_kernel<Bf16> : column_partials_kernel<Fp16>;
  hipLaunchKernelGGL(k, dim3((unsigned)ceil_div(M, 128), (unsigned)ceil_div(N, 64)), dim3(256), 0, s,
                     (const uint16_t*)src->data, src->stride[0], M, (int)N, p);
  return check_launch("column_partials");
}

}  // namespace ffn
}  // namespace maba
