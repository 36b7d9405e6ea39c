// Matrix products of a few rows (decoded tokens): y = x W^T with M <= 16 MT rows, bound by reading W
// once.  A workgroup of eight waves makes the 16 columns of one weight tile (of two tiles, a gate's
// and an up's, with PAIR) for all rows; the waves take every eighth 32-wide chunk of K, load weight
// and input fragments straight into registers, and add their partial tiles through LDS in wave order.
#pragma once

#include "ffn_gemm.h"

namespace maba {
namespace ffn {

struct SkinnyArgs {
  const uint16_t* x; int64_t xs;
  const uint16_t* w[2]; int64_t ws[2];
  int M, N, K;
  int xvec, wvec;     // 16-byte aligned rows of whole 8-element chunks
};

constexpr int SKINNY_NW = 8, SKINNY_U = 4;

// Eight elements at k of a row, zero from K on.
__device__ __forceinline__ u32x4 row8(const uint16_t* row, int k, int K, int vec) {
  u32x4 v = {0, 0, 0, 0};
  if (vec) {
    if (k < K) v = *(const u32x4*)(row + k);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) v[j >> 1] |= (uint32_t)row[k + j] << (16 * (j & 1));
  }
  return v;
}

template <class T, bool PAIR, int MT, class Epi>
__global__ __launch_bounds__(64 * SKINNY_NW) void skinny_kernel(SkinnyArgs a, typename Epi::Args e) {
  constexpr int P = PAIR ? 2 : 1, NW = SKINNY_NW, U = SKINNY_U;
  __shared__ __attribute__((aligned(16))) f32x4 part[NW][P * MT][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int c = lane & 15, q = lane >> 4, n0 = blockIdx.x * 16;
  const int KC = (a.K + 31) / 32;
  const uint16_t* w[P];
#pragma unroll
  for (int p = 0; p < P; ++p) w[p] = a.w[p] + (int64_t)min(n0 + c, a.N - 1) * a.ws[p];
  const uint16_t* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = a.x + (int64_t)min(16 * t + c, a.M - 1) * a.xs;
  f32x4 acc[P][MT];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c0 = wave; c0 < KC; c0 += NW * U) {
    u32x4 fw[U][P], fx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 32 * (c0 + NW * u) + 8 * q;      // past K: zeros
#pragma unroll
      for (int p = 0; p < P; ++p) fw[u][p] = row8(w[p], k, a.K, a.wvec);
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[u][t] = row8(x[t], k, a.K, a.xvec);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[p][t] = T::mma(fw[u][p], fx[u][t], acc[p][t]);
  }
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][p * MT + t][lane] = acc[p][t];
  __syncthreads();
  if (wave < MT) {
    f32x4 v[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      v[p] = part[0][p * MT + wave][lane];
#pragma unroll
      for (int i = 1; i < NW; ++i) v[p] += part[i][p * MT + wave][lane];
    }
    const int m = 16 * wave + c, n = n0 + 4 * q;
    if (m < a.M && n < a.N) Epi::template quad<T>(e, m, n, v[0], v[P - 1]);
  }
}

template <class T, bool PAIR, class Epi>
int skinny(const SkinnyArgs& a, const typename Epi::Args& e, hipStream_t s, const char* who) {
  const dim3 grid((unsigned)ceil_div(a.N, 16));
  auto k = a.M <= 16 ? skinny_kernel<T, PAIR, 1, Epi> : skinny_kernel<T, PAIR, 2, Epi>;
  hipLaunchKernelGGL(k, grid, dim3(64 * SKINNY_NW), 0, s, a, e);
  return check_launch(who);
}
// Whether M rows of K go this way.  Every workgroup reads all of x, so that more than 16 rows of a long k are better
// off in tiles: 32 rows, 2,048 to 2 x 5,504: 19.8 us here and 15.5 there (16 rows: 16.9 here), 1,024 to 2 x 2,816: 7.1 and
// 7.7, and 1,248 to 640, where the tiles need their sum split: 5.0 and 6.9.
inline bool few_rows(int64_t M, int64_t K) { return M <= 16 || (M <= 32 && K <= 1536); }

}  // namespace ffn
}  // namespace maba
