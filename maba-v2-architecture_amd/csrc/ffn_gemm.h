// The matrix-product core of the feed-forward operators: C[m][n] = sum_k A(m, k) B(n, k) in tiles of
// BM x BN, bf16 or fp16 operands, fp32 accumulation on v_mfma_f32_16x16x32.
//
// Each operand lies in memory in one of two ways:
//   rows of k     A[m * lda + k]: the layout of an activation or an nn.Linear weight in y = x W^T
//   columns of k  A[k * lda + m]: the same tensors where the sum runs over their rows (dx = dz W
//                 reads W that way, dW = dz^T x reads both)
// so that no operand is transposed in memory beforehand.  A tile of either kind goes from HBM to LDS by
// direct loads (16 bytes a lane, no registers), ST stages deep.  Rows of k are read back as 16-byte
// fragments, columns of k with the transposing LDS read.  Both layouts XOR the 16-byte chunk index
// with bits of the row, on the global address side since a direct load fills LDS in lane order, so
// that the 16 lanes of a fragment read meet distinct banks.
//
// Out-of-range rows come back as zeros from the buffer descriptor's bounds: it ends at the operand's
// last element.  Chunks past K of a row-of-k operand are sent out of range by their lane offset.
//
// The accumulator holds C transposed (the weight operand is the MFMA's A): a lane has four consecutive
// n of one m, which the epilogues load and store as one 8-byte access.
#pragma once

#include "maba_common.h"

namespace maba {
namespace ffn {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// The two 16-bit types: products, and conversions that round to nearest even.
struct Bf16 {
  static constexpr int CODE = MABA_BF16;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float up(uint32_t h) { return __uint_as_float(h << 16); }
  static __device__ __forceinline__ uint32_t down(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
};
struct Fp16 {
  static constexpr int CODE = MABA_F16;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float up(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }
  static __device__ __forceinline__ uint32_t down(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

// Rows [M, N] of 16-bit elements in global memory that an epilogue reads or writes four columns at a
// time.  vec: every row start is 8-byte aligned, so that whole quads move at once.
struct Rows {
  uint16_t* p;
  int64_t ld;
  int vec;
};
template <class T>
__device__ __forceinline__ f32x4 load4(const Rows& r, int64_t m, int n, int nend) {
  const uint16_t* p = r.p + m * r.ld + n;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (r.vec && n + 4 <= nend) {
    const u32x2 u = *(const u32x2*)p;
    v[0] = T::up(u[0] & 0xffffu); v[1] = T::up(u[0] >> 16); v[2] = T::up(u[1] & 0xffffu); v[3] = T::up(u[1] >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < nend) v[i] = T::up(p[i]);
  }
  return v;
}
template <class T>
__device__ __forceinline__ void store4(const Rows& r, int64_t m, int n, int nend, f32x4 v) {
  uint16_t* p = r.p + m * r.ld + n;
  if (r.vec && n + 4 <= nend) {
    const u32x2 u = {T::down(v[0]) | (T::down(v[1]) << 16), T::down(v[2]) | (T::down(v[3]) << 16)};
    *(u32x2*)p = u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < nend) p[i] = (uint16_t)T::down(v[i]);
  }
}
// Four consecutive elements of a vector [N].
template <class T>
__device__ __forceinline__ f32x4 vec4(const uint16_t* p, int n, int nend) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < nend) v[i] = T::up(p[n + i]);
  return v;
}

enum { K_ROWS = 0, K_ROWS_PAIR = 1, K_COLS = 2, K_COLS_PAIR = 3 };

// One operand.  K_ROWS: p[0] is [rows][K], ld[0] apart.  K_ROWS_PAIR: two such tensors of `rows` rows
// each, whose rows alternate in runs of 16 along the tile (a gate run, then its up run).  K_COLS:
// p[0] is [krows][rows]; k from krows to K (fewer than eight) count as zeros.  K_COLS_PAIR: k < ksplit reads
// p[0], later k row k - ksplit of p[1]; both have krows rows, and rows from there to ksplit count as zeros.
struct Operand {
  const uint16_t* p[2];
  int64_t ld[2];
  int rows;
  int ksplit, krows;
};

struct GemmArgs {
  Operand a, b;
  int64_t K;
  int tiles_m, tiles_n, splits;
  int64_t k_split;      // k of one split, a multiple of the stage depth
};

constexpr uint32_t OUT_OF_RANGE = 0x80000000u;   // a lane offset past every descriptor's end

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t r, uint16_t* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)voff, 0, 0, 0);
}

// Stages R rows (or columns) x BK of an operand.
template <int R, int BK, int NW, int MODE>
struct Stager {
  static constexpr bool COLS = MODE == K_COLS || MODE == K_COLS_PAIR;
  static constexpr int CPR = (COLS ? R : BK) / 8;                  // 16-byte chunks of an LDS row
  static constexpr int RPI = 64 / CPR;                             // LDS rows of one wave instruction
  static constexpr int LOADS = R * BK / (512 * NW);
  static_assert(R * BK % (512 * NW) == 0 && CPR <= 64, "whole instructions");
  static constexpr int PAIRMASK = CPR >= 16 ? 7 : CPR / 2 - 1;

  uint32_t voff[LOADS];        // lane offsets from the tile's base (K_COLS_PAIR: without the row's part)
  uint32_t rowoff[2];          // K_COLS_PAIR: the row's part, with either tensor's stride
  int chunk;                   // rows of k: the lane's chunk of its row, the same for every load
  const char* base[2];         // of the tile, at the first k
  uint32_t span;               // rows of k: bytes from base to the operand's end (rows of this tile)
  int64_t ldb[2];
  int wave, cols;

  // Swizzles: LDS row r keeps chunk c at c ^ key(r).
  static __device__ __forceinline__ int key_rows(int r) { return (r / (16 / CPR)) & (CPR - 1); }
  static __device__ __forceinline__ int key_cols(int k) { return 2 * (((k & 3) | ((k >> 3) & 1) << 2) & PAIRMASK); }

  __device__ __forceinline__ void init(const Operand& o, int64_t K, int64_t kbeg, int r0, int wave_, int lane) {
    wave = wave_;
    ldb[0] = o.ld[0] * 2;
    ldb[1] = o.ld[1] * 2;
    if constexpr (!COLS) {
      static_assert(MODE == K_ROWS || NW * RPI % 32 == 0, "a wave's loads belong to one of the paired tensors");
      chunk = (lane % CPR) ^ key_rows(wave * RPI + lane / CPR);
      const int t = MODE == K_ROWS_PAIR ? (wave * RPI >> 4) & 1 : 0;
      const int first = MODE == K_ROWS_PAIR ? r0 / 2 : r0, most = MODE == K_ROWS_PAIR ? R / 2 : R;
      const int rows = min(o.rows - first, most);
      base[0] = (const char*)(t ? o.p[1] : o.p[0]) + (int64_t)first * ldb[t] + 2 * kbeg;
      span = rows > 0 ? (uint32_t)((rows - 1) * ldb[t] + 2 * (K - kbeg)) : 0u;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        int r = (i * NW + wave) * RPI + lane / CPR;
        if constexpr (MODE == K_ROWS_PAIR) r = ((r >> 5) << 4) | (r & 15);
        voff[i] = (uint32_t)(r * ldb[t]) + 16 * chunk;
      }
    } else {
      cols = 2 * min(o.rows - r0, R);
      base[0] = (const char*)o.p[0] + 2 * (int64_t)r0;
      base[1] = (const char*)o.p[1] + 2 * (int64_t)r0;
      rowoff[0] = (uint32_t)((lane / CPR) * ldb[0]);
      rowoff[1] = (uint32_t)((lane / CPR) * ldb[1]);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int k = (i * NW + wave) * RPI + lane / CPR;
        voff[i] = 16 * ((lane % CPR) ^ key_cols(k)) + (MODE == K_COLS ? (uint32_t)(k * ldb[0]) : 0u);
      }
    }
  }

  // k0: the stage's first k; kend: the end of this workgroup's k range.
  __device__ __forceinline__ void issue(const Operand& o, uint16_t* lds, int64_t k0, int64_t kbeg, int64_t kend) {
    if constexpr (!COLS) {
      const uint32_t adv = 2 * (uint32_t)(k0 - kbeg);
      const uint32_t dead = k0 + 8 * chunk >= kend ? OUT_OF_RANGE : 0u;
      const auto r = rsrc(base[0] + adv, span > adv ? span - adv : 0u);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) lds_load16(r, lds + (i * NW + wave) * 512, voff[i] | dead);
    } else if constexpr (MODE == K_COLS) {
      const uint32_t bytes = (uint32_t)((min(min(kend, (int64_t)o.krows) - k0, (int64_t)BK) - 1) * ldb[0] + cols);
      const auto r = rsrc(base[0] + k0 * ldb[0], bytes);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) lds_load16(r, lds + (i * NW + wave) * 512, voff[i]);
    } else {
      // ksplit is a multiple of 8, so an instruction's rows lie on one side of it; each side has its own
      // stride, and its own end
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int64_t k = k0 + (i * NW + wave) * RPI;
        const int t = k >= o.ksplit;
        const int64_t row = k - (t ? o.ksplit : 0), left = o.krows - row, ld = t ? ldb[1] : ldb[0];
        const uint32_t bytes = left > 0 ? (uint32_t)((min(left, (int64_t)RPI) - 1) * ld + cols) : 0u;
        lds_load16(rsrc((t ? base[1] : base[0]) + row * ld, bytes), lds + (i * NW + wave) * 512,
                   voff[i] + (t ? rowoff[1] : rowoff[0]));
      }
    }
  }
};

// The 16 x 32 fragment of a staged tile at row (column) r0, k step kk: lane (c, q) gets k 8 q .. 8 q + 7 of
// row r0 + c.
template <int R, int BK, int MODE>
__device__ __forceinline__ u32x4 fragment(const uint16_t* lds, int r0, int kk, int c, int q) {
  if constexpr (MODE == K_ROWS || MODE == K_ROWS_PAIR) {
    constexpr int CPR = BK / 8;
    const int key = (c / (16 / CPR)) & (CPR - 1);                  // r0 is a multiple of 16
    return *(const u32x4*)(lds + (r0 + c) * BK + 8 * ((kk * 4 + q) ^ key));
  } else {
    constexpr int CPR = R / 8;
    constexpr int MASK = CPR >= 16 ? 7 : CPR / 2 - 1;
    const int key = ((c >> 2) | (q & 1) << 2) & MASK;
    const uint16_t* p = lds + (kk * 32 + q * 8 + (c >> 2)) * R + 16 * ((r0 >> 4) ^ key) + 4 * (c & 3);
    typedef __attribute__((address_space(3))) i16x4 lds4;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * R)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Tile of this workgroup.  Consecutive ids go to the eight XCDs in turn, each with its own L2: every
// XCD gets a contiguous run of tiles, n fastest, so that its workgroups share a few row panels of A.
struct TileId { int m, n, split; };
__device__ __forceinline__ TileId tile_of(const GemmArgs& g) {
  const uint32_t total = gridDim.x, id = blockIdx.x;
  const uint32_t xcd = id & 7, per = total >> 3, rem = total & 7;
  uint32_t t = xcd * per + min(xcd, rem) + (id >> 3);
  const uint32_t tn = (uint32_t)g.tiles_n, tm = (uint32_t)g.tiles_m;
  TileId r;
  r.n = (int)(t % tn);
  t /= tn;
  r.m = (int)(t % tm);
  r.split = (int)(t / tm);
  return r;
}

template <class T, int BM, int BN, int WM, int WN, int BK, int ST, int AMODE, int BMODE, class Epi>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs g, typename Epi::Args e) {
  constexpr int NW = WM * WN, MI = BM / WM / 16, NI = BN / WN / 16;
  constexpr int A_EL = BM * BK, B_EL = BN * BK;
  typedef Stager<BM, BK, NW, AMODE> SA;
  typedef Stager<BN, BK, NW, BMODE> SB;
  constexpr int LOADS = SA::LOADS + SB::LOADS;
  __shared__ __attribute__((aligned(16))) uint16_t lds[ST * (A_EL + B_EL)];

  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int c = lane & 15, q = lane >> 4;
  const TileId t = tile_of(g);
  const int m0 = t.m * BM, n0 = t.n * BN;
  const int64_t kbeg = t.split * g.k_split, kend = min(g.K, kbeg + g.k_split);
  const int nk = (int)((kend - kbeg + BK - 1) / BK);

  SA sa;
  SB sb;
  sa.init(g.a, g.K, kbeg, m0, wave, lane);
  sb.init(g.b, g.K, kbeg, n0, wave, lane);
  auto issue = [&](int it) {
    uint16_t* p = lds + (it % ST) * (A_EL + B_EL);
    const int64_t k0 = kbeg + (int64_t)it * BK;
    sa.issue(g.a, p, k0, kbeg, kend);
    sb.issue(g.b, p + A_EL, k0, kbeg, kend);
  };

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < nk) issue(s);
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  for (int it = 0; it < nk; ++it) {
    // this wave's loads of the stage have landed, then everyone's; the stage read last is free
    if (ST > 2 && it + ST - 2 < nk) wait_vm<(ST - 2) * LOADS>();
    else wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (it + ST - 1 < nk) issue(it + ST - 1);
    const uint16_t* pa = lds + (it % ST) * (A_EL + B_EL);
    const uint16_t* pb = pa + A_EL;
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      u32x4 fa[MI], fb[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = fragment<BN, BK, BMODE>(pb, wn + 16 * j, kk, c, q);
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = fragment<BM, BK, AMODE>(pa, wm + 16 * i, kk, c, q);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = T::mma(fb[j], fa[i], acc[i][j]);
    }
  }
  Epi::template run<T, BM, BN, WM, WN, MI, NI>(e, acc, t, m0 + wm, n0 + wn, c, q, wave, lds);
}

// Epilogue: C as it is, rounded once to 16 bits.
struct EpiStore {
  struct Args { Rows c; int M, N; };
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + 16 * i + c;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int n = n0 + 16 * j + 4 * q;
        if (m < e.M && n < e.N) store4<T>(e.c, m, n, e.N, acc[i][j]);
      }
    }
  }
};

// Epilogue: fp32 partial products of one k split, [splits][M][N] (N padded to a multiple of 4).
struct EpiPartial {
  struct Args { float* p; int M, N; };
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
    float* p = e.p + (int64_t)t.split * e.M * e.N;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + 16 * i + c;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int n = n0 + 16 * j + 4 * q;
        if (m < e.M && n < e.N) *(f32x4*)(p + (int64_t)m * e.N + n) = acc[i][j];
      }
    }
  }
};

__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.f + fast_exp(-x)); }

// ---------------------------------------------------------------- host side

// Rows [M, N] of `t` (2-D, unit column stride).
inline Rows rows_of(const maba_tensor* t) {
  Rows r;
  r.p = t ? (uint16_t*)t->data : nullptr;
  r.ld = t ? t->stride[0] : 0;
  r.vec = t && t->stride[0] % 4 == 0 && (uintptr_t)t->data % 8 == 0;
  return r;
}

// Whether the core can read `t` in place: 16-byte aligned rows of whole 8-element chunks, at a stride
// whose tile offsets stay far below OUT_OF_RANGE.
inline bool aligned_rows(const maba_tensor* t) {
  return t->stride[0] % 8 == 0 && t->shape[1] % 8 == 0 && (uintptr_t)t->data % 16 == 0 && t->stride[0] <= (1 << 21);
}
inline int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace ffn
}  // namespace maba
