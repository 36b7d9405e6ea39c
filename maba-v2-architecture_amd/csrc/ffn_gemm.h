// The matrix-product core of the feed-forward operators: C[m][n] = sum_k A(m, k) B(n, k) in tiles of
// BM x BN, bf16 or fp16 operands, fp32 accumulation on v_mfma_f32_16x16x32.
//
// Each operand lies in memory in one of two ways:
//   rows of k     A[m * lda + k]: the layout of an activation or an nn.Linear weight in y = x W^T
//   columns of k  A[k * lda + m]: the same tensors where the sum runs over their rows (dx = dz W
//                 reads W that way, dW = dz^T x reads both)
// so that no operand is transposed in memory beforehand.  A tile of either kind goes from HBM to LDS by
// direct loads (16 bytes a lane, no registers).  Rows of k are read back as 16-byte
// fragments, columns of k with the transposing LDS read.  Both layouts XOR the 16-byte chunk index
// with bits of the row, on the global address side since a direct load fills LDS in lane order, so
// that the 16 lanes of a fragment read meet distinct banks.
//
// Out-of-range rows come back as zeros from the buffer descriptor's bounds: it ends at the operand's
// last element.  Chunks past K of a row-of-k operand are sent out of range by their lane offset.
//
// The accumulator holds C transposed (the weight operand is the MFMA's A): a lane has four consecutive
// n of one m.
#pragma once

#include <type_traits>

#include "maba_common.h"

namespace maba {
namespace ffn {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// The two 16-bit types: products, and conversions that round to nearest even.
struct Bf16 {
  static constexpr int CODE = MABA_BF16;
  static constexpr bool SCALED = false;             // operands made on the way are held as they are
  static constexpr float MOST = 3.38953139e38f;     // the largest finite value
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float up(uint32_t h) { return __uint_as_float(h << 16); }
  static __device__ __forceinline__ uint32_t down(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
};
struct Fp16 {
  static constexpr int CODE = MABA_F16;
  static constexpr bool SCALED = true;              // times a power of two (Magnitudes)
  static constexpr float MOST = 65504.f;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float up(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }
  static __device__ __forceinline__ uint32_t down(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

// Rows [M, N] of 16-bit elements in global memory that an epilogue reads or writes, at any alignment of an element
// (global memory takes unaligned vector accesses).
struct Rows {
  uint16_t* p;
  int64_t ld;
};
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
template <class T>
__device__ __forceinline__ f32x4 up4(u32x2 u) {
  return f32x4{T::up(u[0] & 0xffffu), T::up(u[0] >> 16), T::up(u[1] & 0xffffu), T::up(u[1] >> 16)};
}
template <class T>
__device__ __forceinline__ u32x2 down4(f32x4 v) {
  return u32x2{T::down(v[0]) | (T::down(v[1]) << 16), T::down(v[2]) | (T::down(v[3]) << 16)};
}

// The accumulator of two neighbouring 16-column blocks has, in lane (c, q), the quads of columns 4 q and 16 + 4 q
// of row c.  Exchanged between the lane quarters they make the eight columns from 8 q on: one 16-byte access a lane
// instead of two of 8 bytes (the stores of [dg | du] at 16,384 x 2,496 take 10 us less so).
struct Quads { u32x2 a, b; };       // columns 4 q .. and 16 + 4 q ..
__device__ __forceinline__ void swap_quarters(uint32_t& a, uint32_t& b, bool halves) {
  const auto r = halves ? __builtin_amdgcn_permlane32_swap(a, b, false, false) : __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ u32x4 eight_of(Quads v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t a = v.a[i], b = v.b[i];
    swap_quarters(a, b, true);
    swap_quarters(a, b, false);
    v.a[i] = a;
    v.b[i] = b;
  }
  return u32x4{v.a[0], v.a[1], v.b[0], v.b[1]};
}
__device__ __forceinline__ Quads quads_of(u32x4 u) {
  Quads v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t a = u[i], b = u[2 + i];
    swap_quarters(a, b, false);
    swap_quarters(a, b, true);
    v.a[i] = a;
    v.b[i] = b;
  }
  return v;
}
// The raw eight at (m, n); rows from mend and columns from nend on are zeros and are not read.
__device__ __forceinline__ u32x4 load8(const Rows& r, int64_t m, int n, int mend, int nend) {
  u32x4 u = {0, 0, 0, 0};
  if (m >= mend) return u;
  const uint16_t* p = r.p + m * r.ld + n;
  if (n + 8 <= nend) return *(const u32x4_any*)p;
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (n + i < nend) u[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
  return u;
}
__device__ __forceinline__ void store8(const Rows& r, int64_t m, int n, int mend, int nend, u32x4 u) {
  if (m >= mend) return;
  uint16_t* p = r.p + m * r.ld + n;
  if (n + 8 <= nend) {
    *(u32x4_any*)p = u;
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (n + i < nend) p[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
  }
}
// A quad by itself.
__device__ __forceinline__ u32x2 load4(const Rows& r, int64_t m, int n, int nend) {
  const uint16_t* p = r.p + m * r.ld + n;
  if (n + 4 <= nend) return *(const u32x2_any*)p;
  u32x2 u = {0, 0};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (n + i < nend) u[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
  return u;
}
template <class T>
__device__ __forceinline__ void store4(const Rows& r, int64_t m, int n, int nend, f32x4 v) {
  uint16_t* p = r.p + m * r.ld + n;
  const u32x2 u = down4<T>(v);
  if (n + 4 <= nend) {
    *(u32x2_any*)p = u;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (n + i < nend) p[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
  }
}
enum { K_ROWS = 0, K_ROWS_PAIR = 1, K_COLS = 2 };

// One operand.  K_ROWS: p[0] is [rows][K], ld[0] apart.  K_ROWS_PAIR: two such tensors of `rows` rows
// each, whose rows alternate in runs of 16 along the tile (a gate run, then its up run).  K_COLS:
// p[0] is [krows][rows]; k from krows to K (fewer than eight) count as zeros.  A sum of two segments of K each
// (dx = dg Wg + du Wu) goes on with column K of p[0] in K_ROWS, with p[1] in K_COLS.
struct Operand {
  const uint16_t* p[2];
  int64_t ld[2];
  int rows, krows;
};

struct GemmArgs {
  Operand a, b;
  int64_t K;            // of a segment
  int segments;         // 1 or 2
  int tiles_m, tiles_n;
  int split_stages;     // stages of a split's run of the sum (the last split may have fewer)
};

constexpr int GEMM_BK = 64;      // k of a stage: two steps
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;   // a lane offset past every descriptor's end

// The same in every lane; said so to the compiler, which otherwise loops over the lanes' descriptors.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)hi << 32 | lo), 0, (int)__builtin_amdgcn_readfirstlane(bytes),
                                           0x00027000);
}
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t r, uint16_t* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)voff, 0, 0, 0);
}

// Swizzles.  Rows of k: LDS row r (BK elements) keeps 16-byte chunk c at c ^ key_rows(r), so that 16 consecutive
// rows' chunks c lie in the 64 banks once each.  Columns of k: LDS row k (R elements) keeps the pair of chunks p at
// p ^ key_cols(k); a fragment read takes rows 4 j .. 4 j + 3 of two j that differ by 2, whose own offsets (R / 2 banks a
// row) leave log2(128 / gcd(R, 128)) of the three bits that tell the eight rows apart to the row number.
template <int BK>
__device__ __forceinline__ constexpr int key_rows(int r) {
  return (r / (16 / (BK / 8))) & (BK / 8 - 1);
}
template <int R>
__device__ __forceinline__ constexpr int key_cols(int k) {
  return R % 128 == 0 ? (k & 3) | (k >> 3 & 1) << 2 : R % 64 == 0 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : k >> 3 & 1;
}

// Stages R rows (or columns) x BK of an operand.
template <int R, int BK, int NW, int MODE>
struct Stager {
  static constexpr bool COLS = MODE == K_COLS;
  static constexpr int CPR = (COLS ? R : BK) / 8;                  // 16-byte chunks of an LDS row
  static constexpr int LOADS = R * BK / (512 * NW);
  static_assert(R * BK % (512 * NW) == 0 && R % 32 == 0, "whole instructions");

  uint32_t voff[LOADS];        // lane offsets from the tile's base
  int chunk;                   // rows of k: the lane's chunk of its row, the same for every load
  const char* base[2];         // of the tile, at the first k
  uint32_t span;               // rows of k: bytes from base to the operand's end (rows of this tile)
  int64_t ldb;                 // bytes from row to row (both tensors of a K_COLS operand have the same stride)
  int wave, cols;

  __device__ __forceinline__ void init(const Operand& o, const GemmArgs& g, int r0, int wave_, int lane) {
    wave = wave_;
    if constexpr (!COLS) {
      constexpr int RPI = 64 / CPR;                                // LDS rows of one wave instruction
      static_assert(MODE == K_ROWS || NW * RPI % 32 == 0, "a wave's loads belong to one of the paired tensors");
      chunk = (lane % CPR) ^ key_rows<BK>(wave * RPI + lane / CPR);
      const int t = MODE == K_ROWS_PAIR ? (wave * RPI >> 4) & 1 : 0;
      const int first = MODE == K_ROWS_PAIR ? r0 / 2 : r0, most = MODE == K_ROWS_PAIR ? R / 2 : R;
      const int rows = min(o.rows - first, most);
      ldb = (t ? o.ld[1] : o.ld[0]) * 2;
      base[0] = (const char*)(t ? o.p[1] : o.p[0]) + (int64_t)first * ldb;
      base[1] = base[0];
      span = rows > 0 ? (uint32_t)((rows - 1) * ldb + 2 * g.segments * g.K) : 0u;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        int r = (i * NW + wave) * RPI + lane / CPR;
        if constexpr (MODE == K_ROWS_PAIR) r = ((r >> 5) << 4) | (r & 15);
        voff[i] = (uint32_t)(r * ldb) + 16 * chunk;
      }
    } else {
      ldb = o.ld[0] * 2;
      cols = 2 * min(o.rows - r0, R);
      base[0] = (const char*)o.p[0] + 2 * (int64_t)r0;
      base[1] = (const char*)o.p[1] + 2 * (int64_t)r0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int l = (i * NW + wave) * 64 + lane, k = l / CPR, x = l % CPR;
        voff[i] = (uint32_t)(k * ldb) + 16 * ((((x >> 1) ^ key_cols<R>(k)) << 1) | (x & 1));
      }
    }
  }

  // k0: the stage's first k of segment seg.
  __device__ __forceinline__ void issue(const Operand& o, const GemmArgs& g, uint16_t* lds, int seg, int64_t k0) {
    const char* p;
    uint32_t bytes, dead = 0;
    if constexpr (!COLS) {
      const uint32_t adv = 2 * (uint32_t)(seg * g.K + k0);
      p = base[0] + adv;
      bytes = span > adv ? span - adv : 0u;
      dead = k0 + 8 * chunk >= g.K ? OUT_OF_RANGE : 0u;
    } else {
      const int64_t rows = min(min(g.K, (int64_t)o.krows) - k0, (int64_t)BK);
      p = (seg ? base[1] : base[0]) + k0 * ldb;
      bytes = rows > 0 ? (uint32_t)((rows - 1) * ldb + cols) : 0u;
    }
    const auto r = rsrc(p, bytes);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) lds_load16(r, lds + (i * NW + wave) * 512, voff[i] | dead);
  }
};

// The 16 x 32 fragment of a staged tile at row (column) r0, k step kk: lane (c, q) gets k 8 q .. 8 q + 7 of
// row r0 + c.
template <int R, int BK, int MODE>
__device__ __forceinline__ u32x4 fragment(const uint16_t* lds, int r0, int kk, int c, int q) {
  if constexpr (MODE != K_COLS) {
    return *(const u32x4*)(lds + (r0 + c) * BK + 8 * ((kk * 4 + q) ^ key_rows<BK>(c)));   // r0 is a multiple of 16
  } else {
    const uint16_t* p = lds + (kk * 32 + q * 8 + (c >> 2)) * R + 16 * ((r0 >> 4) ^ key_cols<R>(q * 8 + (c >> 2))) + 4 * (c & 3);
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

// Tile of this workgroup.  Consecutive ids go to the eight XCDs in turn, each with its own L2: every XCD gets a
// contiguous run of tiles, in groups of GROUP_M rows of tiles taken column by column, so that the 32 to 64 workgroups
// it runs at once share about as many panels of A as of B.
constexpr uint32_t GROUP_M = 4;
struct TileId { int m, n, split; };
__device__ __forceinline__ TileId tile_of(const GemmArgs& g) {
  const uint32_t total = gridDim.x, id = blockIdx.x;
  const uint32_t xcd = id & 7, per = total >> 3, rem = total & 7;
  uint32_t t = xcd * per + min(xcd, rem) + (id >> 3);
  const uint32_t tn = (uint32_t)g.tiles_n, tm = (uint32_t)g.tiles_m;
  TileId r;
  r.split = (int)(t / (tm * tn));
  t %= tm * tn;
  const uint32_t first = t / (GROUP_M * tn) * GROUP_M, rows = min(GROUP_M, tm - first);
  t -= first * tn;
  r.m = (int)(first + t % rows);
  r.n = (int)(t / rows);
  return r;
}

// The main loop keeps ST stages of 64 k in LDS and the fragments of two steps of 32 k in registers.  While the
// products of one step run, the fragments of the next are read; the one barrier of a stage stands between its two
// steps, where every wave has the stage's last fragments in registers (its buffer is free for the loads of the stage
// ST ahead) and the next stage has landed (its first fragments can be read).  So neither LDS reads nor
// loads are waited for between products, except by the first.
//
// With KG = 2 two groups of WM x WN waves each make the whole tile from every other stage, their own in LDS, and add up
// at the end, half of the rows each.
template <class T, int BM, int BN, int WM, int WN, int ST, int AMODE, int BMODE, class Epi, int KG = 1>
__global__ __launch_bounds__(64 * WM * WN * KG, KG == 2 || BM * BN / (WM * WN) <= 12288 ? 2 : 1) void gemm_kernel(GemmArgs g, typename Epi::Args e) {
  constexpr int NW = WM * WN, MI = BM / WM / 16, NI = BN / WN / 16, BK = GEMM_BK;
  constexpr int A_EL = BM * BK, STAGE = (BM + BN) * BK;
  typedef Stager<BM, BK, NW, AMODE> SA;
  typedef Stager<BN, BK, NW, BMODE> SB;
  __shared__ __attribute__((aligned(16))) uint16_t lds_all[KG * ST * STAGE];

  const int wave_all = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int kg = KG == 1 ? 0 : wave_all / NW, wave = wave_all - kg * NW;       // the wave's group, and its number there
  uint16_t* lds = lds_all + kg * ST * STAGE;
  const int c = lane & 15, q = lane >> 4;
  const TileId t = tile_of(g);
  const int m0 = t.m * BM, n0 = t.n * BN;
  const int nk1 = (int)((g.K + BK - 1) / BK);                                    // stages of a segment
  const int s0 = t.split * g.split_stages, nk = (min(nk1 * g.segments - s0, g.split_stages) + KG - 1) / KG;
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

  SA sa;
  SB sb;
  sa.init(g.a, g, m0, wave, lane);
  sb.init(g.b, g, n0, wave, lane);
  auto issue = [&](int s) {
    uint16_t* p = lds + (s % ST) * STAGE;
    const int at = s0 + KG * s + kg, seg = at >= nk1 && g.segments > 1;         // of an odd number of stages one group's last is past the end: zeros
    const int64_t k0 = (int64_t)(at - seg * nk1) * BK;
    sa.issue(g.a, g, p, seg, k0);
    sb.issue(g.b, g, p + A_EL, seg, k0);
  };
  struct Frags { u32x4 a[MI], b[NI]; };
  auto read = [&](Frags& f, int s, int kk) {
    const uint16_t* p = lds + (s % ST) * STAGE;
#pragma unroll
    for (int j = 0; j < NI; ++j) f.b[j] = fragment<BN, BK, BMODE>(p + A_EL, wn + 16 * j, kk, c, q);
#pragma unroll
    for (int i = 0; i < MI; ++i) f.a[i] = fragment<BM, BK, AMODE>(p, wm + 16 * i, kk, c, q);
  };
  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto products = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = T::mma(f.b[j], f.a[i], acc[i][j]);
  };
  constexpr int LOADS = SA::LOADS + SB::LOADS;
  // An LDS read and, where the step has any, a load before each of the first products.  With all the loads in one place
  // a compute unit with few waves waits for their issue (dx of 8,191 x 640 x 2,496: 45 us against 50).
  auto interleave = [](auto loads) {
    constexpr int READS = MI * (SA::COLS ? 2 : 1) + NI * (SB::COLS ? 2 : 1);
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // LDS read
      if (decltype(loads)::value && i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // MFMA
    }
  };

  Frags f0, f1;
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (s < nk) issue(s);
  if (nk >= ST) wait_vm<(ST - 1) * LOADS>();
  else wait_vm<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read(f0, 0, 0);
  // the steps of stage s; between them the next stage has landed, and every wave holds the fragments of stage s
  auto stage = [&](int s, auto more) {
    constexpr bool MORE = decltype(more)::value;          // there is a stage ST ahead
    read(f1, s, 1);
    products(f0);
    interleave(std::false_type{});
    wait_vm<MORE ? (ST - 2) * LOADS : 0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // past the last stage these are stale values that nothing uses
    read(f0, s + 1, 0);
    // behind the reads: before them, dx of 4,096 x 2,048 x 11,008 takes 151 us against 141, dW of 11,008 x 2,048 x 4,096 in
    // 256 x 256 tiles 206 against 189, the smaller tiles' products the same
    if (MORE) issue(s + ST);
    products(f1);
    interleave(more);
  };
  int s = 0;
  for (; s + ST < nk; ++s) stage(s, std::true_type{});
  for (; s < nk; ++s) stage(s, std::false_type{});
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if constexpr (KG == 1) {
    Epi::template run<T, BM, BN, WM, WN, MI, NI>(e, acc, t, m0 + wm, n0 + wn, c, q, wave, lds);
  } else {
    static_assert(MI % 2 == 0 && BM * BN * 2 <= KG * ST * STAGE, "halves, through the stages' LDS");
    constexpr int HI = MI / 2;
    f32x4* part = (f32x4*)lds_all + (size_t)wave * HI * NI * 64 + lane;       // [2][NW][HI][NI][64]
    constexpr int OTHER = NW * HI * NI * 64;
    __syncthreads();                               // the last stages have been read
    f32x4 sum[HI][NI];
#pragma unroll
    for (int i = 0; i < HI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        sum[i][j] = kg ? acc[HI + i][j] : acc[i][j];
        part[kg * OTHER + (i * NI + j) * 64] = kg ? acc[i][j] : acc[HI + i][j];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) sum[i][j] += part[(1 - kg) * OTHER + (i * NI + j) * 64];
    Epi::template run<T, BM, BN, WM, WN, HI, NI>(e, sum, t, m0 + wm + 16 * HI * kg, n0 + wn, c, q, wave, lds);
  }
}

// 2^e of a scaled operand's exponent, and 2^-e; 1 without one.
template <class T>
__device__ __forceinline__ float power_of(const int* exponent, int sign) {
  if constexpr (T::SCALED) return exponent ? __builtin_amdgcn_ldexpf(1.f, sign * *exponent) : 1.f;
  else return 1.f;
}

// Epilogue: C, times 2^-*exponent where there is one, rounded once to 16 bits; from row `second` on it goes to the
// second tensor's rows (`second` is a multiple of 16).  M: rows of each.
struct EpiStore {
  static constexpr bool LONG = false, GROUPS = true;
  struct Args { Rows c[2]; int second, M, N; const int* exponent; };
  template <class T, int BM, int BN, int WM, int WN, int MI, int NI>
  static __device__ __forceinline__ void run(const Args& e, f32x4 (&acc)[MI][NI], const TileId& t, int m0, int n0, int c,
                                             int q, int wave, uint16_t* lds) {
    const float scale = power_of<T>(e.exponent, -1);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int at = m0 + 16 * i >= e.second, m = m0 + 16 * i - (at ? e.second : 0) + c;
      const Rows r = at ? e.c[1] : e.c[0];
      if (!r.p) continue;
#pragma unroll
      for (int j = 0; j < NI; j += 2)
        store8(r, m, n0 + 16 * j + 8 * q, e.M, e.N, eight_of({down4<T>(acc[i][j] * scale), down4<T>(acc[i][j + 1] * scale)}));
    }
  }
};

// Epilogue: fp32 partial products of one k split, [splits][M][N] (N padded to a multiple of 4).
struct EpiPartial {
  static constexpr bool LONG = false, GROUPS = false;
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

// An unpacked element: code * 2^e, at most `most` in magnitude (a finite value may have rounded up past its type's
// range); NaN stays NaN.
__device__ __forceinline__ float scaled(float code, int e, float most) {
  const float v = __builtin_amdgcn_ldexpf(code, e);
  return v > most ? most : v < -most ? -most : v;
}

__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.f + fast_exp(-x)); }

// Over the 16 lanes of a quarter of the wave, in each of them: neighbours, pairs, quads and eights.
template <class F>
__device__ __forceinline__ float over16(float v, F f) {
  v = f(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, true)));     // lanes 1 0 3 2
  v = f(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, true)));     // lanes 2 3 0 1
  v = f(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true)));    // a half mirrored
  v = f(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true)));    // mirrored
  return v;
}
__device__ __forceinline__ float sum16(float v) { return over16(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float max16(float v) { return over16(v, [](float a, float b) { return fmaxf(a, b); }); }

// ---------------------------------------------------------------- host side

// Rows [M, N] of `t` (2-D, unit column stride).
inline Rows rows_of(const maba_tensor* t) {
  Rows r;
  r.p = t ? (uint16_t*)t->data : nullptr;
  r.ld = t ? t->stride[0] : 0;
  return r;
}

// Whether the core can read `t` in place: 16-byte aligned rows of whole 8-element chunks, at a stride
// whose tile offsets stay far below OUT_OF_RANGE.
inline bool aligned_rows(const maba_tensor* t) {
  return t->stride[0] % 8 == 0 && t->shape[1] % 8 == 0 && (uintptr_t)t->data % 16 == 0 && t->stride[0] <= (1 << 21);
}
// The same for reading it along its columns: rows past the last one are zeros by the descriptor's end, which takes rows
// that lie apart (broadcast or overlapping ones would be read again in their place).
inline bool aligned_columns(const maba_tensor* t) { return aligned_rows(t) && t->stride[0] >= t->shape[1]; }
inline int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace ffn
}  // namespace maba
