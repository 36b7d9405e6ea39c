// Rows of bf16, fp16 or fp32 elements in 16-byte chunks at any alignment of an element (global memory takes unaligned
// vector accesses), sums over the lanes that share a row, and the generator behind dropout.
#pragma once

#include "ffn_common.h"
#include "row_lanes.h"

namespace maba {
namespace rowvec {

using ffn::u32x4;
using ffn::u32x4_any;
using ffn::Bf16;
using ffn::Fp16;
typedef u32x4 u32x4_any4 __attribute__((aligned(4)));
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

struct F32 { static constexpr int CODE = MABA_F32; };
template <class T> struct Traits { typedef uint16_t elem; static constexpr int VEC = 8; };
template <> struct Traits<F32> { typedef float elem; static constexpr int VEC = 4; };

// The elements of a chunk in fp32, and back with one rounding to nearest even.
template <class T>
__device__ __forceinline__ void unpack(u32x4 u, float (&v)[Traits<T>::VEC]) {
  if constexpr (T::CODE == MABA_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = T::up(u[i] & 0xffffu);
      v[2 * i + 1] = T::CODE == MABA_BF16 ? __uint_as_float(u[i] & 0xffff0000u) : T::up(u[i] >> 16);
    }
  }
}
template <class T>
__device__ __forceinline__ u32x4 pack(const float (&v)[Traits<T>::VEC]) {
  u32x4 u;
  if constexpr (T::CODE == MABA_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T::CODE == MABA_BF16) u[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
      else u[i] = T::down(v[2 * i]) | (T::down(v[2 * i + 1]) << 16);
    }
  }
  return u;
}

// The chunk `off` bytes behind `base`, of which `left` elements belong to the row; the rest are zeros that are not read, or
// not written.  `base` is the same in all lanes of a wave: it stays in scalar registers, and an address costs a lane one.
template <class T>
__device__ __forceinline__ u32x4 load_chunk(const void* base, uint32_t off, int left) {
  constexpr int V = Traits<T>::VEC;
  const auto* q = (const typename Traits<T>::elem*)((const char*)base + off);
  u32x4 u = {0, 0, 0, 0};
  if (left >= V) {
    if constexpr (V == 4) u = *(const u32x4_any4*)q;
    else u = *(const u32x4_any*)q;
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < V - 1; ++i) {
      if (i >= left) continue;
      if constexpr (V == 4) u[i] = __float_as_uint(q[i]);
      else u[i >> 1] |= (uint32_t)q[i] << (16 * (i & 1));
    }
  }
  return u;
}
template <class T>
__device__ __forceinline__ void store_chunk(void* base, uint32_t off, int left, u32x4 u) {
  constexpr int V = Traits<T>::VEC;
  auto* q = (typename Traits<T>::elem*)((char*)base + off);
  if (left >= V) {
    if constexpr (V == 4) *(u32x4_any4*)q = u;
    else *(u32x4_any*)q = u;
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < V - 1; ++i) {
      if (i >= left) continue;
      if constexpr (V == 4) q[i] = __uint_as_float(u[i]);
      else q[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Chunks of rows of at least one: loads without a branch.  A chunk that the row's end cuts is loaded as the row's last
// whole chunk, and a lane without a chunk loads that one too; ended() moves the first one's elements to its front and makes
// the others zeros, where they are used.  (Element by element under tests of their own the cut chunks took as long as all the
// rest: 8,192 x 4,095 bf16 forward 90 us, backward 212.)
template <class T>
__device__ __forceinline__ u32x4 ended(u32x4 u, int left) {
  constexpr int V = Traits<T>::VEC;
  if (!__any(left < V)) return u;
  const int k = V - max(min(left, V), 0);                  // elements from the front that belong to the chunk before
  const auto when = [](bool b, uint32_t x, uint32_t y) { return b ? x : y; };
  const int w = V == 8 ? k >> 1 : k;                       // whole words
  u = {when(w & 2, u[2], u[0]), when(w & 2, u[3], u[1]), when(w & 2, 0, u[2]), when(w & 2, 0, u[3])};
  u = {when(w & 1, u[1], u[0]), when(w & 1, u[2], u[1]), when(w & 1, u[3], u[2]), when(w & 1, 0, u[3])};
  if constexpr (V == 8) {
    const bool half = k & 1;
    u = {when(half, __builtin_amdgcn_alignbit(u[1], u[0], 16), u[0]), when(half, __builtin_amdgcn_alignbit(u[2], u[1], 16), u[1]),
         when(half, __builtin_amdgcn_alignbit(u[3], u[2], 16), u[2]), when(half, u[3] >> 16, u[3])};
  }
  return left <= 0 ? u32x4{0, 0, 0, 0} : u;
}

// Rows of a tensor as a wave goes through them: `at` is where chunk 0 of the wave's first row is, `off` how far behind it
// this lane's is.
template <class T>
struct Walk {
  char* p;
  int64_t stride;          // bytes
  uint32_t row_off, off;
  __device__ __forceinline__ Walk(const void* q, int64_t ld, int l, int sub)
      : p((char*)q), stride(ld * (int64_t)sizeof(typename Traits<T>::elem)), row_off(lane_row(sub, stride)), off(row_off + 16 * l) {}
  __device__ __forceinline__ char* at(int64_t row, int chunk) const { return p + row * stride + 16 * (int64_t)chunk; }
};
// A lane's chunks l, l + 2^lg, ... of rows that end inside a chunk, for ended().
template <class T, int NCH>
struct CutRows {
  static constexpr int V = Traits<T>::VEC;
  int64_t last;            // row
  uint32_t in[NCH];        // bytes from a row's start to what is loaded
  __device__ __forceinline__ CutRows(int64_t R, int C, int l, int lg) : last(R - 1) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) in[i] = (uint32_t)min((l + (i << lg)) * V, C - V) * (uint32_t)sizeof(typename Traits<T>::elem);
  }
  // chunk i of the lane's row, or of the last row for a lane past it
  __device__ __forceinline__ u32x4 load(const Walk<T>& w, int64_t row, bool live, int i) const {
    const char* q = w.p + (row < last ? row : last) * w.stride + ((live ? w.row_off : 0u) + in[i]);
    if constexpr (V == 4) return *(const u32x4_any4*)q;
    else return *(const u32x4_any*)q;
  }
};

// The same rows where every row is whole chunks, 16-byte aligned: accesses through a buffer descriptor, which drops those of
// lanes without a chunk or a row, and all of a missing tensor's (whose chunks are zeros), without a branch.
template <class T>
struct WholeWalk : Walk<T> {
  uint32_t bytes;
  __device__ __forceinline__ WholeWalk(const void* q, int64_t ld, int l, int sub) : Walk<T>(q, ld, l, sub), bytes(q ? DESCRIPTOR_END : 0u) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(int64_t row) const { return ffn::rsrc(this->p + row * this->stride, bytes); }
  __device__ __forceinline__ u32x4 load(__amdgpu_buffer_rsrc_t r, uint32_t chunk) const {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_access(this->off, chunk), 0, 0));
  }
  __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t chunk, u32x4 u) const {
    __builtin_amdgcn_raw_buffer_store_b128(u, r, (int)lane_access(this->off, chunk), 0, 0);
  }
};

// A row's lanes: 2^lg of them, lane l of which holds the chunks l, l + 2^lg, ...  Rows narrower than a wave share it.
// `most` is how many elements a lane may have; far: the rows that share a wave would be further apart than 32 bits of bytes tell.
constexpr int MAX_LG = 9, MAX_WIDTH = 16 << MAX_LG;
struct Geometry {
  int lg, nch;
};
inline Geometry row_geometry(int64_t C, int vec, int most, bool far) {      // C <= most << MAX_LG
  const int64_t chunks = ceil_div(C, vec);
  int lg = far ? 6 : 4;
  while (chunks > (int64_t)(most / vec) << lg) ++lg;
  return {lg, (int)ceil_div(chunks, (int64_t)1 << lg)};
}

// v of other lanes for a butterfly whose lanes hold equal values below the step: step 0 and 1 exchange with lane ^ 1 and ^ 2,
// 2 with the other four of eight, 3 with the other eight of sixteen.
template <int STEP>
__device__ __forceinline__ float peer(float v) {
  constexpr int ctrl = STEP == 0 ? 0xb1 : STEP == 1 ? 0x4e : STEP == 2 ? 0x141 : 0x140;
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), ctrl, 0xf, 0xf, true));
}
// The values of the two 16-lane rows of a half, or of the two halves: (first, second) in all their lanes.
struct Pair { float a, b; };
template <bool HALVES>
__device__ __forceinline__ Pair both(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = HALVES ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
// v of all 64 lanes joined by f, which takes its arguments in any order.
template <class F>
__device__ __forceinline__ float wave_joined(float v, F f) {
  v = f(v, peer<0>(v));
  v = f(v, peer<1>(v));
  v = f(v, peer<2>(v));
  v = f(v, peer<3>(v));
  Pair p = both<false>(v);
  p = both<true>(f(p.a, p.b));
  return f(p.a, p.b);
}
// The sums of v over the 2^lg lanes of a row (lg >= 4), the same bits in each of them.  Rows of more than one wave meet in
// `red` [2][M][waves], M being the kernel's largest N; every thread of the workgroup takes part, and the two halves take
// turns, so that one barrier a sum is enough.
template <int N, int M = N>
__device__ __forceinline__ void row_sums(float (&v)[N], int lg, float* red, int& turn) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] += peer<0>(v[n]);
    v[n] += peer<1>(v[n]);
    v[n] += peer<2>(v[n]);
    v[n] += peer<3>(v[n]);
  }
  if (lg > 4)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const Pair p = both<false>(v[n]);
      v[n] = p.a + p.b;
    }
  if (lg > 5)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const Pair p = both<true>(v[n]);
      v[n] = p.a + p.b;
    }
  if (lg > 6) {
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, per = 1 << (lg - 6);
    float* r = red + turn * M * waves;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) r[n * waves + wave] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float* q = r + n * waves + (wave & ~(per - 1));
      float s = 0.f;
      for (int i = 0; i < per; ++i) s += q[i];
      v[n] = s;
    }
    turn ^= 1;
  }
}

// ---------------------------------------------------------------- dropout

// Element (row, column) is dropped where its random word is below p * 2^32.  The words are those of Philox4x32 (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): a block cipher of the counter
// (column / 4, row, stream) under the seed, whose four output words serve four neighbouring columns.  So any part of the
// mask can be made anywhere, in any order, and it is never stored.  Seven rounds, the fewest that pass the statistical
// tests in that paper: with ten dropout of 32,768 x 1,024 bf16 takes 29.2 us instead of 26.6 (without the generator 20.7).
struct Drop {
  const uint64_t* seed;
  uint32_t below, stream;
  float keep;              // 1 / (1 - p)
  int mode;                // 0 nothing is dropped, 1 as above, 2 everything is (p = 1)
};
inline Drop make_drop(double p, const void* seed, uint32_t stream) {
  const double t = __builtin_nearbyint(p * 4294967296.0);       // p is at least 0 and at most 1
  if (t <= 0) return {nullptr, 0, 0, 1.f, 0};
  if (p >= 1.0) return {nullptr, 0, 0, 0.f, 2};
  return {(const uint64_t*)seed, (uint32_t)(t < 4294967295.0 ? t : 4294967295.0), stream, (float)(1.0 / (1.0 - p)), 1};
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
__device__ __forceinline__ u32x4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}
// Bit e of the answer: whether element e of a chunk is kept.
template <int V>
__device__ __forceinline__ uint32_t kept_bits(const Drop& d, uint64_t key, int64_t row, int at) {
  if (d.mode != 1) return d.mode == 0 ? 0xffu : 0u;
  uint32_t bits = 0;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const u32x4 w = philox((uint32_t)(at / 4 + q), (uint32_t)row, (uint32_t)(row >> 32), d.stream, (uint32_t)key, (uint32_t)(key >> 32));
#pragma unroll
    for (int e = 0; e < 4; ++e) bits |= w[e] >= d.below ? 1u << (4 * q + e) : 0u;
    __builtin_amdgcn_sched_barrier(0);
  }
  return bits;
}
// drop_chunk() by such bits, without the factor.
template <int V>
__device__ __forceinline__ void drop_by(float (&v)[V], const Drop& d, uint32_t bits) {
  if (d.mode == 0) return;
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = __uint_as_float(__float_as_uint(v[e]) & (uint32_t)__builtin_amdgcn_sbfe((int)bits, e, 1));
}
// A packed chunk by such bits.
template <class T>
__device__ __forceinline__ u32x4 drop_packed(u32x4 u, const Drop& d, uint32_t bits) {
  if (d.mode == 0) return u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Traits<T>::VEC == 4) {
      u[i] &= (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
    } else {
      const uint32_t lo = (uint32_t)__builtin_amdgcn_sbfe((int)bits, 2 * i, 1), hi = (uint32_t)__builtin_amdgcn_sbfe((int)bits, 2 * i + 1, 1);
      u[i] &= (lo & 0xffffu) | (hi & 0xffff0000u);
    }
  }
  return u;
}
// v where it is kept, times 1 / (1 - p); zero, whatever v is, where it is dropped.  `at` is a multiple of four.
template <int V>
__device__ __forceinline__ void drop_chunk(float (&v)[V], const Drop& d, uint64_t key, int64_t row, int at) {
  if (d.mode == 0) return;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    u32x4 w = {0, 0, 0, 0};
    if (d.mode == 1)
      w = philox((uint32_t)(at / 4 + q), (uint32_t)row, (uint32_t)(row >> 32), d.stream, (uint32_t)key, (uint32_t)(key >> 32));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * q + e] = d.mode == 1 && w[e] >= d.below ? v[4 * q + e] * d.keep : 0.f;
    __builtin_amdgcn_sched_barrier(0);             // one block of the generator after another: fewer registers
  }
}

}  // namespace rowvec
}  // namespace maba
