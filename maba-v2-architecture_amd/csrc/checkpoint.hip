// Activation checkpoints in 8 bits.  Every 32 consecutive elements of a row share a power of two 2^e, the smallest
// with max|x| <= 448 * 2^e (e in [-127, 127], the maximum over the finite ones), kept as the byte e + 127; each element
// is x / 2^e rounded to nearest even as an e4m3 number (448 is the type's largest, so nothing saturates).  NaN and
// infinities become e4m3's NaN: a backward pass that reads one sees it.  The scale costs a byte per 32 elements, and as
// a power of two it costs no accuracy: code * 2^e is exact in fp32 and, but for its subnormals, in bf16.
//
// Bound: HBM.  Four lanes share a group, eight elements each.
#include <algorithm>

#include "ffn_common.h"

namespace maba {
namespace ffn {

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, int n, bool vec, float (&v)[8]) {
  if (vec) {
    if constexpr (DT == MABA_F32) {
      const f32x4 a = *(const f32x4*)((const float*)base + i), b = *(const f32x4*)((const float*)base + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
      const u32x4 u = *(const u32x4*)((const uint16_t*)base + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = DT == MABA_BF16 ? Bf16::up(u[j] & 0xffffu) : Fp16::up(u[j] & 0xffffu);
        v[2 * j + 1] = DT == MABA_BF16 ? Bf16::up(u[j] >> 16) : Fp16::up(u[j] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? load_elem(base, DT, i + j) : 0.f;
  }
}

struct PackArgs {
  const void* x; int64_t xs;
  uint8_t* codes; int64_t cs;
  uint8_t* scales; int64_t ss;
  int64_t rows;
  int C, groups, vec;
};

template <int DT>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
  const int per = a.groups * 4;                       // 8-element slots of a row, whole groups of four
  const int64_t total = a.rows * per;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int slot = (int)(i % per), k = slot * 8, n = min(8, a.C - k);      // n <= 0: a slot past the row
    float v[8];
    if (n > 0) load8<DT>(a.x, r * a.xs + k, n, a.vec, v);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    uint32_t m = 0;                                   // the largest finite magnitude's bits
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
      m = max(m, b < 0x7f800000u ? b : 0u);
    }
    // the four lanes of a group are neighbours, and total is a multiple of four
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    // m = 1.f * 2^(E - 127); 448 = 1.75 * 2^8
    const int e = max((int)(m >> 23) - 127 - 8 + ((m & 0x7fffffu) > 0x600000u), -127);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_ldexpf(v[4 * h + j], -e);
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], p, true);
      w[h] = (uint32_t)p;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((__float_as_uint(v[4 * h + j]) & 0x7fffffffu) >= 0x7f800000u) w[h] = (w[h] & ~(0xffu << (8 * j))) | (0x7fu << (8 * j));
    }
    uint8_t* o = a.codes + r * a.cs + k;
    if (a.vec && n > 0) {
      const u32x2 u = {w[0], w[1]};
      *(u32x2*)o = u;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) o[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
    if ((slot & 3) == 0) a.scales[r * a.ss + (slot >> 2)] = (uint8_t)(e + 127);
  }
}

struct UnpackArgs {
  const uint8_t* codes; int64_t cs;
  const uint8_t* scales; int64_t ss;
  void* y; int64_t ys;
  int64_t rows;
  int C, slots, vec;
};

template <int DT>
__global__ __launch_bounds__(256) void unpack_kernel(UnpackArgs a) {
  const int64_t total = a.rows * a.slots;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / a.slots;
    const int k = (int)(i % a.slots) * 8, n = min(8, a.C - k);
    const uint8_t* p = a.codes + r * a.cs + k;
    const int e = (int)a.scales[r * a.ss + (k >> 5)] - 127;
    u32x2 w = {0, 0};
    if (a.vec) w = *(const u32x2*)p;
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j >> 2] |= (j < n ? (uint32_t)p[j] : 0u) << (8 * (j & 3));
    constexpr float most = DT == MABA_F32 ? 3.40282347e38f : DT == MABA_BF16 ? Bf16::MOST : Fp16::MOST;
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
      v[4 * h] = scaled(lo[0], e, most);
      v[4 * h + 1] = scaled(lo[1], e, most);
      v[4 * h + 2] = scaled(hi[0], e, most);
      v[4 * h + 3] = scaled(hi[1], e, most);
    }
    const int64_t o = r * a.ys + k;
    if (a.vec) {
      if constexpr (DT == MABA_F32) {
        *(f32x4*)((float*)a.y + o) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)((float*)a.y + o + 4) = f32x4{v[4], v[5], v[6], v[7]};
      } else {
        u32x4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          u[j] = DT == MABA_BF16 ? Bf16::down(v[2 * j]) | (Bf16::down(v[2 * j + 1]) << 16)
                                 : Fp16::down(v[2 * j]) | (Fp16::down(v[2 * j + 1]) << 16);
        *(u32x4*)((uint16_t*)a.y + o) = u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= n) continue;
        if constexpr (DT == MABA_F32) ((float*)a.y)[o + j] = v[j];
        else ((uint16_t*)a.y)[o + j] = (uint16_t)(DT == MABA_BF16 ? Bf16::down(v[j]) : Fp16::down(v[j]));
      }
    }
  }
}

// Rows whose 8-element slots are whole and aligned for vector access.
static bool vec_rows(const maba_tensor* t) {
  const int64_t size = t->dtype == MABA_F32 ? 4 : t->dtype == MABA_E4M3 ? 1 : 2;
  return t->shape[1] % 8 == 0 && t->stride[0] % 8 == 0 && (uintptr_t)t->data % std::min<uintptr_t>(16, 8 * size) == 0;
}

static int packed_check(const char* who, const maba_tensor* x, const maba_tensor* codes, const maba_tensor* scales) {
  if (!x || !codes || !scales) return fail(MABA_ERR_INVALID, "%s: three tensors required", who);
  if (!is_float_dt(x->dtype)) return fail(MABA_ERR_DTYPE, "%s: f32, f16 or bf16 only, got dtype code %d", who, x->dtype);
  int rc = check_rows(x, who, "x", x->dtype, -1, -1);
  if (!rc) rc = check_sizes(who, x->shape[0], x->shape[1], x->shape[1]);
  if (!rc) rc = check_rows(codes, who, "codes", MABA_E4M3, x->shape[0], x->shape[1]);
  if (!rc) rc = check_rows(scales, who, "scales", MABA_U8, x->shape[0], ceil_div(x->shape[1], 32));
  return rc;
}

}  // namespace ffn
}  // namespace maba

using namespace maba;
using namespace maba::ffn;

extern "C" int maba_hip_checkpoint_pack(const maba_tensor* x, maba_tensor* codes, maba_tensor* scales, void* stream) {
  const char* who = "checkpoint_pack";
  int rc = packed_check(who, x, codes, scales);
  if (!rc) rc = check_out(codes, who, "codes", MABA_E4M3, -1, -1);
  if (!rc) rc = check_out(scales, who, "scales", MABA_U8, -1, -1);
  if (rc) return rc;
  if (overlap(x, codes) || overlap(x, scales) || overlap(codes, scales)) return fail(MABA_ERR_INVALID, "%s: tensors overlap", who);
  const int C = (int)x->shape[1], groups = (C + 31) / 32;
  const PackArgs a = {x->data, x->stride[0], (uint8_t*)codes->data, codes->stride[0], (uint8_t*)scales->data, scales->stride[0],
                      x->shape[0], C, groups, vec_rows(x) && vec_rows(codes)};
  if (a.rows == 0) return MABA_OK;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(a.rows * groups * 4, 256), 65536));
  auto k = x->dtype == MABA_F32 ? pack_kernel<MABA_F32> : x->dtype == MABA_BF16 ? pack_kernel<MABA_BF16> : pack_kernel<MABA_F16>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(who);
}

extern "C" int maba_hip_checkpoint_unpack(const maba_tensor* codes, const maba_tensor* scales, maba_tensor* out, void* stream) {
  const char* who = "checkpoint_unpack";
  int rc = packed_check(who, out, codes, scales);
  if (!rc) rc = check_out(out, who, "out", out->dtype, -1, -1);
  if (rc) return rc;
  if (overlap(out, codes) || overlap(out, scales)) return fail(MABA_ERR_INVALID, "%s: tensors overlap", who);
  const int C = (int)out->shape[1];
  const UnpackArgs a = {(const uint8_t*)codes->data, codes->stride[0], (const uint8_t*)scales->data, scales->stride[0], out->data,
                        out->stride[0], out->shape[0], C, (C + 7) / 8, vec_rows(out) && vec_rows(codes)};
  if (a.rows == 0) return MABA_OK;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(a.rows * a.slots, 256), 65536));
  auto k = out->dtype == MABA_F32 ? unpack_kernel<MABA_F32> : out->dtype == MABA_BF16 ? unpack_kernel<MABA_BF16> : unpack_kernel<MABA_F16>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(who);
}
