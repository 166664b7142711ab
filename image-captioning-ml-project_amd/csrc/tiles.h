// Matrix-core fragments shared by the sliding-window and 4-bit-cache attention kernels.
//
// A fragment is 8 values per lane.  In a 32x32 product lane l holds row (A) or column (B) l & 31 and
// the contraction slots (h = l >> 5, e = 0..7) of a 16-deep step; in a 16x16 product row / column
// l & 15 and slots (g = l >> 4, e) of a 32-deep step.  bf16 runs one instruction per step; fp32 runs
// eight 2-deep (4-deep) ones, the e-th over slots (., e), so both types share every index below.
// Accumulators: 32x32: lane column l & 31, register i row 8 (i >> 2) + 4 h + (i & 3);
// 16x16: lane column l & 15, register i row 4 g + i.
#pragma once
#include "common.h"

namespace capk {

typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr float kTileLog2e = 1.4426950408889634f, kTileLn2 = 0.6931471805599453f;

template <typename T> struct Tile;
template <> struct Tile<bf16> {
  using V8 = bf16x8;
  __device__ __forceinline__ static V8 load(const bf16* p) { return *(const bf16x8*)p; }
  __device__ __forceinline__ static f32x16 mma32(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static f32x4 mma16(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static void store4(bf16* p, f32x4 v) {
    bf16x4 r = {(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
    *(bf16x4*)p = r;
  }
};
template <> struct Tile<float> {
  using V8 = f32x8;
  __device__ __forceinline__ static V8 load(const float* p) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
    return (V8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  __device__ __forceinline__ static f32x16 mma32(V8 a, V8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static f32x4 mma16(V8 a, V8 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static void store4(float* p, f32x4 v) { *(f32x4*)p = v; }
};

template <typename T> __device__ __forceinline__ typename Tile<T>::V8 tile_zero8() {
  typename Tile<T>::V8 z;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = (T)0.f;
  return z;
}
template <typename V> __device__ __forceinline__ V tile_zero() {
  V z;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) z[i] = 0.f;
  return z;
}

// A fragment of the transpose of a row-major LDS image for a 32-deep-row product: lane column
// c0 + (l & 31), slot (h, e) = image row r0 + 8 (e >> 2) + 4 h + (e & 3) -- the row order in which
// eight accumulator registers of a 32x32 product hold their rows.
__device__ __forceinline__ bf16x8 tile_trans32(const bf16* img, int st, int r0, int c0, int lane) {
  const int i16 = lane & 15;
  const bf16* a = img + (r0 + 4 * (lane >> 5) + (i16 >> 2)) * st + c0 + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
  const bf16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, a));
  const bf16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, a + 8 * st));
  return (bf16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
}
__device__ __forceinline__ f32x8 tile_trans32(const float* img, int st, int r0, int c0, int lane) {
  const float* a = img + (r0 + 4 * (lane >> 5)) * st + c0 + (lane & 31);
  f32x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = a[(8 * (e >> 2) + (e & 3)) * st];
  return r;
}
// The same for a 16x16 product over 32 image rows: lane column c0 + (l & 15), slot (g, e) = image row
// r0 + 16 (e >> 2) + 4 g + (e & 3), the row order of two 16x16 accumulators.
__device__ __forceinline__ bf16x8 tile_trans16(const bf16* img, int st, int r0, int c0, int lane) {
  const int i16 = lane & 15;
  const bf16* a = img + (r0 + 4 * (lane >> 4) + (i16 >> 2)) * st + c0 + 4 * (i16 & 3);
  const bf16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, a));
  const bf16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, a + 16 * st));
  return (bf16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
}
__device__ __forceinline__ f32x8 tile_trans16(const float* img, int st, int r0, int c0, int lane) {
  const float* a = img + (r0 + 4 * (lane >> 4)) * st + c0 + (lane & 15);
  f32x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = a[(16 * (e >> 2) + (e & 3)) * st];
  return r;
}
// v_exp_f32: 2^x; the arguments below are <= 0 or -inf (-> 0)
__device__ __forceinline__ float tile_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace capk
