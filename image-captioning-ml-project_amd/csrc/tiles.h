// Matrix-core fragments shared by the sliding-window and 4-bit-cache attention kernels.
//
// A fragment is 8 values per lane.  In a 32x32 product lane l holds row (A) or column (B) l & 31 and
// the contraction slots (h = l >> 5, e = 0..7) of a 16-deep step; in a 16x16 product row / column
// l & 15 and slots (g = l >> 4, e) of a 32-deep step.  bf16 runs one instruction per step; the fp32 form of
// the latter runs eight 4-deep ones, the e-th over slots (., e), so both types share every index below.
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
  __device__ __forceinline__ static f32x4 mma16(V8 a, V8 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static void store4(float* p, f32x4 v) { *(f32x4*)p = v; }
};

// The operands of the attention products.  bf16 values are fragments as they are.  An fp32 value goes through
// the bf16 unit as three bf16 parts, x = h + m + l to 2^-26 of it, and a product as the six part products
// above 2^-26: 6 x 32 clocks for a 32x32x16 step, where the fp32 instructions take 8 x 64.
struct Split8 {
  bf16x8 h, m, l;
};
template <typename T> struct Mat;
template <> struct Mat<bf16> {
  using V8 = bf16x8;
  __device__ __forceinline__ static V8 pack(const float (&x)[8]) {
    V8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = (bf16)x[e];
    return r;
  }
  __device__ __forceinline__ static void set(V8& r, int e, float x) { r[e] = (bf16)x; }
  __device__ __forceinline__ static V8 from(bf16x8 x) { return x; }
  __device__ __forceinline__ static f32x16 mma32(const V8& a, const V8& b, f32x16 c) { return Tile<bf16>::mma32(a, b, c); }
};
template <> struct Mat<float> {
  using V8 = Split8;
  __device__ __forceinline__ static V8 pack(const float (&x)[8]) {
    V8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) set(r, e, x[e]);
    return r;
  }
  __device__ __forceinline__ static void set(V8& r, int e, float x) {
    r.h[e] = (bf16)x;
    const float y = x - (float)r.h[e];
    r.m[e] = (bf16)y;
    r.l[e] = (bf16)(y - (float)r.m[e]);
  }
  __device__ __forceinline__ static V8 from(f32x8 x) {
    const float y[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
    return pack(y);
  }
  __device__ __forceinline__ static f32x16 mma32(const V8& a, const V8& b, f32x16 c) {
    c = Tile<bf16>::mma32(a.h, b.l, c);
    c = Tile<bf16>::mma32(a.l, b.h, c);
    c = Tile<bf16>::mma32(a.m, b.m, c);
    c = Tile<bf16>::mma32(a.h, b.m, c);
    c = Tile<bf16>::mma32(a.m, b.h, c);
    return Tile<bf16>::mma32(a.h, b.h, c);
  }
};

// Fragments loaded before a loop: waited for here.  Otherwise the compiler waits at their first use, inside
// the loop and in every turn of it, and with them for the copies that are meant to stay in flight.
__device__ __forceinline__ void tile_settle(bf16x8& f) { asm volatile("" : "+v"(f)); }
__device__ __forceinline__ void tile_settle(Split8& f) { asm volatile("" : "+v"(f.h), "+v"(f.m), "+v"(f.l)); }

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

// An LDS image of a [rows][HDP] matrix: unpadded rows of 16-B chunks, chunk c of row r stored at chunk
// c ^ swz(r).  The masks put the 16 lanes that a b128 read serves together ({0-3, 12-15, 20-27} and so on:
// one chunk of 16 rows) and the 32 lanes of a transposed b64 read (four chunks of 4 rows) on distinct
// banks, and leave whole 1-KiB pieces contiguous, as the copy straight from memory needs them.
template <typename T, int HDP> struct TileImg;
template <int HDP> struct TileImg<bf16, HDP> {
  using T = bf16;
  static constexpr int RB = HDP * 2, PER = 8;  // bytes of a row, elements of a chunk
  __device__ __forceinline__ static int swz(int r) {
    if constexpr (HDP == 128) return (r & 3) << 2 | ((r >> 2) & 3);
    else if constexpr (HDP == 64) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  static constexpr int bytes(int rows) { return rows * RB; }

  // Copies rows r0 .. r0 + ROWS - 1 of `src` (row stride rs) into the image, 1 KiB per wave and
  // instruction; rows past `last` repeat it, columns past hd repeat column 0.  src, img, w and the rows are
  // the same for the whole wave; 64 rows span less than 2^31 bytes.  The image is there after the issuing
  // waves waited for vmcnt(0) and met at a barrier.  Written as assembly (it has no destination register):
  // for the builtin the compiler assumes that any transposed LDS read may touch the copy in flight, and
  // waits for it there -- in the middle of the tile that the copy is meant to overlap.
  template <int ROWS, int WAVES>
  __device__ __forceinline__ static void dma(char* img, const T* src, int64_t rs, int r0, int last, int hd, int w, int lane) {
    static_assert(ROWS * RB % (1024 * WAVES) == 0, "whole pieces for every wave");
    constexpr int N = ROWS * RB / 1024 / WAVES;
    constexpr int STEP = 1024 * WAVES / RB;  // rows from one piece of a wave to its next
    constexpr bool SAME = 1024 * WAVES % RB == 0 && STEP % 16 == 0;  // same columns in every piece of a lane
    const uint32_t lds = (uint32_t)(uintptr_t)LDS_PTR(char, img) + w * 1024, rsb = (uint32_t)(rs * (int)sizeof(T));
    const char* base = (const char*)(src + (int64_t)r0 * rs);
    const int left = last - r0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = (SAME ? 0 : i * 1024 * WAVES) + w * 1024 + lane * 16, r = o / RB, c = ((o % RB / 16) ^ swz(r)) * PER;
      const uint32_t col = (c < hd ? c : 0) * (uint32_t)sizeof(T);
      uint32_t off = r * rsb + col;
      const char* at = base;
      if (SAME) at += (int64_t)(i * STEP) * rsb;
      if (left < ROWS - 1) {  // the last rows: clamped one by one
        at = base;
        off = min(r + (SAME ? i * STEP : 0), left) * rsb + col;
      }
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(lds + i * WAVES * 1024), "v"(off), "s"(at)
                   : "memory");
    }
  }
  // zeros in the rows whose bit of `rows` is set (256 threads)
  __device__ __forceinline__ static void clear(char* img, uint64_t rows) {
    for (int o = (threadIdx.x & 255) * 16; o < 64 * RB; o += 256 * 16)
      if (rows >> (o / RB) & 1) *(f32x4*)(img + o) = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  // Byte offsets of a lane's reads: of a row fragment, and of the two halves of a transposed one.
  struct Lane {
    int f, ta, tb;
    __device__ __forceinline__ explicit Lane(int lane) {
      const int r = lane & 31, h = lane >> 5, i16 = lane & 15;
      f = r * RB + ((h ^ swz(r)) << 4);
      const int q = 4 * h + (i16 >> 2), c = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
      ta = q * RB + ((c ^ swz(q)) << 4) + (i16 & 1) * 8;
      tb = (q + 8) * RB + ((c ^ swz(q + 8)) << 4) + (i16 & 1) * 8;
    }
    // Makes the offsets opaque: what derives from them is computed again (an instruction each) where the
    // loop would otherwise hold it in registers that it does not have.
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(f), "+v"(ta), "+v"(tb)); }
  };
  static constexpr bool POW2 = (RB & (RB - 1)) == 0;
  // A / B fragment of a 32x32 product: row r0 + (l & 31), columns 16 s + 8 h (r0 a multiple of 32).  Chunk
  // 2 s beside the mask: an exclusive or, where rows are not a power of two of its masked bits.
  __device__ __forceinline__ static bf16x8 frag(const char* img, int r0, int s, const Lane& l) {
    return *(const bf16x8*)(img + r0 * RB + (POW2 ? l.f ^ (s * 32) : (l.f ^ ((s & 1) * 32)) + (s >> 1) * 64));
  }
  // A fragment of the transpose for a 32x32 product: lane column c0 + (l & 31), slot (h, e) = row
  // r0 + 8 (e >> 2) + 4 h + (e & 3) -- the order in which eight accumulator registers of a 32x32
  // product hold their rows (r0 a multiple of 16, c0 of 32).
  __device__ __forceinline__ static bf16x8 trans(const char* img, int r0, int c0, const Lane& l) {
    const char *a = img + r0 * RB + (POW2 ? l.ta ^ (c0 * 2) : l.ta + c0 * 2), *b = img + r0 * RB + (POW2 ? l.tb ^ (c0 * 2) : l.tb + c0 * 2);
    const bf16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, a));
    const bf16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, b));
    return (bf16x8){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  }
};
// The image of 64 rows of an fp32 matrix: its three bf16 parts one after the other, split once for all waves.
template <int HDP> struct TileImg<float, HDP> {
  using I = TileImg<bf16, HDP>;
  using Lane = typename I::Lane;
  static constexpr int PART = I::bytes(64);
  static constexpr int bytes(int rows) { return 3 * I::bytes(rows); }
  __device__ __forceinline__ static Split8 frag(const char* img, int r0, int s, const Lane& l) {
    return {I::frag(img, r0, s, l), I::frag(img + PART, r0, s, l), I::frag(img + 2 * PART, r0, s, l)};
  }
  __device__ __forceinline__ static Split8 trans(const char* img, int r0, int c0, const Lane& l) {
    return {I::trans(img, r0, c0, l), I::trans(img + PART, r0, c0, l), I::trans(img + 2 * PART, r0, c0, l)};
  }
};
// A fragment of the transpose of a row-major LDS image (row stride st) for a 16x16 product over 32 rows:
// lane column c0 + (l & 15), slot (g, e) = row r0 + 16 (e >> 2) + 4 g + (e & 3), the row order of two
// 16x16 accumulators.
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
// Sum / maximum with the lane 16 (32) away: a swap of the rows' odd and even (upper and lower) halves between two
// copies, in registers (through LDS, as shuffles go, it is 100 cycles and more in the path of every tile).
__device__ __forceinline__ f32x2 tile_swap16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return (f32x2){__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ f32x2 tile_swap32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return (f32x2){__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ float tile_max16(float x) { const f32x2 r = tile_swap16(x); return fmaxf(r[0], r[1]); }
__device__ __forceinline__ float tile_max32(float x) { const f32x2 r = tile_swap32(x); return fmaxf(r[0], r[1]); }
__device__ __forceinline__ float tile_sum16(float x) { const f32x2 r = tile_swap16(x); return r[0] + r[1]; }
__device__ __forceinline__ float tile_sum32(float x) { const f32x2 r = tile_swap32(x); return r[0] + r[1]; }

}  // namespace capk
