// A key / value cache held in 4 bits: e2m1 floats (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one
// power-of-two scale per 32 elements of a head's row, in pages of `page` tokens:
//   codes [pages][2: K, V][Hk][page][hd / 2]   (the first element of a pair in the low half of the byte)
//   scales [pages][2][Hk][page][hd / 32]       (E8M0: 2^(code - 127))
// The scale is the smallest power of two that brings the block's largest magnitude within 6 (nothing is
// clipped; code 127 for a block of zeros, at least 1), a value rounds to the nearest level, ties to the
// even code.  A block with an infinity or a NaN takes code 255 and stands for NaN.  Scaling by a power of
// two is exact, so the codes do not depend on how they are computed.  Bound: HBM, x read once and
// 4.25 bits per element written (append), or the reverse (read).
#include "sliding.h"

namespace capk {

struct Kv4Args {
  int B, n, Hk, hd, pages, page;
  SlideView k, v;  // x or, read back, y
  uint8_t *codes, *scales;
  const int32_t* table;
  int64_t table_ld;
  int table_cols;
  const int32_t *start, *count;
};

// the row of K (V: + Hk * page) of token t of sequence b, -1 where the table has no page for it
__device__ __forceinline__ int64_t kv4_row(const Kv4Args& a, int b, int64_t t, int h) {
  if (t < 0 || t / a.page >= a.table_cols) return -1;
  const int pg = a.table[b * a.table_ld + t / a.page];
  return pg < 0 || pg >= a.pages ? -1 : ((int64_t)pg * 2 * a.Hk + h) * a.page + t % a.page;
}

// Four lanes per block of 32: 8 elements each.  Grid-stride items (b, i, h, K / V, run of 8).
template <typename T>
__global__ __launch_bounds__(256) void kv4_append(Kv4Args a) {
  const int runs = a.hd / 8;
  const int64_t items = (int64_t)a.B * a.n * a.Hk * 2 * runs;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < items; x += (int64_t)gridDim.x * 256) {
    // the four lanes of a block share everything but the run, so they stay together
    const int run = (int)(x % runs), h = (int)(x / runs % a.Hk), kv = (int)(x / runs / a.Hk % 2);
    const int64_t bi = x / runs / a.Hk / 2;
    const int b = (int)(bi / a.n), i = (int)(bi % a.n);
    if (a.count && i >= a.count[b]) continue;
    const int64_t r = kv4_row(a, b, (int64_t)a.start[b] + i, h);
    if (r < 0) continue;
    float v[8];
    Vec8<T>::load(row<T>(kv ? a.v : a.k, b, i, h) + run * 8, v);
    uint32_t amax = 0;  // the largest magnitude, as bits: infinities and NaN compare above every number
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1, 64));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2, 64));
    // amax = 1.f 2^(x - 127) lies within 6 = 1.5 * 2^2 scaled by 2^(x - 129), or the next power past 1.5
    int code = (int)(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x400000u);
    code = amax == 0 ? 127 : amax >= 0x7f800000u ? 255 : code < 1 ? 1 : code;
    const float s = __uint_as_float((uint32_t)code << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    const int64_t at = r + (int64_t)kv * a.Hk * a.page;
    *(uint32_t*)(a.codes + at * (a.hd / 2) + run * 4) = code == 255 ? 0 : c;
    if ((run & 3) == 0) a.scales[at * (a.hd / 32) + run / 4] = (uint8_t)code;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void kv4_read(Kv4Args a) {
  const int runs = a.hd / 8;
  const int64_t items = (int64_t)a.B * a.n * a.Hk * 2 * runs;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < items; x += (int64_t)gridDim.x * 256) {
    const int run = (int)(x % runs), h = (int)(x / runs % a.Hk), kv = (int)(x / runs / a.Hk % 2);
    const int64_t bi = x / runs / a.Hk / 2;
    const int b = (int)(bi / a.n), i = (int)(bi % a.n);
    const int64_t r = kv4_row(a, b, (int64_t)a.start[b] + i, h);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r >= 0) {
      const int64_t at = r + (int64_t)kv * a.Hk * a.page;
      const uint32_t c = *(const uint32_t*)(a.codes + at * (a.hd / 2) + run * 4);
      const float s = kv4_scale(a.scales[at * (a.hd / 32) + run / 4]);
      const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
      const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
      v[0] = p0[0]; v[1] = p0[1]; v[2] = p1[0]; v[3] = p1[1]; v[4] = p2[0]; v[5] = p2[1]; v[6] = p3[0]; v[7] = p3[1];
    }
    Vec8<T>::store(row<T>(kv ? a.v : a.k, b, i, h) + run * 8, v);
  }
}

static int kv4_check(const char* who, int dtype, int B, int n, int Hk, int hd, const SlideView& k, const SlideView& v,
                     const void* codes, const void* scales, int pages, int page, const int32_t* table,
                     int64_t table_ld, int table_cols) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "%s: dtype", who);
  CAPK_CHECK_ARG(B >= 0 && n >= 0 && Hk >= 1, "%s: bad sizes", who);
  CAPK_CHECK_ARG(hd == 32 || hd == 64 || hd == 96 || hd == 128, "%s: hd=%d must be 32, 64, 96 or 128", who, hd);
  CAPK_CHECK_ARG(page >= 16 && page % 16 == 0 && page <= 4096, "%s: page=%d must be a multiple of 16, <= 4096", who, page);
  CAPK_CHECK_ARG(pages >= 1 && codes && scales && (uintptr_t)codes % 16 == 0, "%s: pages must be 16-B aligned", who);
  CAPK_CHECK_ARG(table && table_cols >= 1 && table_ld >= table_cols && (int64_t)table_cols * page <= (1 << 28),
                 "%s: page table of %d columns (at most 2^28 tokens)", who, table_cols);
  const int ea = dtype == CAPK_BF16 ? 8 : 4;
  for (const SlideView* x : {&k, &v})
    CAPK_CHECK_ARG(B == 0 || n == 0 ||
                       (x->p && (uintptr_t)x->p % 16 == 0 && x->bs % ea == 0 && x->rs % ea == 0 && x->hs % ea == 0),
                   "%s: K / V rows must be 16-B aligned with strides that keep it so", who);
  return CAPK_OK;
}

}  // namespace capk

using namespace capk;

static int kv4_blocks(const Kv4Args& a) {
  const int64_t items = (int64_t)a.B * a.n * a.Hk * 2 * (a.hd / 8);
  return (int)(cdiv(items, 256) < 16384 ? cdiv(items, 256) : 16384);
}

extern "C" int capk_kv4_append(int dtype, int B, int n, int Hk, int hd, const void* k, int64_t k_bs, int64_t k_rs,
                               int64_t k_hs, const void* v, int64_t v_bs, int64_t v_rs, int64_t v_hs, void* codes,
                               void* scales, int pages, int page, const int32_t* table, int64_t table_ld,
                               int table_cols, const int32_t* start, const int32_t* count, void* stream) {
  Kv4Args a{B, n, Hk, hd, pages, page, {(void*)k, k_bs, k_rs, k_hs}, {(void*)v, v_bs, v_rs, v_hs},
            (uint8_t*)codes, (uint8_t*)scales, table, table_ld, table_cols, start, count};
  int rc = kv4_check("capk_kv4_append", dtype, B, n, Hk, hd, a.k, a.v, codes, scales, pages, page, table, table_ld, table_cols);
  if (rc) return rc;
  if (B == 0 || n == 0) return CAPK_OK;
  CAPK_CHECK_ARG(start, "capk_kv4_append: start");
  if (dtype == CAPK_BF16) hipLaunchKernelGGL(kv4_append<bf16>, kv4_blocks(a), 256, 0, S(stream), a);
  else hipLaunchKernelGGL(kv4_append<float>, kv4_blocks(a), 256, 0, S(stream), a);
  CAPK_LAUNCH_CHECK("kv4_append");
  return CAPK_OK;
}

extern "C" int capk_kv4_read(int dtype, int B, int n, int Hk, int hd, const void* codes, const void* scales, int pages,
                             int page, const int32_t* table, int64_t table_ld, int table_cols, const int32_t* start,
                             void* k, int64_t k_bs, int64_t k_rs, int64_t k_hs, void* v, int64_t v_bs, int64_t v_rs,
                             int64_t v_hs, void* stream) {
  Kv4Args a{B, n, Hk, hd, pages, page, {k, k_bs, k_rs, k_hs}, {v, v_bs, v_rs, v_hs},
            (uint8_t*)codes, (uint8_t*)scales, table, table_ld, table_cols, start, nullptr};
  int rc = kv4_check("capk_kv4_read", dtype, B, n, Hk, hd, a.k, a.v, codes, scales, pages, page, table, table_ld, table_cols);
  if (rc) return rc;
  if (B == 0 || n == 0) return CAPK_OK;
  CAPK_CHECK_ARG(start, "capk_kv4_read: start");
  if (dtype == CAPK_BF16) hipLaunchKernelGGL(kv4_read<bf16>, kv4_blocks(a), 256, 0, S(stream), a);
  else hipLaunchKernelGGL(kv4_read<float>, kv4_blocks(a), 256, 0, S(stream), a);
  CAPK_LAUNCH_CHECK("kv4_read");
  return CAPK_OK;
}

static StepArgs kv4_step(int B, int H, int Hk, int Nq, int hd, float scale, int window, int sinks, int pages, int page,
                         int table_cols) {
  StepArgs a{};
  a.B = B; a.H = H; a.Hk = Hk; a.Nq = Nq; a.hd = hd; a.scale = scale;
  a.cap = table_cols * page;
  a.window = window == 0 || window > a.cap + Nq ? a.cap + Nq : window;
  a.sinks = sinks > a.cap ? a.cap : sinks;
  a.pages = pages; a.page = page;
  return a;
}

extern "C" size_t capk_kv4_attention_workspace(int dtype, int B, int H, int Hk, int Nq, int hd, int window, int sinks,
                                               int page, int table_cols) {
  if (B < 1 || Hk < 1 || H < Hk || Nq < 1 || hd < 1 || window < 0 || sinks < 0 || page < 1 || table_cols < 1) return 0;
  int splits;
  return step_workspace(dtype, kv4_step(B, H, Hk, Nq, hd, 0.f, window, sinks, 1, page, table_cols), &splits);
}

extern "C" int capk_kv4_attention(int dtype, int B, int H, int Hk, int Nq, int hd, float scale, int window, int sinks,
                                  const void* q, int64_t q_bs, int64_t q_rs, int64_t q_hs, const void* codes,
                                  const void* scales, int pages, int page, const int32_t* table, int64_t table_ld,
                                  int table_cols, const int32_t* kv_len, void* o, int64_t o_bs, int64_t o_rs,
                                  int64_t o_hs, float* lse, void* ws, size_t ws_bytes, void* stream) {
  const SlideView qv = {(void*)q, q_bs, q_rs, q_hs}, ov = {o, o_bs, o_rs, o_hs};
  int rc = kv4_check("capk_kv4_attention", dtype, B, Nq, Hk, hd, qv, ov, codes, scales, pages, page, table, table_ld, table_cols);
  if (rc) return rc;
  if (B == 0) return CAPK_OK;
  CAPK_CHECK_ARG(H >= Hk && H % Hk == 0, "capk_kv4_attention: %d query heads over %d key heads", H, Hk);
  CAPK_CHECK_ARG(Nq >= 1 && Nq <= 64, "capk_kv4_attention: Nq=%d must be 1..64", Nq);
  CAPK_CHECK_ARG(B <= 65535 && Hk * (int64_t)cdiv((int64_t)Nq * (H / Hk), 16) <= 65535, "capk_kv4_attention: too many heads or sequences");
  CAPK_CHECK_ARG(window >= 0 && sinks >= 0, "capk_kv4_attention: window and sinks must not be negative");
  CAPK_CHECK_ARG(scale > 0.f && scale < INFINITY, "capk_kv4_attention: scale must be positive");
  CAPK_CHECK_ARG(kv_len, "capk_kv4_attention: kv_len");
  StepArgs a = kv4_step(B, H, Hk, Nq, hd, scale, window, sinks, pages, page, table_cols);
  a.q = qv; a.o = ov; a.len = kv_len; a.lse = lse;
  a.codes = (const uint8_t*)codes; a.scales = (const uint8_t*)scales;
  a.table = table; a.table_ld = table_ld;
  return step_launch(dtype, a, ws, ws_bytes, S(stream));
}
