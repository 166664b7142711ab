// A key / value cache held in 4 bits: e2m1 floats (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one
// power-of-two scale per 32 elements of a head's row, in pages of `page` tokens:
//   codes [pages][2: K, V][Hk][page][hd / 2]   (the first element of a pair in the low half of the byte)
//   scales [pages][2][Hk][page][hd / 32]       (E8M0: 2^(code - 127))
// The scale is the smallest power of two that brings the block's largest magnitude within 6 (nothing is
// clipped; code 127 for a block of zeros, at least 1), a value rounds to the nearest level, ties to the
// even code.  A block with an infinity or a NaN takes code 255 and stands for NaN.  Scaling by a power of
// two is exact, so the codes do not depend on how they are computed.  Bound: HBM, x read once and
// 4.25 bits per element written (append), or the reverse (read): 14.5 and 13 us for 62 MB (8 x 1500
// tokens, 8 heads of 128 bf16), 4.2 and 4.7 of a copy's 4.7 TB/s; fp32 23 and 26 us for 111 MB.
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
  if (t < 0 || t >= (int64_t)a.table_cols * a.page) return -1;
  const int at = (int)t / a.page, pg = a.table[b * a.table_ld + at];
  return pg < 0 || pg >= a.pages ? -1 : ((int64_t)pg * 2 * a.Hk + h) * a.page + ((int)t - at * a.page);
}

// Grid: (tiles of tokens, Hk x {K, V}, B).  HD / 8 lanes per row of 8 elements each (four to a block of
// 32), so a wave reads whole rows and writes the codes of successive tokens, which lie side by side.
constexpr int kKv4Tile = 64;  // tokens per workgroup
template <int HD> constexpr int kv4_rows() { return 256 / (HD / 8); }

template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_append(Kv4Args a) {
  constexpr int RUNS = HD / 8, ROWS = kv4_rows<HD>(), IT = (kKv4Tile + ROWS - 1) / ROWS;
  const int run = threadIdx.x % RUNS, r0 = threadIdx.x / RUNS, h = blockIdx.y >> 1, kv = blockIdx.y & 1, b = blockIdx.z;
  const int n = a.count ? min(a.n, a.count[b]) : a.n, i0 = blockIdx.x * kKv4Tile;
  const int64_t start = a.start[b];
  const SlideView& x = kv ? a.v : a.k;
  float v[IT][8];
  int64_t at[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {  // every load before the first use
    const int r = r0 + k * ROWS, i = i0 + r;
    at[k] = r0 < ROWS && r < kKv4Tile && i < n ? kv4_row(a, b, start + i, h) : -1;
    Vec8<T>::load(row<T>(x, b, min(i, a.n - 1), h) + run * 8, v[k]);
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    if (at[k] < 0) continue;  // (the four lanes of a block together)
    uint32_t amax = 0;        // the largest magnitude, as bits: infinities and NaN compare above every number
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[k][e]) & 0x7fffffffu);
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1, 64));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2, 64));
    // amax = 1.f 2^(x - 127) lies within 6 = 1.5 * 2^2 scaled by 2^(x - 129), or the next power past 1.5
    int code = (int)(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x400000u);
    code = amax == 0 ? 127 : amax >= 0x7f800000u ? 255 : code < 1 ? 1 : code;
    const float s = __uint_as_float((uint32_t)code << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[k][0], v[k][1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[k][2], v[k][3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[k][4], v[k][5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[k][6], v[k][7], s, 3);
    const int64_t o = at[k] + (int64_t)kv * a.Hk * a.page;
    *(uint32_t*)(a.codes + o * (HD / 2) + run * 4) = code == 255 ? 0 : c;
    if ((run & 3) == 0) a.scales[o * (HD / 32) + run / 4] = (uint8_t)code;
  }
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_read(Kv4Args a) {
  constexpr int RUNS = HD / 8, ROWS = kv4_rows<HD>(), IT = (kKv4Tile + ROWS - 1) / ROWS;
  const int run = threadIdx.x % RUNS, r0 = threadIdx.x / RUNS, h = blockIdx.y >> 1, kv = blockIdx.y & 1, b = blockIdx.z;
  const int i0 = blockIdx.x * kKv4Tile;
  const int64_t start = a.start[b];
  const SlideView& y = kv ? a.v : a.k;
  uint32_t c[IT], e[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int64_t at = kv4_row(a, b, start + i0 + r0 + k * ROWS, h), o = (at < 0 ? 0 : at) + (int64_t)kv * a.Hk * a.page;
    c[k] = *(const uint32_t*)(a.codes + o * (HD / 2) + run * 4);
    e[k] = a.scales[o * (HD / 32) + run / 4];
    if (at < 0) c[k] = 0, e[k] = 127;
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int r = r0 + k * ROWS, i = i0 + r;
    if (r0 >= ROWS || r >= kKv4Tile || i >= a.n) continue;
    const float s = kv4_scale(e[k]);
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], s, 1);
    const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], s, 3);
    const float v[8] = {p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    Vec8<T>::store(row<T>(y, b, i, h) + run * 8, v);
  }
}

static int kv4_check(const char* who, int dtype, int B, int n, int Hk, int hd, const SlideView& k, const SlideView& v,
                     const void* codes, const void* scales, int pages, int page, const int32_t* table,
                     int64_t table_ld, int table_cols) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "%s: dtype", who);
  CAPK_CHECK_ARG(B >= 0 && B <= 65535 && n >= 0 && n <= (1 << 28) && Hk >= 1 && Hk <= 32767, "%s: bad sizes", who);
  CAPK_CHECK_ARG(hd == 32 || hd == 64 || hd == 96 || hd == 128, "%s: hd=%d must be 32, 64, 96 or 128", who, hd);
  CAPK_CHECK_ARG(page >= 16 && page % 16 == 0 && page <= 4096, "%s: page=%d must be a multiple of 16, <= 4096", who, page);
  CAPK_CHECK_ARG(pages >= 1 && codes && scales && (uintptr_t)codes % 16 == 0, "%s: pages must be 16-B aligned", who);
  CAPK_CHECK_ARG((table || B == 0 || n == 0) && table_cols >= 1 && table_ld >= table_cols && (int64_t)table_cols * page <= (1 << 28),
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

#define KV4_LAUNCH(KERNEL)                                                                               \
  {                                                                                                     \
    const dim3 grid(cdiv(n, kKv4Tile), 2 * Hk, B);                                                      \
    SLIDE_HD(hd, {                                                                                      \
      if (dtype == CAPK_BF16) hipLaunchKernelGGL((KERNEL<bf16, HDP>), grid, 256, 0, S(stream), a);      \
      else hipLaunchKernelGGL((KERNEL<float, HDP>), grid, 256, 0, S(stream), a);                        \
    })                                                                                                  \
    CAPK_LAUNCH_CHECK(#KERNEL);                                                                         \
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
  KV4_LAUNCH(kv4_append);
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
  KV4_LAUNCH(kv4_read);
  return CAPK_OK;
}

constexpr int kKv4Heads = 1 << 20;  // query heads: 65535 workgroups of 16 columns (head, query) at most

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
  // (sizes that the entry refuses have no workspace)
  if (B < 1 || B > 65535 || Hk < 1 || H < Hk || H > kKv4Heads || H % Hk || Nq < 1 || Nq > 64 || hd < 1 || hd > 128 ||
      window < 0 || sinks < 0 || page < 1 || table_cols < 1 || (int64_t)table_cols * page > (1 << 28))
    return 0;
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
  CAPK_CHECK_ARG(H >= Hk && H <= kKv4Heads && H % Hk == 0, "capk_kv4_attention: %d query heads over %d key heads", H, Hk);
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
