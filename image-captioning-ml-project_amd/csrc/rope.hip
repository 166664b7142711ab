// Rotary positions over several axes.
//
// Pair i of a head (elements i and i + P of the rotated part in the halved layout, 2i and 2i + 1 in
// the interleaved one, P pairs) turns by a = pos[axis[i]] * freq[i]:
//   y1 = x1 cos a - x2 sin a,   y2 = x1 sin a + x2 cos a,
// and back by -a (the gradient).  The angle depends on the token and the pair only, so a workgroup
// computes the (cos, sin) of its tokens once into LDS and then streams every head of q and k through
// it.  Angles are formed in 64 bits as whole turns plus a fraction: at position 2e5 a 32-bit product
// is off by 1e-2 rad.  Bound: HBM, x read and y written once: 36 us for 154 MB (16 x 1568 tokens, 24 heads of
// 64 bf16), 4.3 of a copy's 4.7 TB/s; fp32 65 us for 309 MB.
#include "common.h"

namespace capk {

struct RopeSide {
  int H;
  const void* x;
  int64_t x_bs, x_rs, x_hs;
  void* y;
  int64_t y_bs, y_rs, y_hs;
};
struct RopeArgs {
  int B, N, hd, pairs, axes, tokens;  // tokens: per workgroup
  uint32_t per_mul, heads_mul;        // ceil(2^32 / .) of the items of a head and of the heads
  const int32_t* pos;
  int64_t pos_as, pos_bs;
  const double* freq;
  const uint8_t* axis;
  float sign;
  RopeSide side[2];
};

template <typename T, int V>
__device__ __forceinline__ void rope_ld(const T* p, float (&f)[V]) {
  typedef T vec __attribute__((ext_vector_type(V), aligned(V * sizeof(T) < 16 ? V * sizeof(T) : 16)));
  const vec v = *(const vec*)p;
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = (float)v[i];
}
template <typename T, int V>
__device__ __forceinline__ void rope_st(T* p, const float (&f)[V]) {
  typedef T vec __attribute__((ext_vector_type(V), aligned(V * sizeof(T) < 16 ? V * sizeof(T) : 16)));
  vec v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (T)f[i];
  *(vec*)p = v;
}

// i / d for i < 2^32 / d, from mul = ceil(2^32 / d) (d = 1: mul wraps to 0); i < 8 tokens x 1024 heads x
// 512 items and d <= 1024 here
__device__ __forceinline__ int rope_div(int i, uint32_t mul) { return mul ? (int)__umulhi((uint32_t)i, mul) : i; }

// V pairs per item; the elements past the rotated part are copied V at a time.  A thread loads four items
// before it stores the first.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  constexpr int U = 4;
  extern __shared__ float2 cs[];  // [tokens][pairs], then [tokens][4] row offsets: q in, q out, k in, k out
  int64_t* offs = (int64_t*)(cs + a.tokens * a.pairs);
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens, all = (int64_t)a.B * a.N;
  const int nt = (int)min((int64_t)a.tokens, all - t0);
  for (int i = threadIdx.x; i < nt * a.pairs; i += 256) {
    const int64_t t = t0 + i / a.pairs, b = t / a.N, n = t % a.N;
    const int p = i % a.pairs, ax = min((int)a.axis[p], a.axes - 1);
    const int pos = a.pos[ax * a.pos_as + b * a.pos_bs + n];
    const double turns = (double)pos * a.freq[p] * 0.15915494309189535;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[i] = make_float2(c, s * a.sign);
  }
  if ((int)threadIdx.x < nt * 4) {
    const int64_t t = t0 + threadIdx.x / 4, b = t / a.N, n = t % a.N;
    const RopeSide& s = a.side[threadIdx.x >> 1 & 1];
    offs[threadIdx.x] = threadIdx.x & 1 ? b * s.y_bs + n * s.y_rs : b * s.x_bs + n * s.x_rs;
  }
  __syncthreads();
  const int rot = 2 * a.pairs, nrot = a.pairs / V, per = nrot + (a.hd - rot) / V;
  const int heads = a.side[0].H + a.side[1].H, items = nt * heads * per;
  for (int base = threadIdx.x; base < items; base += 256 * U) {
    float x1[U][V], x2[U][V];
    T* out[U];
    int d2[U], tr[U];  // second element's offset (0: a copy), the item's first (cos, sin)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(base + u * 256, items - 1);
      const int th = rope_div(i, a.per_mul), c = i - th * per, tl = rope_div(th, a.heads_mul), hh = th - tl * heads;
      const bool k = hh >= a.side[0].H, copy = c >= nrot;
      const RopeSide& s = a.side[k];
      const int h = k ? hh - a.side[0].H : hh, d1 = copy ? rot + (c - nrot) * V : INTER ? 2 * c * V : c * V;
      const T* x = (const T*)s.x + offs[tl * 4 + 2 * k] + h * s.x_hs + d1;
      out[u] = (T*)s.y + offs[tl * 4 + 2 * k + 1] + h * s.y_hs + d1;
      d2[u] = copy ? 0 : INTER ? V : a.pairs;
      tr[u] = copy ? 0 : tl * a.pairs + c * V;
      rope_ld<T, V>(x, x1[u]);
      rope_ld<T, V>(x + d2[u], x2[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * 256 >= items) break;
      if (d2[u] == 0) {
        rope_st<T, V>(out[u], x1[u]);
        continue;
      }
      const float2* r = cs + tr[u];
      float y1[V], y2[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        // interleaved: the 2V elements are V pairs (x1, x2) in a row
        const float f = INTER ? (2 * k < V ? x1[u][2 * k % V] : x2[u][2 * k % V]) : x1[u][k];
        const float g = INTER ? (2 * k + 1 < V ? x1[u][(2 * k + 1) % V] : x2[u][(2 * k + 1) % V]) : x2[u][k];
        const float p = f * r[k].x - g * r[k].y, q = f * r[k].y + g * r[k].x;
        if (INTER) {
          (2 * k < V ? y1[2 * k % V] : y2[2 * k % V]) = p;
          (2 * k + 1 < V ? y1[(2 * k + 1) % V] : y2[(2 * k + 1) % V]) = q;
        } else {
          y1[k] = p;
          y2[k] = q;
        }
      }
      rope_st<T, V>(out[u], y1);
      rope_st<T, V>(out[u] + d2[u], y2);
    }
  }
}

template <typename T>
static int rope_launch(const RopeArgs& a, int V, bool inter, hipStream_t st) {
  const int grid = cdiv((int64_t)a.B * a.N, a.tokens);
  const size_t shm = (size_t)a.tokens * (a.pairs * sizeof(float2) + 4 * sizeof(int64_t));
#define ROPE_CASE(v)                                                                            \
  case v:                                                                                       \
    if (inter) hipLaunchKernelGGL((rope_kernel<T, v, true>), grid, 256, shm, st, a);            \
    else hipLaunchKernelGGL((rope_kernel<T, v, false>), grid, 256, shm, st, a);                 \
    break;
  switch (V) {
    ROPE_CASE(8)
    ROPE_CASE(4)
    ROPE_CASE(1)
  }
#undef ROPE_CASE
  CAPK_LAUNCH_CHECK("rope_kernel");
  return CAPK_OK;
}

}  // namespace capk

using namespace capk;

extern "C" int capk_axis_rope(int dtype, int B, int N, int hd, int pairs, int interleaved, int inverse, int axes,
                              const int32_t* pos, int64_t pos_as, int64_t pos_bs, const double* freq,
                              const uint8_t* axis, int Hq, const void* q, int64_t q_bs, int64_t q_rs, int64_t q_hs,
                              void* qo, int64_t qo_bs, int64_t qo_rs, int64_t qo_hs, int Hk, const void* k,
                              int64_t k_bs, int64_t k_rs, int64_t k_hs, void* ko, int64_t ko_bs, int64_t ko_rs,
                              int64_t ko_hs, void* stream) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "capk_axis_rope: dtype");
  CAPK_CHECK_ARG(B >= 0 && N >= 0 && Hq >= 1 && Hk >= 0 && axes >= 1 && axes <= 255, "capk_axis_rope: bad sizes");
  CAPK_CHECK_ARG(hd >= 2 && hd <= 512 && pairs >= 1 && 2 * pairs <= hd,
                 "capk_axis_rope: need 2 <= 2 * pairs <= hd <= 512 (pairs %d, hd %d)", pairs, hd);
  if (B == 0 || N == 0) return CAPK_OK;
  CAPK_CHECK_ARG(pos && freq && axis && q && qo && (Hk == 0 || (k && ko)), "capk_axis_rope: null pointer");
  RopeArgs a{};
  a.B = B; a.N = N; a.hd = hd; a.pairs = pairs; a.axes = axes;
  a.pos = pos; a.pos_as = pos_as; a.pos_bs = pos_bs; a.freq = freq; a.axis = axis;
  a.sign = inverse ? -1.f : 1.f;
  a.side[0] = {Hq, q, q_bs, q_rs, q_hs, qo, qo_bs, qo_rs, qo_hs};
  a.side[1] = {Hk, k, k_bs, k_rs, k_hs, ko, ko_bs, ko_rs, ko_hs};
  // pairs per item: 8, or 4, where that divides the pairs and the copied rest and every row starts on
  // a whole vector (bf16: 16 B / 8 B; fp32: 32 B / 16 B, two 16-B accesses at most); else 1
  const int es = dtype == CAPK_BF16 ? 2 : 4;
  int V = 8;
  for (; V > 1; V = V == 8 ? 4 : 1) {
    const int align = V * es < 16 ? V * es : 16, ea = align / es;
    bool ok = pairs % V == 0 && (hd - 2 * pairs) % V == 0;
    for (int i = 0; i < 1 + (Hk > 0); ++i) {
      const RopeSide& s = a.side[i];
      ok = ok && (uintptr_t)s.x % align == 0 && (uintptr_t)s.y % align == 0 &&
           (s.x_bs % ea | s.x_rs % ea | s.x_hs % ea | s.y_bs % ea | s.y_rs % ea | s.y_hs % ea) == 0;
    }
    if (ok) break;
  }
  // tokens per workgroup: enough workgroups for every CU first, then up to 8 to share the launch
  const int64_t all = (int64_t)B * N;
  a.tokens = (int)(all / 2048 < 1 ? 1 : all / 2048 > 8 ? 8 : all / 2048);
  CAPK_CHECK_ARG(all / a.tokens < (1 << 24) - 1 && Hq + (int64_t)Hk <= 1024, "capk_axis_rope: too many tokens or heads");
  const int per = pairs / V + (hd - 2 * pairs) / V, heads = Hq + Hk;
  a.per_mul = (uint32_t)(((1ull << 32) + per - 1) / per);
  a.heads_mul = (uint32_t)(((1ull << 32) + heads - 1) / heads);
  return dtype == CAPK_BF16 ? rope_launch<bf16>(a, V, interleaved != 0, S(stream))
                            : rope_launch<float>(a, V, interleaved != 0, S(stream));
}
