// Sliding-window attention whose first tokens stay visible.
//
// The query at position p sees the keys j <= p with j < sinks or p - j < window; queries are the last
// Nq positions of a sequence of len[b] keys (len = Nk without kv_len), H query heads share Hk key
// heads.  o = softmax(scale q k^T) v over the visible keys; lse = log of the softmax's denominator.  A
// query that sees nothing gets o = 0, lse = -inf and no gradient.
//
// Forward: a workgroup owns 128 queries of a head (4 waves x 32), walks the key tiles that hold sinks
// and then those of its window, and keeps a running maximum and sum (one pass).  S^T = K Q^T puts one
// query on each lane, so the row statistics need one shuffle, and P^T, already in B-operand order, is
// multiplied by V^T fragments read transposed from LDS.
// Backward: D = rowsum(do * o); P = exp(s - lse); dS = P (do v^T - D) scale.  One kernel owns queries
// (dQ^T += K^T dS^T), one owns keys and walks their queries over all heads of the group
// (dV^T += dO^T P, dK^T += Q^T dS): every sum has one owner, so results do not depend on timing.  Keys
// that stay visible are seen by all later queries: those far queries are cut into chunks with owners
// of their own, whose 32-bit partial sums one more kernel adds in a fixed order.
#include "sliding.h"

namespace capk {

struct SlideArgs {
  int B, H, Hk, Nq, Nk, hd, window, sinks;
  float scale;
  SlideView q, k, v, o, dout, dq, dk, dv;
  const uint8_t* pad;   // [B, Nk], 1 = hidden
  const int32_t* len;   // [B]
  float* lse;           // [B, H, Nq]
  float* delta;         // [B, H, Nq]
  float* part;          // far-query partial sums of dK and dV
  int sink_tiles, far_chunks, far_rows;
};

__device__ __forceinline__ int slide_len(const SlideArgs& a, int b) {
  return a.len ? min(max(a.len[b], 0), a.Nk) : a.Nk;
}
__device__ __forceinline__ bool slide_sees(const SlideArgs& a, int p, int j) {
  return j <= p && (j < a.sinks || p - j < a.window);
}

// KT rows of a [N, hd] head matrix into LDS (row stride ST), zeros where row_ok says no.
template <typename T, int HDP, int KT, int ST, typename OK>
__device__ __forceinline__ void slide_stage(T* img, const T* src, int64_t rs, int r0, int hd, OK row_ok) {
  constexpr int C = HDP / 8;
  for (int c = threadIdx.x; c < KT * C; c += 256) {
    const int r = c / C, d = c % C * 8;
    typename Tile<T>::V8 x = tile_zero8<T>();
    if (d < hd && row_ok(r0 + r)) x = Tile<T>::load(src + (int64_t)(r0 + r) * rs + d);
    *(typename Tile<T>::V8*)(img + r * ST + d) = x;
  }
}
template <typename T, int HDP>
__device__ __forceinline__ void slide_frags(typename Tile<T>::V8 (&f)[HDP / 16], const T* src, bool ok, int hd, int h) {
#pragma unroll
  for (int s = 0; s < HDP / 16; ++s) {
    f[s] = tile_zero8<T>();
    if (ok && s * 16 + h * 8 < hd) f[s] = Tile<T>::load(src + s * 16 + h * 8);
  }
}
template <typename T> constexpr int slide_st(int hdp) { return hdp + 16 / (int)sizeof(T); }

template <typename T, int HDP>
__device__ __forceinline__ void slide_store(T* dst, const f32x16 (&acc)[HDP / 32], float f, int hd, int h) {
#pragma unroll
  for (int db = 0; db < HDP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * h;
      if (d < hd) Tile<T>::store4(dst + d, (f32x4){acc[db][4 * g] * f, acc[db][4 * g + 1] * f, acc[db][4 * g + 2] * f,
                                                   acc[db][4 * g + 3] * f});
    }
}

// hidden keys of a 64-key tile, one bit each
__device__ __forceinline__ uint64_t slide_hidden(const SlideArgs& a, int b, int j0, int len, int lane) {
  const int j = j0 + lane;
  return __builtin_amdgcn_ballot_w64(j >= len || (a.pad && a.pad[(int64_t)b * a.Nk + j]));
}

template <typename T, int HDP>
__global__ __launch_bounds__(256) void slide_fwd(SlideArgs a) {
  constexpr int KT = 64, ST = slide_st<T>(HDP), NS = HDP / 16, ND = HDP / 32;
  extern __shared__ __align__(16) char smem[];
  T* Ks = (T*)smem;
  T* Vs = Ks + KT * ST;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hh = lane >> 5;
  const int h = blockIdx.y, b = blockIdx.z, kvh = h / (a.H / a.Hk), len = slide_len(a, b), off = len - a.Nq;
  const int q0 = blockIdx.x * 128, qw = q0 + w * 32, qi = qw + (lane & 31), p = off + qi;
  const int p_lo = off + q0, p_hi = off + min(q0 + 127, a.Nq - 1);
  const int pw_lo = off + qw, pw_hi = off + qw + 31;
  const float c = a.scale * kTileLog2e;

  typename Tile<T>::V8 qf[NS];
  slide_frags<T, HDP>(qf, row<T>(a.q, b, qi, h), qi < a.Nq, a.hd, hh);
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = tile_zero<f32x16>();
  float m = -INFINITY, l = 0.f;
  const SlideTiles<KT> tiles(a.window, a.sinks, p_lo, p_hi, len);
  auto ok = [&](int j) {
    return j < len && j <= p_hi && (j < a.sinks || p_lo - j < a.window) && !(a.pad && a.pad[(int64_t)b * a.Nk + j]);
  };
  for (int t = 0; t < tiles.n; ++t) {
    const int j0 = tiles.key0(t);
    __syncthreads();
    slide_stage<T, HDP, KT, ST>(Ks, row<T>(a.k, b, 0, kvh), a.k.rs, j0, a.hd, ok);
    slide_stage<T, HDP, KT, ST>(Vs, row<T>(a.v, b, 0, kvh), a.v.rs, j0, a.hd, ok);
    __syncthreads();
    if (j0 > pw_hi || (j0 >= a.sinks && pw_lo - (j0 + KT - 1) >= a.window)) continue;  // no key for this wave
    const uint64_t hid = slide_hidden(a, b, j0, len, lane);
    const bool full = hid == 0 && j0 + KT - 1 <= pw_lo && (j0 + KT <= a.sinks || pw_hi - j0 < a.window);
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = tile_zero<f32x16>();
#pragma unroll
      for (int st = 0; st < NS; ++st)
        s[kb] = Tile<T>::mma32(Tile<T>::load(Ks + (kb * 32 + (lane & 31)) * ST + st * 16 + hh * 8), qf[st], s[kb]);
    }
    float mt = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int jj = kb * 32 + 8 * (i >> 2) + 4 * hh + (i & 3);
        float x = s[kb][i] * c;
        if (!full && (((hid >> jj) & 1) || !slide_sees(a, p, j0 + jj))) x = -INFINITY;
        s[kb][i] = x;
        mt = fmaxf(mt, x);
      }
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const float mn = fmaxf(m, mt), ms = mn == -INFINITY ? 0.f : mn, alpha = tile_exp2(m - ms);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        typename Tile<T>::V8 pf;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = tile_exp2(s[kb][st * 8 + e] - ms);
          l += x;
          pf[e] = (T)x;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[d] = Tile<T>::mma32(tile_trans32(Vs, ST, kb * 32 + st * 16, d * 32, lane), pf, o[d]);
      }
  }
  l += __shfl_xor(l, 32, 64);
  if (qi >= a.Nq) return;
  slide_store<T, HDP>(row<T>(a.o, b, qi, h), o, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l), a.hd, hh);
  if (a.lse && hh == 0)
    a.lse[((int64_t)b * a.H + h) * a.Nq + qi] = l > 0.f ? (m + __log2f(l)) * kTileLn2 : (l == 0.f ? -INFINITY : l);
}

template <typename T, int HDP>
__global__ __launch_bounds__(256) void slide_dq(SlideArgs a) {
  constexpr int KT = 64, ST = slide_st<T>(HDP), NS = HDP / 16, ND = HDP / 32;
  extern __shared__ __align__(16) char smem[];
  T* Ks = (T*)smem;
  T* Vs = Ks + KT * ST;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hh = lane >> 5;
  const int h = blockIdx.y, b = blockIdx.z, kvh = h / (a.H / a.Hk), len = slide_len(a, b), off = len - a.Nq;
  const int q0 = blockIdx.x * 128, qw = q0 + w * 32, qi = qw + (lane & 31), p = off + qi;
  const int p_lo = off + q0, p_hi = off + min(q0 + 127, a.Nq - 1);
  const int pw_lo = off + qw, pw_hi = off + qw + 31;
  const float c = a.scale * kTileLog2e;

  typename Tile<T>::V8 qf[NS], dof[NS];
  slide_frags<T, HDP>(qf, row<T>(a.q, b, qi, h), qi < a.Nq, a.hd, hh);
  slide_frags<T, HDP>(dof, row<T>(a.dout, b, qi, h), qi < a.Nq, a.hd, hh);
  float delta = 0.f, lse2 = INFINITY;
  {
    typename Tile<T>::V8 of[NS];
    slide_frags<T, HDP>(of, row<T>(a.o, b, qi, h), qi < a.Nq, a.hd, hh);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)of[s][e], (float)dof[s][e], delta);
    delta += __shfl_xor(delta, 32, 64);
    if (qi < a.Nq) {
      const int64_t at = ((int64_t)b * a.H + h) * a.Nq + qi;
      lse2 = a.lse[at] * kTileLog2e;
      if (hh == 0) a.delta[at] = delta;
    }
  }
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = tile_zero<f32x16>();
  const SlideTiles<KT> tiles(a.window, a.sinks, p_lo, p_hi, len);
  auto ok = [&](int j) {
    return j < len && j <= p_hi && (j < a.sinks || p_lo - j < a.window) && !(a.pad && a.pad[(int64_t)b * a.Nk + j]);
  };
  for (int t = 0; t < tiles.n; ++t) {
    const int j0 = tiles.key0(t);
    __syncthreads();
    slide_stage<T, HDP, KT, ST>(Ks, row<T>(a.k, b, 0, kvh), a.k.rs, j0, a.hd, ok);
    slide_stage<T, HDP, KT, ST>(Vs, row<T>(a.v, b, 0, kvh), a.v.rs, j0, a.hd, ok);
    __syncthreads();
    if (j0 > pw_hi || (j0 >= a.sinks && pw_lo - (j0 + KT - 1) >= a.window)) continue;
    const uint64_t hid = slide_hidden(a, b, j0, len, lane);
    const bool full = hid == 0 && j0 + KT - 1 <= pw_lo && (j0 + KT <= a.sinks || pw_hi - j0 < a.window);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s = tile_zero<f32x16>(), dp = tile_zero<f32x16>();
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const int at = (kb * 32 + (lane & 31)) * ST + st * 16 + hh * 8;
        s = Tile<T>::mma32(Tile<T>::load(Ks + at), qf[st], s);
        dp = Tile<T>::mma32(Tile<T>::load(Vs + at), dof[st], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int jj = kb * 32 + 8 * (i >> 2) + 4 * hh + (i & 3);
        const float x = tile_exp2(fmaf(s[i], c, -lse2)) * (dp[i] - delta) * a.scale;
        s[i] = !full && (((hid >> jj) & 1) || !slide_sees(a, p, j0 + jj)) ? 0.f : x;
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        typename Tile<T>::V8 df;
#pragma unroll
        for (int e = 0; e < 8; ++e) df[e] = (T)s[st * 8 + e];
#pragma unroll
        for (int d = 0; d < ND; ++d)
          dq[d] = Tile<T>::mma32(tile_trans32(Ks, ST, kb * 32 + st * 16, d * 32, lane), df, dq[d]);
      }
    }
  }
  if (qi < a.Nq) slide_store<T, HDP>(row<T>(a.dq, b, qi, h), dq, 1.f, a.hd, hh);
}

// Keys [j0, j0 + 128) of a key head against queries [qa, qb) of its group; far = only the sinks among
// the keys, at queries that no longer have them in their window.
constexpr int kSlideKeys = 128;
template <typename T, int HDP>
__global__ __launch_bounds__(256) void slide_dkv(SlideArgs a) {
  constexpr int QT = 64, ST = slide_st<T>(HDP), NS = HDP / 16, ND = HDP / 32;
  extern __shared__ __align__(16) char smem[];
  T* Qs = (T*)smem;
  T* Ds = Qs + QT * ST;
  float* Ls = (float*)(Ds + QT * ST);  // lse (base 2), then delta
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hh = lane >> 5;
  const int kvh = blockIdx.y, b = blockIdx.z, G = a.H / a.Hk, len = slide_len(a, b), off = len - a.Nq;
  const int tiles = (a.Nk + kSlideKeys - 1) / kSlideKeys;
  const bool far = (int)blockIdx.x >= tiles;
  const int tile = far ? ((int)blockIdx.x - tiles) / a.far_chunks : (int)blockIdx.x;
  const int chunk = far ? ((int)blockIdx.x - tiles) % a.far_chunks : a.far_chunks;
  const int j0 = tile * kSlideKeys, jw = j0 + w * 32, j = jw + (lane & 31);
  const bool key_ok = j < len && !(a.pad && a.pad[(int64_t)b * a.Nk + j]) && (!far || j < a.sinks);
  // positions of the queries: near p in [j0, near_end), far p >= near_end in chunks of far_rows
  const int64_t near_end = (int64_t)j0 + kSlideKeys - 1 + a.window;
  const int qn = (int)min((int64_t)a.Nq, max((int64_t)0, near_end - off));
  const int qa = far ? qn + chunk * a.far_rows : max(0, j0 - off);
  const int qb = far ? min(a.Nq, qa + a.far_rows) : (j0 < len ? qn : 0);
  const float c = a.scale * kTileLog2e;

  typename Tile<T>::V8 kf[NS], vf[NS];
  slide_frags<T, HDP>(kf, row<T>(a.k, b, j, kvh), key_ok, a.hd, hh);
  slide_frags<T, HDP>(vf, row<T>(a.v, b, j, kvh), key_ok, a.hd, hh);
  const bool hidden = __builtin_amdgcn_ballot_w64(!key_ok) != 0;
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = tile_zero<f32x16>();
  for (int g = 0; g < G; ++g) {
    const int h = kvh * G + g;
    for (int q0 = qa; q0 < qb; q0 += QT) {
      auto ok = [&](int q) { return q < qb; };
      __syncthreads();
      slide_stage<T, HDP, QT, ST>(Qs, row<T>(a.q, b, 0, h), a.q.rs, q0, a.hd, ok);
      slide_stage<T, HDP, QT, ST>(Ds, row<T>(a.dout, b, 0, h), a.dout.rs, q0, a.hd, ok);
      if (threadIdx.x < QT) {
        const int q = q0 + threadIdx.x;
        const int64_t at = ((int64_t)b * a.H + h) * a.Nq + q;
        Ls[threadIdx.x] = q < qb ? a.lse[at] * kTileLog2e : INFINITY;
        Ls[QT + threadIdx.x] = q < qb ? a.delta[at] : 0.f;
      }
      __syncthreads();
      const int p0 = off + q0;
      // no query of this tile sees a key of this wave
      if (p0 + QT - 1 < jw || (jw >= a.sinks && p0 - (jw + 31) >= a.window)) continue;
      const bool full = !hidden && q0 + QT <= qb && jw + 31 <= p0 && (jw + 32 <= a.sinks || p0 + QT - 1 - jw < a.window);
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        f32x16 s = tile_zero<f32x16>(), dp = tile_zero<f32x16>();
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const int at = (qt * 32 + (lane & 31)) * ST + st * 16 + hh * 8;
          s = Tile<T>::mma32(Tile<T>::load(Qs + at), kf[st], s);
          dp = Tile<T>::mma32(Tile<T>::load(Ds + at), vf[st], dp);
        }
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const int r = qt * 32 + 8 * i4 + 4 * hh;
          const f32x4 ls = *(const f32x4*)(Ls + r), dl = *(const f32x4*)(Ls + QT + r);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * i4 + e;
            float x = tile_exp2(fmaf(s[i], c, -ls[e])), y = x * (dp[i] - dl[e]) * a.scale;
            if (!full && (!key_ok || q0 + r + e >= qb || !slide_sees(a, p0 + r + e, j))) x = y = 0.f;
            s[i] = x;
            dp[i] = y;
          }
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          typename Tile<T>::V8 pf, df;
#pragma unroll
          for (int e = 0; e < 8; ++e) { pf[e] = (T)s[st * 8 + e]; df[e] = (T)dp[st * 8 + e]; }
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            dv[d] = Tile<T>::mma32(tile_trans32(Ds, ST, qt * 32 + st * 16, d * 32, lane), pf, dv[d]);
            dk[d] = Tile<T>::mma32(tile_trans32(Qs, ST, qt * 32 + st * 16, d * 32, lane), df, dk[d]);
          }
        }
      }
    }
  }
  if (tile < a.sink_tiles && a.far_chunks > 0) {  // [B, Hk, sink tile, chunk][dK, dV][128][hd]
    float* dst = a.part + ((((int64_t)b * a.Hk + kvh) * a.sink_tiles + tile) * (a.far_chunks + 1) + chunk) * 2 *
                              kSlideKeys * a.hd + (int64_t)(w * 32 + (lane & 31)) * a.hd;
    slide_store<float, HDP>(dst, dk, 1.f, a.hd, hh);
    slide_store<float, HDP>(dst + (int64_t)kSlideKeys * a.hd, dv, 1.f, a.hd, hh);
  } else if (j < a.Nk) {
    slide_store<T, HDP>(row<T>(a.dk, b, j, kvh), dk, 1.f, a.hd, hh);
    slide_store<T, HDP>(row<T>(a.dv, b, j, kvh), dv, 1.f, a.hd, hh);
  }
}

// dK, dV rows of the sink tiles = the sum of their chunks, in order.  One thread per 4 elements.
template <typename T>
__global__ __launch_bounds__(256) void slide_dkv_sum(SlideArgs a) {
  const int per = kSlideKeys * a.hd / 4;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= per * 2 * a.sink_tiles) return;
  const int e = i % per * 4, which = i / per % 2, tile = i / per / 2, j = tile * kSlideKeys + e / a.hd;
  if (j >= a.Nk) return;
  const float* src = a.part + (((int64_t)blockIdx.z * a.Hk + blockIdx.y) * a.sink_tiles + tile) * (a.far_chunks + 1) * 2 *
                                  kSlideKeys * a.hd + (int64_t)which * kSlideKeys * a.hd + e;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c <= a.far_chunks; ++c) s += *(const f32x4*)(src + (int64_t)c * 2 * kSlideKeys * a.hd);
  Tile<T>::store4(row<T>(which ? a.dv : a.dk, blockIdx.z, j, blockIdx.y) + e % a.hd, s);
}

template <typename K>
static int slide_launch(K kernel, dim3 grid, size_t shm, hipStream_t st, const SlideArgs& a, const char* name) {
  if (shm > 65536) {
    hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shm);
    if (e != hipSuccess) return hip_status(e, name);
  }
  hipLaunchKernelGGL(kernel, grid, dim3(256), shm, st, a);
  CAPK_LAUNCH_CHECK(name);
  return CAPK_OK;
}

static int slide_check(const char* who, int dtype, int B, int H, int Hk, int Nq, int Nk, int hd, int window, int sinks,
                       const SlideView* v, int n) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "%s: dtype", who);
  CAPK_CHECK_ARG(B >= 1 && B <= 65535 && Nq >= 1 && Nk >= 1 && Nq <= (1 << 28) && Nk <= (1 << 28), "%s: bad sizes", who);
  CAPK_CHECK_ARG(Hk >= 1 && H >= Hk && H % Hk == 0 && H <= 65535, "%s: %d query heads over %d key heads", who, H, Hk);
  CAPK_CHECK_ARG(hd >= 8 && hd % 8 == 0 && hd <= 128, "%s: hd=%d must be a multiple of 8, <= 128", who, hd);
  CAPK_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window and sinks must not be negative", who);
  const int ea = dtype == CAPK_BF16 ? 8 : 4;
  for (int i = 0; i < n; ++i)
    CAPK_CHECK_ARG(v[i].p && (uintptr_t)v[i].p % 16 == 0 && v[i].bs % ea == 0 && v[i].rs % ea == 0 && v[i].hs % ea == 0,
                   "%s: operand %d must be 16-B aligned with strides that keep it so", who, i);
  return CAPK_OK;
}

static SlideArgs slide_args(int B, int H, int Hk, int Nq, int Nk, int hd, float scale, int window, int sinks,
                            const uint8_t* pad, const int32_t* len) {
  SlideArgs a{};
  a.B = B; a.H = H; a.Hk = Hk; a.Nq = Nq; a.Nk = Nk; a.hd = hd; a.scale = scale;
  // window 0: every earlier key; a window past all keys changes nothing, and sums of it stay in 32 bits
  a.window = window == 0 || window > Nk + Nq ? Nk + Nq : window;
  a.sinks = sinks > Nk ? Nk : sinks;
  a.pad = pad; a.len = len;
  return a;
}

// The far queries of the sink tiles: chunks of about a window (at least 512), so that no owner of a
// chunk works much longer than the owner of an ordinary key tile.
static void slide_far(SlideArgs& a) {
  a.sink_tiles = cdiv(a.sinks, kSlideKeys);
  a.far_rows = a.window + kSlideKeys > 512 ? (a.window + kSlideKeys + 63) / 64 * 64 : 512;
  // the first sink tile has the most far queries: positions from 127 + window on
  const int64_t most = (int64_t)a.Nk - (kSlideKeys - 1) - a.window;
  const int64_t rows = most < a.Nq ? most : a.Nq;
  a.far_chunks = a.sink_tiles && rows > 0 ? cdiv(rows, a.far_rows) : 0;
}

}  // namespace capk

using namespace capk;

// Few queries (a decoding step, drafted tokens): the kernel that reads the cache once for all of them
static bool slide_few(int Nq) { return Nq <= 16; }
static StepArgs slide_step(const SlideArgs& a) {
  StepArgs s{};
  s.B = a.B; s.H = a.H; s.Hk = a.Hk; s.Nq = a.Nq; s.cap = a.Nk; s.hd = a.hd;
  s.window = a.window; s.sinks = a.sinks; s.scale = a.scale;
  s.q = a.q; s.k = a.k; s.v = a.v; s.o = a.o; s.len = a.len; s.pad = a.pad; s.lse = a.lse;
  return s;
}

extern "C" size_t capk_sliding_attention_fwd_workspace(int dtype, int B, int H, int Hk, int Nq, int Nk, int hd,
                                                       int window, int sinks) {
  if (B < 1 || Hk < 1 || H < Hk || Nq < 1 || Nk < 1 || hd < 1 || window < 0 || sinks < 0 || !slide_few(Nq)) return 0;
  int splits;
  return step_workspace(dtype, slide_step(slide_args(B, H, Hk, Nq, Nk, hd, 0.f, window, sinks, nullptr, nullptr)), &splits);
}

extern "C" int capk_sliding_attention_fwd(int dtype, int B, int H, int Hk, int Nq, int Nk, int hd, float scale,
                                          int window, int sinks, const void* q, int64_t q_bs, int64_t q_rs,
                                          int64_t q_hs, const void* k, int64_t k_bs, int64_t k_rs, int64_t k_hs,
                                          const void* v, int64_t v_bs, int64_t v_rs, int64_t v_hs,
                                          const uint8_t* key_pad, const int32_t* kv_len, void* o, int64_t o_bs,
                                          int64_t o_rs, int64_t o_hs, float* lse, void* ws, size_t ws_bytes,
                                          void* stream) {
  const SlideView vs[] = {{(void*)q, q_bs, q_rs, q_hs}, {(void*)k, k_bs, k_rs, k_hs}, {(void*)v, v_bs, v_rs, v_hs},
                          {o, o_bs, o_rs, o_hs}};
  int rc = slide_check("capk_sliding_attention_fwd", dtype, B, H, Hk, Nq, Nk, hd, window, sinks, vs, 4);
  if (rc) return rc;
  SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, scale, window, sinks, key_pad, kv_len);
  a.q = vs[0]; a.k = vs[1]; a.v = vs[2]; a.o = vs[3]; a.lse = lse;
  if (slide_few(Nq)) return step_launch(dtype, slide_step(a), ws, ws_bytes, S(stream));
  const int hdp = slide_hdp(hd);
  const dim3 grid(cdiv(Nq, 128), H, B);
  SLIDE_HD(hdp, {
    if (dtype == CAPK_BF16)
      return slide_launch(slide_fwd<bf16, HDP>, grid, 2 * 64 * slide_st<bf16>(HDP) * 2, S(stream), a, "slide_fwd");
    return slide_launch(slide_fwd<float, HDP>, grid, 2 * 64 * slide_st<float>(HDP) * 4, S(stream), a, "slide_fwd");
  });
}

extern "C" size_t capk_sliding_attention_bwd_workspace(int B, int H, int Hk, int Nq, int Nk, int hd, int window,
                                                       int sinks) {
  if (B < 1 || H < 1 || Hk < 1 || Nq < 1 || Nk < 1 || hd < 1 || window < 0 || sinks < 0) return 0;
  SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, 0.f, window, sinks, nullptr, nullptr);
  slide_far(a);
  const size_t delta = ((size_t)B * H * Nq * 4 + 15) / 16 * 16;
  return delta + (a.far_chunks ? (size_t)B * Hk * a.sink_tiles * (a.far_chunks + 1) * 2 * kSlideKeys * hd * 4 : 0);
}

extern "C" int capk_sliding_attention_bwd(int dtype, int B, int H, int Hk, int Nq, int Nk, int hd, float scale,
                                          int window, int sinks, const void* q, int64_t q_bs, int64_t q_rs,
                                          int64_t q_hs, const void* k, int64_t k_bs, int64_t k_rs, int64_t k_hs,
                                          const void* v, int64_t v_bs, int64_t v_rs, int64_t v_hs,
                                          const uint8_t* key_pad, const int32_t* kv_len, const void* o, int64_t o_bs,
                                          int64_t o_rs, int64_t o_hs, const void* dout, int64_t do_bs, int64_t do_rs,
                                          int64_t do_hs, const float* lse, void* dq, int64_t dq_bs, int64_t dq_rs,
                                          int64_t dq_hs, void* dk, int64_t dk_bs, int64_t dk_rs, int64_t dk_hs,
                                          void* dv, int64_t dv_bs, int64_t dv_rs, int64_t dv_hs, void* ws,
                                          size_t ws_bytes, void* stream) {
  const SlideView vs[] = {{(void*)q, q_bs, q_rs, q_hs}, {(void*)k, k_bs, k_rs, k_hs}, {(void*)v, v_bs, v_rs, v_hs},
                          {(void*)o, o_bs, o_rs, o_hs}, {(void*)dout, do_bs, do_rs, do_hs}, {dq, dq_bs, dq_rs, dq_hs},
                          {dk, dk_bs, dk_rs, dk_hs}, {dv, dv_bs, dv_rs, dv_hs}};
  int rc = slide_check("capk_sliding_attention_bwd", dtype, B, H, Hk, Nq, Nk, hd, window, sinks, vs, 8);
  if (rc) return rc;
  const size_t need = capk_sliding_attention_bwd_workspace(B, H, Hk, Nq, Nk, hd, window, sinks);
  CAPK_CHECK_ARG(lse && ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0,
                 "capk_sliding_attention_bwd: need lse and a 16-B aligned workspace of %zu bytes", need);
  SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, scale, window, sinks, key_pad, kv_len);
  slide_far(a);
  a.q = vs[0]; a.k = vs[1]; a.v = vs[2]; a.o = vs[3]; a.dout = vs[4]; a.dq = vs[5]; a.dk = vs[6]; a.dv = vs[7];
  a.lse = (float*)lse;
  a.delta = (float*)ws;
  a.part = (float*)((char*)ws + ((size_t)B * H * Nq * 4 + 15) / 16 * 16);
  const int hdp = slide_hdp(hd), es = dtype == CAPK_BF16 ? 2 : 4;
  const dim3 gq(cdiv(Nq, 128), H, B), gk(cdiv(Nk, kSlideKeys) + a.sink_tiles * a.far_chunks, Hk, B);
  hipStream_t st = S(stream);
  SLIDE_HD(hdp, {
    if (dtype == CAPK_BF16) {
      const size_t shm = 2 * 64 * slide_st<bf16>(HDP) * 2;
      if ((rc = slide_launch(slide_dq<bf16, HDP>, gq, shm, st, a, "slide_dq"))) return rc;
      if ((rc = slide_launch(slide_dkv<bf16, HDP>, gk, shm + 512, st, a, "slide_dkv"))) return rc;
    } else {
      const size_t shm = 2 * 64 * slide_st<float>(HDP) * 4;
      if ((rc = slide_launch(slide_dq<float, HDP>, gq, shm, st, a, "slide_dq"))) return rc;
      if ((rc = slide_launch(slide_dkv<float, HDP>, gk, shm + 512, st, a, "slide_dkv"))) return rc;
    }
  });
  if (a.far_chunks) {
    const dim3 gs(cdiv((int64_t)kSlideKeys * hd / 4 * 2 * a.sink_tiles, 256), Hk, B);
    if (es == 2) return slide_launch(slide_dkv_sum<bf16>, gs, 0, st, a, "slide_dkv_sum");
    return slide_launch(slide_dkv_sum<float>, gs, 0, st, a, "slide_dkv_sum");
  }
  return CAPK_OK;
}
