// Attention of few queries (a decoding step, drafted tokens) over a long cache: dense rows, or pages of
// 4-bit floats with one power-of-two scale per 32 elements.
//
// The Nq queries of the G heads that share a key head are the columns of one product, so the cache is
// read once for all of them.  A wave walks tiles of 32 keys: S^T = K Q^T with the keys as rows, running
// maximum and sum per column, then O^T += V^T P^T with P^T straight from the score registers and V^T
// fragments read transposed from the wave's own LDS image.  Loads of the next tile are in flight while a
// tile is computed.  4-bit values become bf16 exactly (two significant bits and a power of two), so
// nothing is lost before the products; 32-bit queries and probabilities go through the bf16 matrix unit
// as three bf16 parts (3 x 8 significant bits: exact).  Bound: HBM, the visible keys' bytes once.  The
// key axis is cut over workgroups (and over the 4 waves of each), whose partial softmaxes are joined.
#include "sliding.h"

namespace capk {

template <bool KV4, typename T> struct StepTypes {
  using F = typename Tile<T>::V8;  // fragments of the products
  using E = T;                     // elements of the LDS image
  static constexpr int PARTS = 1;
};
template <> struct StepTypes<true, float> {
  using F = bf16x8;
  using E = bf16;
  static constexpr int PARTS = 3;
};

// x as PARTS fragments whose sum is x
template <int PARTS, typename F> __device__ __forceinline__ void step_parts(const f32x8& x, F (&f)[PARTS]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float r = x[e];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      f[p][e] = r;
      if (p + 1 < PARTS) r -= (float)f[p][e];
    }
  }
}

__device__ __forceinline__ bf16x8 step_fp4(uint32_t x, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 3);
  return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// One tile of 32 keys in registers: lane l holds, for the keys (l & 15) and 16 + (l & 15), NS runs of 8
// elements: dense from 32 t + 8 g (g = l >> 4), 4-bit from g * HDP / 4 + 8 t (one dword each).
template <bool KV4, typename T, int HDP> struct StepTile;
template <typename T, int HDP> struct StepTile<false, T, HDP> {
  static constexpr int NS = HDP / 32;
  typename Tile<T>::V8 k[2][NS], v[2][NS];
  uint32_t hid;
  __device__ __forceinline__ static int elem(int t, int g) { return 32 * t + 8 * g; }
  __device__ __forceinline__ void load(const StepArgs& a, int b, int kvh, int j0, int last, int lo, int lane) {
    hid = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int j = j0 + 16 * s + (lane & 15);
      const bool ok = j < last && (j < a.sinks || j >= lo) && !(a.pad && a.pad[(int64_t)b * a.cap + j]);
      hid |= (uint32_t)(~__builtin_amdgcn_ballot_w64(ok) & 0xffff) << (16 * s);
      const T *kr = row<T>(a.k, b, j, kvh), *vr = row<T>(a.v, b, j, kvh);
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        const int d = elem(t, lane >> 4);
        k[s][t] = v[s][t] = tile_zero8<T>();
        if (ok && d < a.hd) {
          k[s][t] = Tile<T>::load(kr + d);
          v[s][t] = Tile<T>::load(vr + d);
        }
      }
    }
  }
  __device__ __forceinline__ typename Tile<T>::V8 kf(int s, int t, int) const { return k[s][t]; }
  __device__ __forceinline__ typename Tile<T>::V8 vf(int s, int t, int) const { return v[s][t]; }
};
template <typename T, int HDP> struct StepTile<true, T, HDP> {
  static constexpr int NS = HDP / 32, NB = HDP / 32;
  uint32_t k[2][NS], v[2][NS], ks[2], vs[2], hid;  // ks, vs: scale codes of the first and the last run
  __device__ __forceinline__ static int elem(int t, int g) { return g * (HDP / 4) + 8 * t; }
  __device__ __forceinline__ void load(const StepArgs& a, int b, int kvh, int j0, int last, int lo, int lane) {
    hid = 0;
    const int g = lane >> 4, e0 = elem(0, g) / 32, e1 = elem(NS - 1, g) / 32;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int js = j0 + 16 * s, j = js + (lane & 15);
      // 16 keys from a multiple of 16 lie in one page
      const int pg = js < last ? a.table[(int64_t)b * a.table_ld + js / a.page] : -1;
      const bool ok = j < last && (j < a.sinks || j >= lo) && pg >= 0 && pg < a.pages;
      hid |= (uint32_t)(~__builtin_amdgcn_ballot_w64(ok) & 0xffff) << (16 * s);
      ks[s] = vs[s] = 127 | 127 << 8;
#pragma unroll
      for (int t = 0; t < NS; ++t) k[s][t] = v[s][t] = 0;
      if (ok) {
        const int64_t kr = (((int64_t)pg * 2) * a.Hk + kvh) * a.page + js % a.page + (lane & 15), vr = kr + (int64_t)a.Hk * a.page;
        const uint32_t *kc = (const uint32_t*)(a.codes + kr * (HDP / 2) + g * (HDP / 8)),
                       *vc = (const uint32_t*)(a.codes + vr * (HDP / 2) + g * (HDP / 8));
#pragma unroll
        for (int t = 0; t < NS; ++t) { k[s][t] = kc[t]; v[s][t] = vc[t]; }
        ks[s] = a.scales[kr * NB + e0] | (uint32_t)a.scales[kr * NB + e1] << 8;
        vs[s] = a.scales[vr * NB + e0] | (uint32_t)a.scales[vr * NB + e1] << 8;
      }
    }
  }
  __device__ __forceinline__ static float scale(uint32_t c, int t, int g) {
    // run t lies in the block of the first run or in that of the last
    const bool second = HDP == 96 && elem(t, g) / 32 != elem(0, g) / 32;
    return __uint_as_float((second ? c >> 8 : c & 255) << 23);
  }
  __device__ __forceinline__ bf16x8 kf(int s, int t, int g) const { return step_fp4(k[s][t], scale(ks[s], t, g)); }
  __device__ __forceinline__ bf16x8 vf(int s, int t, int g) const { return step_fp4(v[s][t], scale(vs[s], t, g)); }
};

template <typename T> __device__ __forceinline__ void step_row(const StepArgs& a, int b, int kvh, int r, int& i, int& h) {
  const int G = a.H / a.Hk;
  i = r / G;
  h = kvh * G + r % G;
}

// Grid: (splits, Hk * row groups of 16 NRT, B); 4 waves.
template <bool KV4, typename T, int HDP, int NRT>
__global__ __launch_bounds__(256) void step_attn(StepArgs a) {
  using Ty = StepTypes<KV4, T>;
  using F = typename Ty::F;
  using E = typename Ty::E;
  using St = StepTile<KV4, T, HDP>;
  constexpr int NS = HDP / 32, ND = HDP / 16, PARTS = Ty::PARTS, IST = HDP + 16, OST = HDP + 4;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  const int b = blockIdx.z, kvh = blockIdx.y % a.Hk, r0 = blockIdx.y / a.Hk * 16 * NRT, R = a.Nq * (a.H / a.Hk);
  const int len = a.len ? min(max(a.len[b], 0), a.cap) : a.cap, off = len - a.Nq;
  const float c = a.scale * kTileLog2e;
  E* img = (E*)smem + w * 32 * IST;

  F qf[NRT][NS][PARTS];
  int pos[NRT];
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    const int r = r0 + rt * 16 + (lane & 15);
    int i, h;
    step_row<T>(a, b, kvh, min(r, R - 1), i, h);
    pos[rt] = off + i;
    const T* src = row<T>(a.q, b, i, h);
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      const int d = St::elem(t, g);
      typename Tile<T>::V8 x = tile_zero8<T>();
      if (r < R && d < a.hd) x = Tile<T>::load(src + d);
      if constexpr (PARTS == 1) qf[rt][t][0] = x;
      else step_parts<PARTS, F>(x, qf[rt][t]);
    }
  }
  f32x4 o[NRT][ND];
  float m[NRT], l[NRT];
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[rt][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  const SlideTiles<32> tiles(a.window, a.sinks, off, len - 1, len);
  const int lo = off - a.window + 1;  // first key of the first query's window
  const int t1 = (int)((int64_t)tiles.n * (blockIdx.x + 1) / a.splits);
  int t = (int)((int64_t)tiles.n * blockIdx.x / a.splits) + w;
  St cur, nxt;
  if (t < t1) cur.load(a, b, kvh, tiles.key0(t), len, lo, lane);
  for (; t < t1; t += 4) {
    const int j0 = tiles.key0(t);
    if (t + 4 < t1) nxt.load(a, b, kvh, tiles.key0(t + 4), len, lo, lane);
    // V rows into the wave's own image: a wave's LDS accesses run in order, so the last tile's reads are
    // served before these writes, and these before the reads below (the fences hold the compiler to it)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NS; ++i) *(F*)(img + (16 * s + (lane & 15)) * IST + St::elem(i, g)) = cur.vf(s, i, g);
    asm volatile("" ::: "memory");
    const bool full = cur.hid == 0 && j0 + 31 <= off && (j0 + 32 <= a.sinks || len - 1 - j0 < a.window);
    f32x4 sc[NRT][2];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) sc[rt][0] = sc[rt][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const F k = cur.kf(s, i, g);
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) sc[rt][s] = Tile<E>::mma16(k, qf[rt][i][p], sc[rt][s]);
      }
    F pf[NRT][PARTS];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      float mt = -INFINITY;
      f32x8 x;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int jj = 16 * s + 4 * g + i, j = j0 + jj;
          float y = sc[rt][s][i] * c;
          if (!full && (((cur.hid >> jj) & 1) || j > pos[rt] || (j >= a.sinks && pos[rt] - j >= a.window))) y = -INFINITY;
          x[4 * s + i] = y;
          mt = fmaxf(mt, y);
        }
      mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      const float mn = fmaxf(m[rt], mt), ms = mn == -INFINITY ? 0.f : mn, alpha = tile_exp2(m[rt] - ms);
      m[rt] = mn;
      l[rt] *= alpha;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = tile_exp2(x[e] - ms);
        l[rt] += x[e];
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) o[rt][d] *= alpha;
      step_parts<PARTS, F>(x, pf[rt]);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const F v = tile_trans16(img, IST, 0, d * 16, lane);
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) o[rt][d] = Tile<E>::mma16(v, pf[rt][p], o[rt][d]);
    }
    cur = nxt;
  }
  // join the 4 waves, 16 columns at a time
  float* os = (float*)smem;               // [4][16][OST]
  float* ms = os + 4 * 16 * OST;          // [4][16] maximum, [4][16] sum
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    float lt = l[rt];
    lt += __shfl_xor(lt, 16, 64);
    lt += __shfl_xor(lt, 32, 64);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; ++d) *(f32x4*)(os + (w * 16 + (lane & 15)) * OST + d * 16 + 4 * g) = o[rt][d];
    if (g == 0) { ms[w * 16 + lane] = m[rt]; ms[64 + w * 16 + lane] = lt; }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * HDP / 4; x += 256) {
      const int cr = x / (HDP / 4), d = x % (HDP / 4) * 4, r = r0 + rt * 16 + cr;
      if (r >= R || d >= a.hd) continue;
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) mm = fmaxf(mm, ms[u * 16 + cr]);
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float f = mm == -INFINITY ? 0.f : tile_exp2(ms[u * 16 + cr] - mm);
        ll += f * ms[64 + u * 16 + cr];
        s += *(const f32x4*)(os + (u * 16 + cr) * OST + d) * f;
      }
      int i, h;
      step_row<T>(a, b, kvh, r, i, h);
      const int64_t at = ((int64_t)b * a.H + h) * a.Nq + i;
      if (a.splits > 1) {
        *(f32x4*)(a.po + (at * a.splits + blockIdx.x) * a.hd + d) = s;
        if (d == 0) {
          a.pml[(at * a.splits + blockIdx.x) * 2] = mm;
          a.pml[(at * a.splits + blockIdx.x) * 2 + 1] = ll;
        }
      } else {
        Tile<T>::store4(row<T>(a.o, b, i, h) + d, s * (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll)));
        if (a.lse && d == 0) a.lse[at] = ll > 0.f ? (mm + __log2f(ll)) * kTileLn2 : (ll == 0.f ? -INFINITY : ll);
      }
    }
  }
}

// One wave per (sequence, head, query): the splits' partial softmaxes joined in order.
template <typename T>
__global__ __launch_bounds__(256) void step_join(StepArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= (int64_t)a.B * a.H * a.Nq) return;
  const float* ml = a.pml + at * a.splits * 2;
  float mm = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) mm = fmaxf(mm, ml[2 * s]);
  mm = wave_max(mm);
  float ll = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const float* po = a.po + at * a.splits * a.hd + lane * 4;
  for (int s = 0; s < a.splits; ++s) {
    const float f = mm == -INFINITY ? 0.f : tile_exp2(ml[2 * s] - mm);
    ll += f * ml[2 * s + 1];
    if (lane * 4 < a.hd) o += *(const f32x4*)(po + (int64_t)s * a.hd) * f;
  }
  const int i = (int)(at % a.Nq), h = (int)(at / a.Nq % a.H), b = (int)(at / a.Nq / a.H);
  if (lane * 4 < a.hd) Tile<T>::store4(row<T>(a.o, b, i, h) + lane * 4, o * (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll)));
  if (a.lse && lane == 0) a.lse[at] = ll > 0.f ? (mm + __log2f(ll)) * kTileLn2 : (ll == 0.f ? -INFINITY : ll);
}

// 16-column tiles per wave: all of them up to 4 (fp32, whose queries take two or three times the
// registers: 2); more rows take further workgroups, which read the cache again
static int step_nrt(int dtype, int rows) { return rows <= 16 ? 1 : rows <= 32 || dtype == CAPK_F32 ? 2 : 4; }

size_t step_workspace(int dtype, const StepArgs& a, int* splits) {
  const int rows = a.Nq * (a.H / a.Hk), nrt = step_nrt(dtype, rows);
  const int64_t blocks = (int64_t)a.B * a.Hk * cdiv(rows, 16 * nrt);
  // workgroups for 4 on every CU, with at least a tile of 32 keys for each wave of a split
  int64_t most = (int64_t)a.window + a.Nq + a.sinks + 64;
  if (most > a.cap) most = a.cap;
  int64_t s = 1024 / blocks;
  if (s > cdiv(most, 128)) s = cdiv(most, 128);
  if (s < 1) s = 1;
  *splits = (int)s;
  return s > 1 ? (size_t)a.B * a.H * a.Nq * s * (a.hd + 2) * 4 : 0;
}

template <bool KV4, typename T, int HDP>
static int step_go(const StepArgs& a, hipStream_t st) {
  using E = typename StepTypes<KV4, T>::E;
  const int rows = a.Nq * (a.H / a.Hk), nrt = step_nrt(sizeof(T) == 2 ? CAPK_BF16 : CAPK_F32, rows);
  const dim3 grid(a.splits, a.Hk * cdiv(rows, 16 * nrt), a.B);
  const size_t img = (size_t)4 * 32 * (HDP + 16) * sizeof(E), join = (size_t)4 * 16 * (HDP + 4) * 4 + 512;
  const size_t shm = img > join ? img : join;
  const void* fn = nrt == 1 ? (const void*)step_attn<KV4, T, HDP, 1> : nrt == 2 ? (const void*)step_attn<KV4, T, HDP, 2>
                                                                               : (const void*)step_attn<KV4, T, HDP, (sizeof(T) == 2 ? 4 : 2)>;
  if (shm > 65536) {
    hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shm);
    if (e != hipSuccess) return hip_status(e, "step_attn");
  }
  StepArgs arg = a;
  void* args[] = {&arg};
  hipError_t e = hipLaunchKernel(fn, grid, dim3(256), args, shm, st);
  if (e != hipSuccess) return hip_status(e, "step_attn");
  if (a.splits > 1) {
    hipLaunchKernelGGL(step_join<T>, dim3(cdiv((int64_t)a.B * a.H * a.Nq, 4)), dim3(256), 0, st, a);
    CAPK_LAUNCH_CHECK("step_join");
  }
  return CAPK_OK;
}

int step_launch(int dtype, StepArgs a, void* ws, size_t ws_bytes, hipStream_t st) {
  const size_t need = step_workspace(dtype, a, &a.splits);
  CAPK_CHECK_ARG(need == 0 || (ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0),
                 "attention over a cache: needs a 16-B aligned workspace of %zu bytes", need);
  a.po = (float*)ws;
  a.pml = a.po + (size_t)a.B * a.H * a.Nq * a.splits * a.hd;
  SLIDE_HD(slide_hdp(a.hd), {
    if (a.codes) return dtype == CAPK_BF16 ? step_go<true, bf16, HDP>(a, st) : step_go<true, float, HDP>(a, st);
    return dtype == CAPK_BF16 ? step_go<false, bf16, HDP>(a, st) : step_go<false, float, HDP>(a, st);
  });
  return CAPK_OK;
}

}  // namespace capk
