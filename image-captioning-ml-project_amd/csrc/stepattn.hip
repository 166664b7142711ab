// Attention of few queries (a decoding step, drafted tokens) over a long cache: dense rows, or pages of
// 4-bit floats with one power-of-two scale per 32 elements.
//
// The Nq queries of the G heads that share a key head are the columns of one product, so the cache is
// read once for all of them.  A wave walks tiles of 32 keys: S^T = K Q^T with the keys as rows, running
// maximum and sum per column, then O^T += V^T P^T with P^T straight from the score registers and V^T
// fragments read transposed from the wave's own LDS image.  Loads of the next tile are in flight while a
// tile is computed.  4-bit values become bf16 exactly (two significant bits and a power of two), so
// nothing is lost before the products; 32-bit queries and probabilities go through the bf16 matrix unit
// as three bf16 parts (3 x 8 significant bits: exact).  Bound: HBM, the visible keys' bytes once; with 4 bits
// the conversions (64 per tile and wave) and the softmax take as long as the loads.  The key axis is cut
// over workgroups (and over the 4 waves of each), whose partial softmaxes are joined.  bf16 probabilities are rounded
// (half a bf16 step each) before P V, where the matrix unit takes bf16 operands; sums are 32-bit.
// Heads of 128, 8 key heads of 4 bits: 46 us for 64 sequences of 2048 to 4096 tokens (215 MB, 4.7 TB/s), 36 + 6
// (join) for 5 queries over 131072 tokens (143 MB); dense bf16, 32 windows of 2048, 4 key heads: 32 + 4 us for
// 134 MB.  fp32: 57 us, 67 + 6 over 65536 to 131072 tokens, dense 64 + 4 for 269 MB.
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

// A tile of 32 keys in registers: lane l holds, for the keys (l & 15) and 16 + (l & 15), NS runs of 8
// elements: dense from 32 t + 8 g (g = l >> 4), 4-bit from g * HDP / 4 + 8 t (one dword each).  Loads are
// unconditional, of a valid row where the key is hidden (`hid`, one bit per key), so that nothing waits
// for them before their tile's turn; hidden values become zeros then (they may be anything).
template <bool KV4, typename T, int HDP> struct StepTile;
template <typename T, int HDP> struct StepTile<false, T, HDP> {
  static constexpr int NS = HDP / 32;
  typename Tile<T>::V8 k[2][NS], v[2][NS];
  uint32_t hid;
  __device__ __forceinline__ static int elem(int t, int g) { return 32 * t + 8 * g; }
  __device__ __forceinline__ void load(const StepArgs& a, int b, int kvh, int j0, int last, int lo, uint32_t, int, int lane) {
    hid = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int j = min(j0 + 16 * s + (lane & 15), last - 1);
      const bool ok = (j0 + 16 * s + (lane & 15) < last) & ((j < a.sinks) | (j >= lo));
      hid |= (uint32_t)(~__builtin_amdgcn_ballot_w64(ok) & 0xffff) << (16 * s);
      if (a.pad) hid |= (uint32_t)(__builtin_amdgcn_ballot_w64(a.pad[(int64_t)b * a.cap + j]) & 0xffff) << (16 * s);
      const T *kr = row<T>(a.k, b, j, kvh), *vr = row<T>(a.v, b, j, kvh);
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        const int d = elem(t, lane >> 4) < a.hd ? elem(t, lane >> 4) : 0;
        k[s][t] = Tile<T>::load(kr + d);
        v[s][t] = Tile<T>::load(vr + d);
      }
    }
  }
  __device__ __forceinline__ void clear(int s, bool hidden) {
#pragma unroll
    for (int t = 0; t < NS; ++t)
      if (hidden) v[s][t] = tile_zero8<T>();
  }
  __device__ __forceinline__ typename Tile<T>::V8 kf(int s, int t, int) const { return k[s][t]; }
  __device__ __forceinline__ typename Tile<T>::V8 vf(int s, int t, int) const { return v[s][t]; }
};
template <typename T, int HDP> struct StepTile<true, T, HDP> {
  static constexpr int NS = HDP / 32, NB = HDP / 32;
  uint32_t k[2][NS], v[2][NS];
  uint8_t ks[2][HDP == 96 ? 2 : 1], vs[2][HDP == 96 ? 2 : 1];  // scale codes of the first (and the last) run
  uint32_t hid;
  __device__ __forceinline__ static int elem(int t, int g) { return g * (HDP / 4) + 8 * t; }
  // 16 keys from a multiple of 16 on lie in one page: the sixteenth of the row (of all pages' key rows) where they
  // start, ~0 without a page
  __device__ __forceinline__ static uint32_t piece(const StepArgs& a, int b, int kvh, int j) {
    const int at = j / a.page, pg = a.table[(int64_t)b * a.table_ld + at];
    const int64_t r = ((int64_t)pg * 2 * a.Hk + kvh) * (a.page / 16) + (j - at * a.page) / 16;
    return pg < 0 || pg >= a.pages ? ~0u : (uint32_t)r;  // (2^32 sixteenths are more than memory holds)
  }
  // pieces: those of the next tiles, one per lane; `at` is this tile's first
  __device__ __forceinline__ void load(const StepArgs& a, int b, int kvh, int j0, int last, int lo, uint32_t pieces, int at, int lane) {
    hid = 0;
    const int g = lane >> 4, e0 = elem(0, g) / 32, e1 = elem(NS - 1, g) / 32;
    const int64_t to_v = (int64_t)a.Hk * (a.page / 16);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int j = j0 + 16 * s + (lane & 15);
      const uint32_t pc = __builtin_amdgcn_readlane(pieces, at + s);
      const bool ok = (j < last) & ((j < a.sinks) | (j >= lo)) & (pc != ~0u);
      hid |= (uint32_t)(~__builtin_amdgcn_ballot_w64(ok) & 0xffff) << (16 * s);
      const int64_t kr = pc == ~0u ? 0 : pc, vr = kr + to_v;
      const uint32_t o = (lane & 15) * (HDP / 2) + g * (HDP / 8), so = (lane & 15) * NB;
      const uint32_t *kc = (const uint32_t*)(a.codes + kr * (8 * HDP) + o), *vc = (const uint32_t*)(a.codes + vr * (8 * HDP) + o);
#pragma unroll
      for (int t = 0; t < NS; ++t) { k[s][t] = kc[t]; v[s][t] = vc[t]; }
      const uint8_t *kss = a.scales + kr * (16 * NB) + so, *vss = a.scales + vr * (16 * NB) + so;
      ks[s][0] = kss[e0];
      vs[s][0] = vss[e0];
      if constexpr (HDP == 96) {
        ks[s][1] = kss[e1];
        vs[s][1] = vss[e1];
      }
    }
  }
  __device__ __forceinline__ void clear(int s, bool hidden) {
#pragma unroll
    for (int t = 0; t < NS; ++t) v[s][t] = hidden ? 0 : v[s][t];
    vs[s][0] = hidden ? 127 : vs[s][0];
    if constexpr (HDP == 96) vs[s][1] = hidden ? 127 : vs[s][1];
  }
  __device__ __forceinline__ static float scale(const uint8_t* c, int t, int g) {
    // run t lies in the block of the first run or in that of the last
    if constexpr (HDP == 96) return kv4_scale(elem(t, g) / 32 != elem(0, g) / 32 ? c[1] : c[0]);
    else return kv4_scale(c[0]);
  }
  __device__ __forceinline__ bf16x8 kf(int s, int t, int g) const { return step_fp4(k[s][t], scale(ks[s], t, g)); }
  __device__ __forceinline__ bf16x8 vf(int s, int t, int g) const { return step_fp4(v[s][t], scale(vs[s], t, g)); }
};

template <typename T> __device__ __forceinline__ void step_row(const StepArgs& a, int b, int kvh, int r, int& i, int& h) {
  const int G = a.H / a.Hk;
  i = r / G;
  h = kvh * G + r % G;
}

// waves per SIMD that the registers of each form allow
template <bool KV4, typename T, int HDP, int NRT> constexpr int step_waves() {
  if (NRT == 4 || (NRT == 2 && HDP > 64 && !(KV4 && sizeof(T) == 2))) return 1;
  if (sizeof(T) == 4) return KV4 || (HDP <= 64 && NRT == 1) ? 2 : 1;
  return NRT == 1 && HDP <= 64 ? 3 : 2;
}

// Grid: (splits, Hk * row groups of 16 NRT, B); 4 waves.
template <bool KV4, typename T, int HDP, int NRT>
__global__ __launch_bounds__(256, (step_waves<KV4, T, HDP, NRT>())) void step_attn(StepArgs a) {
  using Ty = StepTypes<KV4, T>;
  using F = typename Ty::F;
  using E = typename Ty::E;
  using St = StepTile<KV4, T, HDP>;
  constexpr int NS = HDP / 32, ND = HDP / 16, PARTS = Ty::PARTS, IST = HDP + 16, OST = HDP + 4;
  constexpr int KT = 32, GROUP = 32;  // keys of a tile; tiles whose pages a wave holds at a time
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int b = blockIdx.z, kvh = blockIdx.y % a.Hk, r0 = blockIdx.y / a.Hk * 16 * NRT, R = a.Nq * (a.H / a.Hk);
  const int len = a.len ? min(max(a.len[b], 0), a.cap) : a.cap, off = len - a.Nq;
  const float c = a.scale * kTileLog2e;
  E* img = (E*)smem + w * 32 * IST;

  const SlideTiles<KT> tiles(a.window, a.sinks, off, len - 1, len);
  const int lo = off - a.window + 1;  // first key of the first query's window
  // this wave's share of the tiles
  const int64_t part = (int64_t)blockIdx.x * 4 + w, parts = (int64_t)a.splits * 4;
  const int ta = (int)(tiles.n * part / parts), tb = (int)(tiles.n * (part + 1) / parts);
  // tiles in flight: 4-bit ones are small, and three of them cover the latency of memory
  constexpr int RING = KV4 ? 3 : 2;
  St ring[RING];
  uint32_t pieces = ~0u;  // where the GROUP tiles from ta + i GROUP on lie, one 16-key piece per lane
  // Every turn fetches a tile (behind the last one, that again, from the caches): with a tile left out now and then
  // the compiler, which has to count loads on every path, would wait for all of them.
  auto fetch = [&](St& st, int t) {
    if constexpr (KV4) {
      if ((t - ta) % GROUP == 0 && t < tb) {
        const int tt = t + lane / 2, j = tt < tb ? tiles.key0(tt) + lane % 2 * 16 : len;
        pieces = j < len ? St::piece(a, b, kvh, j) : ~0u;
      }
    }
    t = min(t, tb - 1);
    st.load(a, b, kvh, tiles.key0(t), len, lo, pieces, (t - ta) % GROUP * 2, lane);
  };
  if (ta < tb) {
#pragma unroll
    for (int i = 0; i + 1 < RING; ++i) fetch(ring[i], ta + i);
  }

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
  float m[NRT], l[NRT];  // m: the exponent that the sums are relative to (c s), within 8 of the running maximum
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[rt][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  auto compute = [&](St& cur, int t) {
    const int j0 = tiles.key0(t);
    const bool full = cur.hid == 0 && j0 + KT - 1 <= off && (j0 + KT <= a.sinks || len - 1 - j0 < a.window);
    f32x4 sc[NRT][2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt) sc[rt][s] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const F k = cur.kf(s, i, g);
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) sc[rt][s] = Tile<E>::mma16(k, qf[rt][i][p], sc[rt][s]);
      }
    }
    if (cur.hid) {
#pragma unroll
      for (int s = 0; s < 2; ++s) cur.clear(s, cur.hid >> (16 * s + (lane & 15)) & 1);
    }
    // V rows into the wave's own image: a wave's LDS accesses run in order, so the last tile's reads are
    // served before these writes, and these before the reads below (the fences hold the compiler to it)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NS; ++i) *(F*)(img + (16 * s + (lane & 15)) * IST + St::elem(i, g)) = cur.vf(s, i, g);
    asm volatile("" ::: "memory");
    F pf[NRT][PARTS];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      f32x8 x = {sc[rt][0][0], sc[rt][0][1], sc[rt][0][2], sc[rt][0][3], sc[rt][1][0], sc[rt][1][1], sc[rt][1][2], sc[rt][1][3]};
      if (!full) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int jj = 16 * (e >> 2) + 4 * g + (e & 3), j = j0 + jj;
          const bool sees = (((unsigned)(pos[rt] - j) < (unsigned)a.window) | ((j < a.sinks) & (j <= pos[rt]))) & !(cur.hid >> jj & 1);
          x[e] = sees ? x[e] : -INFINITY;
        }
      }
      float mt = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mt = fmaxf(mt, x[e]);
      mt = tile_max32(tile_max16(mt)) * c;
      if (__builtin_amdgcn_ballot_w64(mt > m[rt] + 8.f)) {
        const float mn = fmaxf(m[rt], mt), alpha = mn == -INFINITY ? 1.f : tile_exp2(m[rt] - mn);
        m[rt] = mn;
        l[rt] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[rt][d] *= alpha;
      }
      const float ms = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = tile_exp2(fmaf(x[e], c, -ms));
        l[rt] += x[e];
      }
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
  };
  // (a ring by unrolling: copying a tile that is on its way would wait for it)
  for (int t = ta; t < tb; t += RING) {
#pragma unroll
    for (int i = 0; i < RING; ++i) {
      if (t + i >= tb) break;
      fetch(ring[(i + RING - 1) % RING], t + i + RING - 1);
      compute(ring[i], t + i);
    }
  }
  // join the 4 waves, 16 columns at a time
  float* os = (float*)smem;               // [4][16][OST]
  float* ms = os + 4 * 16 * OST;          // [4][16] maximum, [4][16] sum
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    const float lt = tile_sum32(tile_sum16(l[rt]));
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

// One workgroup per (sequence, head, query): 8 groups of 32 lanes (4 elements each) share the splits, and
// their sums are added in order.
template <typename T>
__global__ __launch_bounds__(256) void step_join(StepArgs a) {
  __shared__ f32x4 os[8][32];
  __shared__ float ls[8];
  const int64_t at = blockIdx.x;
  const int lane = threadIdx.x & 63, d = (threadIdx.x & 31) * 4, grp = threadIdx.x >> 5;
  const float* ml = a.pml + at * a.splits * 2;
  float mm = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) mm = fmaxf(mm, ml[2 * s]);
  mm = wave_max(mm);
  float ll = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const float* po = a.po + at * a.splits * a.hd + d;
#pragma unroll 4
  for (int s = grp; s < a.splits; s += 8) {
    const float f = mm == -INFINITY ? 0.f : tile_exp2(ml[2 * s] - mm);
    ll += f * ml[2 * s + 1];
    if (d < a.hd) o += *(const f32x4*)(po + (int64_t)s * a.hd) * f;
  }
  os[grp][threadIdx.x & 31] = o;
  if (d == 0) ls[grp] = ll;
  __syncthreads();
  if (grp || d >= a.hd) return;
  for (int u = 1; u < 8; ++u) {
    o += os[u][threadIdx.x];
    ll += ls[u];
  }
  const int i = (int)(at % a.Nq), h = (int)(at / a.Nq % a.H), b = (int)(at / a.Nq / a.H);
  Tile<T>::store4(row<T>(a.o, b, i, h) + d, o * (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll)));
  if (a.lse && d == 0) a.lse[at] = ll > 0.f ? (mm + __log2f(ll)) * kTileLn2 : (ll == 0.f ? -INFINITY : ll);
}

// 16-column tiles per wave: all of them, up to what registers hold; more rows take further workgroups,
// which read the cache again
static int step_nrt(int dtype, bool kv4, int hd, int rows) {
  const int most = dtype == CAPK_BF16 ? (kv4 || hd <= 96 ? 4 : 2) : kv4 || hd <= 96 ? 2 : 1;
  return rows <= 16 || most == 1 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
}

int64_t step_blocks(int dtype, const StepArgs& a) {
  const int rows = a.Nq * (a.H / a.Hk);  // (entries: 512 queries of 65535 heads, 64 of 2^20)
  return (int64_t)a.B * a.Hk * cdiv(rows, 16 * step_nrt(dtype, a.page != 0, a.hd, rows));
}

size_t step_workspace(int dtype, const StepArgs& a, int* splits) {
  const int64_t blocks = step_blocks(dtype, a);
  // two workgroups (what registers hold) on every CU, with at least a tile of 32 keys for each wave of a
  // split.  65536 to 131072 keys, 8 key heads of 128, 20 columns: 32 + 6 us (join) at 512 workgroups, 37 + 8 at 768,
  // 39 + 10 at 1024
  int64_t most = (int64_t)a.window + a.Nq + a.sinks + 64;
  if (most > a.cap) most = a.cap;
  int64_t s = 512 / blocks;
  if (s > cdiv(most, 128)) s = cdiv(most, 128);
  if (s < 1) s = 1;
  *splits = (int)s;
  return s > 1 ? (size_t)a.B * a.H * a.Nq * s * (a.hd + 2) * 4 : 0;
}

template <bool KV4, typename T, int HDP>
static int step_go(const StepArgs& a, hipStream_t st) {
  using E = typename StepTypes<KV4, T>::E;
  const int rows = a.Nq * (a.H / a.Hk), nrt = step_nrt(sizeof(T) == 2 ? CAPK_BF16 : CAPK_F32, KV4, a.hd, rows);
  const dim3 grid(a.splits, a.Hk * cdiv(rows, 16 * nrt), a.B);
  const size_t img = (size_t)4 * 32 * (HDP + 16) * sizeof(E), join = (size_t)4 * 16 * (HDP + 4) * 4 + 512;
  const size_t shm = img > join ? img : join;
  constexpr int N4 = sizeof(T) == 2 && (KV4 || HDP <= 96) ? 4 : 1, N2 = sizeof(T) == 4 && !KV4 && HDP > 96 ? 1 : 2;
  const void* fn = nrt == 1 ? (const void*)step_attn<KV4, T, HDP, 1> : nrt == 2 ? (const void*)step_attn<KV4, T, HDP, N2>
                                                                               : (const void*)step_attn<KV4, T, HDP, N4>;
  if (shm > 65536) {
    hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shm);
    if (e != hipSuccess) return hip_status(e, "step_attn");
  }
  StepArgs arg = a;
  void* args[] = {&arg};
  hipError_t e = hipLaunchKernel(fn, grid, dim3(256), args, shm, st);
  if (e != hipSuccess) return hip_status(e, "step_attn");
  if (a.splits > 1) {
    hipLaunchKernelGGL(step_join<T>, dim3(a.B * a.H * a.Nq), dim3(256), 0, st, a);
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
