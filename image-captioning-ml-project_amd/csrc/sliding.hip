// Sliding-window attention whose first tokens stay visible.
//
// The query at position p sees the keys j <= p with j < sinks or p - j < window; queries are the last
// Nq positions of a sequence of len[b] keys (len = Nk without kv_len), H query heads share Hk key
// heads.  o = softmax(scale q k^T) v over the visible keys; lse = log of the softmax's denominator.  A
// query that sees nothing gets o = 0, lse = -inf and no gradient.
//
// Forward: a workgroup owns 128 queries of a head (4 waves x 32), walks the key tiles that hold sinks
// and then those of its window, and keeps a running maximum and sum (one pass).  S^T = K Q^T puts one
// query on each lane, so the row statistics need one swap, and P^T, already in B-operand order, is
// multiplied by V^T fragments read transposed from LDS.  A tile's 16 + 16 products of 32 cycles (hd 128)
// stand beside about 1100 cycles of softmax and 1000 of LDS reads (each wave reads the whole tile for its 32
// queries), one after another within a wave, so no unit is saturated: 187 us for 16384 tokens, window 1024, 16 heads
// of 128 (134 GFLOP of visible pairs: 715 TF/s of the 1600 that a large product reaches); 64 queries per wave would
// halve the LDS reads, but its 128 sums then travel between the two halves of the register file every tile (700 us).
// Backward: D = rowsum(do * o); P = exp(s - lse); dS = P (do v^T - D) scale.  One kernel owns queries
// (dQ^T += K^T dS^T), one owns keys and walks their queries over all heads of the group
// (dV^T += dO^T P, dK^T += Q^T dS): every sum has one owner, so results do not depend on timing.  S and dP are
// computed in both (seven products for five): one kernel for all would add dQ through atomics.  The same
// tokens: dQ 236 us (three products: 850 TF/s of visible pairs), dK and dV 300 us (four: 890), with matrix, vector and
// LDS work each about a third of the time, as in the forward.  Keys that stay visible are seen by all later
// queries: those far queries are cut into chunks with owners of their own, whose 32-bit partial sums one more kernel
// adds in a fixed order (7 us).
//
// Roundings of the bf16 forms, besides inputs and results: P before P V and P^T dO, dS before its products (each
// half a bf16 step, 2^-9 to 2^-8 of the value, and independent, so sums of many keys average them), as the matrix
// unit takes bf16 operands and an fp32 operand costs six products; D comes from the rounded output where a row sees
// many keys.  Scores, maxima, sums, lse and D are 32-bit.  16384 tokens: relative error 2.4e-3 against 64 bits, 1.7e-3
// of which are the results' own rounding.
// fp32: three bf16 parts per value and six part products per product (tiles.h), 2.7 times as fast as the fp32 matrix
// instructions.  Magnitudes from 3.39e38 on (the largest bf16) have no finite first part and give NaN.
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
  float* part;          // partial sums of dK and dV
  int sink_tiles, far_chunks, far_rows, near_chunks;
};

constexpr int kSlideKeys = 128;  // keys of a dK / dV workgroup
// Partial sums [B, Hk][part][dK, dV][128][hd]: tiles with sinks have far_chunks + near_chunks parts, the others
// (more than one near chunk) near_chunks.
__host__ __device__ __forceinline__ int slide_parts(const SlideArgs& a) {
  const int tiles = (a.Nk + kSlideKeys - 1) / kSlideKeys;
  if (a.near_chunks > 1) return a.sink_tiles * a.far_chunks + tiles * a.near_chunks;
  return a.far_chunks ? a.sink_tiles * (a.far_chunks + 1) : 0;
}
// the first of a tile's parts; a tile without sinks has no far ones
__device__ __forceinline__ int slide_part(const SlideArgs& a, int tile) {
  return tile * a.near_chunks + min(tile, a.sink_tiles) * a.far_chunks;
}

__device__ __forceinline__ int slide_len(const SlideArgs& a, int b) {
  return a.len ? min(max(a.len[b], 0), a.Nk) : a.Nk;
}
__device__ __forceinline__ bool slide_sees(const SlideArgs& a, int p, int j) {
  return ((unsigned)(p - j) < (unsigned)a.window) | ((j < a.sinks) & (j <= p));  // (no branches: 32 of these per tile)
}

// One-dimensional grids, key heads fastest: workgroups go round-robin over the 8 XCDs, so with B Hk a
// multiple of 8 a key head's tiles run on one XCD and share its L2 (with 4, on two).  Long items first.
struct SlideBlock {
  int b, kvh, rest;
  __device__ __forceinline__ explicit SlideBlock(const SlideArgs& a, int i) {
    const int n = a.B * a.Hk;
    kvh = i % n % a.Hk;
    b = i % n / a.Hk;
    rest = i / n;
  }
};

// Fragments of a row, zeros where !ok or past hd.  The loads are of a valid row in any case and without
// conditions: behind one each would be waited for.
template <typename T, int HDP>
__device__ __forceinline__ void slide_frags(typename Mat<T>::V8 (&f)[HDP / 16], const T* src, bool ok, int hd, int h) {
  typename Tile<T>::V8 x[HDP / 16];
#pragma unroll
  for (int s = 0; s < HDP / 16; ++s) x[s] = Tile<T>::load(src + (s * 16 + h * 8 < hd ? s * 16 + h * 8 : 0));
#pragma unroll
  for (int s = 0; s < HDP / 16; ++s) f[s] = Mat<T>::from(ok && s * 16 + h * 8 < hd ? x[s] : tile_zero8<T>());
}
// The same with conditional loads (src is read only where ok): in slide_dkv of bf16, whose registers are all taken,
// the unconditional form is allocated worse (306 us for 299 at 16384 tokens).
template <typename T, int HDP>
__device__ __forceinline__ void slide_frags_if(typename Mat<T>::V8 (&f)[HDP / 16], const T* src, bool ok, int hd, int h) {
#pragma unroll
  for (int s = 0; s < HDP / 16; ++s) {
    typename Tile<T>::V8 x = tile_zero8<T>();
    if (ok && s * 16 + h * 8 < hd) x = Tile<T>::load(src + s * 16 + h * 8);
    f[s] = Mat<T>::from(x);
  }
}
template <typename V, int N> __device__ __forceinline__ void slide_settle(V (&f)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) tile_settle(f[s]);
}
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

// Tiles of 64 rows of two matrices (K and V, or Q and dO) on their way into LDS images, by 4 waves.
// bf16: copied straight to LDS, into the one pair of images while the other is read.
template <typename T, int HDP> struct SlidePair {
  using Img = TileImg<bf16, HDP>;
  static constexpr int IMG = Img::bytes(64), LDS = 4 * IMG;
  const T *x, *y;
  int64_t xrs, yrs;
  int hd, w, lane;
  char* smem;
  __device__ __forceinline__ void fetch(int r0, int last, int buf) {  // rows past `last` repeat it
    Img::template dma<64, 4>(smem + buf * 2 * IMG, x, xrs, r0, last, hd, w, lane);
    Img::template dma<64, 4>(smem + buf * 2 * IMG + IMG, y, yrs, r0, last, hd, w, lane);
  }
  // Waits for the tile, and for the readers of the one before; rows with a bit in `out` become zeros (they
  // may hold anything).  GROUPS = 2: the barriers meet two groups of waves with tiles of their own, so the
  // second is taken in any case.
  template <int GROUPS = 1> __device__ __forceinline__ void land(int buf, uint64_t out) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (out) {
      Img::clear(smem + buf * 2 * IMG, out);
      Img::clear(smem + buf * 2 * IMG + IMG, out);
    }
    if (GROUPS == 2 || out) __syncthreads();
  }
  __device__ __forceinline__ const char* first(int buf) const { return smem + buf * 2 * IMG; }
  __device__ __forceinline__ const char* second(int buf) const { return smem + buf * 2 * IMG + IMG; }
};
// fp32: through registers, split into the parts of the one pair of images when its readers are done.
template <int HDP> struct SlidePair<float, HDP> {
  using Img = TileImg<float, HDP>;
  static constexpr int IMG = Img::bytes(64), LDS = 2 * IMG, C = HDP / 8, N = C / 4;  // chunks of 8: per row, per thread
  const float *x, *y;
  int64_t xrs, yrs;
  int hd, w, lane;
  char* smem;
  f32x8 rx[N], ry[N];
  __device__ __forceinline__ void fetch(int r0, int last, int) {
    const int t = threadIdx.x & 255;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = i * 256 + t, c = o % C * 8, col = c < hd ? c : 0;
      const int64_t r = min(r0 + o / C, last);
      rx[i] = Tile<float>::load(x + r * xrs + col);
      ry[i] = Tile<float>::load(y + r * yrs + col);
    }
  }
  template <int GROUPS = 1> __device__ __forceinline__ void land(int, uint64_t out) {
    __syncthreads();
    const int t = threadIdx.x & 255;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = i * 256 + t, r = o / C, at = r * TileImg<bf16, HDP>::RB + ((o % C ^ TileImg<bf16, HDP>::swz(r)) << 4);
      if (out >> r & 1) rx[i] = ry[i] = tile_zero8<float>();
      const Split8 a = Mat<float>::from(rx[i]), b = Mat<float>::from(ry[i]);
      *(bf16x8*)(smem + at) = a.h;
      *(bf16x8*)(smem + at + Img::PART) = a.m;
      *(bf16x8*)(smem + at + 2 * Img::PART) = a.l;
      *(bf16x8*)(smem + at + IMG) = b.h;
      *(bf16x8*)(smem + at + IMG + Img::PART) = b.m;
      *(bf16x8*)(smem + at + IMG + 2 * Img::PART) = b.l;
    }
    __syncthreads();
  }
  __device__ __forceinline__ const char* first(int) const { return smem; }
  __device__ __forceinline__ const char* second(int) const { return smem + IMG; }
};

// One bit per key of the tile at j0: past the length or padded; seen by no query at p_lo..p_hi.
__device__ __forceinline__ uint64_t slide_hidden(const SlideArgs& a, int b, int j, int len) {
  return __builtin_amdgcn_ballot_w64(j >= len || (a.pad && a.pad[(int64_t)b * a.Nk + j]));
}
__device__ __forceinline__ uint64_t slide_unseen(const SlideArgs& a, int j, int p_lo, int p_hi) {
  return __builtin_amdgcn_ballot_w64((j > p_hi) | ((j >= a.sinks) & (p_lo - j >= a.window)));
}

// n products whose LDS operands are requested D ahead: the order is written down, as the compiler would
// request each operand right before its use and wait for it
template <int D, int N, typename L, typename M> __device__ __forceinline__ void slide_pipe(L load, M mul) {
  decltype(load(0)) f[D];
#pragma unroll
  for (int i = 0; i < D && i < N; ++i) f[i] = load(i);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    mul(i, f[i % D]);
    if (i + D < N) f[i % D] = load(i + D);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// whether queries at positions p_lo..p_hi see none, or all, of the keys j0 .. j0 + n - 1
__device__ __forceinline__ bool slide_none(const SlideArgs& a, int j0, int n, int p_lo, int p_hi) {
  return j0 > p_hi || (j0 >= a.sinks && p_lo - (j0 + n - 1) >= a.window);
}
__device__ __forceinline__ bool slide_full(const SlideArgs& a, int j0, int n, int p_lo, int p_hi) {
  return j0 + n - 1 <= p_lo && (j0 + n <= a.sinks || p_hi - j0 < a.window);
}

// GROUPS = 2: a second group of 4 waves, with images of its own, takes every other tile of the same queries.
template <typename T, int HDP, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, sizeof(T) == 4 ? (HDP <= 64 ? 2 : 1) : GROUPS == 2 || HDP > 96 ? 2 : 3) void slide_fwd(SlideArgs a) {
  using KV = SlidePair<T, HDP>;
  using Img = typename KV::Img;
  constexpr int NS = HDP / 16, ND = HDP / 32;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3), hh = lane >> 5;
  const int grp = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const SlideBlock at(a, blockIdx.x);
  const int b = at.b, kvh = at.kvh, G = a.H / a.Hk, h = kvh * G + at.rest % G, len = slide_len(a, b), off = len - a.Nq;
  const int q0 = ((a.Nq + 127) / 128 - 1 - at.rest / G) * 128, qw = q0 + w * 32, qi = qw + (lane & 31), p = off + qi;
  const int qr = min(qi, a.Nq - 1);  // a row to load
  const int p_lo = off + q0, p_hi = off + min(q0 + 127, a.Nq - 1);
  const int pw_lo = off + qw, pw_hi = off + qw + 31;
  const float c = a.scale * kTileLog2e;
  typename Img::Lane ln(lane);
  const SlideTiles<64> tiles(a.window, a.sinks, p_lo, p_hi, len);
  const int last = min(len, p_hi + 1) - 1;
  KV kv{row<T>(a.k, b, 0, kvh), row<T>(a.v, b, 0, kvh), a.k.rs, a.v.rs, a.hd, w, lane, smem + grp * KV::LDS};
  if (grp < tiles.n) kv.fetch(tiles.key0(grp), last, 0);

  typename Mat<T>::V8 qf[NS];
  slide_frags<T, HDP>(qf, row<T>(a.q, b, qr, h), qi < a.Nq, a.hd, hh);
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = tile_zero<f32x16>();
  // mc: the exponent that the sums are relative to, the running maximum of c s or up to 8 below it (so
  // that o is rescaled when the maximum has grown 2^8-fold, not with every step of it)
  float mc = -INFINITY, l = 0.f;
  slide_settle(qf);
  for (int u = 0; u * GROUPS < tiles.n; ++u) {  // (as many turns, and barriers, in both groups)
    const int t = u * GROUPS + grp, j0 = tiles.key0(t);
    const int j = t < tiles.n ? j0 + lane : p_hi;
    const uint64_t hid = slide_hidden(a, b, j, len);
    kv.template land<GROUPS>(u & 1, hid | slide_unseen(a, j, p_lo, p_hi));
    if (t >= tiles.n) continue;
    const char *ki = kv.first(u & 1), *vi = kv.second(u & 1);
    if (t + GROUPS < tiles.n) kv.fetch(tiles.key0(t + GROUPS), last, (u + 1) & 1);
    if (slide_none(a, j0, 64, pw_lo, pw_hi)) continue;
    f32x16 s[2] = {tile_zero<f32x16>(), tile_zero<f32x16>()};
    slide_pipe<4, 2 * NS>([&](int i) { return Img::frag(ki, (i & 1) * 32, i >> 1, ln); },
                  [&](int i, const auto& k) { s[i & 1] = Mat<T>::mma32(k, qf[i >> 1], s[i & 1]); });
    typename Mat<T>::V8 vf[2][ND];  // V^T fragments of a 16-key step, requested a step ahead
#pragma unroll
    for (int d = 0; d < ND; ++d) vf[0][d] = Img::trans(vi, 0, d * 32, ln);
    // most masked tiles: three instructions per score, not eight (at 96, where three waves share a SIMD, the second
    // form of the mask spills: 97 us for 65 over 16 x 1024 tokens)
    if (HDP != 96 && !hid && j0 >= a.sinks) {
      if (!slide_full(a, j0, 64, pw_lo, pw_hi)) {
        const int d = p - j0 - 4 * hh;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[kb][i] = (unsigned)(d - (kb * 32 + 8 * (i >> 2) + (i & 3))) < (unsigned)a.window ? s[kb][i] : -INFINITY;
      }
    } else if (hid || !slide_full(a, j0, 64, pw_lo, pw_hi)) {
      const uint32_t hl[2] = {(uint32_t)hid >> (4 * hh), (uint32_t)(hid >> 32) >> (4 * hh)};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = 8 * (i >> 2) + (i & 3);
          const bool sees = slide_sees(a, p, j0 + kb * 32 + 4 * hh + r) & !(hl[kb] >> r & 1);
          s[kb][i] = sees ? s[kb][i] : -INFINITY;
        }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mt = fmaxf(fmaxf(mt, s[0][i]), s[1][i]);
    mt = tile_max32(mt) * c;
    if (__builtin_amdgcn_ballot_w64(mt > mc + 8.f)) {
      const float mn = fmaxf(mc, mt), alpha = mn == -INFINITY ? 1.f : tile_exp2(mc - mn);
      mc = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
    }
    const float ms = mc == -INFINITY ? 0.f : mc;
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // 16 keys each
      __builtin_amdgcn_sched_barrier(0);
      if (u < 3)
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[(u + 1) & 1][d] = Img::trans(vi, (u + 1) * 16, d * 32, ln);
      __builtin_amdgcn_sched_barrier(0);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = tile_exp2(fmaf(s[u >> 1][(u & 1) * 8 + e], c, -ms));
        l += x[e];
      }
      const typename Mat<T>::V8 pf = Mat<T>::pack(x);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = Mat<T>::mma32(vf[u & 1][d], pf, o[d]);
    }
  }
  l = tile_sum32(l);
  if constexpr (GROUPS == 2) {  // the groups' partial softmaxes joined: registers of the second through LDS
    __syncthreads();
    float* x = (float*)smem + (threadIdx.x & 255);
    if (grp == 1) {
      x[0] = mc;
      x[256] = l;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[(2 + d * 16 + i) * 256] = o[d][i];
    }
    __syncthreads();
    if (grp == 1) return;
    const float m1 = x[0], mn = fmaxf(mc, m1), f0 = mn == -INFINITY ? 0.f : tile_exp2(mc - mn), f1 = mn == -INFINITY ? 0.f : tile_exp2(m1 - mn);
    mc = mn;
    l = l * f0 + x[256] * f1;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * f0 + x[(2 + d * 16 + i) * 256] * f1;
  }
  if (qi >= a.Nq) return;
  slide_store<T, HDP>(row<T>(a.o, b, qi, h), o, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l), a.hd, hh);
  if (a.lse && hh == 0)
    a.lse[((int64_t)b * a.H + h) * a.Nq + qi] = l > 0.f ? (mc + __log2f(l)) * kTileLn2 : (l == 0.f ? -INFINITY : l);
}

template <typename T, int HDP>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? (HDP <= 64 ? 2 : 1) : HDP <= 64 ? 3 : 2) void slide_dq(SlideArgs a) {
  using KV = SlidePair<T, HDP>;
  using Img = typename KV::Img;
  constexpr int NS = HDP / 16, ND = HDP / 32;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const SlideBlock at(a, blockIdx.x);
  const int b = at.b, kvh = at.kvh, G = a.H / a.Hk, h = kvh * G + at.rest % G, len = slide_len(a, b), off = len - a.Nq;
  const int q0 = ((a.Nq + 127) / 128 - 1 - at.rest / G) * 128, qw = q0 + w * 32, qi = qw + (lane & 31), p = off + qi;
  const int qr = min(qi, a.Nq - 1);  // a row to load
  const int p_lo = off + q0, p_hi = off + min(q0 + 127, a.Nq - 1);
  const int pw_lo = off + qw, pw_hi = off + qw + 31;
  const float c = a.scale * kTileLog2e;
  typename Img::Lane ln(lane);
  const SlideTiles<64> tiles(a.window, a.sinks, p_lo, p_hi, len);
  const int last = min(len, p_hi + 1) - 1;
  KV kv{row<T>(a.k, b, 0, kvh), row<T>(a.v, b, 0, kvh), a.k.rs, a.v.rs, a.hd, w, lane, smem};
  if (tiles.n) kv.fetch(tiles.key0(0), last, 0);

  typename Mat<T>::V8 qf[NS], dof[NS];
  slide_frags<T, HDP>(qf, row<T>(a.q, b, qr, h), qi < a.Nq, a.hd, hh);
  slide_frags<T, HDP>(dof, row<T>(a.dout, b, qr, h), qi < a.Nq, a.hd, hh);
  const int64_t stat = ((int64_t)b * a.H + h) * a.Nq + qi;
  const float lse = a.lse[stat - qi + qr], lse2 = qi < a.Nq ? lse * kTileLog2e : INFINITY;
  // D from the saved output costs a pass over one row, but inherits that output's rounding, which weighs
  // where few keys share a row.  With at most 4 tiles of keys D is summed from P (do v^T) itself, in a
  // walk of its own.
  const bool walk = tiles.n <= 4;
  float delta = 0.f;
  if (!walk) {
    const T *o = row<T>(a.o, b, qr, h), *d = row<T>(a.dout, b, qr, h);
    typename Tile<T>::V8 x[NS], y[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int at = s * 16 + hh * 8 < a.hd ? s * 16 + hh * 8 : 0;
      x[s] = Tile<T>::load(o + at);
      y[s] = Tile<T>::load(d + at);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float f = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f = fmaf((float)x[s][e], (float)y[s][e], f);
      if (s * 16 + hh * 8 < a.hd) delta += f;
    }
    delta = tile_sum32(delta);
    if (lse2 == -INFINITY) delta = 0.f;  // (it sees nothing, and its do may be anything)
  }
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = tile_zero<f32x16>();
  slide_settle(qf);
  slide_settle(dof);
  // P and do v^T of 32 keys of a tile, zeros where the query does not see the key
  auto scores = [&](const char* ki, const char* vi, int j0, int kb, uint64_t hid, f32x16& s, f32x16& dp) {
    const uint32_t hidden = (uint32_t)(hid >> (32 * kb));
    s = dp = tile_zero<f32x16>();
    slide_pipe<(sizeof(T) == 2 ? 4 : 2), 2 * NS>([&](int i) { return Img::frag(i & 1 ? vi : ki, kb * 32, i >> 1, ln); },
                          [&](int i, const auto& f) {
                            if (i & 1) dp = Mat<T>::mma32(f, dof[i >> 1], dp);
                            else s = Mat<T>::mma32(f, qf[i >> 1], s);
                          });
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = tile_exp2(fmaf(s[i], c, -lse2));
    if (hidden || !slide_full(a, j0 + kb * 32, 32, pw_lo, pw_hi)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 8 * (i >> 2) + (i & 3);
        const bool sees = slide_sees(a, p, j0 + kb * 32 + 4 * hh + r) & !(hidden >> (4 * hh + r) & 1);
        s[i] = sees ? s[i] : 0.f;
        dp[i] = sees ? dp[i] : 0.f;
      }
    }
  };
  int buf = 0;
  if (walk) {
    for (int t = 0; t < tiles.n; ++t, buf ^= 1) {
      const int j0 = tiles.key0(t);
      const uint64_t hid = slide_hidden(a, b, j0 + lane, len);
      kv.land(buf, hid | slide_unseen(a, j0 + lane, p_lo, p_hi));
      const char *ki = kv.first(buf), *vi = kv.second(buf);
      kv.fetch(tiles.key0(t + 1 < tiles.n ? t + 1 : 0), last, buf ^ 1);
#pragma unroll 1
      for (int kb = 0; kb < 2; ++kb) {
        if (slide_none(a, j0 + kb * 32, 32, pw_lo, pw_hi)) continue;
        f32x16 s, dp;
        scores(ki, vi, j0, kb, hid, s, dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) delta = fmaf(s[i], dp[i], delta);
      }
    }
    delta = tile_sum32(delta);
  }
  for (int t = 0; t < tiles.n; ++t, buf ^= 1) {
    const int j0 = tiles.key0(t);
    const uint64_t hid = slide_hidden(a, b, j0 + lane, len);
    kv.land(buf, hid | slide_unseen(a, j0 + lane, p_lo, p_hi));
    const char *ki = kv.first(buf), *vi = kv.second(buf);
    if (t + 1 < tiles.n) kv.fetch(tiles.key0(t + 1), last, buf ^ 1);
#pragma unroll 1
    for (int kb = 0; kb < 2; ++kb) {
      if (slide_none(a, j0 + kb * 32, 32, pw_lo, pw_hi)) continue;
      f32x16 s, dp;
      scores(ki, vi, j0, kb, hid, s, dp);
      typename Mat<T>::V8 df[2];
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[st * 8 + e] * (dp[st * 8 + e] - delta);
        df[st] = Mat<T>::pack(x);
      }
      slide_pipe<(sizeof(T) == 2 ? 4 : 2), 2 * ND>([&](int i) { return Img::trans(ki, kb * 32 + i / ND * 16, i % ND * 32, ln); },
                            [&](int i, const auto& f) { dq[i % ND] = Mat<T>::mma32(f, df[i / ND], dq[i % ND]); });
    }
  }
  if (qi >= a.Nq) return;
  if (hh == 0) a.delta[stat] = delta;
  slide_store<T, HDP>(row<T>(a.dq, b, qi, h), dq, a.scale, a.hd, hh);
}

// The key tile and chunk of an item of dK / dV: near chunks of every tile first, then the far ones.
struct SlideChunk : SlideBlock {
  bool far;
  int tile, chunk;
  __device__ __forceinline__ SlideChunk(const SlideArgs& a, int i, int near_chunks) : SlideBlock(a, i) {
    const int near = (a.Nk + kSlideKeys - 1) / kSlideKeys * near_chunks;
    far = rest >= near;
    const int at = far ? rest - near : rest, cut = far ? a.far_chunks : near_chunks;
    tile = at / cut;
    chunk = at % cut;
  }
};

// Keys [j0, j0 + 128) of a key head against queries [qa, qb) of its group, a chunk of their tiles; far = only the
// sinks among the keys, at queries that no longer have them in their window.  CUT: more than one near chunk (a form
// of its own: with it the other would hold a few registers in memory, 307 us for 300 at 16384 tokens).
template <typename T, int HDP, bool CUT>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : HDP <= 64 ? 3 : 2) void slide_dkv(SlideArgs a) {
  using Pair = SlidePair<T, HDP>;
  using Img = typename Pair::Img;
  constexpr int QT = 64, NS = HDP / 16, ND = HDP / 32;
  extern __shared__ __align__(16) char smem[];
  float* Ls = (float*)(smem + Pair::LDS);  // per buffer: lse (base 2) and D of 64 queries
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int cuts = CUT ? a.near_chunks : 1;
  const SlideChunk at(a, blockIdx.x, cuts);
  const int b = at.b, kvh = at.kvh, G = a.H / a.Hk, len = slide_len(a, b), off = len - a.Nq;
  const bool far = at.far;
  const int tile = at.tile, chunk = at.chunk;
  const int j0 = tile * kSlideKeys, jw = j0 + w * 32, j = jw + (lane & 31);
  const bool key_ok = j < len && !(a.pad && a.pad[(int64_t)b * a.Nk + j]) && (!far || j < a.sinks);
  // positions of the queries: near p in [j0, near_end), far p >= near_end in chunks of far_rows (no
  // chunks: the owner of a tile with sinks walks all of them)
  const int64_t near_end = tile < a.sink_tiles && a.far_chunks == 0 ? (int64_t)1 << 40 : (int64_t)j0 + kSlideKeys - 1 + a.window;
  const int qn = (int)min((int64_t)a.Nq, max((int64_t)0, near_end - off));
  int qa = far ? qn + chunk * a.far_rows : max(0, j0 - off);
  int qb = far ? min(a.Nq, qa + a.far_rows) : (j0 < len ? qn : 0);
  if (CUT && !far) {  // a share of the range's tiles of 64
    const int64_t n = qb > qa ? (qb - qa + QT - 1) / QT : 0;
    const int lo = (int)(n * chunk / cuts), hi = (int)(n * (chunk + 1) / cuts);
    qb = min(qb, qa + hi * QT);
    qa += lo * QT;
  }
  const float c = a.scale * kTileLog2e;
  typename Img::Lane ln(lane);
  const int nq = qb > qa ? (qb - qa + QT - 1) / QT : 0, all = nq * G;

  // the tile of 64 queries t: head kvh G + t / nq, queries qa + 64 (t % nq)
  const float* stat = (threadIdx.x & 64 ? a.delta : a.lse) + (int64_t)b * a.H * a.Nq;
  float ld = 0.f;  // threads 0..63 carry lse, 64..127 D (unconditional loads: nothing waits for them here)
  Pair qd{nullptr, nullptr, a.q.rs, a.dout.rs, a.hd, w, lane, smem};
  auto fetch = [&](int t, int buf) {
    const int h = kvh * G + t / nq, q0 = qa + t % nq * QT;
    ld = stat[(int64_t)h * a.Nq + min(q0 + lane, qb - 1)];
    qd.x = row<T>(a.q, b, 0, h);
    qd.y = row<T>(a.dout, b, 0, h);
    qd.fetch(q0, qb - 1, buf);
  };
  if (all > 0) fetch(0, 0);
  typename Mat<T>::V8 kf[NS], vf[NS];
  if constexpr (sizeof(T) == 4) {
    const int jr = min(j, a.Nk - 1);
    slide_frags<T, HDP>(kf, row<T>(a.k, b, jr, kvh), key_ok, a.hd, hh);
    slide_frags<T, HDP>(vf, row<T>(a.v, b, jr, kvh), key_ok, a.hd, hh);
  } else {
    slide_frags_if<T, HDP>(kf, row<T>(a.k, b, j, kvh), key_ok, a.hd, hh);
    slide_frags_if<T, HDP>(vf, row<T>(a.v, b, j, kvh), key_ok, a.hd, hh);
  }
  const bool hidden = __builtin_amdgcn_ballot_w64(!key_ok) != 0;
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = tile_zero<f32x16>();
  slide_settle(kf);
  slide_settle(vf);
  for (int t = 0; t < all; ++t) {
    const float* ls = Ls + (t & 1) * 128;
    const int q0 = qa + t % nq * QT, p0 = off + q0;
    if (w < 2) Ls[(t & 1) * 128 + threadIdx.x] = q0 + lane >= qb ? (w ? 0.f : INFINITY) : (w ? ld : ld * kTileLog2e);
    qd.land(t & 1, 0);
    const char *qi = qd.first(t & 1), *di = qd.second(t & 1);
    if (t + 1 < all) fetch(t + 1, (t + 1) & 1);
#pragma unroll 1
    for (int qt = 0; qt < 2; ++qt) {
      const int pq = p0 + qt * 32;
      if (slide_none(a, jw, 32, pq, pq + 31)) continue;
      const bool full = !hidden && q0 + qt * 32 + 32 <= qb && slide_full(a, jw, 32, pq, pq + 31);
      if constexpr (sizeof(T) == 2 || HDP > 96) ln.forget();
      f32x16 s = tile_zero<f32x16>(), dp = tile_zero<f32x16>();
      slide_pipe<2, 2 * NS>([&](int i) { return Img::frag(i & 1 ? di : qi, qt * 32, i >> 1, ln); },
                            [&](int i, const auto& f) {
                              if (i & 1) dp = Mat<T>::mma32(f, vf[i >> 1], dp);
                              else s = Mat<T>::mma32(f, kf[i >> 1], s);
                            });
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int r = qt * 32 + 8 * i4 + 4 * hh;
        const f32x4 lv = *(const f32x4*)(ls + r), dl = *(const f32x4*)(ls + 64 + r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * i4 + e;
          const float x = tile_exp2(fmaf(s[i], c, -lv[e]));
          s[i] = x;
          dp[i] = x * (dp[i] - dl[e]);
        }
      }
      if (!full) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = qt * 32 + 8 * (i >> 2) + 4 * hh + (i & 3);
          const bool sees = key_ok & (q0 + r < qb) & slide_sees(a, p0 + r, j);
          s[i] = sees ? s[i] : 0.f;
          dp[i] = sees ? dp[i] : 0.f;
        }
      }
      typename Mat<T>::V8 pf[2], df[2];
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = s[st * 8 + e]; y[e] = dp[st * 8 + e]; }
        pf[st] = Mat<T>::pack(x);
        df[st] = Mat<T>::pack(y);
      }
      slide_pipe<2, 4 * ND>([&](int i) { return Img::trans(i & 1 ? qi : di, qt * 32 + i / (2 * ND) * 16, (i >> 1) % ND * 32, ln); },
                            [&](int i, const auto& f) {
                              const int d = (i >> 1) % ND, st = i / (2 * ND);
                              if (i & 1) dk[d] = Mat<T>::mma32(f, df[st], dk[d]);
                              else dv[d] = Mat<T>::mma32(f, pf[st], dv[d]);
                            });
    }
  }
  SlideChunk to = at;
  if constexpr (CUT) {  // (found again: the loop has no registers to keep it)
    int item = blockIdx.x;
    asm volatile("" : "+s"(item));
    to = SlideChunk(a, item, cuts);
  }
  if (to.far && j >= a.sinks) return;
  if (CUT || (to.tile < a.sink_tiles && a.far_chunks > 0)) {
    const int part = slide_part(a, to.tile) + (to.far || to.tile >= a.sink_tiles ? to.chunk : a.far_chunks + to.chunk);
    float* dst = a.part + (((int64_t)to.b * a.Hk + to.kvh) * slide_parts(a) + part) * 2 * kSlideKeys * a.hd +
                 (int64_t)(w * 32 + (lane & 31)) * a.hd;
    slide_store<float, HDP>(dst, dk, a.scale, a.hd, hh);
    slide_store<float, HDP>(dst + (int64_t)kSlideKeys * a.hd, dv, 1.f, a.hd, hh);
  } else if (j < a.Nk) {
    slide_store<T, HDP>(row<T>(a.dk, to.b, j, to.kvh), dk, a.scale, a.hd, hh);
    slide_store<T, HDP>(row<T>(a.dv, to.b, j, to.kvh), dv, 1.f, a.hd, hh);
  }
}

// dK, dV rows of the tiles with partial sums = their sum, in order.  One thread per 4 elements.
template <typename T>
__global__ __launch_bounds__(256) void slide_dkv_sum(SlideArgs a) {
  const int per = kSlideKeys * a.hd / 4;
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int e = i % per * 4, which = i / per % 2, tile = i / per / 2, j = tile * kSlideKeys + e / a.hd;
  if (j >= a.Nk || (a.near_chunks == 1 && tile >= a.sink_tiles)) return;
  const int far = tile < a.sink_tiles ? a.far_chunks : 0;
  const float* src = a.part + (((int64_t)blockIdx.z * a.Hk + blockIdx.y) * slide_parts(a) + slide_part(a, tile)) * 2 *
                                  kSlideKeys * a.hd + (int64_t)which * kSlideKeys * a.hd + e;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int c = j < a.sinks ? 0 : far; c < far + a.near_chunks; ++c) s += *(const f32x4*)(src + (int64_t)c * 2 * kSlideKeys * a.hd);
  Tile<T>::store4(row<T>(which ? a.dv : a.dk, blockIdx.z, j, blockIdx.y) + e % a.hd, s);
}

template <typename K>
static int slide_launch(K kernel, dim3 grid, size_t shm, hipStream_t st, const SlideArgs& a, const char* name,
                        int threads = 256) {
  if (shm > 65536) {
    hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shm);
    if (e != hipSuccess) return hip_status(e, name);
  }
  hipLaunchKernelGGL(kernel, grid, dim3(threads), shm, st, a);
  CAPK_LAUNCH_CHECK(name);
  return CAPK_OK;
}

// sizes that a workspace query may compute with (the entries refuse the others, with a message)
static bool slide_sizes(int B, int H, int Hk, int Nq, int Nk, int hd, int window, int sinks) {
  return B >= 1 && B <= 65535 && Hk >= 1 && H >= Hk && H <= 65535 && H % Hk == 0 && Nq >= 1 && Nq <= (1 << 28) && Nk >= 1 && Nk <= (1 << 28) &&
         hd >= 1 && hd <= 128 && window >= 0 && sinks >= 0;
}

static int slide_check(const char* who, int dtype, int B, int H, int Hk, int Nq, int Nk, int hd, int window, int sinks,
                       float scale, const SlideView* v, int n) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "%s: dtype", who);
  CAPK_CHECK_ARG(B >= 1 && B <= 65535 && Nq >= 1 && Nk >= 1 && Nq <= (1 << 28) && Nk <= (1 << 28), "%s: bad sizes", who);
  CAPK_CHECK_ARG(Hk >= 1 && H >= Hk && H % Hk == 0 && H <= 65535, "%s: %d query heads over %d key heads", who, H, Hk);
  CAPK_CHECK_ARG(hd >= 8 && hd % 8 == 0 && hd <= 128, "%s: hd=%d must be a multiple of 8, <= 128", who, hd);
  CAPK_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window and sinks must not be negative", who);
  CAPK_CHECK_ARG((int64_t)B * H * (cdiv(Nq, 128) + 2 * (int64_t)cdiv(Nk, 128)) < (1 << 24), "%s: too many tiles", who);
  CAPK_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: scale must be positive", who);
  const int ea = dtype == CAPK_BF16 ? 8 : 4;
  for (int i = 0; i < n; ++i)
    CAPK_CHECK_ARG(v[i].p && (uintptr_t)v[i].p % 16 == 0 && v[i].bs % ea == 0 && v[i].rs % ea == 0 && v[i].hs % ea == 0 &&
                       v[i].rs >= 0 && v[i].rs < (1 << 22),
                   "%s: operand %d must be 16-B aligned with strides that keep it so, and tokens less than 2^22 elements apart",
                   who, i);
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

// How the queries of the key tiles are cut.  An item's length is its 64-query tiles over all heads of the group.
// Near queries: where the tiles alone leave CUs without a workgroup (fewer than 256), each tile's range goes in chunks
// whose length is a CU's share of the whole (at least two).  Measured, dK and dV with their sum: 80 to 34 us (one
// sequence of 2956, 2 key heads of 64, window 489), 586 to 207 (4096, 4 of 128, no window), 60 to 20 (2 x 500, 2 of
// 64), fp32 78 to 50 (3 x 777, 3 of 80, window 100).  Far queries of the sink tiles: on such small grids in chunks of that length too; else the launch runs about
// `slots` workgroups at a time, and where even the longest item (a sink tile with every query) is within a slot's
// share of the whole, each sink tile has one owner; else its far queries go in chunks of a quarter of that share (at
// least 256 queries), so the partial sums stay below 2^29 bytes.
static void slide_cut(SlideArgs& a) {
  const int64_t slots = 512, G = a.H / a.Hk, heads = a.B * (int64_t)a.Hk, tiles = cdiv(a.Nk, kSlideKeys);
  a.sink_tiles = cdiv(a.sinks, kSlideKeys);
  a.far_rows = a.far_chunks = 0;
  a.near_chunks = 1;
  // the first sink tile has the most far queries: positions from 127 + window on
  const int64_t most = (int64_t)a.Nk - (kSlideKeys - 1) - a.window, rows = most < a.Nq ? most : a.Nq;
  const bool whole = a.window + kSlideKeys >= a.Nq;  // no window to speak of: later tiles have fewer queries
  const int64_t walk = cdiv(whole ? a.Nq : a.window + kSlideKeys, 64), near = walk * G;
  const int64_t far = a.sink_tiles && rows > 0 ? cdiv(rows, 64) * G : 0;
  int64_t n;
  if (heads * tiles < 256) {
    int64_t share = heads * (tiles * (whole ? near / 2 + 1 : near) + a.sink_tiles * far) / 256 + 1;
    if (share < 2) share = 2;
    const int64_t cut = cdiv(near, share);
    a.near_chunks = (int)(cut < walk ? cut : walk);
    n = cdiv(share, G) * 64;
  } else {
    const int64_t share = heads * (tiles * near + a.sink_tiles * far) / slots;
    if (near + far <= share) return;
    n = share / 4 / G * 64;
    if (n < 256) n = 256;
  }
  if (!far) return;
  a.far_rows = (int)n;
  a.far_chunks = cdiv(rows, n);
}

}  // namespace capk

using namespace capk;

static StepArgs slide_step(const SlideArgs& a) {
  StepArgs s{};
  s.B = a.B; s.H = a.H; s.Hk = a.Hk; s.Nq = a.Nq; s.cap = a.Nk; s.hd = a.hd;
  s.window = a.window; s.sinks = a.sinks; s.scale = a.scale;
  s.q = a.q; s.k = a.k; s.v = a.v; s.o = a.o; s.len = a.len; s.pad = a.pad; s.lse = a.lse;
  return s;
}
// Few queries for their keys (a decoding step, drafted tokens, a chunk of a prompt): the kernel that splits the keys
// over workgroups.  slide_fwd walks a query tile's keys in one chain, whatever else is idle: 10 to 14 ns a key in bf16
// (heads of 64 to 128), 41 to 99 in fp32, as long as its workgroups find a CU each.  The other takes 0.05 ns (fp32 0.1)
// times the keys times its workgroups of up to 64 columns (query, head), and about 20 us: even at 210 to 260 of them
// (fp32 430 to 900) on long caches.  The rule stays below that, and lower on shorter caches.  Measured, us, slide_fwd /
// this: bf16, 16 / 4 heads of 128, 131072 keys 1905 / 114 (17 queries), 1907 / 253 (64), 1912 / 917 (256); 8192 keys 122 /
// 26, 123 / 35, 126 / 81; eight sequences of 8192 126 / 65, 128 / 137, 153 / 476; 2048 keys 35 / 15, 36 / 26, 37 / 37; 12
// heads of 64, 8192 keys 90 / 17, 91 / 30, 92 / 53; 512 keys 12 to 16 / 15 to 26.  fp32, 16 / 4 heads of 128, 512 keys
// 57 / 17, 57 / 19, 59 / 41; 32768 3240 / 107, 3243 / 257, 3260 / 916; 512 queries
// of 12 heads of 64 over 512 keys 27 / 33.  At most 512 queries (four tiles): beyond, a whole pass is meant, where
// later queries see more keys than earlier ones and slide_fwd does not compute the difference.
// Up to 16 queries are the step's own case, on short caches too (512 keys: 14.8 / 15.1).
static bool slide_few(int dtype, const SlideArgs& a) {
  if (a.Nq <= 16) return true;
  if (a.Nq > 512) return false;
  // keys that a tile of 128 queries sees, and those that all queries together see
  const int64_t w = (int64_t)a.window + a.sinks, keys = w + 128 < a.Nk ? w + 128 : a.Nk, span = w + a.Nq < a.Nk ? w + a.Nq : a.Nk;
  const int64_t blocks = step_blocks(dtype, slide_step(a));
  if (dtype == CAPK_BF16) return keys >= 2048 && blocks * 64 <= keys && blocks * span <= 128 * keys;
  return keys >= 512 && blocks * 3 <= keys && blocks * span <= 384 * keys;
}

extern "C" size_t capk_sliding_attention_fwd_workspace(int dtype, int B, int H, int Hk, int Nq, int Nk, int hd,
                                                       int window, int sinks) {
  if (!slide_sizes(B, H, Hk, Nq, Nk, hd, window, sinks)) return 0;
  const SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, 0.f, window, sinks, nullptr, nullptr);
  int splits;
  return slide_few(dtype, a) ? step_workspace(dtype, slide_step(a), &splits) : 0;
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
  int rc = slide_check("capk_sliding_attention_fwd", dtype, B, H, Hk, Nq, Nk, hd, window, sinks, scale, vs, 4);
  if (rc) return rc;
  SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, scale, window, sinks, key_pad, kv_len);
  a.q = vs[0]; a.k = vs[1]; a.v = vs[2]; a.o = vs[3]; a.lse = lse;
  if (slide_few(dtype, a)) return step_launch(dtype, slide_step(a), ws, ws_bytes, S(stream));
  const int hdp = slide_hdp(hd);
  const dim3 grid(cdiv(Nq, 128) * H * B);
  // up to one workgroup per CU: a second group of waves shares its tiles (117 to 82 us at 256 workgroups of
  // 66 tiles, heads of 128).  fp32: at 128 the second pair of images does not fit in LDS, at 96 (144 of 160 KiB) two
  // waves per SIMD leave 256 registers and the kernel spills 76
  const bool two = grid.x <= 256;
  SLIDE_HD(hdp, {
    constexpr int L16 = SlidePair<bf16, HDP>::LDS, L32 = SlidePair<float, HDP>::LDS, G32 = HDP <= 64 ? 2 : 1;
    if (dtype == CAPK_BF16)
      return two ? slide_launch(slide_fwd<bf16, HDP, 2>, grid, 2 * L16, S(stream), a, "slide_fwd", 512)
                 : slide_launch(slide_fwd<bf16, HDP, 1>, grid, L16, S(stream), a, "slide_fwd");
    return two && G32 == 2 ? slide_launch(slide_fwd<float, HDP, G32>, grid, G32 * L32, S(stream), a, "slide_fwd", 256 * G32)
                           : slide_launch(slide_fwd<float, HDP, 1>, grid, L32, S(stream), a, "slide_fwd");
  });
}

extern "C" size_t capk_sliding_attention_bwd_workspace(int B, int H, int Hk, int Nq, int Nk, int hd, int window,
                                                       int sinks) {
  if (!slide_sizes(B, H, Hk, Nq, Nk, hd, window, sinks)) return 0;
  SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, 0.f, window, sinks, nullptr, nullptr);
  slide_cut(a);
  const size_t delta = ((size_t)B * H * Nq * 4 + 15) / 16 * 16;
  return delta + (size_t)B * Hk * slide_parts(a) * 2 * kSlideKeys * hd * 4;
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
  int rc = slide_check("capk_sliding_attention_bwd", dtype, B, H, Hk, Nq, Nk, hd, window, sinks, scale, vs, 8);
  if (rc) return rc;
  const size_t need = capk_sliding_attention_bwd_workspace(B, H, Hk, Nq, Nk, hd, window, sinks);
  CAPK_CHECK_ARG(lse && ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0,
                 "capk_sliding_attention_bwd: need lse and a 16-B aligned workspace of %zu bytes", need);
  SlideArgs a = slide_args(B, H, Hk, Nq, Nk, hd, scale, window, sinks, key_pad, kv_len);
  slide_cut(a);
  a.q = vs[0]; a.k = vs[1]; a.v = vs[2]; a.o = vs[3]; a.dout = vs[4]; a.dq = vs[5]; a.dk = vs[6]; a.dv = vs[7];
  a.lse = (float*)lse;
  a.delta = (float*)ws;
  a.part = (float*)((char*)ws + ((size_t)B * H * Nq * 4 + 15) / 16 * 16);
  const int hdp = slide_hdp(hd), es = dtype == CAPK_BF16 ? 2 : 4;
  const dim3 gq(cdiv(Nq, 128) * H * B), gk((cdiv(Nk, kSlideKeys) * a.near_chunks + a.sink_tiles * a.far_chunks) * Hk * B);
  hipStream_t st = S(stream);
  const bool cut = a.near_chunks > 1;
  SLIDE_HD(hdp, {
    if (dtype == CAPK_BF16) {
      const size_t shm = SlidePair<bf16, HDP>::LDS;
      if ((rc = slide_launch(slide_dq<bf16, HDP>, gq, shm, st, a, "slide_dq"))) return rc;
      rc = cut ? slide_launch(slide_dkv<bf16, HDP, true>, gk, shm + 1024, st, a, "slide_dkv")
               : slide_launch(slide_dkv<bf16, HDP, false>, gk, shm + 1024, st, a, "slide_dkv");
    } else {
      const size_t shm = SlidePair<float, HDP>::LDS;
      if ((rc = slide_launch(slide_dq<float, HDP>, gq, shm, st, a, "slide_dq"))) return rc;
      rc = cut ? slide_launch(slide_dkv<float, HDP, true>, gk, shm + 1024, st, a, "slide_dkv")
               : slide_launch(slide_dkv<float, HDP, false>, gk, shm + 1024, st, a, "slide_dkv");
    }
    if (rc) return rc;
  });
  if (slide_parts(a)) {
    const int64_t n = a.near_chunks > 1 ? cdiv(Nk, kSlideKeys) : a.sink_tiles;
    const dim3 gs(cdiv((int64_t)kSlideKeys * hd / 4 * 2 * n, 256), Hk, B);
    if (es == 2) return slide_launch(slide_dkv_sum<bf16>, gs, 0, st, a, "slide_dkv_sum");
    return slide_launch(slide_dkv_sum<float>, gs, 0, st, a, "slide_dkv_sum");
  }
  return CAPK_OK;
}
