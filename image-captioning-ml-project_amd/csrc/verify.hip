// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// p_i = softmax(target row i / T), q_i = softmax(draft row i / T), or a one-hot q_i at the drafted token
// where there are no draft logits.  Draft i is accepted while u_i q_i(x_i) < p_i(x_i); at the first
// refusal the next token is drawn from max(p_n - q_n, 0), after len acceptances from p_n, as the first
// token whose cumulative mass exceeds u_K times the whole (inverse CDF).  Sums and probabilities are
// held in 64 bits: over a vocabulary of 5e4 a 32-bit cumulative sum would put every hundredth draw
// on the wrong side of a border.
// Three launches: (maximum, sum of exp) of every row in chunks; acceptance and the residual's mass in
// chunks; the draw within its chunk.  Bound: HBM (each logit once, and the chosen rows again) beside a
// 64-bit exp per logit.
#include "common.h"

namespace capk {

constexpr int kVerChunk = 4096, kVerRun = kVerChunk / 256;  // logits per workgroup, per thread

struct VerArgs {
  int B, K, V, chunks;
  int64_t t_bs, t_rs, d_bs, d_rs;
  const void *target, *draft;
  const int64_t* ids;
  int64_t ids_bs;
  const float* u;
  int64_t u_bs;
  const int32_t* draft_len;
  double inv_t;
  int32_t* accepted;
  int64_t* tokens;
  int64_t tok_bs;
  double *zs, *rest;  // [B][2K + 1][chunks] sums, [B][chunks][2] masses (residual, target)
  float* ms;          // [B][2K + 1][chunks] maxima
};

__device__ __forceinline__ int ver_len(const VerArgs& a, int b) {
  return a.draft_len ? min(max(a.draft_len[b], 0), a.K) : a.K;
}
// row i of sequence b: the K + 1 target rows, then the K draft rows
template <typename T> __device__ __forceinline__ const T* ver_row(const VerArgs& a, int b, int i) {
  return i <= a.K ? (const T*)a.target + b * a.t_bs + i * a.t_rs : (const T*)a.draft + b * a.d_bs + (i - a.K - 1) * a.d_rs;
}
__device__ __forceinline__ double ver_exp(const VerArgs& a, float x, float m) {
  return m == -INFINITY ? 0.0 : exp(((double)x - (double)m) * a.inv_t);
}

__device__ __forceinline__ double ver_wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double ver_block_sum(double v) {
  __shared__ double s[4];
  v = ver_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <typename T>
__global__ __launch_bounds__(256) void verify_rows(VerArgs a) {
  __shared__ float sm[4];
  const int rows = a.draft ? 2 * a.K + 1 : a.K + 1, b = blockIdx.y / rows, i = blockIdx.y % rows, c = blockIdx.x;
  const int len = ver_len(a, b);
  if (i <= a.K ? i > len : i - a.K - 1 >= len) return;  // never asked for
  const T* x = ver_row<T>(a, b, i);
  const int v0 = c * kVerChunk;
  float r[kVerRun], m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kVerRun; ++k) {
    const int v = v0 + k * 256 + threadIdx.x;
    r[k] = v < a.V ? to_f32(x[v]) : -INFINITY;
    m = fmaxf(m, r[k]);
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  double z = 0.0;
#pragma unroll
  for (int k = 0; k < kVerRun; ++k) z += ver_exp(a, r[k], m);
  z = ver_block_sum(z);
  if (threadIdx.x == 0) {
    const int64_t at = ((int64_t)b * (2 * a.K + 1) + i) * a.chunks + c;
    a.ms[at] = m;
    a.zs[at] = z;
  }
}

// maximum and whole sum of row i from its chunks
__device__ __forceinline__ void ver_stats(const VerArgs& a, int b, int i, float& m, double& z) {
  const int64_t at = ((int64_t)b * (2 * a.K + 1) + i) * a.chunks;
  m = -INFINITY;
  for (int c = 0; c < a.chunks; ++c) m = fmaxf(m, a.ms[at + c]);
  z = 0.0;
  for (int c = 0; c < a.chunks; ++c) z += a.zs[at + c] * ver_exp(a, a.ms[at + c], m);
}

struct VerPick {
  int n, len;
  float mp, mq;
  double zp, zq;
  int64_t id;
};
// How many drafts are accepted, and the statistics of the row to draw from (whole workgroup).
template <typename T>
__device__ __forceinline__ VerPick ver_pick(const VerArgs& a, int b) {
  __shared__ int first;
  VerPick p;
  p.len = ver_len(a, b);
  if (threadIdx.x == 0) first = p.len;
  __syncthreads();
  for (int i = threadIdx.x; i < p.len; i += 256) {
    const int64_t id = a.ids[b * a.ids_bs + i];
    bool ok = id >= 0 && id < a.V;
    if (ok) {
      float m;
      double z, q = 1.0;
      ver_stats(a, b, i, m, z);
      const double pr = ver_exp(a, to_f32(ver_row<T>(a, b, i)[id]), m) / z;
      if (a.draft) {
        ver_stats(a, b, a.K + 1 + i, m, z);
        q = ver_exp(a, to_f32(ver_row<T>(a, b, a.K + 1 + i)[id]), m) / z;
      }
      ok = (double)a.u[b * a.u_bs + i] * q < pr;
    }
    if (!ok) atomicMin(&first, i);  // the smallest refused index: the same in every order
  }
  __syncthreads();
  p.n = first;
  p.id = p.n < p.len ? a.ids[b * a.ids_bs + p.n] : -1;
  ver_stats(a, b, p.n, p.mp, p.zp);
  p.mq = -INFINITY;
  p.zq = 1.0;
  if (p.n < p.len && a.draft) ver_stats(a, b, a.K + 1 + p.n, p.mq, p.zq);
  return p;
}
// mass of token v: the residual where a draft was refused, else (or with `whole`) the target's
template <typename T>
__device__ __forceinline__ double ver_mass(const VerArgs& a, const VerPick& p, const T* tr, const T* dr, int v, bool whole) {
  const double pv = ver_exp(a, to_f32(tr[v]), p.mp) / p.zp;
  if (whole || p.n >= p.len) return pv;
  const double qv = dr ? ver_exp(a, to_f32(dr[v]), p.mq) / p.zq : (v == p.id ? 1.0 : 0.0);
  return fmax(pv - qv, 0.0);
}

template <typename T>
__global__ __launch_bounds__(256) void verify_mass(VerArgs a) {
  const int b = blockIdx.y, c = blockIdx.x, v0 = c * kVerChunk;
  const VerPick p = ver_pick<T>(a, b);
  const T *tr = ver_row<T>(a, b, p.n), *dr = a.draft && p.n < p.len ? ver_row<T>(a, b, a.K + 1 + p.n) : nullptr;
  double r = 0.0, w = 0.0;
#pragma unroll 4
  for (int k = 0; k < kVerRun; ++k) {
    const int v = v0 + k * 256 + threadIdx.x;
    if (v < a.V) {
      r += ver_mass(a, p, tr, dr, v, false);
      w += ver_mass(a, p, tr, dr, v, true);
    }
  }
  r = ver_block_sum(r);
  w = ver_block_sum(w);
  if (threadIdx.x == 0) {
    a.rest[((int64_t)b * a.chunks + c) * 2] = r;
    a.rest[((int64_t)b * a.chunks + c) * 2 + 1] = w;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void verify_draw(VerArgs a) {
  __shared__ double ws[4];
  __shared__ int best;
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const VerPick p = ver_pick<T>(a, b);
  const T *tr = ver_row<T>(a, b, p.n), *dr = a.draft && p.n < p.len ? ver_row<T>(a, b, a.K + 1 + p.n) : nullptr;
  const double* rest = a.rest + (int64_t)b * a.chunks * 2;
  double all = 0.0;
  for (int c = 0; c < a.chunks; ++c) all += rest[2 * c];
  const bool whole = !(all > 0.0);  // a refused draft equal to its target leaves no residual: draw from the target
  if (whole) {
    all = 0.0;
    for (int c = 0; c < a.chunks; ++c) all += rest[2 * c + 1];
  }
  const double goal = (double)a.u[b * a.u_bs + a.K] * all;
  // the chunk whose cumulative mass first exceeds the goal; rounding can leave none: the last with mass
  int pick = -1, last = 0;
  double before = 0.0, sum = 0.0, last_before = 0.0;
  for (int c = 0; c < a.chunks && pick < 0; ++c) {
    const double x = rest[2 * c + whole];
    if (x > 0.0) { last = c; last_before = sum; }
    if (sum + x > goal) { pick = c; before = sum; }
    sum += x;
  }
  if (pick < 0) { pick = last; before = last_before; }
  const int v0 = pick * kVerChunk + threadIdx.x * kVerRun;  // kVerRun tokens in a row per thread
  double run[kVerRun], mine = 0.0;
#pragma unroll
  for (int k = 0; k < kVerRun; ++k) {
    run[k] = v0 + k < a.V ? ver_mass(a, p, tr, dr, v0 + k, whole) : 0.0;
    mine += run[k];
  }
  double scan = mine;  // inclusive over the wave's lanes
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(scan, o, 64);
    if (lane >= o) scan += y;
  }
  if (threadIdx.x == 0) best = 0x7fffffff;
  if (lane == 63) ws[threadIdx.x >> 6] = scan;
  __syncthreads();
  double at = before + scan - mine;
  for (int u = 0; u < (int)(threadIdx.x >> 6); ++u) at += ws[u];
  int found = 0x7fffffff, some = -1;
#pragma unroll
  for (int k = kVerRun - 1; k >= 0; --k)
    if (run[k] > 0.0 && some < 0) some = v0 + k;  // this thread's last token with mass
#pragma unroll
  for (int k = 0; k < kVerRun; ++k) {
    at += run[k];
    if (run[k] > 0.0 && at > goal && found == 0x7fffffff) found = v0 + k;
  }
  if (found != 0x7fffffff) atomicMin(&best, found);
  __syncthreads();
  const bool none = best == 0x7fffffff;
  __syncthreads();
  if (none) {  // rounding at the chunk's end: its last token with mass (0 where the row has no mass at all)
    if (threadIdx.x == 0) best = 0;
    __syncthreads();
    if (some >= 0) atomicMax(&best, some);
    __syncthreads();
  }
  if (threadIdx.x == 0) a.accepted[b] = p.n;
  for (int i = threadIdx.x; i <= a.K; i += 256)
    a.tokens[b * a.tok_bs + i] = i < p.n ? a.ids[b * a.ids_bs + i] : i == p.n ? (int64_t)best : -1;
}

template <typename T>
static int verify_go(const VerArgs& a, hipStream_t st) {
  const int rows = a.draft ? 2 * a.K + 1 : a.K + 1;
  hipLaunchKernelGGL(verify_rows<T>, dim3(a.chunks, a.B * rows), dim3(256), 0, st, a);
  CAPK_LAUNCH_CHECK("verify_rows");
  hipLaunchKernelGGL(verify_mass<T>, dim3(a.chunks, a.B), dim3(256), 0, st, a);
  CAPK_LAUNCH_CHECK("verify_mass");
  hipLaunchKernelGGL(verify_draw<T>, dim3(a.B), dim3(256), 0, st, a);
  CAPK_LAUNCH_CHECK("verify_draw");
  return CAPK_OK;
}

}  // namespace capk

using namespace capk;

extern "C" size_t capk_verify_drafts_workspace(int B, int K, int V) {
  if (B < 1 || K < 0 || V < 1) return 0;
  const size_t c = cdiv(V, kVerChunk), rows = (size_t)B * (2 * (size_t)K + 1) * c;
  return rows * 8 + (size_t)B * c * 16 + rows * 4;
}

extern "C" int capk_verify_drafts(int dtype, int B, int K, int V, const void* target, int64_t t_bs, int64_t t_rs,
                                  const void* draft, int64_t d_bs, int64_t d_rs, const int64_t* ids, int64_t ids_bs,
                                  const float* u, int64_t u_bs, const int32_t* draft_len, double temperature,
                                  int32_t* accepted, int64_t* tokens, int64_t tok_bs, void* ws, size_t ws_bytes,
                                  void* stream) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "capk_verify_drafts: dtype");
  CAPK_CHECK_ARG(B >= 0 && K >= 0 && K <= 1024 && V >= 1 && (int64_t)B * (2 * K + 1) <= 65535 && V <= (1 << 28),
                 "capk_verify_drafts: need 0 <= K <= 1024, V >= 1 and B (2 K + 1) <= 65535 (B %d, K %d, V %d)", B, K, V);
  CAPK_CHECK_ARG(temperature > 0.0 && temperature < (double)INFINITY, "capk_verify_drafts: temperature must be positive");
  if (B == 0) return CAPK_OK;
  CAPK_CHECK_ARG(target && (K == 0 || ids) && u && accepted && tokens, "capk_verify_drafts: null pointer");
  const size_t need = capk_verify_drafts_workspace(B, K, V);
  CAPK_CHECK_ARG(ws && ws_bytes >= need && (uintptr_t)ws % 8 == 0,
                 "capk_verify_drafts: needs an 8-B aligned workspace of %zu bytes", need);
  VerArgs a{};
  a.B = B; a.K = K; a.V = V; a.chunks = cdiv(V, kVerChunk);
  a.target = target; a.t_bs = t_bs; a.t_rs = t_rs;
  a.draft = K ? draft : nullptr; a.d_bs = d_bs; a.d_rs = d_rs;
  a.ids = ids; a.ids_bs = ids_bs; a.u = u; a.u_bs = u_bs; a.draft_len = draft_len;
  a.inv_t = 1.0 / temperature;
  a.accepted = accepted; a.tokens = tokens; a.tok_bs = tok_bs;
  const size_t rows = (size_t)B * (2 * (size_t)K + 1) * a.chunks;
  a.zs = (double*)ws;
  a.rest = a.zs + rows;
  a.ms = (float*)(a.rest + (size_t)B * a.chunks * 2);
  return dtype == CAPK_BF16 ? verify_go<bf16>(a, S(stream)) : verify_go<float>(a, S(stream));
}
