// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// p_i = softmax(target row i / T), q_i = softmax(draft row i / T), or a one-hot q_i at the drafted token
// where there are no draft logits.  Draft i is accepted while u_i q_i(x_i) < p_i(x_i); at the first
// refusal the next token is drawn from max(p_n - q_n, 0), after len acceptances from p_n, as the first
// token whose cumulative mass exceeds u_K times the whole (inverse CDF).  Sums and probabilities are
// held in 64 bits: over a vocabulary of 5e4 a 32-bit cumulative sum would put every hundredth draw
// on the wrong side of a border.
// Three launches: (maximum, sum of exp) of every row in chunks; acceptance and the mass of the row to draw
// from in chunks; the draw within its chunk.  (Drawing in the last workgroup of the second launch was
// slower, 27 for 10 us alone and 80 for 22 us at 64 sequences: its fences write the L2 back.)
// Bound: a 64-bit exp per logit, about 26 vector instructions, of which the first launch runs nine tenths of
// the time (25 us over 8 of 64 x 15 rows of 50257 bf16 logits in the mean, 2 TB/s; the second 13, the third 8; fp32 the
// same; without draft logits 15, 10 and 7).
#include "common.h"

namespace capk {

// logits per workgroup (chunk) = 256 RUN: 4096 where that gives workgroups for every CU, else 1024
template <int RUN> constexpr int ver_chunk() { return 256 * RUN; }
static int ver_run(int B, int K, int V) { return (int64_t)B * (2 * K + 1) * cdiv(V, 4096) >= 1024 ? 16 : 4; }

struct VerArgs {
  int B, K, V, chunks;
  int64_t t_bs, t_rs, d_bs, d_rs;
  const void *target, *draft;
  const int64_t* ids;
  int64_t ids_bs;
  const float* u;
  int64_t u_bs;
  const int32_t* draft_len;
  double scale64;  // 64 log2(e) / T
  int32_t* accepted;
  int64_t* tokens;
  int64_t tok_bs;
  double *zs, *rest;  // [B][2K + 1][chunks] sums, [B][chunks][2] masses (residual, target)
  float *ms, *lx;     // [B][2K + 1][chunks] maxima, [B][2K + 1] each row's logit of its drafted token
  struct VerPick* pick;  // [B]
};

__device__ __forceinline__ int ver_len(const VerArgs& a, int b) {
  return a.draft_len ? min(max(a.draft_len[b], 0), a.K) : a.K;
}
// row i of sequence b: the K + 1 target rows, then the K draft rows
template <typename T> __device__ __forceinline__ const T* ver_row(const VerArgs& a, int b, int i) {
  return i <= a.K ? (const T*)a.target + b * a.t_bs + i * a.t_rs : (const T*)a.draft + b * a.d_bs + (i - a.K - 1) * a.d_rs;
}
// e^((x - m) / T) in 64 bits: with t = 64 log2(e) (x - m) / T = 64 e + j + f, 2^e times 2^(j / 64) from a
// table times the series of 2^(f / 64), |f| <= 1/2, whose fifth term is below 4e-14.  (A series for
// |f| <= 1/2 of a whole octave takes eleven terms: 36 us over 64 x 8 rows of 50257.)  x - m is exact
// enough at any size of either, so t is too, however small T; below 2^-3000 there is no mass, nor has
// -inf, NaN or a row whose m is -inf.
__device__ const double kVerPow[64] = {  // 2^(j / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};
struct VerTable {
  double at[64];
  // requested before a kernel's own loads, stored once those are on their way; a barrier has to follow
  __device__ __forceinline__ static double load() { return kVerPow[threadIdx.x & 63]; }
  __device__ __forceinline__ void store(double x) { if (threadIdx.x < 64) at[threadIdx.x] = x; }
};
struct VerExp {
  double scale, top;  // 64 log2(e) / T, m
  const VerTable& tab;
  __device__ __forceinline__ VerExp(const VerArgs& a, const VerTable& tb, float m)
      : scale(a.scale64), top(m == -INFINITY ? INFINITY : (double)m), tab(tb) {}
  __device__ __forceinline__ double operator()(float x) const {
    constexpr double round = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to whole numbers, in the low bits
    const double t = fmax(((double)x - top) * scale, -64 * 3000.0), u = t + round, f = t - (u - round);
    const int i = __double2loint(u);
    constexpr double c1 = 0.69314718055994530942 / 64, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
    return __builtin_ldexp(fma(f, fma(f, fma(f, fma(f, c4, c3), c2), c1), 1.0) * tab.at[i & 63], i >> 6);
  }
};

__device__ __forceinline__ double ver_block_sum(double v) {
  __shared__ double s[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}
// inclusive sum over the wave's lanes
__device__ __forceinline__ double ver_wave_scan(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  return v;
}

// Chunks are cut at 16-B (8-B) borders of memory, as a row of an odd vocabulary starts anywhere: chunk c
// holds the elements from head + c * chunk on, chunk 0 also those before; every thread takes whole vectors.
template <typename T, int RUN>
__global__ __launch_bounds__(256) void verify_rows(VerArgs a) {
  constexpr int PER = RUN * (int)sizeof(T) < 16 ? RUN : 16 / (int)sizeof(T), NV = RUN / PER, AL = PER * (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(PER)));
  __shared__ float sm[4];
  __shared__ VerTable tab;
  const int rows = a.draft ? 2 * a.K + 1 : a.K + 1, b = blockIdx.y / rows, i = blockIdx.y % rows, c = blockIdx.x;
  const int len = ver_len(a, b);
  if (i <= a.K ? i > len : i - a.K - 1 >= len) return;  // never asked for
  const double pow = VerTable::load();
  const T* x = ver_row<T>(a, b, i);
  const int head = min(a.V, (int)((AL - ((uintptr_t)x & (AL - 1))) & (AL - 1)) / (int)sizeof(T));
  const int v0 = head + c * ver_chunk<RUN>();
  float r[RUN], first = -INFINITY, m = -INFINITY;
  if (c == 0 && (int)threadIdx.x < head) m = first = to_f32(x[threadIdx.x]);
  if (v0 + ver_chunk<RUN>() <= a.V) {
    vec y[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) y[k] = *(const vec*)(x + v0 + (k * 256 + threadIdx.x) * PER);
    tab.store(pow);
#pragma unroll
    for (int k = 0; k < RUN; ++k) r[k] = (float)y[k / PER][k % PER];
  } else {
    tab.store(pow);
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const int v = v0 + (k / PER * 256 + (int)threadIdx.x) * PER + k % PER;
      const float z = to_f32(x[min(v, a.V - 1)]);
      r[k] = v < a.V ? z : -INFINITY;
    }
  }
#pragma unroll
  for (int k = 0; k < RUN; ++k) m = fmaxf(m, r[k]);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const VerExp mass(a, tab, m);
  double z = head && c == 0 ? mass(first) : 0.0;
#pragma unroll
  for (int k = 0; k < RUN; ++k) z += mass(r[k]);
  z = ver_block_sum(z);
  if (threadIdx.x == 0) {
    const int64_t at = ((int64_t)b * (2 * a.K + 1) + i) * a.chunks + c;
    a.ms[at] = m;
    a.zs[at] = z;
  }
  if (c == 0 && threadIdx.x == 255 && i != a.K) {
    const int64_t id = a.ids[b * a.ids_bs + (i < a.K ? i : i - a.K - 1)];
    a.lx[(int64_t)b * (2 * a.K + 1) + i] = id >= 0 && id < a.V ? to_f32(x[id]) : -INFINITY;
  }
}

struct VerPick {
  int n, len;
  float mp, mq;
  double zp, zq;  // reciprocals of the sums
  int64_t id;
};
// How many drafts are accepted, and the statistics of the row to draw from (whole workgroup).  What it
// reads does not depend on what it reads and is requested at once (of the drafts past 256, later), so it
// pays memory's latency once.  Fills the table.
struct VerDraft {
  float xp, xq, u;
  int64_t id;
  __device__ __forceinline__ void load(const VerArgs& a, int b, int i) {
    const float* lx = a.lx + (int64_t)b * (2 * a.K + 1);
    xp = lx[i];
    xq = a.draft ? lx[a.K + 1 + i] : 0.f;
    id = a.ids[b * a.ids_bs + i];
    u = a.u[b * a.u_bs + i];
  }
};
struct VerStats {  // lane l of a row's 16: chunks l, l + 16, .. of the first 64
  float m[4];
  double z[4];
  __device__ __forceinline__ void load(const VerArgs& a, int64_t at, int l) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = l + 16 * k, cc = min(c, a.chunks - 1);
      m[k] = a.ms[at + cc];
      z[k] = a.zs[at + cc];
      if (c >= a.chunks) m[k] = -INFINITY, z[k] = 0.0;
    }
  }
};
__device__ __forceinline__ VerPick ver_pick(const VerArgs& a, VerTable& tab, int b, double* zs, float* ms) {
  __shared__ int first;
  VerPick p;
  const double pow = VerTable::load();
  p.len = ver_len(a, b);
  const int rows = a.draft ? 2 * a.K + 1 : a.K + 1, l = threadIdx.x & 15;
  const int64_t at0 = (int64_t)b * (2 * a.K + 1) * a.chunks;
  VerDraft mine{};
  if (a.K > 0) mine.load(a, b, min((int)threadIdx.x, a.K - 1));
  VerStats st;
  st.load(a, at0 + (int64_t)min((int)threadIdx.x >> 4, rows - 1) * a.chunks, l);
  tab.store(pow);
  if (threadIdx.x == 0) first = p.len;
  __syncthreads();
  for (int i = threadIdx.x >> 4; i < rows; i += 16) {  // 16 lanes per row
    const int64_t at = at0 + (int64_t)i * a.chunks;
    if (i >= 16) st.load(a, at, l);
    float m = fmaxf(fmaxf(st.m[0], st.m[1]), fmaxf(st.m[2], st.m[3]));
    for (int c = l + 64; c < a.chunks; c += 16) m = fmaxf(m, a.ms[at + c]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 16));
    const VerExp mass(a, tab, m);
    double z = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) z += st.z[k] * mass(st.m[k]);
    for (int c = l + 64; c < a.chunks; c += 16) z += a.zs[at + c] * mass(a.ms[at + c]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) z += __shfl_xor(z, o, 16);
    if (l == 0) { ms[i] = m; zs[i] = z; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.len; i += 256) {
    if (i >= 256) mine.load(a, b, i);
    const double q = a.draft ? VerExp(a, tab, ms[a.K + 1 + i])(mine.xq) / zs[a.K + 1 + i] : 1.0;
    // the smallest refused index: the same in every order
    if (mine.id < 0 || mine.id >= a.V || !(mine.u * q < VerExp(a, tab, ms[i])(mine.xp) / zs[i])) atomicMin(&first, i);
  }
  __syncthreads();
  p.n = first;
  p.id = p.n < p.len ? a.ids[b * a.ids_bs + p.n] : -1;
  p.mp = ms[p.n];
  p.zp = 1.0 / zs[p.n];
  p.mq = -INFINITY;
  p.zq = 0.0;
  if (p.n < p.len && a.draft) {
    p.mq = ms[a.K + 1 + p.n];
    p.zq = 1.0 / zs[a.K + 1 + p.n];
  }
  return p;
}
// masses of token v: the residual where a draft was refused (else the target's), and the target's
struct VerMass {
  VerExp ep, eq;
  const VerPick& p;
  bool soft;  // the draft has probabilities of its own
  __device__ __forceinline__ VerMass(const VerArgs& a, const VerTable& tab, const VerPick& pk)
      : ep(a, tab, pk.mp), eq(a, tab, pk.mq), p(pk), soft(a.draft != nullptr) {}
  __device__ __forceinline__ double operator()(float t, float d, int v, double& whole) const {
    whole = ep(t) * p.zp;
    if (p.n >= p.len) return whole;
    return fmax(whole - (soft ? eq(d) * p.zq : v == p.id ? 1.0 : 0.0), 0.0);
  }
};

template <typename T, int RUN>
__global__ __launch_bounds__(256) void verify_mass(VerArgs a) {
  __shared__ VerTable tab;
  extern __shared__ double zs[];  // [rows] sums, [rows] maxima
  const int b = blockIdx.y, v0 = blockIdx.x * ver_chunk<RUN>();
  const VerPick p = ver_pick(a, tab, b, zs, (float*)(zs + 2 * a.K + 1));
  if (blockIdx.x == 0 && threadIdx.x == 0) a.pick[b] = p;
  const bool two = a.draft && p.n < p.len;
  const T *tr = ver_row<T>(a, b, p.n), *dr = two ? ver_row<T>(a, b, a.K + 1 + p.n) : tr;
  const VerMass mass(a, tab, p);
  T t[RUN], d[RUN];  // (loads without a condition: behind one each would be waited for)
#pragma unroll
  for (int k = 0; k < RUN; ++k) {
    const int v = min(v0 + k * 256 + (int)threadIdx.x, a.V - 1);
    t[k] = tr[v];
    d[k] = dr[v];
  }
  double r = 0.0, w = 0.0;
#pragma unroll
  for (int k = 0; k < RUN; ++k) {
    const int v = v0 + k * 256 + threadIdx.x;
    double y;
    const double x = mass(v < a.V ? to_f32(t[k]) : -INFINITY, to_f32(d[k]), v, y);
    r += x;
    w += y;
  }
  r = ver_block_sum(r);
  w = ver_block_sum(w);
  if (threadIdx.x == 0) {
    double* rest = a.rest + ((int64_t)b * a.chunks + blockIdx.x) * 2;
    rest[0] = r;
    rest[1] = w;
  }
}

template <typename T, int RUN>
__global__ __launch_bounds__(1024) void verify_draw(VerArgs a) {
  constexpr int PER = ver_chunk<RUN>() / 1024;  // tokens per thread
  __shared__ VerTable tab;
  __shared__ int best, last;
  __shared__ double ws[16];
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const double pow = VerTable::load();
  const VerPick p = a.pick[b];
  const double u = a.u[b * a.u_bs + a.K];
  const int64_t my_id = (int)threadIdx.x < a.K ? a.ids[b * a.ids_bs + threadIdx.x] : -1;  // (K <= 1024)
  const double* rest = a.rest + (int64_t)b * a.chunks * 2;
  if (threadIdx.x == 0) best = 0x7fffffff, last = 0;
  // every wave for itself: the whole mass, then the chunk whose cumulative mass first exceeds u times it
  // (rounding can leave none: the last with mass)
  double r = 0.0, t = 0.0;
  for (int c = lane; c < a.chunks; c += 64) { r += rest[2 * c]; t += rest[2 * c + 1]; }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { r += __shfl_xor(r, o, 64); t += __shfl_xor(t, o, 64); }
  // a refused draft equal to its target leaves no residual: draw from the target
  const bool whole = !(r > 0.0);
  const double goal = u * (whole ? t : r);
  int pick = 0;
  double before = 0.0, carry = 0.0;
  for (int c0 = 0; c0 < a.chunks; c0 += 64) {
    const double x = c0 + lane < a.chunks ? rest[2 * (c0 + lane) + whole] : 0.0;
    const double at = carry + ver_wave_scan(x);
    const uint64_t has = __builtin_amdgcn_ballot_w64(x > 0.0), past = __builtin_amdgcn_ballot_w64(x > 0.0 && at > goal);
    if (has) {
      const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(has);
      pick = c0 + l;
      before = __shfl(at - x, l, 64);
    }
    if (past) break;
    carry = __shfl(at, 63, 64);
  }
  // the same within the chunk
  const T *tr = ver_row<T>(a, b, p.n), *dr = a.draft && p.n < p.len ? ver_row<T>(a, b, a.K + 1 + p.n) : tr;
  const int v0 = pick * ver_chunk<RUN>() + threadIdx.x * PER;
  T xt[PER], xd[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int v = min(v0 + k, a.V - 1);
    xt[k] = tr[v];
    xd[k] = dr[v];
  }
  tab.store(pow);
  __syncthreads();
  const VerMass mass(a, tab, p);
  double run[PER], mine = 0.0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    double y;
    run[k] = mass(v0 + k < a.V ? to_f32(xt[k]) : -INFINITY, to_f32(xd[k]), v0 + k, y);
    if (whole) run[k] = y;
    mine += run[k];
  }
  const double scan = ver_wave_scan(mine);
  if (lane == 63) ws[w] = scan;
  __syncthreads();
  double at = before + scan - mine;
  for (int i = 0; i < w; ++i) at += ws[i];
  int found = 0x7fffffff, some = -1;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    at += run[k];
    if (run[k] > 0.0) some = v0 + k;
    if (run[k] > 0.0 && at > goal && found == 0x7fffffff) found = v0 + k;
  }
  // the first of a wave is its first lane's; the last, its last lane's
  const uint64_t hit = __builtin_amdgcn_ballot_w64(found != 0x7fffffff), has = __builtin_amdgcn_ballot_w64(some >= 0);
  if (hit && lane == __builtin_ctzll(hit)) atomicMin(&best, found);
  if (has && lane == 63 - __builtin_clzll(has)) atomicMax(&last, some);
  __syncthreads();
  const int token = best != 0x7fffffff ? best : last;  // (0 where the row has no mass at all)
  if (threadIdx.x == 0) a.accepted[b] = p.n;
  for (int i = threadIdx.x; i <= a.K; i += 1024) a.tokens[b * a.tok_bs + i] = i < p.n ? my_id : i == p.n ? (int64_t)token : -1;
}

template <typename T, int RUN>
static int verify_go(const VerArgs& a, hipStream_t st) {
  const int rows = a.draft ? 2 * a.K + 1 : a.K + 1;
  hipLaunchKernelGGL((verify_rows<T, RUN>), dim3(a.chunks, a.B * rows), dim3(256), 0, st, a);
  CAPK_LAUNCH_CHECK("verify_rows");
  hipLaunchKernelGGL((verify_mass<T, RUN>), dim3(a.chunks, a.B), dim3(256), (size_t)(2 * a.K + 1) * 12, st, a);
  CAPK_LAUNCH_CHECK("verify_mass");
  hipLaunchKernelGGL((verify_draw<T, RUN>), dim3(a.B), dim3(1024), 0, st, a);
  CAPK_LAUNCH_CHECK("verify_draw");
  return CAPK_OK;
}

}  // namespace capk

using namespace capk;

extern "C" size_t capk_verify_drafts_workspace(int B, int K, int V) {
  if (B < 1 || K < 0 || V < 1) return 0;
  const size_t c = cdiv(V, 256 * ver_run(B, K, V)), rows = (size_t)B * (2 * (size_t)K + 1) * c;
  return rows * 8 + (size_t)B * c * 16 + (size_t)B * sizeof(VerPick) + rows * 4 + (size_t)B * (2 * (size_t)K + 1) * 4;
}

extern "C" int capk_verify_drafts(int dtype, int B, int K, int V, const void* target, int64_t t_bs, int64_t t_rs,
                                  const void* draft, int64_t d_bs, int64_t d_rs, const int64_t* ids, int64_t ids_bs,
                                  const float* u, int64_t u_bs, const int32_t* draft_len, double temperature,
                                  int32_t* accepted, int64_t* tokens, int64_t tok_bs, void* ws, size_t ws_bytes,
                                  void* stream) {
  CAPK_CHECK_ARG(dtype == CAPK_F32 || dtype == CAPK_BF16, "capk_verify_drafts: dtype");
  CAPK_CHECK_ARG(B >= 0 && K >= 0 && K <= 1024 && V >= 1 && (int64_t)B * (2 * K + 1) <= 65535 && V <= (1 << 28),
                 "capk_verify_drafts: need 0 <= K <= 1024, V >= 1 and B (2 K + 1) <= 65535 (B %d, K %d, V %d)", B, K, V);
  CAPK_CHECK_ARG(temperature >= 1e-300 && temperature < (double)INFINITY, "capk_verify_drafts: temperature must be positive");
  if (B == 0) return CAPK_OK;
  CAPK_CHECK_ARG(target && (K == 0 || ids) && u && accepted && tokens, "capk_verify_drafts: null pointer");
  const size_t need = capk_verify_drafts_workspace(B, K, V);
  CAPK_CHECK_ARG(ws && ws_bytes >= need && (uintptr_t)ws % 8 == 0,
                 "capk_verify_drafts: needs an 8-B aligned workspace of %zu bytes", need);
  VerArgs a{};
  a.B = B; a.K = K; a.V = V; a.chunks = cdiv(V, 256 * ver_run(B, K, V));
  a.target = target; a.t_bs = t_bs; a.t_rs = t_rs;
  a.draft = K ? draft : nullptr; a.d_bs = d_bs; a.d_rs = d_rs;
  a.ids = ids; a.ids_bs = ids_bs; a.u = u; a.u_bs = u_bs; a.draft_len = draft_len;
  a.scale64 = 64 * 1.4426950408889634074 / temperature;
  a.accepted = accepted; a.tokens = tokens; a.tok_bs = tok_bs;
  const size_t rows = (size_t)B * (2 * (size_t)K + 1) * a.chunks;
  a.zs = (double*)ws;
  a.rest = a.zs + rows;
  a.pick = (VerPick*)(a.rest + (size_t)B * a.chunks * 2);
  a.ms = (float*)(a.pick + B);
  a.lx = a.ms + rows;
  if (ver_run(B, K, V) == 16) return dtype == CAPK_BF16 ? verify_go<bf16, 16>(a, S(stream)) : verify_go<float, 16>(a, S(stream));
  return dtype == CAPK_BF16 ? verify_go<bf16, 4>(a, S(stream)) : verify_go<float, 4>(a, S(stream));
}
