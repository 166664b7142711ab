// Views, key tiles and dispatch shared by sliding.hip (many queries) and stepattn.hip (few queries).
#pragma once
#include "tiles.h"

namespace capk {

struct SlideView {
  void* p;
  int64_t bs, rs, hs;
};
template <typename T>
__device__ __forceinline__ T* row(const SlideView& v, int b, int n, int h) {
  return (T*)v.p + b * v.bs + n * v.rs + h * v.hs;
}

// The key tiles (KT keys each) that queries at positions p_lo..p_hi see: those with sinks, then the window's.
template <int KT> struct SlideTiles {
  int ns, w0, n;
  __device__ __forceinline__ SlideTiles(int window, int sinks, int p_lo, int p_hi, int len) {
    const int last = min(p_hi + 1, len);  // keys [0, last)
    ns = w0 = n = 0;
    if (last <= 0) return;
    const int end = (last + KT - 1) / KT;
    ns = min((min(sinks, last) + KT - 1) / KT, end);
    w0 = max(ns, max(0, p_lo - window + 1) / KT);
    n = ns + max(0, end - w0);
  }
  __device__ __forceinline__ int key0(int i) const { return (i < ns ? i : w0 + i - ns) * KT; }
};

inline int slide_hdp(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : 128; }

#define SLIDE_HD(hdp, ...)                                     \
  switch (hdp) {                                               \
    case 32: { constexpr int HDP = 32; __VA_ARGS__; break; }   \
    case 64: { constexpr int HDP = 64; __VA_ARGS__; break; }   \
    case 96: { constexpr int HDP = 96; __VA_ARGS__; break; }   \
    default: { constexpr int HDP = 128; __VA_ARGS__; break; }  \
  }

// the power of two that an E8M0 scale code of the 4-bit cache stands for (255: NaN)
__device__ __forceinline__ float kv4_scale(uint32_t code) {
  return code == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(code << 23);
}

// Attention of few queries over a dense cache or over 4-bit pages (stepattn.hip).
struct StepArgs {
  int B, H, Hk, Nq, cap, hd, window, sinks;  // cap: no sequence holds more keys
  float scale;
  SlideView q, o;
  const int32_t* len;  // [B], nullptr: cap
  float* lse;          // [B, H, Nq], optional
  // dense: key / value rows, hidden keys
  SlideView k, v;
  const uint8_t* pad;
  // 4-bit pages: codes [pages][2][Hk][page][hd / 2], scales [pages][2][Hk][page][hd / 32]
  const uint8_t *codes, *scales;
  const int32_t* table;  // [B][table_ld] page of every `page` tokens
  int64_t table_ld;
  int pages, page;
  // partial results of the splits of the key axis: [B H Nq][splits][hd] sums, [B H Nq][splits] max and sum
  float *po, *pml;
  int splits;
};
// workgroups without a split of the keys, bytes of partial results (0: the keys are not split), and the launch
int64_t step_blocks(int dtype, const StepArgs& a);
size_t step_workspace(int dtype, const StepArgs& a, int* splits);
int step_launch(int dtype, StepArgs a, void* ws, size_t ws_bytes, hipStream_t st);

}  // namespace capk
