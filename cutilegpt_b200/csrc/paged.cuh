// The paged key/value cache as its kernels see it: where positions, rows and
// partial results are, shared by paged_append.cu, paged_simt.cu and paged.cu.
#pragma once

#include <float.h>

#include "common.cuh"

namespace gpt {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

// A score times the scale is subtracted from the reference point in one fused operation, which does not round the
// product, as the reference point was rounded: of a score of 2^b the two differ by up to 2^(b - 25), more than an exponential
// can hold from about 2^32 on. From this size on the few-row kernel rounds the product first; paged_tc.cu has a size of its own.
constexpr float kHugeScore = 1 << 20;
__device__ __forceinline__ float scaled(float s, float scale) { return __fmul_rn(s, scale); }   // in no fused operation

// What a launch of an attention kernel looks at.
//   kPrefix  the rows of all sequences of a group against the group's prefix
//   kOwn     the rows of one sequence against its own positions
//   kAll     the rows of one sequence against its prefix and then its own
// The rows of a sequence and key head are (t, head of the group): r = t * share + h;
// those of a group follow each other sequence by sequence.
enum Phase { kPrefix = 0, kOwn = 1, kAll = 2 };

// Division of 0 <= n < 2^31 by a number that the host knows: q = n m >> (31 + s) with s = ceil(log2 d),
// m = ceil(2^(31 + s) / d) < 2^32; m d exceeds 2^(31 + s) by less than 2^s, too little to change q. A few
// clocks, where a division by a variable is about a hundred, and a launch's first loads wait for several.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(int64_t div) : d((uint32_t)div), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> (31 + s)); }
  __device__ __forceinline__ int mod(int n) const { return n - div(n) * (int)d; }
};

struct Attn {
  const void* q;
  void* out;
  int64_t q_b, q_h, q_t, o_b, o_h, o_t;   // element strides
  const void* k;
  const void* v;
  int64_t page_stride, head_stride, slot_stride;
  int n_pages, page;
  const int32_t* table;
  int64_t ld_table;
  int cap;                  // own positions a table row can list
  const int32_t* seq_lens;
  const int32_t* ptable;
  int64_t ld_ptable;
  int pcap;
  const int32_t* plens;
  int B, T, H, K, share;    // share = H / K
  int per;                  // sequences of a group (B without groups)
  int D;
  FastDiv by_page, by_K, by_share, by_rows, by_per;   // by_rows: T * share, the rows of a sequence
  float scale_log2;
  // Partial results, slot by slot: acc [slot][row][D] (sum of 2^(s - m) v), ml [slot][row] (m, sum of
  // 2^(s - m)), row = (b * T + t) * H + h. Prefix parts are slots [0, n_pre), own parts n_pre ...
  float* acc;
  float2* ml;
  int n_pre, n_own;
};

// Row r of a phase's row space: sequence, token and head.
struct Row {
  int b, t, h;
  __device__ __forceinline__ Row(const Attn& p, int b0, int kh, int r) {
    const int i = p.by_rows.div(r), rr = r - i * (int)p.by_rows.d;
    t = p.by_share.div(rr);
    b = b0 + i;
    h = kh * p.share + rr - t * p.share;
  }
};

__device__ __forceinline__ int64_t row_id(const Attn& p, int b, int t, int h) {
  return ((int64_t)b * p.T + t) * p.H + h;
}

// A length from device memory, clamped to what its table row can list.
__device__ __forceinline__ int clamped_len(const int32_t* lens, int i, int cap) {
  const int n = lens[i];
  if (n < 0 || n > cap) {
    record_device_error(GPT_DEVERR_INDEX);
    return n < 0 ? 0 : cap;
  }
  return n;
}
__device__ __forceinline__ int own_len(const Attn& p, int b) { return clamped_len(p.seq_lens, b, p.cap); }
__device__ __forceinline__ int prefix_len(const Attn& p, int g) {
  return p.plens ? clamped_len(p.plens, g, p.pcap) : 0;
}

// Page id of a table entry, -1 (and the device error word) for one outside the pool.
__device__ __forceinline__ int page_id(int id, int n_pages) {
  if ((unsigned)id >= (unsigned)n_pages) {
    record_device_error(GPT_DEVERR_INDEX);
    return -1;
  }
  return id;
}

// The keys of a phase are positions 0 .. n_pre + n_own - 1: the prefix's first, then the own ones.
struct Keys {
  const int32_t* pre;
  const int32_t* own;
  int n_pre, n_own;
  __device__ Keys(const Attn& p, int phase, int seq_or_group) {
    const int b = phase == kPrefix ? seq_or_group * p.per : seq_or_group;
    const int g = phase == kPrefix ? seq_or_group : p.by_per.div(b);
    n_pre = phase == kOwn ? 0 : prefix_len(p, g);
    n_own = phase == kPrefix ? 0 : own_len(p, b);
    pre = p.ptable + (int64_t)g * p.ld_ptable;
    own = p.table + (int64_t)b * p.ld_table;
  }
  __device__ int n() const { return n_pre + n_own; }
  // element offset of position j's row of head `kh`, -1 for a page outside the pool
  __device__ int64_t offset(const Attn& p, int j, int kh) const {
    const bool own_part = j >= n_pre;
    const int i = own_part ? j - n_pre : j;
    const int at = p.by_page.div(i);
    const int id = page_id((own_part ? own : pre)[at], p.n_pages);
    return id < 0 ? -1 : id * p.page_stride + kh * p.head_stride + (int64_t)(i - at * p.page) * p.slot_stride;
  }
};

// A column's mean of values, acc times inv = 1 / l. The largest fp32 numbers come out of their split parts rounded
// up by 2^-24 (paged_rows.cu), past the range; a mean is never past it.
template <typename T>
__device__ __forceinline__ float mean(float acc, float inv) {
  const float x = acc * inv;
  return sizeof(T) == 4 && isinf(x) && !isinf(acc) ? copysignf(FLT_MAX, x) : x;
}

// ---- infinities and NaN in values that not every row of a tile sees -----------
// The tensor-core kernels give such a value the probability 0 for the rows that do not see it, and multiply:
// 0 x inf would reach outputs it has no part in. They look through the value tiles at the causal edge (T > 1 only)
// and, where one holds such a value, compute the CTA's rows again here, key by key.
template <typename T>
__device__ __forceinline__ bool non_finite(uint32_t w) {   // either bf16 of the pair, or the fp32
  if constexpr (sizeof(T) == 2)
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  else
    return (w & 0x7f800000u) == 0x7f800000u;
}
template <typename T>
__device__ __forceinline__ bool non_finite(uint4 v) {
  return non_finite<T>(v.x) || non_finite<T>(v.y) || non_finite<T>(v.z) || non_finite<T>(v.w);
}

// Row `q` against keys j0 .. j1 - 1 by one warp: m, l and acc (columns lane + 32 c), D <= 128.
template <typename T>
__device__ __noinline__ void slow_row(const Attn& p, const Keys keys, int kh, const T* q, int j0, int j1, int lane, float& m,
                                      float& l, float (&acc)[4]) {
  float x[4];
  m = -INFINITY;
  l = 0.f;
  for (int c = 0; c < 4; ++c) {
    x[c] = lane + 32 * c < p.D ? Tr<T>::to_f(q[lane + 32 * c]) : 0.f;
    acc[c] = 0.f;
  }
  for (int j = j0; j < j1; ++j) {
    const int64_t off = keys.offset(p, j, kh);
    float s = 0.f;
    for (int c = 0; c < 4; ++c)
      if (off >= 0 && lane + 32 * c < p.D) s = fmaf(x[c], Tr<T>::to_f(((const T*)p.k)[off + lane + 32 * c]), s);
    s = scaled(warp_sum(s), p.scale_log2);
    // a NaN score leaves m where it is, -inf at first: its exponential is NaN all the same
    const float to = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - to), e = s == -INFINITY ? 0.f : exp2f(s - to);
    m = to;
    l = l * a + e;
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < p.D) acc[c] = acc[c] * a + (off < 0 ? 0.f : e * Tr<T>::to_f(((const T*)p.v)[off + lane + 32 * c]));
  }
}

}  // namespace paged
}  // namespace gpt
