// New tokens into the paged key/value cache, their rotation on the way.
//
// A pair of values (x0, x1) of a query or key head at position n becomes
// (x0 c - x1 s, x0 s + x1 c) with c, s from the caller's fp32 table; values
// are copied. Everything is read once and written once, so the kernel is
// bound by HBM: 2 (2 K + H) D e bytes per token with rotation, 4 K D e without.
// B200: 8 prompts of 4093 tokens, 32 + 2 x 8 heads of 128 in bf16 (806 MB), 138.6 us = 5.8 TB/s, 0.89 of
// a measured copy; 5 x 1021 tokens, 3 x 25 heads of 64 in fp32, 33.1 us = 5.9 TB/s; a step of 256 sequences 3.1 us.
//
// One thread handles two vectors of V elements of one head (16 bytes each
// when sizes and alignment allow, single elements otherwise): for halves
// style rotation the vectors at j and j + rot/2, which hold both members of
// V pairs, else 2 V neighbouring elements. Heads of a token are numbered keys,
// values, then queries, so a launch without rotation just has fewer of them.
#include "paged.cuh"

namespace gpt {
namespace paged {

struct Append {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  int64_t q_s[3], k_s[3], v_s[3], o_s[3];   // element strides of (b, h, t)
  void* k_pages;
  void* v_pages;
  int64_t page_stride, head_stride, slot_stride;
  int n_pages, page;
  const int32_t* table;
  int64_t ld_table;
  int cap;
  const int32_t* seq_lens;
  const int32_t* plens;
  int pcap, per;
  const float* cos_sin;
  int64_t n_pos;
  int rot, interleaved;
  int T, K, D;
  int B;
  int total;     // threads with work for a sequence: tokens x heads x pairs of vectors of a head
  FastDiv by_heads, by_units, by_page;   // heads: 2 K, or 2 K + H with rotation
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// A vector that nobody reads again: evicted first, so that the pages and the queries written stay in L2.
template <typename W>
__device__ __forceinline__ W load_once(const void* p) {
  if constexpr (sizeof(W) == 16) {
    const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const W*>(&x);
  } else {
    return *reinterpret_cast<const W*>(p);
  }
}

// One thread's share of sequence b: N pairs of vectors of one head, `units` / N pairs apart, so that their
// lookups and addresses are computed once.
template <typename T, int V, int N>
__device__ __forceinline__ void append_one(const Append& p, int b, int id) {
  const int token_head = p.by_units.div(id), u0 = id - token_head * (int)p.by_units.d;
  const int t = p.by_heads.div(token_head);
  int h = token_head - t * (int)p.by_heads.d;
  const int kind = h < p.K ? 0 : h < 2 * p.K ? 1 : 2;   // key, value, query
  h -= kind * p.K;

  const int rot = kind == 1 ? 0 : p.rot, half = rot / 2;
  using W = Vec<T, V>;
  // the values are on their way while the length and the page are looked up
  const int64_t* s = kind == 0 ? p.k_s : kind == 1 ? p.v_s : p.q_s;
  const T* src = (const T*)(kind == 0 ? p.k : kind == 1 ? p.v : p.q) + b * s[0] + h * s[1] + t * s[2];
  int d0[N], d1[N];   // first elements of the two vectors
  W a[N], c[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = u0 + k * (int)p.by_units.d;
    // halves' pairs first, behind them the rest of the head in order
    const bool halves = rot > 0 && !p.interleaved && u * V < half;
    d0[k] = halves ? u * V : (rot > 0 && !p.interleaved) ? rot + 2 * (u * V - half) : 2 * u * V;
    d1[k] = halves ? half + u * V : d0[k] + V;
    a[k] = load_once<W>(src + d0[k]);
    c[k] = W{};
    if (d1[k] < p.D) c[k] = load_once<W>(src + d1[k]);
  }

  const int pre = p.plens ? clamped_len(p.plens, b / p.per, p.pcap) : 0;
  // A length past the table keeps its tokens' positions, and those without a slot are treated as padding: clamped like a
  // length that is only read, the new tokens would land on earlier ones.
  const int len = p.seq_lens[b], at = max(len, 0) - p.T + t, i = at < p.cap ? at : -1;
  if (len < 0 || len > p.cap) record_device_error(GPT_DEVERR_INDEX);
  T* dst;
  if (kind == 2) {
    dst = (T*)p.q_out + b * p.o_s[0] + h * p.o_s[1] + t * p.o_s[2];
  } else {
    if (i < 0) return;   // padding
    const int page = p.by_page.div(i), pid = page_id(p.table[b * p.ld_table + page], p.n_pages);
    if (pid < 0) return;
    dst = (T*)(kind == 0 ? p.k_pages : p.v_pages) + pid * p.page_stride + h * p.head_stride +
          (int64_t)(i - page * p.page) * p.slot_stride;
  }
  if (rot > 0) {
    const int64_t n = (int64_t)pre + i;
    // a position without a table row gives a row of zeros, its unrotated part included, as does a padding query
    const bool known = i >= 0 && n < p.n_pos;
    if (i >= 0 && !known) record_device_error(GPT_DEVERR_INDEX);
    const float* cs = p.cos_sin + n * rot;
    using F = Vec<float, V % 4 == 0 ? 4 : 1>;
    constexpr int FV = sizeof(F) / sizeof(float);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (!known) {
        a[k] = W{};
        c[k] = W{};
      } else if (d0[k] < rot) {
        // halves: element j of the one vector with element j of the other; interleaved: V neighbouring
        // pairs of 2 V elements, the pairs at and past rot (a multiple of 2 FV where FV > 1) stay
        const int j_first = p.interleaved ? d0[k] / 2 : d0[k];
#pragma unroll
        for (int j0 = 0; j0 < V; j0 += FV) {
          if (p.interleaved && d0[k] + 2 * j0 >= rot) break;
          const F co = *reinterpret_cast<const F*>(cs + j_first + j0), si = *reinterpret_cast<const F*>(cs + half + j_first + j0);
#pragma unroll
          for (int j = 0; j < FV; ++j) {
            const int e = 2 * (j0 + j);
            T& e0 = !p.interleaved ? a[k].e[j0 + j] : e < V ? a[k].e[e % V] : c[k].e[e % V];
            T& e1 = !p.interleaved ? c[k].e[j0 + j] : e + 1 < V ? a[k].e[(e + 1) % V] : c[k].e[(e + 1) % V];
            const float x0 = Tr<T>::to_f(e0), x1 = Tr<T>::to_f(e1);
            e0 = Tr<T>::from_f(x0 * co.e[j] - x1 * si.e[j]);
            e1 = Tr<T>::from_f(x0 * si.e[j] + x1 * co.e[j]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    *reinterpret_cast<W*>(dst + d0[k]) = a[k];
    if (d1[k] < p.D) *reinterpret_cast<W*>(dst + d1[k]) = c[k];
  }
}

constexpr int kAppendThreads = 128;

template <typename T, int V, int N>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const Append p) {
  pdl_wait();
  pdl_trigger();
  const int id = (int)blockIdx.x * kAppendThreads + threadIdx.x;
  if (id >= p.total) return;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) append_one<T, V, N>(p, b, id);
}

template <typename T, int V, int N>
static int launch_append_n(Append p, int64_t heads, int64_t units, cudaStream_t st) {
  const int64_t total = p.T * heads * units;
  GPT_CHECK_SHAPE(total < (1LL << 31) - kAppendThreads, "gpt_paged_kv_append: too many elements of one sequence for one call");
  p.total = (int)total;
  p.by_heads = FastDiv(heads);
  p.by_units = FastDiv(units);
  p.by_page = FastDiv(p.page);
  const unsigned blocks = (unsigned)((total + kAppendThreads - 1) / kAppendThreads);
  launch_pdl(paged_append_kernel<T, V, N>, dim3(blocks, (unsigned)(p.B < 65535 ? p.B : 65535)), dim3(kAppendThreads), 0, st, p);
  return launch_status("paged_kv_append");
}

template <typename T, int V>
static int launch_append(const Append& p, int64_t heads, cudaStream_t st) {
  const int64_t units = (p.D + 2 * V - 1) / (2 * V);
  // Two pairs of vectors a thread where that leaves threads enough to fill the GPU (8 prompts of 4093 tokens: 172 us,
  // 144 with two).
  if constexpr (V > 1)
    if (units % 2 == 0 && (int64_t)p.B * p.T * heads * units >= (1 << 20)) return launch_append_n<T, V, 2>(p, heads, units / 2, st);
  return launch_append_n<T, V, 1>(p, heads, units, st);
}

}  // namespace paged
}  // namespace gpt
