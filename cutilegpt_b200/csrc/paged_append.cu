// New tokens into the paged key/value cache, their rotation on the way.
//
// A pair of values (x0, x1) of a query or key head at position n becomes
// (x0 c - x1 s, x0 s + x1 c) with c, s from the caller's fp32 table; values
// are copied. Everything is read once and written once, so the kernel is
// bound by HBM: 2 (2 K + H) D e bytes per token with rotation, 4 K D e without.
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

// One thread's share of sequence b.
template <typename T, int V>
__device__ __forceinline__ void append_one(const Append& p, int b, int id) {
  const int token_head = p.by_units.div(id), u = id - token_head * (int)p.by_units.d;
  const int t = p.by_heads.div(token_head);
  int h = token_head - t * (int)p.by_heads.d;
  const int kind = h < p.K ? 0 : h < 2 * p.K ? 1 : 2;   // key, value, query
  h -= kind * p.K;

  const int rot = kind == 1 ? 0 : p.rot, half = rot / 2;
  const bool halves = rot > 0 && !p.interleaved && u * V < half;
  // first elements of the two vectors; behind the halves' pairs the rest of the head in order
  const int d0 = halves ? u * V : (rot > 0 && !p.interleaved) ? rot + 2 * (u * V - half) : 2 * u * V;
  const int d1 = halves ? half + u * V : d0 + V;
  const bool second = d1 < p.D;
  using W = Vec<T, V>;
  // the values are on their way while the length and the page are looked up
  const int64_t* s = kind == 0 ? p.k_s : kind == 1 ? p.v_s : p.q_s;
  const T* src = (const T*)(kind == 0 ? p.k : kind == 1 ? p.v : p.q) + b * s[0] + h * s[1] + t * s[2];
  W a = *reinterpret_cast<const W*>(src + d0), c = {};
  if (second) c = *reinterpret_cast<const W*>(src + d1);

  const int pre = p.plens ? clamped_len(p.plens, b / p.per, p.pcap) : 0;
  const int i = clamped_len(p.seq_lens, b, p.cap) - p.T + t;
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
  if (d0 < rot) {
    const int64_t n = (int64_t)pre + i;
    const bool known = i >= 0 && n >= 0 && n < p.n_pos;
    if (i >= 0 && !known) record_device_error(GPT_DEVERR_INDEX);
    const float* cs = p.cos_sin + n * rot;
    using F = Vec<float, V % 4 == 0 ? 4 : 1>;
    constexpr int FV = sizeof(F) / sizeof(float);
    if (!known) {
      a = {};
      c = {};
    } else if (halves) {
#pragma unroll
      for (int j0 = 0; j0 < V; j0 += FV) {
        const F co = *reinterpret_cast<const F*>(cs + d0 + j0), si = *reinterpret_cast<const F*>(cs + half + d0 + j0);
#pragma unroll
        for (int j = 0; j < FV; ++j) {
          const float x0 = Tr<T>::to_f(a.e[j0 + j]), x1 = Tr<T>::to_f(c.e[j0 + j]);
          a.e[j0 + j] = Tr<T>::from_f(x0 * co.e[j] - x1 * si.e[j]);
          c.e[j0 + j] = Tr<T>::from_f(x0 * si.e[j] + x1 * co.e[j]);
        }
      }
    } else {
      // 2 V neighbouring elements, V pairs; the pairs at and past rot stay
#pragma unroll
      for (int j0 = 0; j0 < V; j0 += FV) {
        if (d0 + 2 * j0 >= rot) break;   // rot is a multiple of 2 FV where FV > 1
        const F co = *reinterpret_cast<const F*>(cs + d0 / 2 + j0), si = *reinterpret_cast<const F*>(cs + half + d0 / 2 + j0);
#pragma unroll
        for (int j = 0; j < FV; ++j) {
          const int e = 2 * (j0 + j);
          T& e0 = e < V ? a.e[e % V] : c.e[e % V];
          T& e1 = e + 1 < V ? a.e[(e + 1) % V] : c.e[(e + 1) % V];
          const float x0 = Tr<T>::to_f(e0), x1 = Tr<T>::to_f(e1);
          e0 = Tr<T>::from_f(x0 * co.e[j] - x1 * si.e[j]);
          e1 = Tr<T>::from_f(x0 * si.e[j] + x1 * co.e[j]);
        }
      }
    }
  } else if (kind == 2 && i < 0) {
    a = {};
    c = {};
  }
  if (kind != 1 && rot > 0 && d0 >= rot && i >= 0 && (int64_t)pre + i >= p.n_pos) {
    a = {};   // a position without a table row gives a row of zeros, its unrotated part included
    c = {};
  }
  *reinterpret_cast<W*>(dst + d0) = a;
  if (second) *reinterpret_cast<W*>(dst + d1) = c;
}

constexpr int kAppendThreads = 128;

template <typename T, int V>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const Append p) {
  pdl_wait();
  pdl_trigger();
  const int id = (int)blockIdx.x * kAppendThreads + threadIdx.x;
  if (id >= p.total) return;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) append_one<T, V>(p, b, id);
}

template <typename T, int V>
static int launch_append(Append p, int64_t heads, cudaStream_t st) {
  const int64_t units = (p.D + 2 * V - 1) / (2 * V), total = p.T * heads * units;
  GPT_CHECK_SHAPE(total < (1LL << 31) - kAppendThreads, "gpt_paged_kv_append: too many elements of one sequence for one call");
  p.total = (int)total;
  p.by_heads = FastDiv(heads);
  p.by_units = FastDiv(units);
  p.by_page = FastDiv(p.page);
  const unsigned blocks = (unsigned)((total + kAppendThreads - 1) / kAppendThreads);
  launch_pdl(paged_append_kernel<T, V>, dim3(blocks, (unsigned)(p.B < 65535 ? p.B : 65535)), dim3(kAppendThreads), 0, st, p);
  return launch_status("paged_kv_append");
}

}  // namespace paged
}  // namespace gpt
