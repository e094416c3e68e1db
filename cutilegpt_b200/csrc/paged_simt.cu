// Attention over the paged cache on the CUDA cores, in fp32: any head size up
// to 256, any page size, strides and alignment, both types. It serves what the tensor-core kernels'
// conditions leave over (13 sequences behind 1003 positions, 12 heads of 64 in fp32, in views at odd
// elements: 98 us a call; aligned, in the few-row kernel, 12.0).
//
// A CTA of four warps takes up to RB rows of one key head (see Phase in
// paged.cuh) and one of `splits` equal shares of the phase's keys, 32 keys a
// step: the keys and values of the step go to shared memory as fp32; warp w
// owns rows w, w + 4, ..., lane j computes the score of key j, the warp keeps the row's
// running maximum m and its share of the sum l, and the accumulator's columns
// lane, lane + 32, ...:
//   s_j = scale q.k_j,  m' = max(m, max_j s_j),  l' = l 2^(m-m') + sum_j 2^(s_j-m'),
//   acc' = acc 2^(m-m') + sum_j 2^(s_j-m') v_j
// (scores in units of log2). A masked key is left out by its probability 0 and,
// so that what a cache slot behind the length holds has no say, by zeros in
// its place.
#include "paged.cuh"

namespace gpt {
namespace paged {

constexpr int kSimtKeys = 32;
constexpr int kSimtWarps = 4;
constexpr int kSimtMaxD = 256;

// Index of the last own position row (b, t) sees, below 0 for a padding token.
__device__ __forceinline__ int last_key(const Attn& p, int b, int t) { return own_len(p, b) - p.T + t; }

// acc / l of one row joined with `n` partial slots from `first` on; one warp, lane holds columns
// lane + 32 c. Slots without keys have l = 0.
template <int NC>
__device__ __forceinline__ void join_slots(const Attn& p, int first, int n, int64_t row, int lane, float& m, float& l,
                                           float (&acc)[NC]) {
  const int64_t rows = (int64_t)p.B * p.T * p.H;
  for (int s = first; s < first + n; ++s) {
    const float2 o = p.ml[s * rows + row];
    if (o.y == 0.f) continue;
    const float mn = fmaxf(m, o.x);
    const float a = l == 0.f ? 0.f : exp2f(m - mn), c = exp2f(o.x - mn);
    const float* part = p.acc + (s * rows + row) * p.D;
    m = mn;
    l = l * a + o.y * c;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int d = lane + 32 * k;
      acc[k] = acc[k] * a + (d < p.D ? part[d] * c : 0.f);
    }
  }
}

template <typename T, int RB>
__global__ void __launch_bounds__(kSimtWarps * 32) paged_simt_kernel(const Attn p, int phase, int splits, int blocks,
                                                                     int slot0, int direct) {
  constexpr int RW = (RB + kSimtWarps - 1) / kSimtWarps;   // rows of a warp
  constexpr int NC = kSimtMaxD / 32;
  extern __shared__ float simt_smem[];
  const int pitch = p.D | 1;                               // odd: no bank conflicts between keys
  float* sk = simt_smem;                                   // [32][pitch]
  float* sv = sk + kSimtKeys * pitch;
  float* sq = sv + kSimtKeys * pitch;                      // [RB][D], scaled
  __shared__ int64_t soff[kSimtKeys];
  pdl_wait();
  pdl_trigger();
  int item = blockIdx.x;
  const int split = item % splits;
  item /= splits;
  const int block = item % blocks;
  item /= blocks;
  const int kh = item % p.K, who = item / p.K;
  const int b0 = phase == kPrefix ? who * p.per : who;
  const int rows = p.T * p.share * (phase == kPrefix ? p.per : 1);
  const int r0 = block * RB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Keys keys(p, phase, who);
  const int n = keys.n();
  const int chunk = ((n + splits - 1) / splits + kSimtKeys - 1) / kSimtKeys * kSimtKeys;
  const int j0 = min(n, split * chunk), j1 = min(n, j0 + chunk);

  for (int i = threadIdx.x; i < RB * p.D; i += blockDim.x) {
    const int r = r0 + i / p.D, d = i % p.D;
    float x = 0.f;
    if (r < rows) {
      const int b = b0 + r / (p.T * p.share), rr = r % (p.T * p.share);
      x = Tr<T>::to_f(((const T*)p.q)[b * p.q_b + (int64_t)(kh * p.share + rr % p.share) * p.q_h +
                                      (rr / p.share) * p.q_t + d]) * p.scale_log2;
    }
    sq[i] = x;
  }
  int seen[RW];   // keys below this one are the row's
  float m[RW], l[RW], acc[RW][NC];
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int r = r0 + warp + i * kSimtWarps;
    seen[i] = 0;
    if (r < rows) seen[i] = phase == kPrefix ? n : keys.n_pre + last_key(p, b0, r / p.share) + 1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) acc[i][k] = 0.f;
  }

  for (int j = j0; j < j1; j += kSimtKeys) {
    __syncthreads();
    if (threadIdx.x < kSimtKeys) soff[threadIdx.x] = j + threadIdx.x < j1 ? keys.offset(p, j + threadIdx.x, kh) : -1;
    __syncthreads();
    for (int i = threadIdx.x; i < kSimtKeys * p.D; i += blockDim.x) {
      const int key = i / p.D, d = i % p.D;
      const int64_t off = soff[key];
      sk[key * pitch + d] = off < 0 ? 0.f : Tr<T>::to_f(((const T*)p.k)[off + d]);
      sv[key * pitch + d] = off < 0 ? 0.f : Tr<T>::to_f(((const T*)p.v)[off + d]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int rl = warp + i * kSimtWarps;
      if (rl >= RB || j >= seen[i]) continue;   // uniform in the warp
      float s = 0.f;
      for (int d = 0; d < p.D; ++d) s = fmaf(sq[rl * p.D + d], sk[lane * pitch + d], s);
      if (j + lane >= min(seen[i], j1)) s = -INFINITY;
      const float mn = fmaxf(m[i], warp_max(s));
      const float a = m[i] == -INFINITY ? 0.f : exp2f(m[i] - mn);
      const float e = s == -INFINITY ? 0.f : exp2f(s - mn);   // NaN for a NaN score, which leaves the maximum alone
      m[i] = mn;
      l[i] = l[i] * a + warp_sum(e);
#pragma unroll
      for (int k = 0; k < NC; ++k) acc[i][k] *= a;
      for (int key = 0; key < min(kSimtKeys, seen[i] - j); ++key) {   // a value that the row does not see has no part in it
        const float w = __shfl_sync(0xffffffffu, e, key);
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if (lane + 32 * k < p.D) acc[i][k] = fmaf(w, sv[key * pitch + lane + 32 * k], acc[i][k]);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int rl = warp + i * kSimtWarps, r = r0 + rl;
    if (rl >= RB || r >= rows) continue;
    const int rs = p.T * p.share, b = b0 + r / rs, t = r % rs / p.share, h = kh * p.share + r % rs % p.share;
    const int64_t row = row_id(p, b, t, h);
    if (direct) {
      const bool padding = last_key(p, b, t) < 0;
      if (!padding) join_slots<NC>(p, 0, p.n_pre, row, lane, m[i], l[i], acc[i]);
      T* out = (T*)p.out + b * p.o_b + h * p.o_h + t * p.o_t;
      const float inv = padding ? 0.f : 1.f / l[i];
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (lane + 32 * k < p.D) out[lane + 32 * k] = Tr<T>::from_f(padding ? 0.f : acc[i][k] * inv);
    } else {
      const int64_t at = (int64_t)(slot0 + split) * p.B * p.T * p.H + row;
      if (lane == 0) p.ml[at] = make_float2(m[i], l[i]);
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (l[i] != 0.f && lane + 32 * k < p.D) p.acc[at * p.D + lane + 32 * k] = acc[i][k];
    }
  }
}

// out of all partial slots: `groups` teams of D / 4 threads a row (four columns a thread; D threads, one column
// each, where D is no multiple of 4), team g takes slots g, g + groups, ..., eight loads at a time, and the teams are
// joined in order through shared memory.
constexpr int kJoinThreads = 256;

template <typename T, int V>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const Attn p, int groups, int rows_cta) {
  struct alignas(4 * V) Cols {
    float c[V];
  };
  __shared__ float2 sm_ml[kJoinThreads];
  __shared__ Cols sm_acc[kJoinThreads];
  pdl_wait();
  pdl_trigger();
  const int team = p.D / V, who = threadIdx.x / team, d = (threadIdx.x - who * team) * V;
  const int64_t rows = (int64_t)p.B * p.T * p.H, row = (int64_t)blockIdx.x * rows_cta + who / groups;
  const int group = who % groups, n = p.n_pre + p.n_own;
  const bool mine = who < rows_cta * groups && row < rows;
  float m = -INFINITY, l = 0.f;
  Cols acc = {};
  auto add = [&](float2 ml, const Cols& v) {   // a slot without keys has l = 0 and was not written
    if (ml.y == 0.f) return;
    const float to = fmaxf(m, ml.x), a = l == 0.f ? 0.f : exp2f(m - to), b = exp2f(ml.x - to);
    m = to;
    l = l * a + ml.y * b;
#pragma unroll
    for (int i = 0; i < V; ++i) acc.c[i] = acc.c[i] * a + v.c[i] * b;
  };
  for (int s0 = group; mine && s0 < n; s0 += 8 * groups) {
    float2 ml[8];
    Cols v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + i * groups;
      ml[i] = make_float2(0.f, 0.f);
      if (s >= n) continue;
      ml[i] = p.ml[s * rows + row];
      v[i] = *reinterpret_cast<const Cols*>(p.acc + (s * rows + row) * p.D + d);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) add(ml[i], v[i]);
  }
  if (groups > 1) {
    sm_ml[threadIdx.x] = make_float2(m, l);
    sm_acc[threadIdx.x] = acc;
    __syncthreads();
    if (group != 0) return;
    for (int g = 1; mine && g < groups; ++g) add(sm_ml[threadIdx.x + g * team], sm_acc[threadIdx.x + g * team]);
  }
  if (!mine || group != 0) return;
  const int h = (int)(row % p.H), t = (int)(row / p.H % p.T), b = (int)(row / p.H / p.T);
  const bool padding = last_key(p, b, t) < 0;
  const float inv = 1.f / l;   // l = 0: every score is -inf, the row is 0 / 0
  T* out = (T*)p.out + b * p.o_b + h * p.o_h + t * p.o_t + d;
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = Tr<T>::from_f(padding ? 0.f : mean<T>(acc.c[i], inv));
}

template <typename T, int RB>
static int launch_simt_rb(const Attn& p, int phase, int splits, int slot0, int direct, cudaStream_t st) {
  const int64_t rows = (int64_t)p.T * p.share * (phase == kPrefix ? p.per : 1);
  const int64_t blocks = (rows + RB - 1) / RB;
  const int64_t grid = blocks * splits * p.K * (phase == kPrefix ? p.B / p.per : p.B);
  GPT_CHECK_SHAPE(grid < (1LL << 31), "gpt_attention_shared_prefix: too many rows for one call");
  constexpr auto bytes = [](int D) { return (2 * kSimtKeys * (D | 1) + RB * D) * (int)sizeof(float); };
  // The limit belongs to the kernel on the device, not to the call: the largest head's, once, as a smaller one set by
  // another thread would have this launch refused.
  static bool done[64] = {false};
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> g(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(paged_simt_kernel<T, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(kSimtMaxD));
      if (e != cudaSuccess) return fail(GPT_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      done[dev] = true;
    }
  }
  const size_t smem = bytes(p.D);
  launch_pdl(paged_simt_kernel<T, RB>, dim3((unsigned)grid), dim3(kSimtWarps * 32), smem, st, p, phase, splits,
             (int)blocks, slot0, direct);
  return launch_status("paged_simt");
}

template <typename T>
static int launch_simt(const Attn& p, int phase, int splits, int slot0, int direct, cudaStream_t st) {
  const int64_t rows = (int64_t)p.T * p.share * (phase == kPrefix ? p.per : 1);
  return rows <= 4 ? launch_simt_rb<T, 4>(p, phase, splits, slot0, direct, st)
                   : launch_simt_rb<T, 16>(p, phase, splits, slot0, direct, st);
}

template <typename T, int V>
static int launch_join_v(const Attn& p, cudaStream_t st) {
  const int team = p.D / V, teams = kJoinThreads / team, n = p.n_pre + p.n_own;
  // teams for a row: as many as the slots keep busy with eight loads, so that many slots cost few rounds
  int groups = 1;
  while (groups * 8 < n && groups * 2 <= teams) groups *= 2;
  const int rows_cta = teams / groups;
  const int64_t rows = (int64_t)p.B * p.T * p.H;
  launch_pdl(paged_join_kernel<T, V>, dim3((unsigned)((rows + rows_cta - 1) / rows_cta)), dim3(kJoinThreads), 0, st, p, groups,
             rows_cta);
  return launch_status("paged_join");
}

template <typename T>
static int launch_join(const Attn& p, cudaStream_t st) {
  return p.D % 4 == 0 ? launch_join_v<T, 4>(p, st) : launch_join_v<T, 1>(p, st);
}

}  // namespace paged
}  // namespace gpt
