// Attention over the paged cache for few rows a key head: one decode step, or
// the few tokens of a draft.
//
// Every key and value is read once and meets at most 16 rows, so the kernel is
// bound by HBM: 2 D e bytes a key against 32 D multiply-adds. A CTA takes 16 rows
// of one key head (phases as in paged.cuh) and one of `splits` equal shares of
// the phase's keys. Its W warps work alone until the end: warp w takes the
// steps of KS keys w, w + W, ... of the share, copies them by cp.async
// (16 bytes a lane, addresses from the page table, zeros behind the length) into its
// own ring, and keeps running maxima, sums and the 16 x D accumulator in
// registers. S = Q Kᵀ and O += P V are tensor-core products of 16 rows
// (mma.sync: 16 rows cannot fill the 128 rows of a tcgen05 tile; those run in paged_tc.cu).
// No barrier stands between a warp's loads and its products; 12 to 16 warps of an
// SM keep 96 to 144 KB in flight (fp32: 8 warps, 64 KB).
// B200: 128 sequences of up to 4096 positions, 8 key heads of 128 in bf16 (1.08 GB): 173 us = 6.2 TB/s, 0.96 of a
// measured copy; 67 of up to 1024: 36 us = 4.1 TB/s (the last CTAs alone). Below some 300 keys a CTA its fixed
// chain rules (length, page table, first copies, join: about 5 us): 64 of up to 256, 12 heads of 64: 13.2 us.
//
// bf16: m16n8k16. P is rounded to bf16 for its product with V, its sum is taken before.
// fp32: m16n8k8 on TF32 parts. A value x is hi + lo, hi = x to 11 bits, lo = (x - hi) to
// 11 bits: x is met to 2^-22, and hi hi + hi lo + lo hi leaves out 2^-22 of a product. The tensor cores
// cut sums off towards zero, so a product chain is short (16 elements of a score, a step's keys of
// the output) and is added to the running sum by a rounding add (13 samples of 1003 + 77 positions against
// 64 bits: 1.2e-6 off with chains through, 4.5e-7 so). The order of a contraction is free, so a lane's operands are
// those that one 16-byte read gives it.
#include "paged.cuh"

namespace gpt {
namespace paged {

constexpr int kRowTile = 16;
constexpr int kMaxSlots = 32;    // prefix slots that the kernel joins itself

template <typename T, int DP, int W>   // DP: head size padded to a power of two
struct Rows {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kKeys = kWide ? (DP == 128 ? 8 : DP == 64 ? 16 : 32) : (DP >= 64 ? 16 : 1024 / DP);   // of a warp's step
  static constexpr int kTile = kKeys * DP * (int)sizeof(T);    // bytes of a step's keys
  // Steps of a warp's ring. Deeper ones cost resident CTAs: with four warps a fourth step pays (48 drafts of 5 tokens,
  // D = 64: 31.5 -> 30.0 us), with two it does not (64 samples of 768 + 256 positions: 13.4 us, 18.7 with four steps).
  static constexpr int kRing = kTile > 2048 ? 2 : W == 4 ? 4 : 3;
  // Q fragments in shared memory, read at every step, where they would take too many registers
  static constexpr bool kQShared = kWide || DP == 128;
  static constexpr int kQSteps = kWide ? DP / 4 : DP / 16;     // uint4 of a lane
  static constexpr int kQ = kQShared ? kQSteps * 512 : 0;
  static constexpr int kRings = W * kRing * 2 * kTile;
  static constexpr int kMerge = W * kRowTile * (DP + 2) * 4 + kRowTile * kMaxSlots * 8;
  static constexpr int kSmem = (kRings > kMerge ? kRings : kMerge) + kQ;
  // CTAs of an SM: as many as its registers give room for (8, 12 or 16 warps), or its shared memory
  static constexpr int kByRegs = (kWide ? 8 : DP == 128 ? 12 : 16) / W, kBySmem = 227 * 1024 / (kSmem + 1024);
  static constexpr int kCtas = kByRegs < kBySmem ? kByRegs : kBySmem;
};

// Byte offset of 16-byte chunk c of row r in a tile of rows of DP values, chunks permuted
// inside a row so that the chunks that one read touches lie in different bank groups.
template <typename T, int DP>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  constexpr int kChunks = DP * (int)sizeof(T) / 16;
  int x;
  if (sizeof(T) == 4)   // reads of rows 0..7 by 4 chunks, and of rows 0, 2, 4, 6 by 8 floats
    x = (((r ^ (r >> 1)) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 1) & 1);
  else                  // reads of 8 rows of one chunk column
    x = kChunks >= 8 ? (r & 7) : kChunks == 4 ? ((r >> 1) & 3) : ((r >> 2) & 1);
  return (uint32_t)(r * DP * (int)sizeof(T) + ((c ^ x) << 4));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, float (&r)[4]) {
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// hi is never rounded to infinity: of a number near the largest it is the largest TF32, of an infinity too, and lo
// is the rest, an infinity then. Products with both parts thus have the infinity once; NaN is NaN in both.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.satfinite.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = to_tf32(x - __uint_as_float(hi));
}
// c += a b in three TF32 products, the small ones first. kLarge: a may exceed 1 so far that its low part by an
// infinity's high one overflows against the infinity's sign: that product is left out.
template <bool kLarge>
__device__ __forceinline__ void mma_split(float (&c)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  if (kLarge)
    mma1688(c, al, isinf(b0) ? 0u : h0, isinf(b1) ? 0u : h1);
  else
    mma1688(c, al, h0, h1);
  mma1688(c, ah, l0, l1);
  mma1688(c, ah, h0, h1);
}

template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 v) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(dst) = v;
  else
    *reinterpret_cast<uint2*>(dst) = make_uint2(tc::pack2_bf16(v.x, v.y), tc::pack2_bf16(v.z, v.w));
}

struct RowsArgs {
  int phase, splits, slot0, direct;
  int early;                // behind this call's prefix launch: 1 waits for it before the end, 2 runs beside it
  int two_warps;            // CTAs of two warps, not four
  FastDiv by_splits, by_blocks;
};

// kEdge: several tokens a sequence and own keys, so that rows of the tile see different keys.
template <typename T, int DP, int W, bool kEdge>
__global__ void __launch_bounds__(W * 32, (Rows<T, DP, W>::kCtas)) paged_rows_kernel(const __grid_constant__ Attn p,
                                                                                     const RowsArgs a) {
  using C = Rows<T, DP, W>;
  constexpr bool kWide = C::kWide;
  constexpr int KS = C::kKeys, kPer = 16 / (int)sizeof(T), kChunks = DP / kPer, kLoads = KS * kChunks / 32;
  constexpr int kTile = C::kTile, kRing = C::kRing;
  extern __shared__ __align__(128) uint8_t rows_smem_dyn[];
  // With early the launch before is this call's prefix launch, whose every CTA has waited for all
  // that came before it: what is read and written here is then safe, but for the prefix's partial results.
  if (!a.early) pdl_wait();
  pdl_trigger();
  const int split_item = a.by_splits.div((int)blockIdx.x), split = (int)blockIdx.x - split_item * a.splits;
  const int block_item = a.by_blocks.div(split_item), block = split_item - block_item * (int)a.by_blocks.d;
  const int who = p.by_K.div(block_item), kh = block_item - who * p.K;
  const int b0 = a.phase == kPrefix ? who * p.per : who;
  const int rows = (int)p.by_rows.d * (a.phase == kPrefix ? p.per : 1);
  const int r0 = block * kRowTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3;
  const Keys keys(p, a.phase, who);
  const int n = keys.n();
  const int chunk = (a.by_splits.div(n + a.splits - 1) + KS - 1) / KS * KS;
  const int j0 = min(n, split * chunk);
  int j1 = min(n, j0 + chunk);

  // rows lane / 4 and lane / 4 + 8 of the tile
  const T* src[2];
  bool live[2];
  int seen[2];                      // keys below this one are the row's
  int most = 0, least = n;          // the largest and the smallest of the tile's
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + lane / 4 + 8 * h;
    live[h] = r < rows;
    const Row at(p, b0, kh, live[h] ? r : r0);
    const int last = keys.n_own - p.T + at.t;         // own key; below 0 the row is padding and sees nothing
    seen[h] = !live[h] ? 0 : a.phase == kPrefix ? n : last < 0 ? 0 : keys.n_pre + last + 1;
    most = max(most, seen[h]);
    if (live[h]) least = min(least, seen[h]);
    src[h] = (const T*)p.q + at.b * p.q_b + at.h * p.q_h + at.t * p.q_t;
  }
  j1 = min(j1, (int)__reduce_max_sync(0xffffffffu, (unsigned)most));
  least = min(j1, (int)__reduce_min_sync(0xffffffffu, (unsigned)least));

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(rows_smem_dyn) + C::kQ + warp * (kRing * 2 * kTile);
  if (p.D < DP) {   // columns behind D stay zeros
    for (int i = threadIdx.x; i < C::kRings / 16; i += blockDim.x) reinterpret_cast<uint4*>(rows_smem_dyn + C::kQ)[i] = uint4{};
    __syncthreads();
  }
  const int steps = j1 > j0 + warp * KS ? (j1 - j0 - warp * KS + W * KS - 1) / (W * KS) : 0;
  // lane i holds the offsets of keys i, i + 32, ... of a step, -1 where there is none
  constexpr int kOffs = (KS + 31) / 32;
  int64_t off[kRing][kOffs];                       // the first steps' are looked up side by side
  auto locate = [&](int s, int64_t (&to)[kOffs]) {
#pragma unroll
    for (int i = 0; i < kOffs; ++i) {
      const int in = lane + 32 * i, j = j0 + (s * W + warp) * KS + in;
      to[i] = in < KS && s < steps && j < j1 ? keys.offset(p, j, kh) : -1;
    }
  };
  auto fetch = [&](int s, const int64_t (&from)[kOffs]) {
    const uint32_t dst = ring + (uint32_t)(s % kRing) * (2 * kTile);
    const int c = lane % kChunks;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * (32 / kChunks) + lane / kChunks;
      const int64_t o = __shfl_sync(0xffffffffu, from[i * (32 / kChunks) / 32], r & 31);
      if (c * kPer < p.D) {
        const int64_t at = (o < 0 ? 0 : o) + c * kPer;
        cp_async16(dst + swz<T, DP>(r, c), (const T*)p.k + at, o >= 0);
        cp_async16(dst + kTile + swz<T, DP>(r, c), (const T*)p.v + at, o >= 0);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < kRing; ++s) locate(s, off[s]);
#pragma unroll
  for (int s = 0; s < kRing - 1; ++s) fetch(s, off[s]);

  // Q in the A fragments, with kQShared in shared memory as [step][lane]
  uint4* sq = reinterpret_cast<uint4*>(rows_smem_dyn);
  uint4 qf[C::kQShared ? 1 : C::kQSteps];
  if constexpr (kWide) {
    constexpr int kMine = (DP / 8 + W - 1) / W;      // contraction steps of this warp, all loads first
    float x[kMine][4];
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      // the step's elements of this lane: 16 (k / 2) + 4 quad + 2 (k % 2) and the next one
      const int k = warp + u * W, d = 16 * (k / 2) + 4 * quad + 2 * (k % 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] = live[i & 1] && d + (i >> 1) < p.D ? src[i & 1][d + (i >> 1)] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      const int k = warp + u * W;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split_tf32(x[u][i], hi[i], lo[i]);
      sq[2 * k * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      sq[(2 * k + 1) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  } else {
    auto load = [&](int k) {
      uint32_t f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = k * 16 + (i >> 1) * 8 + quad * 2;
        f[i] = live[i & 1] && d < p.D ? *reinterpret_cast<const uint32_t*>(src[i & 1] + d) : 0u;
      }
      return make_uint4(f[0], f[1], f[2], f[3]);
    };
    if constexpr (C::kQShared) {
      uint4 x[DP / 16 / W];
#pragma unroll
      for (int u = 0; u < DP / 16 / W; ++u) x[u] = load(warp + u * W);
#pragma unroll
      for (int u = 0; u < DP / 16 / W; ++u) sq[(warp + u * W) * 32 + lane] = x[u];
    } else {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) qf[k] = load(k);
    }
  }
  if (C::kQShared) __syncthreads();
  auto q_frag = [&](int k, uint32_t (&f)[4]) {
    const uint4 x = C::kQShared ? sq[k * 32 + lane] : qf[C::kQShared ? 0 : k];
    f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
  };

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
  const bool edge = least < j1;     // some rows see keys of this share that others do not
  bool odd = false;
  for (int s = 0; s < steps; ++s) {
    cp_wait<kRing - 2>();
    __syncwarp();
    fetch(s + kRing - 1, off[kRing - 1]);   // into the slot of step s - 1, which every lane has left
    locate(s + kRing, off[kRing - 1]);      // the table read is on its way while this step computes
    const uint32_t sk = ring + (uint32_t)(s % kRing) * (2 * kTile), sv = sk + kTile;
    const int j = j0 + (s * W + warp) * KS;
    float sc[KS / 8][4];
#pragma unroll
    for (int i = 0; i < KS / 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) sc[i][k] = 0.f;
    if constexpr (kWide) {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t ah[2][4], al[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          q_frag(4 * k + 2 * u, ah[u]);
          q_frag(4 * k + 2 * u + 1, al[u]);
        }
#pragma unroll
        for (int i = 0; i < KS / 8; ++i) {
          float kv[4], part[4] = {0.f, 0.f, 0.f, 0.f};
          lds128(sk + swz<T, DP>(i * 8 + lane / 4, k * 4 + quad), kv);
          mma_split<true>(part, ah[0], al[0], kv[0], kv[1]);
          mma_split<true>(part, ah[1], al[1], kv[2], kv[3]);
#pragma unroll
          for (int u = 0; u < 4; ++u) sc[i][u] += part[u];
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t f[4];
        q_frag(k, f);
#pragma unroll
        for (int i = 0; i < KS / 16; ++i) {
          uint32_t kb[4];
          ldsm4(sk + swz<T, DP>(i * 16 + (lane >> 4) * 8 + (lane & 7), k * 2 + ((lane >> 3) & 1)), kb);
          mma16816(sc[2 * i], f, kb[0], kb[1]);
          mma16816(sc[2 * i + 1], f, kb[2], kb[3]);
        }
      }
    }
    if (j + KS > least) {   // keys that some row does not see
      if (kEdge && edge)    // see slow_row
        for (int i = lane; i < kTile / 16; i += 32) odd |= non_finite<T>(lds_u4(sv + i * 16));
#pragma unroll
      for (int i = 0; i < KS / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (j + i * 8 + quad * 2 + (k & 1) >= min(j1, seen[k >> 1])) sc[i][k] = -INFINITY;
    }
    float mx[2] = {-INFINITY, -INFINITY}, base[2];
#pragma unroll
    for (int i = 0; i < KS / 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) mx[k >> 1] = fmaxf(mx[k >> 1], sc[i][k]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      // fp32: P is at most 1/2, so that a value near the largest number stays in range while its parts are added
      mx[h] = scaled(fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2)), p.scale_log2) + (kWide ? 1.f : 0.f);
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
      float by[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mn = fmaxf(m[h], mx[h]);
        by[h] = mn == -INFINITY ? 1.f : exp2f(m[h] - mn);
        m[h] = mn;
        l[h] *= by[h];
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] *= by[k >> 1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) base[h] = m[h] == -INFINITY ? 0.f : m[h];   // a row without keys so far: every 2^(s - base) is 0
    float unit = p.scale_log2;
    if (__any_sync(0xffffffffu, fmaxf(fabsf(base[0]), fabsf(base[1])) > kHugeScore)) {
      unit = 1.f;
#pragma unroll
      for (int i = 0; i < KS / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) sc[i][k] = scaled(sc[i][k], p.scale_log2);
    }
#pragma unroll
    for (int i = 0; i < KS / 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sc[i][k] = attn_tc::ex2(fmaf(sc[i][k], unit, -base[k >> 1]));
        l[k >> 1] += sc[i][k];
      }
    if constexpr (kWide) {
      uint32_t ah[KS / 8][4], al[KS / 8][4];
#pragma unroll
      for (int i = 0; i < KS / 8; ++i) {   // contraction index quad is key 2 quad, quad + 4 is key 2 quad + 1
        split_tf32(sc[i][0], ah[i][0], al[i][0]);
        split_tf32(sc[i][2], ah[i][1], al[i][1]);
        split_tf32(sc[i][1], ah[i][2], al[i][2]);
        split_tf32(sc[i][3], ah[i][3], al[i][3]);
      }
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {   // column index g of product u is element 32 d + 4 g + u
        float part[4][4] = {};
#pragma unroll
        for (int i = 0; i < KS / 8; ++i) {
          float v0[4], v1[4];
          lds128(sv + swz<T, DP>(i * 8 + 2 * quad, d * 8 + lane / 4), v0);
          lds128(sv + swz<T, DP>(i * 8 + 2 * quad + 1, d * 8 + lane / 4), v1);
#pragma unroll
          for (int u = 0; u < 4; ++u) mma_split<false>(part[u], ah[i], al[i], v0[u], v1[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[4 * d + u][k] += part[u][k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < KS / 16; ++i) {
        uint32_t pf[4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) pf[h + 2 * c] = tc::pack2_bf16(sc[2 * i + c][2 * h], sc[2 * i + c][2 * h + 1]);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          uint32_t vb[4];
          ldsm4_t(sv + swz<T, DP>(i * 16 + (lane & 15), d * 2 + (lane >> 4)), vb);
          mma16816(o[2 * d], pf, vb[0], vb[1]);
          mma16816(o[2 * d + 1], pf, vb[2], vb[3]);
        }
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }

  // the warps' results joined through shared memory, where the rings were
  cp_wait<0>();
  bool again = false;
  if (kEdge)
    again = __syncthreads_or(odd);
  else
    __syncthreads();
  float* sm_o = reinterpret_cast<float*>(rows_smem_dyn + C::kQ);         // [warp][16][DP]
  float2* sm_ml = reinterpret_cast<float2*>(sm_o + W * kRowTile * DP);   // [warp][16]
  float2* sm_w = sm_ml + W * kRowTile;                                   // [16][kMaxSlots]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = lane / 4 + 8 * h;
    if (quad == 0) sm_ml[warp * kRowTile + r] = make_float2(m[h], l[h]);
    float* dst = sm_o + (warp * kRowTile + r) * DP;
    if constexpr (kWide) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float4*>(dst + 32 * d + 4 * (2 * quad + e)) =
              make_float4(o[4 * d][2 * h + e], o[4 * d + 1][2 * h + e], o[4 * d + 2][2 * h + e], o[4 * d + 3][2 * h + e]);
    } else {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
        *reinterpret_cast<float2*>(dst + i * 8 + quad * 2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
  }
  __syncthreads();
  if (kEdge && again) {
    for (int rl = warp; rl < kRowTile; rl += W) {
      float rm = -INFINITY, rls = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
      if (r0 + rl < rows) {
        const Row at(p, b0, kh, r0 + rl);
        const int last = keys.n_own - p.T + at.t;
        slow_row<T>(p, keys, kh, (const T*)p.q + at.b * p.q_b + at.h * p.q_h + at.t * p.q_t, j0,
                    last < 0 ? j0 : min(j1, keys.n_pre + last + 1), lane, rm, rls, acc);
      }
      if (lane < W) sm_ml[lane * kRowTile + rl] = lane == 0 ? make_float2(rm, rls) : make_float2(-INFINITY, 0.f);
      for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < p.D) sm_o[rl * DP + lane + 32 * c] = acc[c];
    }
    __syncthreads();
  }
  // the prefix launch's partial results; its end, which the launch that joins must not come before: for
  // that one CTA's wait is enough, and the others make room for the next
  if (a.early == 1 || (a.early == 2 && blockIdx.x == 0)) pdl_wait();
  // A row's parts: the prefix's slots and the CTA's warps, in that order. Everything that comes from global
  // memory is asked for at once: the slots' (m, l) of all rows, by all threads, and the first slots'
  // columns of the thread's first item.
  const int n_live = min(kRowTile, rows - r0), quads = p.D / 4, n_pre = a.direct ? p.n_pre : 0;
  const int64_t all_rows = (int64_t)p.B * p.T * p.H;
  for (int i = threadIdx.x; i < n_live * n_pre; i += W * 32) {
    const int rl = i / n_pre, s = i - rl * n_pre;
    const Row at(p, b0, kh, r0 + rl);
    sm_w[rl * kMaxSlots + s] = __ldcg(p.ml + s * all_rows + row_id(p, at.b, at.t, at.h));
  }
  bool first = true;
#pragma unroll 1
  for (int i = threadIdx.x; first || i < n_live * quads; i += W * 32) {
    const bool mine = i < n_live * quads;            // the first round is everyone's, for its barrier
    const int rl = mine ? i / quads : 0, d = mine ? (i - rl * quads) * 4 : 0;
    const Row at(p, b0, kh, r0 + rl);
    const int64_t row = row_id(p, at.b, at.t, at.h);
    const float* part = p.acc + row * p.D + d;
    float4 v[8];
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (mine && s < n_pre) v[s] = __ldcg(reinterpret_cast<const float4*>(part + s * all_rows * p.D));
    if (first) __syncthreads();
    first = false;
    if (!mine) break;
    const float2* slots = sm_w + rl * kMaxSlots;
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < n_pre; ++s) top = slots[s].y != 0.f ? fmaxf(top, slots[s].x) : top;
#pragma unroll
    for (int u = 0; u < W; ++u) top = fmaxf(top, sm_ml[u * kRowTile + rl].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // A part without keys has l = 0 and anything in x. One whose scores are all NaN has m = -inf, as a maximum
    // passes NaN over, but a NaN l: at the weight 0 it still joins.
    auto add = [&](float2 ml, float4 x) {
      if (ml.y == 0.f) return;
      const float w = exp2f(ml.x - top);
      sum = fmaf(ml.y, w, sum);
      acc.x = fmaf(x.x, w, acc.x);
      acc.y = fmaf(x.y, w, acc.y);
      acc.z = fmaf(x.z, w, acc.z);
      acc.w = fmaf(x.w, w, acc.w);
    };
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s < n_pre) add(slots[s], v[s]);
#pragma unroll 4
    for (int s = 8; s < n_pre; ++s) add(slots[s], __ldcg(reinterpret_cast<const float4*>(part + s * all_rows * p.D)));
#pragma unroll
    for (int u = 0; u < W; ++u)
      add(sm_ml[u * kRowTile + rl], *reinterpret_cast<const float4*>(sm_o + (u * kRowTile + rl) * DP + d));
    if (a.direct) {
      const bool padding = keys.n_own - p.T + at.t < 0;
      const float inv = 1.f / sum;   // sum = 0: every score is -inf, the row is 0 / 0
      store4((T*)p.out + at.b * p.o_b + at.h * p.o_h + at.t * p.o_t + d,
             padding ? make_float4(0.f, 0.f, 0.f, 0.f)
                     : make_float4(mean<T>(acc.x, inv), mean<T>(acc.y, inv), mean<T>(acc.z, inv), mean<T>(acc.w, inv)));
    } else {
      const int64_t to = (int64_t)(a.slot0 + split) * all_rows + row;
      if (d == 0) p.ml[to] = make_float2(top, sum);
      *reinterpret_cast<float4*>(p.acc + to * p.D + d) = acc;
    }
  }
}

// Whether the kernel serves the call: 16-byte rows of keys and values, pairs of q for bf16, quads of out.
static bool rows_eligible(const Attn& p, int size) {
  const int per = 16 / size;
  if (p.D % per || p.D > 128 || !aligned(p.k, 16) || !aligned(p.v, 16) || !aligned(p.q, 4) || !aligned(p.out, 4 * size)) return false;
  for (int64_t s : {p.page_stride, p.head_stride, p.slot_stride})
    if (s % per) return false;
  for (int64_t s : {p.q_b, p.q_h, p.q_t})
    if (s % (size == 2 ? 2 : 1)) return false;
  for (int64_t s : {p.o_b, p.o_h, p.o_t})
    if (s % 4) return false;
  return true;
}

template <typename T, int DP, int W, bool kEdge>
static int launch_rows_w(const Attn& p, RowsArgs a, cudaStream_t st) {
  using C = Rows<T, DP, W>;
  static bool done[64] = {false};
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> g(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<T, DP, W, kEdge>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return fail(GPT_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      done[dev] = true;
    }
  }
  const int64_t rows = (int64_t)p.T * p.share * (a.phase == kPrefix ? p.per : 1);
  const int64_t blocks = (rows + kRowTile - 1) / kRowTile;
  const int64_t grid = blocks * a.splits * p.K * (a.phase == kPrefix ? p.B / p.per : p.B);
  GPT_CHECK_SHAPE(grid < (1LL << 31), "gpt_attention_shared_prefix: too many rows for one call");
  a.by_splits = FastDiv(a.splits);
  a.by_blocks = FastDiv(blocks);
  launch_pdl(paged_rows_kernel<T, DP, W, kEdge>, dim3((unsigned)grid), dim3(W * 32), C::kSmem, st, p, a);
  return launch_status("paged_rows");
}

template <typename T, int DP>
static int launch_rows_dp(const Attn& p, RowsArgs a, cudaStream_t st) {
  if (a.phase != kPrefix && p.T > 1)
    return a.two_warps ? launch_rows_w<T, DP, 2, true>(p, a, st) : launch_rows_w<T, DP, 4, true>(p, a, st);
  return a.two_warps ? launch_rows_w<T, DP, 2, false>(p, a, st) : launch_rows_w<T, DP, 4, false>(p, a, st);
}

template <typename T>
static int launch_rows(const Attn& p, const RowsArgs& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (p.D <= 16) return launch_rows_dp<T, 16>(p, a, st);
  if (p.D <= 32) return launch_rows_dp<T, 32>(p, a, st);
  if (p.D <= 64) return launch_rows_dp<T, 64>(p, a, st);
  return launch_rows_dp<T, 128>(p, a, st);
}

}  // namespace paged
}  // namespace gpt
