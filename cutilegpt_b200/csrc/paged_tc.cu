// Attention over the paged cache on the 5th-generation tensor cores (bf16,
// head sizes 64 and 128): the rows of all sequences of a group against the
// prefix that they share, and the many rows of long questions.
//
// A CTA takes 128 or 256 rows of one key head (phases and rows as in paged.cuh) and
// one of `splits` equal shares of the phase's key tiles. A tile is up to 128 keys:
// whole pages, each copied by one TMA box per 64 columns from {D, slot, head, page} maps (a page past the
// pool is out of the map's bounds: zeros). Two pipelines of one softmax
// warpgroup (one thread per row = TMEM lane) and one MMA-issuing lane work on
//   two != 0: the same tiles, pipeline s on rows 128 s .. of the block, so that 256
//             rows share one reading of the keys,
//   two == 0: the same 128 rows, pipeline s on tiles s, s + 2, ... of the share; the results are joined at the end,
// so that one's products run while the other's softmax does. Per tile:
//   S = Q Kᵀ      tcgen05.mma M=128 N=128 K=D -> TMEM
//   softmax       the row's 128 scores are read into registers, masked (the row's keys end inside a
//                 tile), P = 2^(scale S - m) to TMEM as bf16, the sum of P before its rounding in fp32
//   O += P V      A = P from TMEM, B = V MN-major as its boxes arrive; only the 16-key steps
//                 that hold keys are issued, and the last one's rows behind the keys are cleared
//                 first: what the cache holds there must not meet P = 0
// The exponentials do not wait for the tile's maximum: m is 16 above the largest score (in powers of two) that earlier
// tiles left, a tile whose maximum lies 8 above that one makes the next tile move m (O and the sum are rescaled), one
// 16 above moves it at once and starts over. P = 2^(s - m) is thus at most 1, and a value of any size stays in range;
// weights below 2^-110 of the largest are 0. The PV of a tile's first 64 keys runs under the exponentials of the others. With D = 64 P has
// TMEM columns of its own and the next S is computed under the softmax; with D = 128
// P takes the place of S (256 columns a pipeline), and the next S follows the PV.
// Keys and values have separate rings; every wait is bounded.
// Bound by the softmax warps' issue: a pair of 128 x 128 tiles at D = 128 takes 4300 clocks, of which the products
// and the special-function unit need 2048 each. B200: 8 questions of 256 tokens behind 4096 + 700 positions, 32 heads
// (149 GFLOP): 175 us = 853 TF/s; 512 rows of each of 8 key heads against 65536 keys: 148 to 162 us = 851 to 926 TF/s.
#include "paged.cuh"

namespace gpt {
namespace paged {

using attn_tc::ex2;
using attn_tc::fadd2;
using attn_tc::ffma2;
using attn_tc::fmax3;
using attn_tc::pack_f2;
using attn_tc::pack_u2;
using attn_tc::tc_mma_ts;
using attn_tc::tmem_ld32_nw;
using attn_tc::tmem_st16;
using attn_tc::tmem_st32;
using attn_tc::tmem_wait_ld;
using attn_tc::tmem_wait_st;
using attn_tc::tma_load_4d;
using attn_tc::unpack_f2;
using tc::desc_sw128;
using tc::mbar_arrive;
using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mbar_wait;
using tc::smem_addr;
using tc::tc_commit;
using tc::tc_fence_after;
using tc::tc_fence_before;
using tc::tc_mma;
using tc::tmem_ld32;

constexpr int kTcThreads = 12 * 32;      // 2 x 4 softmax warps, 2 MMA warps, K and V copy warps
constexpr int kPanel = 128 * 128;        // 128 rows of 64 bf16, 128-byte swizzled
constexpr float kTcRescale = 8.f;        // rise of the largest score, in powers of two, from which the next tile moves m
constexpr float kTcFar = 16.f;           // and from which the tile itself moves m and starts over; m lies this far above
constexpr float kTcHugeScore = 1 << 30;  // from which a row is computed again

template <int D>
struct Tc {
  static constexpr int kPanels = D / 64;
  static constexpr int kTile = kPanels * kPanel;         // a Q, K or V tile
  static constexpr int kStages = D == 64 ? 5 : 2;        // of each ring: 160 or 128 KB in flight
  static constexpr int kSmem = 1024 + 2 * kTile + 2 * kStages * kTile + 512 + 256 * (int)sizeof(float2);
  static constexpr bool kAlias = D == 128;               // P in the columns of S
  static constexpr uint32_t kP = kAlias ? 0 : 128, kO = kAlias ? 128 : 192;
};

struct TcArgs {
  int phase, splits, blocks, slot0, direct, early, two;
  int tile;   // keys of a tile
  int box;    // keys of a TMA box
  FastDiv by_splits, by_blocks, by_tile;
};

// kEdge: several tokens a sequence and own keys, so that rows of a tile see different keys.
template <int D, bool kEdge>
__global__ void __launch_bounds__(kTcThreads, 1) paged_tc_kernel(const __grid_constant__ CUtensorMap tk,
                                                                 const __grid_constant__ CUtensorMap tv,
                                                                 const __grid_constant__ Attn p, const TcArgs a) {
  using C = Tc<D>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t tc_smem_dyn[];
  uint8_t* base = (uint8_t*)(((uintptr_t)tc_smem_dyn + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = base;                       // [2][kTile]
  uint8_t* sK = sQ + 2 * C::kTile;          // [ST][kTile]
  uint8_t* sV = sK + ST * C::kTile;         // [ST][kTile]
  uint64_t* bars = (uint64_t*)(sV + ST * C::kTile);
  uint64_t *k_full = bars, *k_empty = bars + ST, *v_full = bars + 2 * ST, *v_empty = bars + 3 * ST;
  uint64_t* pipe_bars = bars + 4 * ST;      // per pipeline: q_full, s_full, s_free, p_full (two halves), o_full
  uint64_t* turns = pipe_bars + 12;         // [pipeline][warp of the warpgroup]: its exponentials may begin
  uint32_t* tmem_slot = (uint32_t*)(turns + 8);
  volatile uint32_t* again = tmem_slot + 1;            // the rows are computed again by slow_row
  float2* ml_smem = (float2*)((uint8_t*)bars + 512);   // [pipeline][row]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (!a.early) pdl_wait();   // see paged_rows.cu
  pdl_trigger();
  const int split_item = a.by_splits.div((int)blockIdx.x), split = (int)blockIdx.x - split_item * a.splits;
  const int block_item = a.by_blocks.div(split_item), block = split_item - block_item * a.blocks;
  const int who = p.by_K.div(block_item), kh = block_item - who * p.K;
  const int b0 = a.phase == kPrefix ? who * p.per : who;
  const int rows = (int)p.by_rows.d * (a.phase == kPrefix ? p.per : 1);
  const int r0 = block * (a.two ? 256 : 128);
  const Keys keys(p, a.phase, who);
  // own keys that the block's last row sees
  const int r_last = min(rows, r0 + (a.two ? 256 : 128)) - 1;
  const int n_own = a.phase == kPrefix ? 0 : max(0, keys.n_own - p.T + p.by_share.div(r_last) + 1);
  const int nt_pre = a.by_tile.div(keys.n_pre + a.tile - 1), nt = nt_pre + a.by_tile.div(n_own + a.tile - 1);
  const int per_split = a.by_splits.div(nt + a.splits - 1);
  const int t0 = min(nt, split * per_split), n_tiles = min(nt, t0 + per_split) - t0;
  // pipelines with work, and the consumers of a ring slot
  const int pipes = n_tiles == 0 ? 0 : a.two ? (r0 + 128 < rows ? 2 : 1) : (n_tiles > 1 ? 2 : 1);
  const int consumers = a.two ? pipes : 1;

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(smem_addr(&k_full[i]), 1);
      mbar_init(smem_addr(&k_empty[i]), max(1, consumers));
      mbar_init(smem_addr(&v_full[i]), 1);
      mbar_init(smem_addr(&v_empty[i]), max(1, consumers));
    }
    for (int s = 0; s < 2; ++s) {
      uint64_t* b = pipe_bars + 6 * s;
      mbar_init(smem_addr(&b[0]), 4);
      mbar_init(smem_addr(&b[1]), 1);
      mbar_init(smem_addr(&b[2]), 4);
      mbar_init(smem_addr(&b[3]), 4);
      mbar_init(smem_addr(&b[4]), 4);
      mbar_init(smem_addr(&b[5]), 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(smem_addr(&turns[i]), 1);
    *again = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  bool ok = true;

  if (warp >= 10) {
    // ------------------------------------------------ K (warp 10) and V (warp 11) copies, one lane per box
    const bool is_v = warp == 11;
    uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    uint8_t* ring = is_v ? sV : sK;
    const CUtensorMap* map = is_v ? &tv : &tk;
    // this lane's box of tile i: page id (-1: none) and slot
    auto look = [&](int i, int& slot, int& boxes) -> int {
      const int t = t0 + i;
      const bool own = t >= nt_pre;
      const int at = (own ? t - nt_pre : t) * a.tile, valid = min(a.tile, (own ? n_own : keys.n_pre) - at);
      boxes = p.page <= 128 ? p.by_page.div(valid + a.box - 1) : 1;   // a box is a page, or 128 keys of one
      if (lane >= boxes) return -1;
      const int pos = at + lane * a.box, page = p.by_page.div(pos);
      slot = pos - page * p.page;
      const int id = page_id((own ? keys.own : keys.pre)[page], p.n_pages);
      return id < 0 ? p.n_pages : id;   // past the pool: the map's fill value
    };
    int slot = 0, boxes = 0, id = n_tiles ? look(0, slot, boxes) : -1;
    int i = 0;
    for (; i < n_tiles && ok; ++i) {
      const int st = i % ST;
      int next_slot = 0, next_boxes = 0;
      const int next = i + 1 < n_tiles ? look(i + 1, next_slot, next_boxes) : -1;
      if (i >= ST && !mbar_wait(smem_addr(&empty[st]), (uint32_t)((i / ST - 1) & 1))) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(smem_addr(&full[st]), (uint32_t)(boxes * a.box * 128 * C::kPanels));
      __syncwarp();
      if (id >= 0) {
        const uint32_t dst = smem_addr(ring + st * C::kTile) + (uint32_t)(lane * a.box * 128);
#pragma unroll
        for (int c = 0; c < C::kPanels; ++c)
          tma_load_4d(dst + (uint32_t)(c * kPanel), map, smem_addr(&full[st]), c * 64, slot, kh, id);
      }
      id = next;
      slot = next_slot;
      boxes = next_boxes;
      if constexpr (kEdge) {
        // values that some row of the block does not see: see slow_row. This warp has the time, and the slot
        // is not filled again before it goes on.
        const int t = t0 + i, at = (t - nt_pre) * a.tile, valid = min(a.tile, n_own - at);
        const int edge = max(0, keys.n_own - p.T + p.by_share.div(r0) + 1);   // keys below: seen by all
        if (is_v && t >= nt_pre && at + valid > edge) {
          if (!mbar_wait(smem_addr(&full[st]), (uint32_t)((i / ST) & 1))) ok = false;
          bool odd = false;
#pragma unroll 4
          for (int k = lane; k < valid * 8 * C::kPanels; k += 32) {
            const int panel = k >= valid * 8;
            odd |= non_finite<__nv_bfloat16>(
                *reinterpret_cast<const uint4*>(ring + st * C::kTile + panel * kPanel + (k - panel * valid * 8) * 16));
          }
          if (odd) *again = 1;
        }
      }
    }
    // given up: the copies in flight land before the CTA's shared memory goes
    if (!ok)
      for (int j = max(0, i - ST); j < i; ++j) mbar_wait(smem_addr(&full[j % ST]), (uint32_t)((j / ST) & 1));
    if (kEdge && is_v) {
      __syncwarp();
      asm volatile("bar.sync 2, 288;" ::: "memory");   // with the softmax warps: `again` is said
    }
  } else if (warp >= 8) {
    // ------------------------------------------------ MMA issue, one lane per pipeline
    const int pipe = warp - 8;
    if (lane == 0 && pipe < pipes) {
      uint64_t* pb = pipe_bars + 6 * pipe;
      const uint32_t tm = *tmem_slot + (uint32_t)(pipe * 256);
      constexpr uint32_t idS = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t idO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
                               ((uint32_t)(128 >> 4) << 24);
      const int step = a.two ? 1 : 2, first = a.two ? 0 : pipe;
      // The lane's own instructions stand between a tile's softmax and its products, so what they
      // need is at hand before the waits: addresses, stage-0 descriptors, stages and parities.
      const uint32_t s_full = smem_addr(&pb[1]), s_free = smem_addr(&pb[2]), p_half0 = smem_addr(&pb[3]),
                     p_half1 = smem_addr(&pb[4]), o_full = smem_addr(&pb[5]);
      const uint32_t kf = smem_addr(k_full), ke = smem_addr(k_empty), vf = smem_addr(v_full), ve = smem_addr(v_empty);
      const uint64_t qd = desc_sw128(smem_addr(sQ + (a.two ? pipe : 0) * C::kTile));
      const uint64_t kd0 = desc_sw128(smem_addr(sK));
      // MN-major: the leading byte offset is the distance of the 64-column panels
      const uint64_t vd0 = desc_sw128(smem_addr(sV)) + ((uint64_t)((kPanel >> 4) - 1) << 16);
      int ks = first % ST, vs = ks;              // ring slots of the next S and the next PV
      uint32_t kpar = 0, vpar = 0;
      auto issue_s = [&](int g) {                // the pipeline's g-th tile
        const uint64_t kd = kd0 + (uint64_t)(ks * (C::kTile >> 4));
        if (!mbar_wait(kf + 8 * ks, kpar)) return false;
        if (!C::kAlias && g > 0 && !mbar_wait(s_free, (uint32_t)((g - 1) & 1))) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t o = (uint64_t)((k / 4) * (kPanel >> 4) + (k % 4) * 2);
          tc_mma(tm, qd + o, kd + o, idS, k > 0);
        }
        tc_commit(s_full);
        tc_commit(ke + 8 * ks);
        ks += step;
        if (ks >= ST) ks -= ST, kpar ^= 1;
        return true;
      };
      ok = mbar_wait(smem_addr(&pipe_bars[a.two ? 6 * pipe : 0]), 0) && issue_s(0);
      int g = 0;
      for (int i = first; ok && i < n_tiles; i += step, ++g) {
        const int t = t0 + i;
        const int valid = min(a.tile, t < nt_pre ? keys.n_pre - t * a.tile : n_own - (t - nt_pre) * a.tile);
        const int steps = (valid + 15) / 16;     // 16 keys: 8 columns of packed P, 2 KB of V rows
        const uint64_t vd = vd0 + (uint64_t)(vs * (C::kTile >> 4));
        const bool more = i + step < n_tiles;
        if (!C::kAlias && more && !(ok = issue_s(g + 1))) break;
        if (!(ok = mbar_wait(vf + 8 * vs, vpar) && mbar_wait(p_half0, (uint32_t)(g & 1)))) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < steps) tc_mma_ts(tm + C::kO, tm + C::kP + (uint32_t)(k * 8), vd + (uint64_t)(k * 128), idO, (k > 0 || g > 0) ? 1u : 0u);
        if (!(ok = mbar_wait(p_half1, (uint32_t)(g & 1)))) break;
        tc_fence_after();
        if (steps == 8) {
#pragma unroll
          for (int k = 4; k < 8; ++k) tc_mma_ts(tm + C::kO, tm + C::kP + (uint32_t)(k * 8), vd + (uint64_t)(k * 128), idO, 1u);
        } else {
          for (int k = 4; k < steps; ++k) tc_mma_ts(tm + C::kO, tm + C::kP + (uint32_t)(k * 8), vd + (uint64_t)(k * 128), idO, 1u);
        }
        if (C::kAlias && more) {                 // the arrival of the next S says that this PV is done
          tc_commit(ve + 8 * vs);
          if (!(ok = issue_s(g + 1))) break;
        } else {
          tc_commit(o_full);
          tc_commit(ve + 8 * vs);
        }
        vs += step;
        if (vs >= ST) vs -= ST, vpar ^= 1;
      }
    }
  } else {
    // ------------------------------------------------ softmax: thread = row = TMEM lane
    const int pipe = warp >> 2, rl = tid & 127;
    uint64_t* pb = pipe_bars + 6 * pipe;
    const int r = r0 + (a.two ? pipe * 128 : 0) + rl;
    const bool live = r < rows;
    int last;   // last own key of the row; below 0: padding
    {
      const Row at(p, b0, kh, live ? r : r0);
      last = a.phase == kPrefix ? 0 : keys.n_own - p.T + at.t;
      // Q into its tile (with two == 0 by pipeline 0 for both)
      if (pipes > 0 && (pipe == 0 || a.two)) {
        uint8_t* dst = sQ + (a.two ? pipe : 0) * C::kTile + rl * 128;
        const uint4* src = reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.q + at.b * p.q_b + at.h * p.q_h + at.t * p.q_t);
        uint4 x[D / 8];   // all of the row's loads before the first store
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = live ? src[c] : uint4{};
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4*>(dst + (c / 8) * kPanel + (((c & 7) ^ (rl & 7)) << 4)) = x[c];
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&pb[0]));
      }
    }
    const uint32_t tm = *tmem_slot + (uint32_t)(pipe * 256) + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = tm, tP = tm + C::kP, tO = tm + C::kO;
    const int seen_own = live ? max(0, last + 1) : 0;
    const int seen_pre = live && (a.phase == kPrefix || last >= 0) ? keys.n_pre : 0;
    float m = -INFINITY, l = 0.f, top = -INFINITY;   // top: the largest scaled score so far
    int g = 0;
    if (pipe < pipes) {
      const uint64_t sc2 = pack_f2(p.scale_log2, p.scale_log2);
      const int step = a.two ? 1 : 2;
      for (int i = a.two ? 0 : pipe; i < n_tiles; i += step, ++g) {
        const int tt = t0 + i;
        const bool own = tt >= nt_pre;
        const int at = (own ? tt - nt_pre : tt) * a.tile;
        const int nvalid = min(a.tile, (own ? seen_own : seen_pre) - at);   // of this row
        const int valid = min(a.tile, (own ? n_own : keys.n_pre) - at);     // of the tile
        if (ok && !mbar_wait(smem_addr(&pb[1]), (uint32_t)(g & 1))) ok = false;
        tc_fence_after();
        uint32_t s[128];
        auto load = [&](int n) {   // the first n scores, -inf for what the row does not see
#pragma unroll
          for (int c = 0; c < n; c += 32) tmem_ld32_nw(tS + (uint32_t)c, s + c);
          tmem_wait_ld();
          if (nvalid < n) {
#pragma unroll
            for (int k = 0; k < n; ++k)
              if (k >= nvalid) s[k] = 0xff800000u;
          }
        };
        load(128);
        auto row_max = [&]() {
          float m8[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) m8[k] = fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 8]));
#pragma unroll
          for (int k = 16; k < 128; k += 16)
#pragma unroll
            for (int c = 0; c < 8; ++c) m8[c] = fmax3(m8[c], __uint_as_float(s[k + c]), __uint_as_float(s[k + 8 + c]));
          return scaled(fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7])), p.scale_log2);
        };
        bool rescale = false;
        float alpha = 1.f;
        auto move_to = [&](float to) {   // also from m = -inf, no keys so far
          const float f = ex2(m - to);
          alpha *= f;
          l *= f;
          m = to;
          rescale = g > 0;
        };
        if (g == 0)
          m = row_max() + kTcFar;
        else if (top > m + (kTcRescale - kTcFar))
          move_to(top + kTcFar);
        // The two warps of a scheduler take turns at the exponentials, pipeline 0 first: while one's fill
        // the special-function unit the other's products run. Left alone the pipelines fall into step
        // and neither overlaps the other.
        if (pipes == 2 && (pipe == 1 || g > 0)) {
          if (ok && !mbar_wait(smem_addr(&turns[warp]), (uint32_t)((pipe == 1 ? g : g - 1) & 1))) ok = false;
        }
        uint64_t sum2[2];
        uint32_t w[32];
        // 64 keys from column c on: P into w, their sum
        auto exps = [&](int c, bool fresh) {
          const float from = m == -INFINITY ? 0.f : m;
          const uint64_t nm2 = pack_f2(-from, -from);
          if (fresh) sum2[0] = sum2[1] = 0ull;
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float x0, x1;
            unpack_f2(ffma2(pack_u2(s[c + 2 * k], s[c + 2 * k + 1]), sc2, nm2), x0, x1);
            const float p0 = ex2(x0), p1 = ex2(x1);
            sum2[k & 1] = fadd2(sum2[k & 1], pack_f2(p0, p1));
            w[k] = tc::pack2_bf16(p0, p1);
          }
        };
        exps(0, true);
        const float mx = row_max();   // beside the exponentials
        if (__any_sync(0xffffffffu, mx > m)) {
          if (mx > m) move_to(mx + kTcFar);
          load(64);
          exps(0, true);
        }
        top = mx;
        if (!C::kAlias) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&pb[2]));
        }
        // P's columns and O are free once the PV before has completed (aliased: before this S)
        if (!C::kAlias && g > 0) {
          if (ok && !mbar_wait(smem_addr(&pb[5]), (uint32_t)((g - 1) & 1))) ok = false;
          tc_fence_after();
        }
        tmem_st16(tP, w);
        tmem_st16(tP + 16, w + 16);
        if (__any_sync(0xffffffffu, rescale)) {   // whole warp: tcgen05.ld / st are warp-wide
          uint32_t o[32];
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            tmem_ld32(tO + (uint32_t)c, o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st32(tO + (uint32_t)c, o);
          }
        }
        if (valid & 15) {   // the last step's V rows behind the keys
          const int st = i % ST;
          if (ok && !mbar_wait(smem_addr(&v_full[st]), (uint32_t)((i / ST) & 1))) ok = false;
          const int clear = 16 - (valid & 15);
          for (int k = rl; k < clear * 8 * C::kPanels; k += 128)
            *reinterpret_cast<uint4*>(sV + st * C::kTile + (k / (clear * 8)) * kPanel + valid * 128 + (k % (clear * 8)) * 16) =
                uint4{};
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&pb[3]));   // the PV of the first 64 keys may run
        exps(64, false);
        tmem_st16(tP + 32, w);
        tmem_st16(tP + 48, w + 16);
        // the turn passes on behind the stores: without them the compiler moves the exponentials past it
        __syncwarp();
        if (pipes == 2 && lane == 0) mbar_arrive(smem_addr(&turns[warp ^ 4]));
        float s0, s1, s2, s3;
        unpack_f2(sum2[0], s0, s1);
        unpack_f2(sum2[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&pb[4]));
      }
      // the last PV: with aliased P the only one that arrives here
      if (ok && !mbar_wait(smem_addr(&pb[5]), C::kAlias ? 0u : (uint32_t)((g - 1) & 1))) ok = false;
      tc_fence_after();
    }
    // Row rr of the phase once more, key by key, by this warp.
    auto compute_again = [&](int rr) {
      const int te = t0 + n_tiles;
      const int j0 = t0 < nt_pre ? t0 * a.tile : keys.n_pre + (t0 - nt_pre) * a.tile;
      const int j1 = te <= nt_pre ? min(keys.n_pre, te * a.tile) : keys.n_pre + min(n_own, (te - nt_pre) * a.tile);
      const Row to(p, b0, kh, rr);
      const int end = keys.n_own - p.T + to.t;
      float rm, rls, acc[4];
      slow_row<__nv_bfloat16>(p, keys, kh, (const __nv_bfloat16*)p.q + to.b * p.q_b + to.h * p.q_h + to.t * p.q_t, j0,
                              a.phase == kPrefix ? j1 : end < 0 ? j0 : min(j1, keys.n_pre + end + 1), lane, rm, rls, acc);
      const int64_t at = ((int64_t)a.slot0 + split) * p.B * p.T * p.H + row_id(p, to.b, to.t, to.h);
      if (!a.direct && lane == 0) p.ml[at] = make_float2(rm, rls);
      for (int c = 0; c < D / 32; ++c) {
        if (a.direct)
          ((__nv_bfloat16*)p.out)[to.b * p.o_b + to.h * p.o_h + to.t * p.o_t + lane + 32 * c] =
              __float2bfloat16_rn(end < 0 ? 0.f : acc[c] / rls);
        else if (rls != 0.f)
          p.acc[at * D + lane + 32 * c] = acc[c];
      }
    };
    bool done = false;
    if constexpr (kEdge) {
      asm volatile("bar.sync 2, 288;" ::: "memory");
      done = *again != 0;
      if (done) {   // an infinity or NaN at the causal edge: the block's rows, a warp for each
        if (a.early) pdl_wait();
        for (int rr = r0 + warp; rr < min(rows, r0 + (a.two ? 256 : 128)); rr += 8) compute_again(rr);
      }
    }
    // The row's result: out, or its slot of partial results. Two pipelines on the same rows see each
    // other's (m, l) through shared memory and O in TMEM (same lanes), and write half the columns each.
    float scale0 = 1.f, scale1 = 0.f;   // of this pipeline's O, of the other's
    const bool shared_rows = !a.two && pipes == 2;
    if (shared_rows) {
      tc_fence_before();
      ml_smem[pipe * 128 + rl] = make_float2(m, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      tc_fence_after();
      const float2 o = ml_smem[(1 - pipe) * 128 + rl];
      const float to = fmaxf(m, o.x);
      scale0 = l == 0.f ? 0.f : ex2(m - to);
      scale1 = o.y == 0.f ? 0.f : ex2(o.x - to);
      l = l * scale0 + o.y * scale1;
      m = to;
    }
    if (a.early) pdl_wait();
    // Scores of 2^30 and more lose more in the fused operation (see kHugeScore) than the 2^16 between 1 and P can make
    // up for. Looking for them in every tile costs 1 to 4%: such rows are computed again.
    const bool huge = live && pipe < pipes && fabsf(m) > kTcHugeScore && !isinf(m);
    if (const uint32_t rest = __ballot_sync(0xffffffffu, huge); rest && !done && (a.two || pipe == 0))
      for (uint32_t left = rest; left; left &= left - 1) compute_again(r - lane + __ffs(left) - 1);
    const Row to_row(p, b0, kh, live ? r : r0);
    const int64_t at = ((int64_t)a.slot0 + split) * p.B * p.T * p.H + row_id(p, to_row.b, to_row.t, to_row.h);
    const bool mine = live && !done && !huge && (a.two || shared_rows || pipe == 0), none = l == 0.f;
    const uint32_t no_keys = last < 0 ? 0u : 0x7fc07fc0u;   // zeros for padding, else every score is -inf: 0 / 0
    if (mine && !a.direct && (a.two || pipe == 0)) p.ml[at] = make_float2(m, l);
    if (a.direct) {
      const float inv = none ? 0.f : 1.f / l;
      scale0 *= inv;
      scale1 *= inv;
    }
    auto put = [&](int c, const uint32_t (&o)[32]) {   // columns c .. c + 31 of the row
      if (!mine) return;
      if (a.direct) {
        uint4* dst = reinterpret_cast<uint4*>((__nv_bfloat16*)p.out + to_row.b * p.o_b + to_row.h * p.o_h + to_row.t * p.o_t + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t w[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            w[u] = none ? no_keys : tc::pack2_bf16(__uint_as_float(o[8 * k + 2 * u]), __uint_as_float(o[8 * k + 2 * u + 1]));
          dst[k] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else if (!none) {
        uint4* dst = reinterpret_cast<uint4*>(p.acc + at * D + c);
#pragma unroll
        for (int k = 0; k < 8; ++k) dst[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
      }
    };
    if (shared_rows) {
#pragma unroll 1
      for (int c = pipe * (D / 2); c < (pipe + 1) * (D / 2); c += 32) {
        uint32_t o[32], x[32];
        tmem_ld32(tO + (uint32_t)c, o);
        tmem_ld32((pipe == 0 ? tO + 256 : tO - 256) + (uint32_t)c, x);
#pragma unroll
        for (int k = 0; k < 32; ++k)
          o[k] = __float_as_uint(__uint_as_float(o[k]) * scale0 + __uint_as_float(x[k]) * scale1);
        put(c, o);
      }
    } else {
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32] = {};
        if (pipe < pipes) tmem_ld32(tO + (uint32_t)c, o);
        if (a.direct) {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * scale0);
        }
        put(c, o);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512u));
  }
}

// Whether the kernel serves the call: head size, pages that make tiles of whole 8-row swizzle atoms, 16-byte rows.
static bool tc_eligible(const Attn& p) {
  if (p.D != 64 && p.D != 128) return false;
  if (p.page % 8 || (p.page > 128 && p.page % 128)) return false;
  for (const void* x : {p.q, (const void*)p.out, p.k, p.v})
    if (!aligned(x, 16)) return false;
  for (int64_t s : {p.page_stride, p.head_stride, p.slot_stride})
    if (s % 8 || s <= 0 || s >= (1LL << 38)) return false;
  for (int64_t s : {p.q_b, p.q_h, p.q_t, p.o_b, p.o_h, p.o_t})
    if (s % 8) return false;
  return true;
}

static int page_map(CUtensorMap* map, const void* pages, const Attn& p, int box) {
  auto enc = tc::get_encode();
  if (!enc) return fail(GPT_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  cuuint64_t dims[4] = {(cuuint64_t)p.D, (cuuint64_t)p.page, (cuuint64_t)p.K, (cuuint64_t)p.n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)p.slot_stride * 2, (cuuint64_t)p.head_stride * 2, (cuuint64_t)p.page_stride * 2};
  cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pages), dims, strides, boxes, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GPT_ERR_CUDA, "cuTensorMapEncodeTiled (paged cache) failed (%d)", (int)r);
  return GPT_OK;
}

template <int D, bool kEdge>
static int launch_tc_d(const Attn& p, TcArgs a, cudaStream_t st) {
  static bool done[64] = {false};
  static std::mutex mu;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> g(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(paged_tc_kernel<D, kEdge>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc<D>::kSmem);
      if (e != cudaSuccess) return fail(GPT_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      done[dev] = true;
    }
  }
  a.box = p.page < 128 ? p.page : 128;
  a.tile = 128 / a.box * a.box;
  CUtensorMap mk, mv;
  int s = page_map(&mk, p.k, p, a.box);
  if (!s) s = page_map(&mv, p.v, p, a.box);
  if (s) return s;
  const int64_t rows = (int64_t)p.T * p.share * (a.phase == kPrefix ? p.per : 1), block = a.two ? 256 : 128;
  const int64_t blocks = (rows + block - 1) / block;
  const int64_t grid = blocks * a.splits * p.K * (a.phase == kPrefix ? p.B / p.per : p.B);
  GPT_CHECK_SHAPE(grid < (1LL << 31), "gpt_attention_shared_prefix: too many rows for one call");
  a.blocks = (int)blocks;
  a.by_splits = FastDiv(a.splits);
  a.by_blocks = FastDiv(blocks);
  a.by_tile = FastDiv(a.tile);
  launch_pdl(paged_tc_kernel<D, kEdge>, dim3((unsigned)grid), dim3(kTcThreads), Tc<D>::kSmem, st, mk, mv, p, a);
  return launch_status("paged_tc");
}

static int launch_tc(const Attn& p, const TcArgs& a, cudaStream_t st) {
  if (a.phase != kPrefix && p.T > 1)
    return p.D == 64 ? launch_tc_d<64, true>(p, a, st) : launch_tc_d<128, true>(p, a, st);
  return p.D == 64 ? launch_tc_d<64, false>(p, a, st) : launch_tc_d<128, false>(p, a, st);
}

}  // namespace paged
}  // namespace gpt
