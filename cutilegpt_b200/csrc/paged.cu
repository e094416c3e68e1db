// C entry points of the paged key/value cache and the plan of an attention
// call: which kernels run, over how many shares of the keys.
#include <math.h>

#include "paged.cuh"

namespace gpt {
namespace paged {

// Checks what both operators need of a cache description.
static int check_kv(const gpt_paged_kv* kv, const char* what) {
  GPT_CHECK_ARG(kv, "%s: null cache description", what);
  GPT_CHECK_SHAPE(kv->batch >= 0 && kv->batch < (1LL << 24) && kv->kv_heads > 0 && kv->kv_heads < (1 << 20) &&
                      kv->head_dim > 0 && kv->head_dim <= 256,
                  "%s: bad sizes batch=%lld kv_heads=%lld head_dim=%lld (1..256)", what, (long long)kv->batch,
                  (long long)kv->kv_heads, (long long)kv->head_dim);
  GPT_CHECK_SHAPE(kv->n_pages > 0 && kv->n_pages < (1LL << 31) && kv->page_size > 0 && kv->page_size < (1LL << 29),
                  "%s: bad sizes n_pages=%lld page_size=%lld", what, (long long)kv->n_pages, (long long)kv->page_size);
  GPT_CHECK_SHAPE(kv->page_stride >= 0 && kv->head_stride >= 0 && kv->slot_stride >= 0,
                  "%s: negative cache stride", what);
  GPT_CHECK_SHAPE(kv->max_pages > 0 && kv->max_pages <= (1LL << 29) / kv->page_size &&
                      kv->ld_page_table >= kv->max_pages,
                  "%s: page_table rows list %lld pages (row stride %lld) of %lld positions; a row lists 1 to 2^29 positions",
                  what, (long long)kv->max_pages, (long long)kv->ld_page_table, (long long)kv->page_size);
  GPT_CHECK_SHAPE(kv->n_groups >= 0 && (kv->n_groups == 0 || kv->batch % kv->n_groups == 0),
                  "%s: n_groups=%lld does not divide batch=%lld", what, (long long)kv->n_groups, (long long)kv->batch);
  if (kv->n_groups > 0)
    GPT_CHECK_SHAPE(kv->max_prefix_pages > 0 && kv->max_prefix_pages <= (1LL << 29) / kv->page_size &&
                        kv->ld_prefix_table >= kv->max_prefix_pages,
                    "%s: prefix_table rows list %lld pages (row stride %lld) of %lld positions; a row lists 1 to 2^29 positions",
                    what, (long long)kv->max_prefix_pages, (long long)kv->ld_prefix_table, (long long)kv->page_size);
  return GPT_OK;
}

static int check_kv_pointers(const gpt_paged_kv* kv, const char* what) {
  GPT_CHECK_ARG(kv->k_pages && kv->v_pages && kv->page_table && kv->seq_lens, "%s: null cache pointer", what);
  GPT_CHECK_ARG(kv->n_groups == 0 || (kv->prefix_table && kv->prefix_lens), "%s: null prefix pointer", what);
  return GPT_OK;
}

// The kernels of an attention call, in the order of preference for the calls that they can serve.
enum Kernel { kSimt = 0, kRows = 1, kTc = 2 };

// The stride of a dimension of one element says nothing: 8 keeps every alignment.
static int64_t used_stride(int64_t size, int64_t stride) { return size == 1 ? 8 : stride; }

// How an attention call runs.
struct Plan {
  int shared;              // the prefix apart from the own positions, once for a group
  Kernel pre, own;         // kernels of the two launches (own: of the only one without `shared`)
  int pre_splits, pre_two, own_splits, own_two;
  int n_pre, n_own;        // slots of partial results; n_own = 0: the own launch writes out
  int beside;              // the own launch runs beside the prefix launch and does not wait for it
  int64_t acc_floats;      // of the workspace: the accumulators, then the rows' (m, l)
  int64_t bytes;           // workspace
};

// Rows of a sequence and key head up to which the few-row kernel takes them.
constexpr int kFewRows = 16;
// Rows from which a sequence reads its group's prefix by itself: it fills a 128-row tile alone.
constexpr int kOwnTile = 128;

// Equal shares of `keys` keys for `items` CTAs: enough for `per_sm` CTAs on every SM, at least `least` keys in a share.
static int shares(int64_t items, int64_t keys, int sms, int per_sm, int64_t least) {
  const int64_t want = (per_sm * (int64_t)sms + items - 1) / (items > 0 ? items : 1);
  const int64_t most = (keys + least - 1) / least;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

static void plan_launch(Kernel kernel, int64_t rows, int64_t items, int64_t keys, int sms, int* splits, int* two,
                        int* slots) {
  // 256 rows on the same tiles, but for three 128-row blocks, which two pipelines of their own serve in 1.5 passes, not 2
  const int64_t tiles128 = (rows + 127) / 128;
  *two = kernel == kTc && tiles128 > 1 && tiles128 != 3;
  if (kernel == kTc) {
    // one CTA on an SM: no more than fit at once, a tile at least for a pipeline
    items *= (rows + (*two ? 255 : 127)) / (*two ? 256 : 128);
    const int64_t tile = *two ? 128 : 256, most = (keys + tile - 1) / tile, want = sms / (items > 0 ? items : 1);
    *splits = (int)(want < 1 ? 1 : want < most ? want : most < 1 ? 1 : most);
  } else {
    *splits = shares(items * ((rows + 15) / 16), keys, sms, 2, 128);
  }
  *slots = *splits;
}

// The plan for the best kernel allowed.
static Plan make_plan(int64_t T, int64_t H, const gpt_paged_kv* kv, int dtype, Kernel best) {
  int sms = device_sm_count();
  if (sms <= 0) sms = 148;
  Plan pl = {};
  const int64_t groups = kv->n_groups, per = groups > 0 ? kv->batch / groups : kv->batch;
  const int64_t rows = T * (H / kv->kv_heads), own_keys = kv->max_pages * kv->page_size;
  const int64_t pre_keys = groups > 0 ? kv->max_prefix_pages * kv->page_size : 0;
  // A prefix that is cheap to read for every sequence anew (from L2, by the CTAs that run anyway) saves a launch:
  // 4 samples behind 96 positions, 12 heads: 14 us a call with a launch of its own, 11 without.
  const int64_t size = dtype == GPT_F32 ? 4 : 2;
  const bool cheap = rows <= kFewRows && pre_keys <= 256 &&
                     kv->batch * kv->kv_heads * pre_keys * 2 * kv->head_dim * size <= (8 << 20);
  pl.shared = groups > 0 && per > 1 && !cheap && (best != kTc || rows < kOwnTile);
  // Few rows in all fill no 128-row tile: 8 prompts with 8 samples each, 25 heads: 37 us with the tcgen05 kernel
  // for the prefixes, 29 with the few-row one, whose CTAs run among the own launch's.
  pl.pre = best == kTc && rows * per <= kFewRows ? kRows : best;
  pl.own = best == kTc && rows <= kFewRows ? kRows : best;
  if (pl.shared) plan_launch(pl.pre, rows * per, groups * kv->kv_heads, pre_keys, sms, &pl.pre_splits, &pl.pre_two, &pl.n_pre);
  plan_launch(pl.own, rows, kv->batch * kv->kv_heads, own_keys + (pl.shared ? 0 : pre_keys), sms, &pl.own_splits, &pl.own_two,
              &pl.n_own);
  if (pl.shared && pl.pre == kTc && pl.own == kRows) {
    // A long prefix keeps the tensor cores busy, long own parts HBM: run beside each other they share the time. The
    // prefix gets n of the SMs (one CTA each), the own launch fills the others at once and the prefix's when they
    // end. Both times are estimated on the whole GPU, in us: pair of tiles 2.3 (D = 128) or 1.5, own keys (half of the
    // table's positions) at 5500 GB/s, or at 55 GB/s for each SM where fewer read; both end together with
    // sms pre / n = 100 own / (sms - n). B200, 128 sequences behind 64k positions, up to 4k own: 348 us one after
    // the other, 322 beside; 67 sequences behind 8k, up to 1k own (pre = 11 us): 54 and 53, so not for short ones.
    const int64_t blocks = groups * kv->kv_heads * ((rows * per + (pl.pre_two ? 255 : 127)) / (pl.pre_two ? 256 : 128));
    const double passes = (double)blocks * ((pre_keys + 127) / 128) / (pl.pre_two ? 1 : 2);
    const double pre = passes * (kv->head_dim > 64 ? 2.3 : 1.5) / sms;
    const double own = (double)kv->batch * kv->kv_heads * own_keys * 4 * kv->head_dim / 2 / 5.5e6;
    if (pre > 20 && own > 20) {
      const double n = (double)sms * sms * pre / (100 * own + sms * pre);
      const int splits = (int)(n / blocks + 0.999);
      if (splits < pl.pre_splits) {
        pl.pre_splits = pl.n_pre = splits < 1 ? 1 : splits;
        pl.beside = 1;
      }
    }
  }
  // one share: the kernel joins the prefix's slots itself and writes out (the tcgen05 kernel: where there are none;
  // the few-row kernel: as many as it has room for)
  if (pl.n_own == 1 && !pl.beside && (pl.own == kTc ? pl.n_pre == 0 : pl.own == kRows ? pl.n_pre <= kMaxSlots : true)) pl.n_own = 0;
  const int64_t parts = (int64_t)(pl.n_pre + pl.n_own) * kv->batch * T * H;
  pl.acc_floats = (parts * kv->head_dim + 3) / 4 * 4;
  pl.bytes = (pl.acc_floats + 2 * parts) * (int64_t)sizeof(float);
  return pl;
}

// The largest workspace over the kernels that the alignment of q and out may ask for.
static int64_t workspace_bytes(int64_t T, int64_t H, const gpt_paged_kv* kv, int dtype) {
  int64_t most = 0;
  for (int k = kSimt; k <= (dtype == GPT_BF16 ? kTc : kRows); ++k) {
    const int64_t n = make_plan(T, H, kv, dtype, (Kernel)k).bytes;
    most = n > most ? n : most;
  }
  return most;
}

template <typename T>
static int launch(Kernel kernel, const Attn& p, int phase, int splits, int two, int slot0, int direct, int early,
                  cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (kernel == kTc) {
      TcArgs a = {};
      a.phase = phase;
      a.splits = splits;
      a.two = two;
      a.slot0 = slot0;
      a.direct = direct;
      a.early = early;
      return launch_tc(p, a, st);
    }
  }
  if (kernel == kRows) {
    RowsArgs a = {};
    a.phase = phase;
    a.splits = splits;
    a.slot0 = slot0;
    a.direct = direct;
    a.early = early;
    // Two warps a CTA where four would not fit at once and a share's keys are few: a CTA's start and end then
    // weigh more than its steps, and smaller CTAs overlap more of them (B200, 768 and 1600 CTAs of up to 256
    // keys, D = 64: 14 and 37 us, with four warps 21 and 42; 536 CTAs of up to 1024 keys, D = 128: 69, with four 56).
    const int64_t rows = (int64_t)p.T * p.share * (phase == kPrefix ? p.per : 1);
    const int64_t ctas = (rows + 15) / 16 * splits * p.K * (phase == kPrefix ? p.B / p.per : p.B);
    const int64_t share_keys = ((int64_t)(phase == kOwn ? 0 : p.pcap) + (phase == kPrefix ? 0 : p.cap)) / splits;
    constexpr int fit = Rows<T, 64, 4>::kCtas;   // CTAs of four warps on an SM
    static_assert(fit == Rows<T, 32, 4>::kCtas && fit == Rows<T, 128, 4>::kCtas, "the same at every head size");
    a.two_warps = ctas > (int64_t)fit * device_sm_count() && share_keys <= 512;
    return launch_rows<T>(p, a, st);
  }
  return launch_simt<T>(p, phase, splits, slot0, direct, st);
}

template <typename T>
static int run(Attn& p, const Plan& pl, cudaStream_t st) {
  p.n_pre = pl.n_pre;
  p.n_own = pl.n_own;
  int s = GPT_OK;
  if (pl.shared) s = launch<T>(pl.pre, p, kPrefix, pl.pre_splits, pl.pre_two, 0, 0, 0, st);
  if (!s) s = launch<T>(pl.own, p, pl.shared ? kOwn : kAll, pl.own_splits, pl.own_two, pl.n_pre, pl.n_own == 0, pl.shared ? 1 + pl.beside : 0, st);
  if (!s && pl.n_own > 0) s = launch_join<T>(p, st);
  return s;
}

}  // namespace paged
}  // namespace gpt

extern "C" {

int gpt_paged_kv_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, void* q_out, const int64_t* q_out_strides, int64_t T, int64_t H,
                        const gpt_paged_kv* kv, const float* cos_sin, int64_t n_pos, int64_t rot, int interleaved,
                        int dtype, void* stream) {
  const char* what = "gpt_paged_kv_append";
  GPT_CHECK_DTYPE(dtype);
  int s = gpt::paged::check_kv(kv, what);
  if (s) return s;
  GPT_CHECK_SHAPE(T >= 0 && T < (1LL << 30) && H > 0 && H < (1 << 20), "%s: bad sizes T=%lld H=%lld", what, (long long)T,
                  (long long)H);
  GPT_CHECK_SHAPE(rot >= 0 && rot % 2 == 0 && rot <= kv->head_dim, "%s: rot=%lld must be even and at most head_dim=%lld",
                  what, (long long)rot, (long long)kv->head_dim);
  GPT_CHECK_SHAPE(rot == 0 || n_pos > 0, "%s: rotation needs a table of at least one position", what);
  if (kv->batch == 0 || T == 0) return GPT_OK;
  s = gpt::paged::check_kv_pointers(kv, what);
  if (s) return s;
  GPT_CHECK_ARG(k && v && k_strides && v_strides, "%s: null pointer", what);
  GPT_CHECK_ARG(rot == 0 || (q && q_out && q_strides && q_out_strides && cos_sin), "%s: rotation needs q, q_out and cos_sin",
                what);
  gpt::paged::Append p = {};
  const size_t es = dtype == GPT_F32 ? 4 : 2;
  bool wide = kv->head_dim * es % 16 == 0 && gpt::aligned(k, 16) && gpt::aligned(v, 16) && gpt::aligned(kv->k_pages, 16) &&
              gpt::aligned(kv->v_pages, 16) && kv->page_stride * es % 16 == 0 && kv->head_stride * es % 16 == 0 &&
              kv->slot_stride * es % 16 == 0;
  for (int i = 0; i < 3; ++i) {
    p.k_s[i] = k_strides[i];
    p.v_s[i] = v_strides[i];
    wide = wide && k_strides[i] * (int64_t)es % 16 == 0 && v_strides[i] * (int64_t)es % 16 == 0;
    if (rot) {
      p.q_s[i] = q_strides[i];
      p.o_s[i] = q_out_strides[i];
      wide = wide && q_strides[i] * (int64_t)es % 16 == 0 && q_out_strides[i] * (int64_t)es % 16 == 0;
    }
  }
  if (rot) {
    // the members of a pair in vectors of their own, or pairs inside a vector
    wide = wide && gpt::aligned(q, 16) && gpt::aligned(q_out, 16) && gpt::aligned(cos_sin, 16) &&
           (interleaved ? rot : rot / 2) * es % 16 == 0 && rot % 8 == 0;
  }
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.k_pages = kv->k_pages;
  p.v_pages = kv->v_pages;
  p.page_stride = kv->page_stride;
  p.head_stride = kv->head_stride;
  p.slot_stride = kv->slot_stride;
  p.n_pages = (int)kv->n_pages;
  p.page = (int)kv->page_size;
  p.table = kv->page_table;
  p.ld_table = kv->ld_page_table;
  p.cap = (int)(kv->max_pages * kv->page_size);
  p.seq_lens = kv->seq_lens;
  p.plens = kv->n_groups > 0 ? kv->prefix_lens : nullptr;
  p.pcap = kv->n_groups > 0 ? (int)(kv->max_prefix_pages * kv->page_size) : 0;
  p.per = (int)(kv->n_groups > 0 ? kv->batch / kv->n_groups : kv->batch);
  p.cos_sin = cos_sin;
  p.n_pos = n_pos;
  p.rot = (int)rot;
  p.interleaved = interleaved != 0;
  p.T = (int)T;
  p.K = (int)kv->kv_heads;
  p.D = (int)kv->head_dim;
  p.B = (int)kv->batch;
  const int64_t heads = 2 * kv->kv_heads + (rot ? H : 0);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == GPT_BF16)
    return wide ? gpt::paged::launch_append<__nv_bfloat16, 8>(p, heads, st)
                : gpt::paged::launch_append<__nv_bfloat16, 1>(p, heads, st);
  return wide ? gpt::paged::launch_append<float, 4>(p, heads, st) : gpt::paged::launch_append<float, 1>(p, heads, st);
}

int64_t gpt_attention_shared_prefix_workspace_size(int64_t T, int64_t H, const gpt_paged_kv* kv, int dtype) {
  if (gpt::paged::check_kv(kv, "gpt_attention_shared_prefix_workspace_size") || (dtype != GPT_F32 && dtype != GPT_BF16) ||
      T <= 0 || H <= 0 || H % kv->kv_heads || kv->batch == 0)
    return 0;
  return gpt::paged::workspace_bytes(T, H, kv, dtype);
}

int gpt_attention_shared_prefix(const void* q, const int64_t* q_strides, void* out, const int64_t* out_strides, int64_t T,
                                int64_t H, const gpt_paged_kv* kv, float scale, void* workspace, int64_t workspace_bytes,
                                int dtype, void* stream) {
  const char* what = "gpt_attention_shared_prefix";
  GPT_CHECK_DTYPE(dtype);
  int s = gpt::paged::check_kv(kv, what);
  if (s) return s;
  GPT_CHECK_SHAPE(T >= 0 && H > 0 && H % kv->kv_heads == 0, "%s: H=%lld must be a multiple of kv_heads=%lld, T=%lld", what,
                  (long long)H, (long long)kv->kv_heads, (long long)T);
  GPT_CHECK_SHAPE(T < (1LL << 30) && H < (1 << 20) && (kv->batch == 0 || T * H <= (1LL << 30) / kv->batch),
                  "%s: more than 2^30 rows", what);
  GPT_CHECK_ARG(scale > 0.f && isfinite(scale), "%s: scale must be positive and finite", what);
  if (kv->batch == 0 || T == 0) return GPT_OK;
  s = gpt::paged::check_kv_pointers(kv, what);
  if (s) return s;
  GPT_CHECK_ARG(q && out && q_strides && out_strides, "%s: null pointer", what);
  gpt::paged::Attn p = {};
  p.q = q;
  p.out = out;
  using gpt::paged::used_stride;
  p.q_b = used_stride(kv->batch, q_strides[0]);
  p.q_h = used_stride(H, q_strides[1]);
  p.q_t = used_stride(T, q_strides[2]);
  p.o_b = used_stride(kv->batch, out_strides[0]);
  p.o_h = used_stride(H, out_strides[1]);
  p.o_t = used_stride(T, out_strides[2]);
  p.k = kv->k_pages;
  p.v = kv->v_pages;
  p.page_stride = used_stride(kv->n_pages, kv->page_stride);
  p.head_stride = used_stride(kv->kv_heads, kv->head_stride);
  p.slot_stride = used_stride(kv->page_size, kv->slot_stride);
  p.n_pages = (int)kv->n_pages;
  p.page = (int)kv->page_size;
  p.table = kv->page_table;
  p.ld_table = kv->ld_page_table;
  p.cap = (int)(kv->max_pages * kv->page_size);
  p.seq_lens = kv->seq_lens;
  p.per = (int)kv->batch;
  if (kv->n_groups > 0) {
    p.ptable = kv->prefix_table;
    p.ld_ptable = kv->ld_prefix_table;
    p.pcap = (int)(kv->max_prefix_pages * kv->page_size);
    p.plens = kv->prefix_lens;
    p.per = (int)(kv->batch / kv->n_groups);
  }
  p.B = (int)kv->batch;
  p.T = (int)T;
  p.H = (int)H;
  p.K = (int)kv->kv_heads;
  p.share = (int)(H / kv->kv_heads);
  p.D = (int)kv->head_dim;
  p.by_page = gpt::paged::FastDiv(p.page);
  p.by_K = gpt::paged::FastDiv(p.K);
  p.by_share = gpt::paged::FastDiv(p.share);
  p.by_rows = gpt::paged::FastDiv((int64_t)p.T * p.share);
  p.by_per = gpt::paged::FastDiv(p.per);
  p.scale_log2 = scale * gpt::paged::kLog2e;
  const gpt::paged::Kernel best = dtype == GPT_BF16 && gpt::paged::tc_eligible(p)              ? gpt::paged::kTc
                                  : gpt::paged::rows_eligible(p, dtype == GPT_BF16 ? 2 : 4) ? gpt::paged::kRows
                                                                                            : gpt::paged::kSimt;
  const gpt::paged::Plan pl = gpt::paged::make_plan(T, H, kv, dtype, best);
  const int64_t need = gpt::paged::workspace_bytes(T, H, kv, dtype);
  GPT_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace of %lld bytes required", what,
                (long long)need);
  GPT_CHECK_ALIGN(need == 0 || gpt::aligned(workspace, 16), "%s: workspace needs 16-byte alignment", what);
  p.acc = (float*)workspace;
  p.ml = (float2*)((float*)workspace + pl.acc_floats);
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == GPT_BF16 ? gpt::paged::run<__nv_bfloat16>(p, pl, st) : gpt::paged::run<float>(p, pl, st);
}

}  // extern "C"
