"""The paged key/value cache at the edges of its contract: infinities, NaN and huge values against the definition,
lengths past a table, calls from several threads, outputs given by the caller.

The tolerance of a finite result is that of test_paged_kv_gpu.py, with the keys of weight 0 (a score of -inf) left out
of its largest score: A (2 u + off) in bf16, A (u + off) in fp32, A = sum_j p_j |v_j| and off = 2 (head_dim + 2) 2^-24 S
+ (n + 32) 2^-24. NaN and infinities have to be where the definition has them.
"""
import threading

import pytest
import torch

import cutilegpt_b200 as cg
from cutilegpt_b200 import _lib as L
from test_paged_kv_gpu import BF, F32, U, make

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def definition(q, kv, scale):
    """fp64 outputs and tolerances, row by row: only what a row sees is looked at."""
    B, H, T, D = q.shape
    page = kv.k_pages.shape[2]
    kp, vp, qc = kv.k_pages.double().cpu(), kv.v_pages.double().cpu(), q.double().cpu()
    table, seq = kv.page_table.cpu().long(), kv.seq_lens.tolist()
    G = kv.prefix_table.shape[0] if kv.prefix_table is not None else 0
    out, tol = torch.zeros(B, H, T, D, dtype=torch.float64), torch.zeros(B, H, T, D, dtype=torch.float64)
    for b in range(B):
        i = torch.arange(seq[b])
        pages, slots = table[b][i // page], i % page
        if G:
            g = b // (B // G)
            i = torch.arange(int(kv.prefix_lens[g]))
            pages = torch.cat([kv.prefix_table[g].cpu().long()[i // page], pages])
            slots = torch.cat([i % page, slots])
        for t in range(T):
            if seq[b] - T + t < 0:
                continue
            n = len(pages) - T + t + 1
            k, v = (x[pages[:n], :, slots[:n]].repeat_interleave(H // kv.n_kv_head, dim=1) for x in (kp, vp))
            terms = qc[b, :, t] * k * scale                                  # [n, H, D]
            s = terms.sum(-1)
            S = torch.where(s.isfinite(), terms.abs().sum(-1), 0.0).amax(0)   # [H]
            p = torch.softmax(s, 0)[..., None]
            out[b, :, t] = (p * v).sum(0)
            off = 2 * (D + 2) * 2.0 ** -24 * S + (n + 32) * 2.0 ** -24
            tol[b, :, t] = (p * v.abs()).sum(0) * ((2 if q.dtype == BF else 1) * U[q.dtype] + off)[:, None]
    return out, tol


def check(q, kv, scale=None):
    got = cg.cutile_shared_prefix_attention(q, kv, scale).double().cpu()
    ref, tol = definition(q, kv, q.shape[-1] ** -0.5 if scale is None else scale)
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.isinf(), ref.isinf()) and torch.equal(got[ref.isinf()], ref[ref.isinf()])
    fin = ref.isfinite()
    off = (got - ref).abs()[fin] / tol[fin].clamp_min(1e-300)
    assert off.numel() == 0 or off.max() <= 1, f"off by {off.max().item()} of the tolerance"
    assert L.device_error() == 0
    return ref


def spot(kv, b, i):
    """Page and slot of own position i of sequence b."""
    page = kv.k_pages.shape[2]
    return int(kv.page_table[b, i // page]), i % page


def prefix_spot(kv, g, i):
    page = kv.k_pages.shape[2]
    return int(kv.prefix_table[g, i // page]), i % page


# ------------------------------------------------------------------ NaN in keys
FEW_ROWS = [
    # dtype, B, G, T, H, K, D, page, prefix, seq: served by the few-row kernel
    (BF, 2, 0, 1, 4, 2, 64, 16, [], [17, 40]),
    (BF, 2, 0, 1, 4, 2, 128, 16, [], [17, 65]),
    (F32, 2, 0, 1, 4, 2, 64, 16, [], [17, 40]),
    (BF, 2, 1, 1, 8, 4, 32, 16, [40], [17, 3]),
    (BF, 3, 1, 1, 4, 4, 64, 16, [700], [5, 33, 17]),        # the prefix in slots of its own
    (F32, 3, 1, 1, 2, 2, 128, 16, [700], [5, 33, 9]),
    (BF, 1, 0, 3, 4, 4, 64, 16, [], [35]),
]


def nan_keys_one_by_one(case):
    """NaN in the key of one position at a time, then in the keys of one page."""
    kv, q = make(*case)
    seq, prefix, page = case[9], case[8], case[7]
    clean = kv.k_pages.clone()
    for b, n in enumerate(seq):
        for i in sorted({0, n // 2, n - 1}):
            pid, slot = spot(kv, b, i)
            kv.k_pages[pid, :, slot] = NAN
            assert check(q, kv)[b].isnan().any()
            kv.k_pages.copy_(clean)
    for g, n in enumerate(prefix):
        for i in sorted({0, n // 2, n - 1}):
            pid, slot = prefix_spot(kv, g, i)
            kv.k_pages[pid, :, slot] = NAN
            assert check(q, kv).isnan().any()
            kv.k_pages[pid] = NAN                             # a whole page
            assert check(q, kv).isnan().any()
            kv.k_pages.copy_(clean)


@pytest.mark.parametrize("case", FEW_ROWS, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_nan_keys_few_rows(case):
    """A key that is alone among what a warp, or a share of the keys, has met for a row."""
    nan_keys_one_by_one(case)


@pytest.mark.parametrize("case", [(BF, 3, 1, 1, 32, 1, 64, 16, [700], [5, 33, 17]), (BF, 1, 1, 40, 2, 1, 128, 64, [260], [140])],
                         ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_nan_keys_many_rows(case):
    nan_keys_one_by_one(case)


# ------------------------------------------------------------------ rows that are computed again
@pytest.mark.parametrize("case", [(BF, 2, 0, 4, 4, 4, 64, 16, [], [20, 50]), (F32, 2, 0, 4, 4, 4, 64, 16, [], [20, 50]),
                                  (BF, 1, 0, 40, 4, 1, 128, 64, [], [140])],
                         ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_nan_keys_beside_infinite_values(case):
    """An infinite value of the last token, and NaN in the first keys: every row sees these."""
    kv, q = make(*case)
    for b, n in enumerate(case[9]):
        for i in (0, 1):
            pid, slot = spot(kv, b, i)
            kv.k_pages[pid, :, slot] = NAN
        pid, slot = spot(kv, b, n - 1)
        kv.v_pages[pid, :, slot] = INF
    assert check(q, kv).isnan().all()


# ------------------------------------------------------------------ the kernel for all other sizes
SIMT = [
    (BF, 2, 0, 1, 3, 1, 7, 16, [], [40, 33]),
    (F32, 2, 0, 1, 3, 1, 7, 16, [], [70, 20]),
    (F32, 1, 0, 2, 2, 1, 7, 16, [], [3000]),                 # dozens of shares
    (BF, 2, 1, 1, 4, 2, 256, 16, [40], [3, 20]),
]


@pytest.mark.parametrize("case", SIMT, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_nan_keys_any_size(case):
    """NaN in the first keys, as many as a step takes, and in all of a query."""
    kv, q = make(*case)
    clean = kv.k_pages.clone()
    for b, n in enumerate(case[9]):
        for i in range(min(32, n)):
            pid, slot = spot(kv, b, i)
            kv.k_pages[pid, :, slot] = NAN
    assert check(q, kv).isnan().all()
    kv.k_pages.copy_(clean)
    q = q.clone()
    q[0, 0] = NAN
    assert check(q, kv)[0, 0].isnan().all()


# ------------------------------------------------------------------ scores of -inf
ALL_KERNELS = FEW_ROWS + SIMT + [
    (BF, 40, 1, 1, 2, 1, 64, 16, [517], [1 + i % 5 for i in range(40)]),     # 128-row tiles, the prefix in slots
    (BF, 1, 0, 150, 2, 1, 128, 64, [], [150]),
    (BF, 2, 1, 33, 2, 1, 64, 64, [190], [40, 33]),
    (BF, 1, 0, 300, 1, 1, 64, 64, [], [300]),
]


@pytest.mark.parametrize("case", ALL_KERNELS, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_rows_without_a_finite_score(case):
    """Every score of a row is -inf: 0 / 0, whichever kernel serves the call; padding stays zeros."""
    kv, q = make(*case, garbage=False)
    q = q.clone()
    q[..., 0] = q[..., 0].abs() + 0.5
    kv.k_pages[..., 0] = -INF
    assert check(q, kv).isnan().all()
    kv.seq_lens[0] = 0
    ref = check(q, kv)
    assert (ref[0] == 0).all() and ref[1:].isnan().all()


# ------------------------------------------------------------------ infinite and huge operands in fp32
FP32 = [
    (F32, 2, 0, 1, 4, 2, 64, 16, [], [17, 40]),
    (F32, 3, 1, 1, 2, 2, 128, 16, [700], [5, 33, 9]),
    (F32, 3, 1, 4, 4, 2, 32, 16, [50], [4, 20, 77]),
    (F32, 2, 0, 1, 3, 1, 7, 16, [], [17, 40]),               # the plain kernel
]


@pytest.mark.parametrize("case", FP32, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_fp32_infinite_keys_and_values(case):
    kv, q = make(*case, garbage=False)
    T, seq = case[3], case[9]
    clean = kv.k_pages.clone(), kv.v_pages.clone()
    q = q.clone()
    # first elements that fill fp32, that have 11 bits, and that lie just below and above such a number
    first = torch.tensor([0.7, 1.0, 1.5 - 2.0 ** -20, 1.5 + 2.0 ** -20, 4097.0 - 2.0 ** -9], device="cuda")
    q[..., 0] = first[torch.arange(q[..., 0].numel(), device="cuda") % 5].view(q.shape[:3])
    for b, n in enumerate(seq):
        pid, slot = spot(kv, b, (n - T) // 2)
        kv.k_pages[pid, :, slot, 0] = -INF                    # weight 0
        kv.v_pages[pid, :, slot] = 1000.0
    kv.k_pages[..., 0].clamp_(-INF, 1e-3)
    assert check(q, kv, 0.01).isfinite().all()
    for b, n in enumerate(seq):                               # seen by every row: +inf, -inf, and both
        for i, x in ((0, INF), (1, -INF)):
            pid, slot = spot(kv, b, max(0, min(i, n - T)))
            kv.k_pages[pid, :, slot] = 0.0
            kv.v_pages[pid, :, slot, 2 * i:2 * i + 3] = x
    ref = check(q, kv, 0.01)
    assert ref.isinf().any() and not ref.isnan().all()
    kv.k_pages.copy_(clean[0])
    kv.v_pages.copy_(clean[1])
    big = 3.4028234e38
    for b, n in enumerate(seq):                               # the largest number, of either sign, in one key's values
        pid, slot = spot(kv, b, n - 1)
        kv.v_pages[pid, :, slot, 0] = big
        kv.v_pages[pid, :, slot, 1] = -big
    assert check(q, kv, 0.01).isfinite().all()


@pytest.mark.parametrize("n,D", [(1, 64), (1, 128), (33, 32), (700, 64)])
def test_fp32_largest_numbers(n, D):
    """One key has all the weight, and its values are the largest numbers."""
    kv, q = make(F32, 1, 0, 1, 2, 2, D, 16, [], [n])
    q = torch.zeros_like(q)
    q[..., 0] = 1.0
    top = torch.tensor([3.4028235e38, 3.4028233e38, 3.402e38, -3.4028235e38], device="cuda")
    kv.k_pages[..., 0] = 0.0
    for i in {0, n // 2, n - 1}:
        pid, slot = spot(kv, 0, i)
        kv.k_pages[pid, :, slot, 0] = 900.0
        kv.v_pages[pid, :, slot] = top[torch.arange(D, device="cuda") % 4]
        assert check(q, kv, 0.5).isfinite().all()
        kv.k_pages[pid, :, slot, 0] = 0.0
        kv.v_pages[pid, :, slot] = 1.0


# ------------------------------------------------------------------ huge scores
RISING = [
    # enough sequences, groups and key heads that a CTA sees several tiles
    (BF, 40, 0, 17, 2, 2, 64, 64, [], [700 - i for i in range(40)]),
    (BF, 40, 0, 17, 2, 2, 128, 64, [], [700 - i for i in range(40)]),
    (BF, 40, 0, 17, 16, 2, 64, 64, [], [450 - i for i in range(40)]),        # 256 rows on the same tiles
    (BF, 40, 0, 17, 16, 2, 128, 64, [], [450 - i for i in range(40)]),
    (BF, 80, 40, 1, 18, 2, 64, 64, [600] * 40, [1 + i % 5 for i in range(80)]),
    (BF, 4, 1, 1, 2, 2, 64, 16, [517], [1, 2, 40, 300]),                     # the few-row kernel
]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("exponent", [20, 35, 60, 110])
@pytest.mark.parametrize("case", ALL_KERNELS + RISING[1:5:3], ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_huge_scores(case, exponent, sign):
    """Scores of 7 to 11 times 2^exponent, all exact: the keys with the largest share the weight, whatever its size."""
    kv, q = make(*case)
    q = torch.zeros_like(q)
    q[..., 0] = sign * 2.0 ** (exponent // 2)
    level = torch.arange(kv.k_pages[..., 0].numel(), device="cuda").view(kv.k_pages.shape[:3]) * 7 % 11 % 5 + 7
    kv.k_pages[..., 0] = level * 2.0 ** (exponent - exponent // 2)
    kv.k_pages[..., 1:] = 0.0
    for scale in (0.3, 0.123, 0.0717):
        assert check(q, kv, scale).isfinite().all()
    if case[3] > 1:                                          # rows that are computed again
        for b, n in enumerate(case[9]):
            pid, slot = spot(kv, b, n - 1)
            kv.v_pages[pid, :, slot] = INF
        check(q, kv, 0.123)


# ------------------------------------------------------------------ every row beside damaged tokens
DAMAGED = [
    (BF, 3, 1, 4, 8, 2, 64, 16, [100], [4, 40, 77]), (F32, 3, 1, 4, 8, 2, 64, 16, [100], [4, 40, 77]),
    (BF, 3, 1, 33, 4, 2, 64, 64, [190], [33, 40, 64]), (BF, 2, 1, 150, 4, 1, 128, 64, [260], [150, 400]),
    (BF, 2, 0, 9, 2, 2, 128, 16, [], [9, 300]), (BF, 2, 1, 3, 2, 1, 7, 16, [20], [3, 30]),
    (BF, 2, 1, 5, 2, 2, 64, 16, [700], [2, 30]), (F32, 2, 1, 5, 2, 2, 64, 16, [700], [2, 30]),   # padding among the rows
]


@pytest.mark.parametrize("what", ["values", "keys", "both"])
@pytest.mark.parametrize("case", DAMAGED, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_every_row_beside_damaged_tokens(case, what):
    """Two of the new tokens hold infinities and NaN: all rows, before, at and behind them, against the definition."""
    kv, q = make(*case)
    T, seq = case[3], case[9]
    for pages, junk in ((kv.v_pages, (INF, -INF, NAN)), (kv.k_pages, (-INF, NAN, INF))):
        if what != "both" and (pages is kv.v_pages) != (what == "values"):
            continue
        for b, n in enumerate(seq):
            for t, x in ((T // 2, junk[0]), (T - 1, junk[1 + b % 2])):
                i = n - T + t
                if i >= 0:
                    pid, slot = spot(kv, b, i)
                    pages[pid, :, slot] = x
    ref = check(q, kv)
    live = [b for b, n in enumerate(seq) if n >= T]
    assert ref[live, :, :T // 2].isfinite().all() and not ref[live, :, T - 1].isfinite().any()


# ------------------------------------------------------------------ tables for a server's longest context
WIDE = [
    (BF, 4, 1, 1, 12, 12, 64, 16, [96], [1, 5, 16, 17]),
    (BF, 67, 1, 1, 8, 2, 128, 64, [810], [i % 103 for i in range(67)]),
    (F32, 13, 1, 1, 3, 3, 64, 16, [103], [i % 8 for i in range(13)]),
    (BF, 48, 3, 5, 6, 2, 64, 32, [200, 33, 7], [5 + i % 50 for i in range(48)]),
    (BF, 2, 1, 40, 8, 2, 128, 64, [300], [40, 90]), (BF, 2, 0, 3, 2, 1, 7, 16, [], [3, 30]),
]


@pytest.mark.parametrize("width", [1000, 65536])
@pytest.mark.parametrize("case", WIDE, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_tables_wider_than_the_lengths(case, width):
    """Shares, joins and launches go by the tables' width; entries behind a length are no pages and are not read."""
    kv, q = make(*case)
    want = cg.cutile_shared_prefix_attention(q, kv).double().cpu()

    def widen(table):
        if table is None:
            return None
        wide = torch.full((table.shape[0], width // case[7]), -7, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        return wide

    kv2 = cg.PagedKV(kv.k_pages, kv.v_pages, widen(kv.page_table), kv.seq_lens, widen(kv.prefix_table), kv.prefix_lens)
    check(q, kv2)
    ref, tol = definition(q, kv, q.shape[-1] ** -0.5)
    assert ((want - ref).abs() <= tol).all()


# ------------------------------------------------------------------ the range of values
@pytest.mark.parametrize("exponent", [100, -100])
@pytest.mark.parametrize("case", RISING, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_large_values_behind_rising_scores(case, exponent):
    """Values of 2^100 whose scores rise by 12 to 27 (in powers of two) from tile to tile: the weights of the first
    tiles are what the sums are in units of until the kernel notices. And small values, which must not get lost."""
    kv, q = make(*case, garbage=False)
    page = case[7]
    q = torch.zeros_like(q)
    q[..., 0] = 1.0
    lists = [(kv.page_table[b], n) for b, n in enumerate(case[9])] + [(kv.prefix_table[g], n) for g, n in enumerate(case[8])]
    for row, n in lists:
        level = 0
        for i, pid in zip(range(0, n, page), row.tolist()):
            if i % 128 == 0 and i > 0:
                level += 10 + (i // 128 * 17) % 20
            kv.k_pages[pid, ..., 0] = level
    kv.v_pages.mul_(2.0 ** exponent)
    assert check(q, kv, 0.693).isfinite().all()


# ------------------------------------------------------------------ append past a table
@pytest.mark.parametrize("dtype,D,rot", [(BF, 64, 0), (BF, 64, 64), (F32, 64, 32), (BF, 7, 4), (F32, 7, 0)])
@pytest.mark.parametrize("T,past", [(1, 1), (5, 2), (5, 5), (5, 100), (3, 2 ** 31 - 1 - 48)])
def test_append_past_the_table(dtype, D, rot, T, past):
    """Tokens that fit go to their own positions, the others nowhere; no earlier position changes."""
    page, cap = 16, 48
    kv, _ = make(dtype, 2, 1, T, 4, 2, D, page, [20], [cap - 17, cap - 17], garbage=False)
    assert kv.page_table.shape[1] * page == cap
    kv.seq_lens.copy_(torch.tensor([cap + past, 30]))
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, h, T, D, generator=g).to(dtype).cuda() for h in (4, 2, 2))
    table = torch.randn(20 + cap + 8, rot, generator=g).cuda() if rot else None
    before = kv.k_pages.clone(), kv.v_pages.clone()
    L.device_error()
    got = cg.cutile_paged_kv_append(q, k, v, kv, table)
    with pytest.raises(L.GptError):
        L.device_error()
    after = kv.k_pages.clone(), kv.v_pages.clone()
    # the same with one call for each token that has a place
    kv.k_pages.copy_(before[0])
    kv.v_pages.copy_(before[1])
    want = torch.zeros_like(q) if rot else q
    for b, n in enumerate((cap + past, 30)):
        for t in range(T):
            i = n - T + t
            if i >= cap:
                continue
            one = cg.PagedKV(kv.k_pages, kv.v_pages, kv.page_table[b:b + 1], torch.tensor([i + 1], dtype=torch.int32).cuda(),
                             kv.prefix_table, kv.prefix_lens)
            x = cg.cutile_paged_kv_append(q[b:b + 1, :, t:t + 1], k[b:b + 1, :, t:t + 1], v[b:b + 1, :, t:t + 1], one, table)
            if rot:
                want[b, :, t] = x[0, :, 0]
    assert L.device_error() == 0
    assert torch.equal(after[0], kv.k_pages) and torch.equal(after[1], kv.v_pages)
    assert torch.equal(got, want)


# ------------------------------------------------------------------ steps that follow each other
@pytest.mark.parametrize("dtype,B,T,H,K,D,prefix,own", [
    (BF, 64, 1, 12, 12, 64, 768, 200), (BF, 60, 1, 32, 8, 128, 1100, 300), (BF, 48, 5, 24, 8, 64, 517, 130),
    (BF, 8, 20, 8, 2, 64, 700, 200), (F32, 13, 1, 12, 12, 64, 1003, 77), (BF, 4, 1, 12, 12, 64, 96, 16),
    (BF, 64, 1, 32, 8, 128, 33000, 2000)])
def test_steps_back_to_back(dtype, B, T, H, K, D, prefix, own):
    """Append and attention over and over on the same buffers, nothing between them: no step sees an earlier one's
    queries or keys, though the launches overlap. Lengths and tables change between two rounds."""
    steps = 24
    kv, _ = make(dtype, B, 1, T, H, K, D, 64, [prefix], [T + (i * 7) % (own - T) for i in range(B)], garbage=False)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(steps, B, T, H + 2 * K, D, generator=g, device="cuda").to(dtype)
    table = torch.randn(prefix + own + 64, D, generator=g, device="cuda")
    ws = torch.empty(max(16, kv.workspace_bytes(H, T)), dtype=torch.uint8, device="cuda")
    qbuf = torch.empty(B, H, T, D, dtype=dtype, device="cuda")
    outs = torch.empty(steps, B, H, T, D, dtype=dtype, device="cuda")
    lens = kv.seq_lens.clone(), kv.seq_lens.flip(0).contiguous()
    tables = kv.page_table.clone(), kv.page_table.flip(0).contiguous()

    def run(wait):
        for i in range(steps):
            if i % 8 == 0:
                kv.seq_lens.copy_(lens[i // 8 % 2])
                kv.page_table.copy_(tables[i // 8 % 2])
            q, k, v = (y.transpose(1, 2) for y in x[i].split([H, K, K], dim=2))
            cg.cutile_paged_kv_append(q, k, v, kv, table, q_out=qbuf)
            if wait:
                torch.cuda.synchronize()
            cg.cutile_shared_prefix_attention(qbuf, kv, out=outs[i], workspace=ws)
            if wait:
                torch.cuda.synchronize()
                qbuf.fill_(NAN)
                ws.fill_(255)

    pages = kv.k_pages.clone(), kv.v_pages.clone()
    run(True)
    want = outs.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(False)
    for again in (lambda: run(False), graph.replay, graph.replay):
        kv.k_pages.copy_(pages[0])
        kv.v_pages.copy_(pages[1])
        outs.fill_(NAN)
        again()
        assert torch.equal(outs, want)
    assert L.device_error() == 0


# ------------------------------------------------------------------ calls from several threads
def test_attention_from_several_threads():
    """Head sizes whose tiles need different amounts of shared memory, at the same time."""
    calls, kept = [], []
    for D in (256, 160, 200, 136) * 2:
        kv, q = make(F32, 2, 1, 5, 4, 1, D, 16, [40], [5, 20])
        want, out = cg.cutile_shared_prefix_attention(q, kv), torch.zeros(q.shape, device="cuda")
        ws = torch.empty(max(16, kv.workspace_bytes(4, 5)), dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        calls.append((q.data_ptr(), L.strides3(*q.stride()[:3]), out.data_ptr(), L.strides3(*out.stride()[:3]), 5, 4, kv._ref,
                      D ** -0.5, ws.data_ptr(), ws.numel(), L.GPT_F32, stream.cuda_stream))
        kept.append((kv, q, want, out, ws, stream))
    torch.cuda.synchronize()
    statuses, attend = [], L.lib().gpt_attention_shared_prefix

    def work(args):
        statuses.extend({attend(*args) for _ in range(2000)})

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert set(statuses) == {L.GPT_OK}
    for _, _, want, out, _, _ in kept:
        assert torch.equal(out, want)
    assert L.device_error() == 0


# ------------------------------------------------------------------ outputs given by the caller
class Producer:
    """An array of another library: DLPack and nothing else."""

    def __init__(self, t):
        self.t = t

    def __dlpack__(self, **kw):
        return self.t.__dlpack__(**kw)

    def __dlpack_device__(self):
        return self.t.__dlpack_device__()


def test_outputs_of_another_library():
    kv, q = make(BF, 3, 1, 2, 4, 2, 64, 16, [40], [3, 17, 30])
    want = cg.cutile_shared_prefix_attention(q, kv)
    out = torch.empty(q.shape, dtype=BF, device="cuda")
    got = cg.cutile_shared_prefix_attention(q, kv, out=Producer(out))
    assert torch.equal(out, want) and torch.equal(got, want)
    k = torch.randn(3, 2, 2, 64, device="cuda").to(BF)
    table = torch.randn(100, 64, device="cuda")
    want = cg.cutile_paged_kv_append(q, k, k, kv, table)
    got = cg.cutile_paged_kv_append(q, k, k, kv, table, q_out=Producer(out))
    assert torch.equal(out, want) and torch.equal(got, want)


def test_outputs_in_the_way_are_refused():
    kv, q = make(BF, 3, 1, 2, 4, 2, 64, 16, [40], [3, 17, 30])
    with pytest.raises(ValueError, match="memory"):
        cg.cutile_shared_prefix_attention(q, kv, out=q)
    square = torch.randn(3, 2, 2, 64, device="cuda").to(BF)
    kv2 = cg.PagedKV(kv.k_pages, kv.v_pages, kv.page_table, kv.seq_lens)
    table = torch.randn(100, 64, device="cuda")
    with pytest.raises(ValueError, match="strides"):
        cg.cutile_paged_kv_append(square, square.clone(), square.clone(), kv2, table, q_out=square.transpose(1, 2))
    got = cg.cutile_paged_kv_append(square.clone(), square, square, kv2, table)
    x = square.clone()
    assert torch.equal(cg.cutile_paged_kv_append(x, square, square, kv2, table, q_out=x), got)
    one = square[:, :, :1].clone()               # the stride of a dimension of size 1 says nothing
    want = cg.cutile_paged_kv_append(one, one, one, kv2, table)
    x = one.clone()
    other = torch.as_strided(x, x.shape, (x.stride(0), x.stride(1), 8, 1))
    assert torch.equal(cg.cutile_paged_kv_append(x, one, one, kv2, table, q_out=other), want) and torch.equal(x, want)


def test_tables_and_workspaces_of_another_library():
    kv, q = make(BF, 3, 1, 2, 4, 2, 64, 16, [900], [3, 17, 30])
    ws = torch.empty(kv.workspace_bytes(4, 2), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0
    assert torch.equal(cg.cutile_shared_prefix_attention(q, kv, workspace=Producer(ws)), cg.cutile_shared_prefix_attention(q, kv))
    k, table = torch.randn(3, 2, 2, 64, device="cuda").to(BF), torch.randn(950, 64, device="cuda")
    want = cg.cutile_paged_kv_append(q, k, k, kv, table)
    assert torch.equal(cg.cutile_paged_kv_append(q, k, k, kv, Producer(table)), want)
    for bad in ([1.0, 2.0], "table", Producer(table.double())):
        with pytest.raises(ValueError):
            cg.cutile_paged_kv_append(q, k, k, kv, bad)
