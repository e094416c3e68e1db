"""The paged key/value cache: appending (with rotation) and shared-prefix attention, against plain fp64.

Tolerances, with u the unit roundoff of the type (2^-8 for bf16, 2^-24 for fp32) and A = sum_j p_j |v_j|
computed beside the reference: the output is rounded once (u A) and, in bf16, the probabilities are rounded
before they meet the values (u A more); a score is a sum of head_dim products in fp32, off by at most
(head_dim + 2) 2^-24 S with S = max sum_d |q_d k_d| scale, which moves a probability by twice that relatively; the
exponential, the sums over n keys and the joins add (n + 32) 2^-24 A. A rotated pair is two products and a sum in
fp32 and one rounding: 4 * 2^-24 (|x0| + |x1|) + u |y|. Copies are exact.
"""
import math

import pytest
import torch

import cutilegpt_b200 as cg
from cutilegpt_b200 import _lib as L

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make(dtype, B, G, T, H, K, D, page, prefix, seq, seed=0, nhd=False, extra_pages=3, garbage=True, fused=True):
    """A cache with shuffled pages; slots behind a length hold NaN and infinities. prefix, seq: lists of lengths."""
    g = torch.Generator().manual_seed(seed)
    n_own = max(1, -(-max(list(seq) + [1]) // page)) + 1
    n_pre = -(-max(list(prefix) + [1]) // page) + 1 if G else 0
    total = B * n_own + G * n_pre + extra_pages
    order = torch.randperm(total, generator=g).int()
    shape = (total, page, K, D) if nhd else (total, K, page, D)
    kp, vp = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if nhd:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    table, ptable = order[:B * n_own].view(B, n_own), order[B * n_own:B * n_own + G * n_pre].view(G, n_pre) if G else None
    if garbage:
        junk = torch.tensor([float("nan"), float("inf"), -float("inf")])
        keep = torch.zeros(total, page, dtype=torch.bool)
        for tab, lens in ((table, seq), (ptable, prefix)):
            for row, n in enumerate(lens or []):
                i = torch.arange(n)
                if n:
                    keep[tab[row, i // page].long(), i % page] = True
        bad = (~keep)[:, None, :, None].expand(kp.shape)
        fill = junk[torch.arange(kp.numel()) % 3].view(kp.shape).to(dtype)
        kp.copy_(torch.where(bad, fill, kp))
        vp.copy_(torch.where(bad, fill, vp))
    cuda_pages = [x.transpose(1, 2).contiguous().cuda().transpose(1, 2) if nhd else x.contiguous().cuda() for x in (kp, vp)]
    args = [table.contiguous().cuda(), torch.tensor(seq, dtype=torch.int32).cuda()]
    if G:
        args += [ptable.contiguous().cuda(), torch.tensor(prefix, dtype=torch.int32).cuda()]
    q = torch.randn(B, T, H + 2 * K, D, generator=g).to(dtype) * 2
    qd = q.cuda()[:, :, :H].transpose(1, 2) if fused else q[:, :, :H].transpose(1, 2).contiguous().cuda()
    return cg.PagedKV(*cuda_pages, *args), qd


def reference(q, kv, scale):
    """fp64 outputs and their tolerances, row by row from the definition."""
    B, H, T, D = q.shape
    K, page = kv.n_kv_head, kv.k_pages.shape[2]
    kp, vp, qc = kv.k_pages.double().cpu(), kv.v_pages.double().cpu(), q.double().cpu()
    table, seq = kv.page_table.cpu().long(), kv.seq_lens.tolist()
    G = kv.prefix_table.shape[0] if kv.prefix_table is not None else 0
    out, tol = torch.zeros(B, H, T, D, dtype=torch.float64), torch.zeros(B, H, T, D, dtype=torch.float64)
    u = U[q.dtype]
    for b in range(B):
        rows = []
        if G:
            g = b // (B // G)
            i = torch.arange(int(kv.prefix_lens[g]))
            rows.append((kv.prefix_table[g].cpu().long()[i // page], i % page))
        i = torch.arange(seq[b])
        rows.append((table[b][i // page], i % page))
        pages, slots = torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows])
        m = len(pages) - seq[b]
        k, v = kp[pages, :, slots], vp[pages, :, slots]          # [n, K, D]
        for t in range(T):
            n = seq[b] - T + t + 1
            if n <= 0:
                continue
            n += m
            kk, vv = (x[:n].repeat_interleave(H // K, dim=1) for x in (k, v))
            s = torch.einsum("hd,nhd->hn", qc[b, :, t], kk) * scale
            S = (torch.einsum("hd,nhd->hn", qc[b, :, t].abs(), kk.abs()) * scale).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            out[b, :, t] = torch.einsum("hn,nhd->hd", p, vv)
            A = torch.einsum("hn,nhd->hd", p, vv.abs())
            off = 2 * (D + 2) * 2.0 ** -24 * S + (n + 32) * 2.0 ** -24
            tol[b, :, t] = A * ((2 * u if q.dtype == torch.bfloat16 else u) + off)
    return out, tol


def check_attention(q, kv, scale=None, **kw):
    got = cg.cutile_shared_prefix_attention(q, kv, scale, **kw)
    ref, tol = reference(q, kv, q.shape[-1] ** -0.5 if scale is None else scale)
    err = (got.double().cpu() - ref).abs()
    assert not got.isnan().any()
    assert (err <= tol).all(), f"off by {(err / tol.clamp_min(1e-300)).max().item()} of the tolerance"
    assert L.device_error() == 0
    return got


BF, F32 = torch.bfloat16, torch.float32
ATTENTION = [
    # dtype, B, G, T, H, K, D, page, prefix, seq
    (BF, 4, 1, 1, 12, 12, 64, 16, [96], [1, 5, 16, 17]),
    (BF, 3, 1, 1, 8, 2, 128, 64, [128], [64, 65, 1]),
    (F32, 5, 1, 1, 4, 4, 64, 16, [33], [1, 0, 31, 32, 47]),
    (BF, 6, 2, 1, 4, 4, 32, 32, [70, 1], [3, 0, 40, 1, 33, 64]),
    (BF, 6, 3, 5, 8, 2, 64, 32, [100, 5, 64], [5, 9, 3, 0, 77, 33]),      # rows of padding in sequences 2 and 3
    (F32, 6, 3, 5, 8, 2, 64, 32, [100, 5, 64], [5, 9, 3, 0, 77, 33]),
    (BF, 2, 0, 1, 8, 1, 128, 16, [], [513, 700]),                         # no prefix, one key head
    (BF, 2, 2, 1, 8, 1, 64, 16, [300, 40], [1, 130]),                     # a prefix each: nothing shared
    (BF, 3, 1, 1, 16, 1, 128, 128, [1000], [129, 1, 300]),
    (BF, 40, 1, 1, 8, 2, 64, 16, [517], [(7 * i) % 50 for i in range(40)]),
    (BF, 9, 1, 33, 4, 2, 64, 64, [190], [33, 40, 64, 65, 33, 10, 0, 100, 34]),
    (BF, 2, 1, 150, 4, 1, 128, 64, [260], [150, 400]),
    (BF, 1, 0, 300, 2, 2, 64, 64, [], [300]),                             # a plain causal prompt
    (BF, 2, 1, 257, 2, 2, 128, 16, [0], [257, 300]),                      # an empty prefix
    (F32, 2, 1, 40, 2, 1, 64, 16, [77], [40, 55]),
    (BF, 3, 1, 2, 6, 3, 80, 24, [50], [2, 25, 49]),                       # head and page sizes off the usual ones
    (BF, 3, 1, 2, 6, 3, 64, 24, [250], [2, 25, 149]),
    (BF, 3, 1, 1, 2, 2, 64, 1, [9], [2, 1, 5]),                           # pages of one position
    (BF, 3, 1, 1, 2, 2, 64, 256, [700], [2, 257, 300]),
    (BF, 3, 1, 1, 2, 2, 64, 200, [700], [2, 257, 400]),
    (F32, 3, 1, 3, 2, 1, 7, 5, [11], [3, 4, 20]),
    (BF, 3, 1, 3, 2, 1, 7, 5, [11], [3, 4, 20]),
    (BF, 2, 1, 1, 2, 1, 256, 16, [40], [3, 20]),
    (F32, 2, 1, 1, 2, 1, 256, 16, [40], [3, 20]),
    (BF, 70, 1, 2, 8, 2, 128, 16, [300], [2 + i for i in range(70)]),
    (BF, 1, 1, 1, 1, 1, 64, 16, [1], [1]),
    (BF, 130, 1, 1, 2, 1, 128, 64, [1025], [(i * 5) % 9 for i in range(130)]),
    (BF, 1, 0, 1, 2, 1, 128, 64, [], [9000]),                             # one sequence, dozens of shares of its keys
    (F32, 1, 0, 1, 1, 1, 64, 32, [], [5001]),
    (BF, 1, 0, 2, 3, 1, 7, 16, [], [3000]),
    (BF, 8, 1, 1, 1, 1, 64, 128, [20000], [9, 3, 1, 4, 100, 2, 7, 8]),    # many shares of the prefix
    (F32, 20, 1, 1, 4, 2, 32, 16, [700], [i % 7 for i in range(20)]),
    (BF, 3, 1, 20, 8, 1, 64, 16, [333], [20, 47, 90]),                    # rows of a sequence fill no tile, prefix shared
    (BF, 64, 1, 1, 32, 8, 128, 128, [33000], [(37 * i) % 2000 + 1 for i in range(64)]),   # prefix beside own parts
]


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_attention(case):
    kv, q = make(*case)
    check_attention(q, kv)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_nhd_pages_scale_and_given_out(dtype):
    kv, q = make(dtype, 4, 2, 2, 8, 4, 64, 16, [90, 20], [2, 40, 1, 33], seed=3, nhd=True)
    out = torch.full((4, 2, 8, 64), float("nan"), dtype=dtype, device="cuda")      # (B, T, H, D) layout
    got = check_attention(q, kv, scale=0.3, out=out.transpose(1, 2))
    assert got.data_ptr() == out.data_ptr() and not out.isnan().any()
    again = check_attention(q, kv, scale=0.3)
    assert torch.equal(again, out.transpose(1, 2))                                 # same order of sums every time


def test_attention_unaligned_views():
    """Rows and pages that start at odd elements."""
    kv, q = make(BF, 3, 1, 1, 4, 2, 64, 16, [40], [3, 17, 30], garbage=False)
    flat = torch.empty(kv.k_pages.numel() * 2 + 64, dtype=BF, device="cuda")
    n = kv.k_pages.numel()
    pages = [flat[1 + i * n:1 + (i + 1) * n].view(kv.k_pages.shape) for i in range(2)]
    pages[0].copy_(kv.k_pages)
    pages[1].copy_(kv.v_pages)
    odd = torch.empty(q.numel() + 3, dtype=BF, device="cuda")[3:].view(3, 4, 1, 64)
    odd.copy_(q)
    out = torch.empty(q.numel() + 5, dtype=BF, device="cuda")[5:].view(3, 4, 1, 64)
    check_attention(odd, cg.PagedKV(*pages, kv.page_table, kv.seq_lens, kv.prefix_table, kv.prefix_lens), out=out)
    check_attention(q, kv, out=out)


def test_attention_strides_of_single_dimensions():
    """The stride of a dimension of size 1 is never used, whatever it says."""
    kv, q = make(BF, 2, 1, 1, 4, 1, 64, 16, [40], [3, 17])
    kp, vp = (torch.as_strided(x, x.shape, (x.stride(0), 3, x.stride(2), 1)) for x in (kv.k_pages, kv.v_pages))
    odd = cg.PagedKV(kp, vp, kv.page_table, kv.seq_lens, kv.prefix_table, kv.prefix_lens)
    q1 = torch.as_strided(q, q.shape, (q.stride(0), q.stride(1), 5, 1), q.storage_offset())
    assert torch.equal(check_attention(q1, odd), cg.cutile_shared_prefix_attention(q, kv))


def test_attention_peaked_and_huge_scores():
    """Scores far apart (one key has all the weight) and near fp32's exponent range of 2^x."""
    kv, q = make(BF, 5, 1, 1, 4, 2, 64, 16, [300], [3, 17, 30, 1, 200], seed=5)
    check_attention(q, kv, scale=8.0)
    kv.k_pages.mul_(32)
    check_attention(q, kv, scale=4.0)


def test_attention_lengths_follow_device_memory():
    """Tables and lengths are read on the device: a captured call follows them."""
    kv, q = make(BF, 4, 1, 1, 4, 4, 64, 16, [128], [60, 33, 5, 1], garbage=False)
    out = torch.empty(q.shape, dtype=BF, device="cuda")
    ws = torch.empty(max(1, kv.workspace_bytes(4, 1)), dtype=torch.uint8, device="cuda")
    cg.cutile_shared_prefix_attention(q, kv, out=out, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cg.cutile_shared_prefix_attention(q, kv, out=out, workspace=ws)
    for seq, prefix in (([1, 2, 3, 4], [100]), ([64, 0, 64, 17], [0]), ([7, 40, 0, 1], [77])):
        kv.seq_lens.copy_(torch.tensor(seq))
        kv.prefix_lens.copy_(torch.tensor(prefix))
        g.replay()
        ref, tol = reference(q, kv, 0.125)
        assert ((out.double().cpu() - ref).abs() <= tol).all(), (seq, prefix)


def test_attention_on_another_stream():
    kv, q = make(BF, 4, 1, 1, 4, 4, 64, 16, [128], [60, 33, 5, 1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cg.cutile_shared_prefix_attention(q, kv)
    s.synchronize()
    ref, tol = reference(q, kv, 0.125)
    assert ((got.double().cpu() - ref).abs() <= tol).all()


def test_attention_bad_tables_and_lengths_are_reported():
    """A page id outside the pool reads as zeros, a length past the table is clamped; both are reported."""
    for dtype, T in ((BF, 1), (F32, 1), (BF, 40)):
        kv, q = make(dtype, 2, 1, T, 2, 2, 64, 16, [40], [T, T + 20], garbage=False)
        L.device_error()
        kv.page_table[1, 0] = kv.k_pages.shape[0] + 7
        kv.prefix_table[0, 1] = -5
        got = cg.cutile_shared_prefix_attention(q, kv)
        with pytest.raises(L.GptError):
            L.device_error()
        zero = torch.zeros(1, *kv.k_pages.shape[1:], dtype=dtype, device="cuda")
        pages = [torch.cat([x, zero]) for x in (kv.k_pages, kv.v_pages)]
        n = pages[0].shape[0] - 1
        table, ptable = kv.page_table.clone(), kv.prefix_table.clone()
        table[1, 0], ptable[0, 1] = n, n
        mended = cg.PagedKV(*pages, table, kv.seq_lens, ptable, kv.prefix_lens)
        ref, tol = reference(q, mended, 0.125)
        assert ((got.double().cpu() - ref).abs() <= tol).all()
        cap = kv.page_table.shape[1] * 16
        kv.page_table[1, 0] = 0
        kv.prefix_table[0, 1] = 1
        kv.seq_lens.copy_(torch.tensor([cap + 9, -3]))
        got = cg.cutile_shared_prefix_attention(q, kv)
        with pytest.raises(L.GptError):
            L.device_error()
        kv.seq_lens.copy_(torch.tensor([cap, 0]))
        ref, tol = reference(q, kv, 0.125)
        assert ((got.double().cpu() - ref).abs() <= tol).all()


def test_attention_long_pool_offsets():
    """Pages whose offsets pass 2^31 elements."""
    page, D = 64, 128
    n_pages = 2 ** 31 // (page * D) + 8
    kp = torch.empty(n_pages, 1, page, D, dtype=BF, device="cuda")
    vp = torch.empty(n_pages, 1, page, D, dtype=BF, device="cuda")
    last = [n_pages - 1, n_pages - 2, n_pages - 3]
    g = torch.Generator().manual_seed(1)
    kv = cg.PagedKV(kp, vp, torch.tensor([[last[0]], [last[1]]], dtype=torch.int32, device="cuda"),
                    torch.tensor([64, 3], dtype=torch.int32, device="cuda"),
                    torch.tensor([[last[2]]], dtype=torch.int32, device="cuda"),
                    torch.tensor([50], dtype=torch.int32, device="cuda"))
    k, v = (torch.randn(2, 1, 64, D, generator=g).to(BF).cuda() for _ in range(2))
    for i in last:
        kp[i].copy_(k[0])
        vp[i].copy_(v[1])
    kv2_seq = kv.seq_lens.clone()
    kv.seq_lens.fill_(64)
    cg.cutile_paged_kv_append(None, k, v, kv)                                      # all 64 slots of both sequences
    assert torch.equal(kp[last[1]], k[1]) and torch.equal(vp[last[0]], v[0])
    kv.seq_lens.copy_(kv2_seq)
    q = torch.randn(2, 4, 1, D, generator=g).to(BF).cuda()
    got = cg.cutile_shared_prefix_attention(q, kv)
    pages = [torch.stack([x[i] for i in last]) for x in (kp, vp)]
    small = cg.PagedKV(*pages, torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"), kv.seq_lens,
                       torch.tensor([[2]], dtype=torch.int32, device="cuda"), kv.prefix_lens)
    ref, tol = reference(q, small, D ** -0.5)
    assert ((got.double().cpu() - ref).abs() <= tol).all()


def test_attention_empty_batch_and_no_tokens():
    kv, q = make(BF, 2, 1, 1, 2, 2, 64, 16, [40], [3, 4])
    assert cg.cutile_shared_prefix_attention(q[:, :, :0], kv).shape == (2, 2, 0, 64)
    none = cg.PagedKV(kv.k_pages, kv.v_pages, kv.page_table[:0], kv.seq_lens[:0])
    assert cg.cutile_shared_prefix_attention(q[:0], none).shape == (0, 2, 1, 64)
    cg.cutile_paged_kv_append(None, q[:0], q[:0], none)


# ----------------------------------------------------------------- append
def turned(x, table, rot, interleaved):
    x = x.double().clone()
    half = rot // 2
    cos, sin = table[..., :half].double(), table[..., half:].double()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :half], x[..., half:rot])
    y0, y1 = a * cos - b * sin, a * sin + b * cos
    mag = a.abs() + b.abs()
    y, m = x.clone(), torch.zeros_like(x)
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = y0, y1
        m[..., 0:rot:2], m[..., 1:rot:2] = mag, mag
    else:
        y[..., :half], y[..., half:rot] = y0, y1
        m[..., :half], m[..., half:rot] = mag, mag
    return y, m


APPEND = [
    # dtype, B, G, T, H, K, D, page, rot, interleaved, seq, nhd, fused
    (BF, 4, 0, 1, 12, 12, 64, 16, 0, False, [1, 16, 17, 40], False, True),
    (BF, 3, 0, 1, 8, 2, 128, 64, 128, False, [1, 64, 65], False, True),
    (BF, 3, 1, 5, 8, 2, 128, 16, 64, True, [5, 20, 33], True, True),
    (F32, 4, 2, 7, 5, 5, 64, 16, 64, False, [7, 3, 0, 40], False, True),     # padding tokens, an idle sequence
    (F32, 2, 1, 33, 4, 1, 64, 32, 32, True, [33, 90], False, False),
    (BF, 2, 1, 3, 4, 2, 32, 16, 8, False, [3, 17], False, True),             # rotated part below a 16-byte vector
    (BF, 2, 1, 3, 4, 2, 80, 24, 48, False, [3, 50], False, True),
    (BF, 2, 1, 3, 4, 2, 80, 24, 20, True, [3, 50], False, True),
    (F32, 2, 0, 2, 3, 3, 7, 5, 6, False, [2, 11], False, True),
    (BF, 2, 0, 2, 3, 3, 7, 5, 4, True, [2, 11], True, True),
    (BF, 3, 1, 300, 4, 2, 64, 64, 64, False, [300, 301, 350], False, True),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:10]))
@pytest.mark.parametrize("in_place", [False, True])
def test_append(case, in_place):
    dtype, B, G, T, H, K, D, page, rot, interleaved, seq, nhd, fused = case
    prefix = [13 + 5 * g for g in range(G)]
    kv, _ = make(dtype, B, G, T, H, K, D, page, prefix, seq, seed=2, nhd=nhd, garbage=False)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(B, T, H + 2 * K, D, generator=g).to(dtype).cuda()
    q, k, v = (y.transpose(1, 2) if fused else y.transpose(1, 2).contiguous() for y in x.split([H, K, K], dim=2))
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    before = kv.k_pages.clone(), kv.v_pages.clone()
    n_pos = 13 + 5 * G + max(seq) + 1
    cos_sin = None
    if rot:
        angle = torch.arange(n_pos).double()[:, None] * 10000.0 ** (-torch.arange(rot // 2).double() / (rot // 2))
        cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
    got = cg.cutile_paged_kv_append(q, k, v, kv, cos_sin, interleaved, q_out=q if in_place and rot else None)
    assert L.device_error() == 0
    if not rot:
        assert got is q and torch.equal(q, q0)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    u = U[dtype]
    want_k, want_v = before[0].clone(), before[1].clone()
    tol_k = torch.zeros(want_k.shape, dtype=torch.float64, device="cuda")
    want_k = want_k.double()
    for b in range(B):
        for t in range(T):
            i = seq[b] - T + t
            if i < 0:
                if rot:
                    assert (got[b, :, t] == 0).all()
                continue
            pid, slot = int(kv.page_table[b, i // page]), i % page
            want_v[pid, :, slot] = v0[b, :, t]
            if rot:
                row = cos_sin[(prefix[b // (B // G)] if G else 0) + i]
                for src, is_q in ((q0, True), (k0, False)):
                    y, m = turned(src[b, :, t], row, rot, interleaved)
                    tol = (4 * 2.0 ** -24 * m + u * y.abs()) * (m > 0)
                    if is_q:
                        assert ((got[b, :, t].double() - y).abs() <= tol).all()
                    else:
                        want_k[pid, :, slot], tol_k[pid, :, slot] = y, tol
            else:
                want_k[pid, :, slot] = k0[b, :, t].double()
    assert torch.equal(kv.v_pages, want_v)
    assert ((kv.k_pages.double() - want_k).abs() <= tol_k).all()


def test_append_reports_positions_without_table_rows_and_bad_pages():
    kv, _ = make(BF, 2, 0, 1, 2, 2, 64, 16, [], [5, 9], garbage=False)
    x = torch.randn(3, 2, 2, 1, 64, device="cuda", dtype=BF)
    cos_sin = torch.ones(6, 32, device="cuda")
    before = kv.k_pages.clone()
    L.device_error()
    q = cg.cutile_paged_kv_append(x[0], x[1], x[2], kv, cos_sin)        # position 8 has no row
    with pytest.raises(L.GptError):
        L.device_error()
    assert (q[1] == 0).all() and (q[0] != 0).any()
    pid = int(kv.page_table[1, 0])
    assert (kv.k_pages[pid, :, 8] == 0).all() and torch.equal(kv.v_pages[pid, :, 8], x[2][1, :, 0])
    assert torch.equal(kv.k_pages[pid, :, :8], before[pid, :, :8])
    pages = kv.k_pages.clone(), kv.v_pages.clone()
    kv.page_table[:, 0] = torch.tensor([-1, kv.k_pages.shape[0]])
    cg.cutile_paged_kv_append(x[0], x[1], x[2], kv)
    with pytest.raises(L.GptError):
        L.device_error()
    assert torch.equal(kv.k_pages, pages[0]) and torch.equal(kv.v_pages, pages[1])


def test_append_then_attend_equals_causal_attention():
    """A prompt that goes through the paged cache attends like the framework's causal attention."""
    for dtype in (BF, F32):
        B, H, T, D, page = 2, 4, 200, 64, 16
        g = torch.Generator().manual_seed(4)
        q, k, v = (torch.randn(B, H, T, D, generator=g).to(dtype).cuda() for _ in range(3))
        n = -(-T // page)
        pages = torch.zeros(2, B * n + 1, H, page, D, dtype=dtype, device="cuda")
        kv = cg.PagedKV(pages[0], pages[1], torch.arange(1, B * n + 1, dtype=torch.int32, device="cuda").view(B, n),
                        torch.full((B,), T, dtype=torch.int32, device="cuda"))
        cg.cutile_paged_kv_append(None, k, v, kv)
        a = cg.cutile_shared_prefix_attention(q, kv).double()
        b = cg.cutile_causal_attention(q, k, v, H).double()
        # both are within (2 u + small) sum p |v| <= (2 u + small) max |v| of the same values
        assert (a - b).abs().max() <= 2 * (2 * U[dtype] + 1e-5) * v.double().abs().max()


# ----------------------------------------------------------------- refusals
def test_refusals():
    kv, q = make(BF, 4, 2, 1, 4, 2, 64, 16, [40, 3], [3, 4, 5, 6])
    kp, vp, pt, sl, ft, fl = kv._tensors
    bad = [
        (kp.cpu(), vp.cpu(), pt, sl), (kp, vp.float(), pt, sl), (kp.half(), vp.half(), pt, sl), (kp[0], vp[0], pt, sl),
        (kp, vp[:, :1], pt, sl), (kp.transpose(2, 3), vp.transpose(2, 3), pt, sl), (kp, vp, pt.long(), sl),
        (kp, vp, pt, sl.long()), (kp, vp, pt, sl[:3]), (kp, vp, pt[0], sl), (kp, vp, pt.t(), sl), (kp, vp, pt[:, :0], sl),
        (kp, vp, pt.cpu(), sl), (kp, vp, pt, sl, ft), (kp, vp, pt, sl, None, fl), (kp, vp, pt[:3], sl[:3], ft, fl),
        (kp, vp, pt, sl, ft, fl[:1]), (kp, vp, pt, sl, ft[:0], fl[:0]), (kp, None, pt, sl),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            cg.PagedKV(*args)
    for x in (q.cpu(), q.float(), q[:3], q[..., :32], q[:, :3], q[0]):
        with pytest.raises(ValueError):
            cg.cutile_shared_prefix_attention(x, kv)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            cg.cutile_shared_prefix_attention(q, kv, scale)
    with pytest.raises(ValueError):
        cg.cutile_shared_prefix_attention(q, kv, out=torch.empty(4, 4, 1, 32, dtype=BF, device="cuda"))
    with pytest.raises(ValueError):
        cg.cutile_shared_prefix_attention(q, kv, out=torch.empty(4, 4, 64, 1, dtype=BF, device="cuda"))
    need = kv.workspace_bytes(4, 1)
    if need:
        for ws in (torch.empty(need - 1, dtype=torch.uint8, device="cuda"), torch.empty(need, dtype=torch.uint8),
                   torch.empty(need + 16, dtype=torch.uint8, device="cuda")[3:]):
            with pytest.raises(ValueError):
                cg.cutile_shared_prefix_attention(q, kv, workspace=ws)
    k = torch.randn(4, 2, 1, 64, device="cuda", dtype=BF)
    table = torch.ones(50, 64, device="cuda")
    for args in ((q, k[:, :1], k, kv), (q, k, k[:, :, :0], kv), (q, k.float(), k, kv), (q, k, k.cpu(), kv),
                 (q, k, k, kv, table.double()), (q, k, k, kv, table[:, :63]), (q, k, k, kv, table.cpu()), (q, k, k, kv, table[0]),
                 (q, k, k, kv, torch.ones(50, 66, device="cuda")), (q, k, k, kv, table[:0]), (q[:3], k, k, kv, table),
                 (q, k, k, kv, table, False, q[:, :2]), (q, k, k, kv, None, False, q)):
        with pytest.raises(ValueError):
            cg.cutile_paged_kv_append(*args)
    assert L.device_error() == 0


def test_workspace_refusals():
    kv, q = make(BF, 4, 1, 1, 4, 2, 64, 16, [900], [3, 4, 5, 6])
    need = kv.workspace_bytes(4, 1)
    assert need > 0
    for ws in (torch.empty(need - 1, dtype=torch.uint8, device="cuda"), torch.empty(need, dtype=torch.uint8),
               torch.empty(need + 16, dtype=torch.uint8, device="cuda")[3:]):
        with pytest.raises(ValueError):
            cg.cutile_shared_prefix_attention(q, kv, workspace=ws)
    check_attention(q, kv, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dtype,interleaved,rot", [(BF, False, 128), (BF, True, 64), (F32, False, 64), (BF, False, 0)])
def test_append_many_tokens(dtype, interleaved, rot):
    """Prompts long enough for the variant that gives a thread two pairs of vectors."""
    B, T, H, K, D, page = 2, 2100, 24, 8, 128, 64
    n = -(-T // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = torch.zeros(2, B * n, K, page, D, dtype=dtype, device="cuda")
    order = torch.randperm(B * n, generator=g, device="cuda").int().view(B, n)
    kv = cg.PagedKV(pages[0], pages[1], order, torch.full((B,), T, dtype=torch.int32, device="cuda"))
    x = torch.randn(B, T, H + 2 * K, D, generator=g, device="cuda").to(dtype)
    q, k, v = (y.transpose(1, 2) for y in x.split([H, K, K], dim=2))
    table = torch.randn(T, rot, generator=g, device="cuda") if rot else None
    got = cg.cutile_paged_kv_append(q, k, v, kv, table, interleaved)
    in_order = [p[order.long()].transpose(1, 2).reshape(B, K, n * page, D)[:, :, :T] for p in pages]
    assert torch.equal(in_order[1], v)
    u = U[dtype]
    for have, src in ((got, q), (in_order[0], k)):
        if rot:
            y, m = turned(src, table, rot, interleaved)
            assert ((have.double() - y).abs() <= (4 * 2.0 ** -24 * m + u * y.abs()) * (m > 0)).all()
        else:
            assert torch.equal(have, src)


@pytest.mark.parametrize("case", [(BF, 3, 1, 4, 8, 2, 64, 16, [100], [4, 40, 77]), (F32, 3, 1, 4, 8, 2, 64, 16, [100], [4, 40, 77]),
                                  (BF, 3, 1, 33, 4, 2, 64, 64, [190], [33, 40, 64]), (BF, 2, 1, 150, 4, 1, 128, 64, [260], [150, 400]),
                                  (BF, 2, 0, 9, 2, 2, 128, 16, [], [9, 300]), (BF, 2, 1, 3, 2, 1, 7, 16, [20], [3, 30])],
                         ids=lambda c: "-".join(str(x) for x in (str(c[0])[6:],) + c[1:8]))
def test_attention_non_finite_values_of_later_tokens(case):
    """Keys and values of a token that hold infinities and NaN reach its own row and later ones, no earlier one."""
    kv, q = make(*case)
    dtype, B, G, T, page = case[0], case[1], case[2], case[3], case[7]
    seq, at = case[9], T // 2
    clean, tol = reference(q, kv, q.shape[-1] ** -0.5)
    for n, (pages, junk) in enumerate(((kv.v_pages, [float("inf"), float("nan")]), (kv.k_pages, [float("nan"), float("-inf")]))):
        for b in range(B):
            for t, x in zip((at, T - 1), junk):
                i = seq[b] - T + t
                pages[int(kv.page_table[b, i // page]), :, i % page] = x
        got = cg.cutile_shared_prefix_attention(q, kv).double().cpu()
        assert ((got[:, :, :at] - clean[:, :, :at]).abs() <= tol[:, :, :at]).all(), n
        assert not got[:, :, T - 1].isfinite().all(), n
    assert L.device_error() == 0
