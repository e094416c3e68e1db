"""What is measured of the paged key/value cache: appending to it and attention over it.

Two operators. ``append`` takes the queries, keys and values of T new tokens of each of B sequences, turns
the queries and keys by their positions (or leaves them, for learned positions) and writes the keys and
values into the pages of the cache. ``attention`` lets the queries of the new tokens look at the cache:
first at the pages of a prefix that the sequences of a group have in common, then at the pages of their own
sequence, causally. Sequence b belongs to group b // (B // groups).

``seq_lens[b]`` counts the own keys of sequence b with the new tokens among them, so query t of sequence b
has index ``seq_lens[b] - T + t`` in it and sees the whole prefix and the own keys up to that index. A
sequence of length 0 is an idle slot of a batch: nothing is appended for it and its outputs are zeros.
"""
import math

import torch

own = False


# ------------------------------------------------------------------ the cases
def _append(name, batch, tokens, heads, kv_heads, dim, rot, interleaved, page, context, dtype):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "interleaved": interleaved, "page": page, "context": context, "dtype": dtype}


def _attention(name, batch, groups, tokens, heads, kv_heads, dim, page, prefix, suffix, idle, dtype):
    return {"name": name, "op": "attention", "batch": batch, "groups": groups, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "prefix": prefix, "suffix": suffix, "idle": idle,
            "dtype": dtype}


def listed():
    return [
        # one decode step of four samples of a 12-head model with learned positions: latency is all there is
        _append("append step small", 4, 1, 12, 12, 64, 0, False, 16, 100, "bf16"),
        # one decode step of a full serving batch, shared key heads, rotation over the whole head
        _append("append step batch", 256, 1, 32, 8, 128, 128, False, 64, 2000, "bf16"),
        # the prompts of a batch going into the cache, rotation of neighbouring pairs over a part of the head
        _append("append prompts", 8, 4093, 32, 8, 128, 64, True, 64, 4093, "bf16"),
        # odd sizes in full precision: 25 heads, 1021 tokens that end inside a page
        _append("append f32 odd", 5, 1021, 25, 25, 64, 64, False, 16, 1500, "f32"),
        # four samples of one short prompt, first steps of the generation
        _attention("samples small", 4, 1, 1, 12, 12, 64, 16, 96, 16, 0, "bf16"),
        # 64 samples of one prompt of 768 tokens, up to 256 generated: the benchmark's decode lengths
        _attention("samples 768+256", 64, 1, 1, 12, 12, 64, 16, 768, 256, 0, "bf16"),
        # eight prompts with eight samples each, 25 heads
        _attention("prompts x samples", 64, 8, 1, 25, 25, 64, 32, 700, 260, 0, "bf16"),
        # chat requests behind a long instruction, shared key heads, a few slots of the batch idle
        _attention("chat 8k", 67, 1, 1, 32, 8, 128, 64, 8100, 1024, 3, "bf16"),
        # the same with a book as the prefix and long answers: the largest traffic
        _attention("book 64k", 128, 1, 1, 32, 8, 128, 128, 65536, 4096, 0, "bf16"),
        # drafts of five tokens checked in one call, three groups
        _attention("drafts of 5", 48, 3, 5, 24, 8, 64, 32, 2047, 513, 0, "bf16"),
        # questions of 256 tokens behind a shared document, some after earlier ones: the largest arithmetic
        _attention("questions", 8, 1, 256, 32, 8, 128, 64, 4096, 700, 0, "bf16"),
        # full precision, lengths that end inside pages
        _attention("samples f32 odd", 13, 1, 1, 12, 12, 64, 16, 1003, 77, 1, "f32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    most = {op: [max(c[k] for c in costs) for k in ("bytes", "flops")] for op in ("append", "attention")
            for costs in [[work(c) for c in listed() if c["op"] == op]]}
    while True:
        dtype = "f32" if rng.random() < 0.15 else "bf16"
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12, 16, 25])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
        dim = rng.choice([64, 64, 128, 128, 32])
        page = rng.choice([16, 32, 64, 128])
        if heads > 64:
            continue
        if rng.random() < 0.3:
            batch, tokens = _log(rng, 1, 300), 1 if rng.random() < 0.4 else _log(rng, 2, 5000)
            case = _append("", batch, tokens, heads, kv_heads, dim, rng.choice([0, dim // 2, dim, dim]),
                           rng.random() < 0.5, page, tokens + rng.randrange(0, 2000), dtype)
            if work(case)["bytes"] > most["append"][0]:
                continue
        else:
            groups = rng.choice([1, 1, 1, 2, 3, 8])
            batch = groups * max(1, _log(rng, 1, 256) // groups)
            tokens = rng.choice([1, 1, 1, rng.randrange(2, 9), _log(rng, 16, 384)])
            prefix = _log(rng, 16, 40000)
            suffix = max(tokens, _log(rng, 1, 4500))
            idle = rng.choice([0, 0, min(batch - 1, 2)])
            if dtype == "f32":
                tokens, prefix, suffix = min(tokens, 8), min(prefix, 3000), max(min(tokens, 8), min(suffix, 500))
            case = _attention("", batch, groups, tokens, heads, kv_heads, dim, page, prefix, suffix, idle, dtype)
            cost, scores = work(case), batch * tokens * heads * (prefix + suffix)
            if cost["bytes"] > most["attention"][0] or cost["flops"] > most["attention"][1] or scores > 3e8:
                continue
        del case["name"]
        return case


# ------------------------------------------------------------------ sizes
def _lens(case):
    """Own lengths and prefix lengths as lists: the same ones for every seed (prepare shuffles the own ones)."""
    B, T = case["batch"], case["tokens"]
    if case["op"] == "append":
        return [T + (b * (case["context"] - T)) // max(1, B - 1) for b in range(B)], [0]
    live = B - case["idle"]
    seq = [0] * case["idle"] + [T + (b * (case["suffix"] - T)) // max(1, live - 1) for b in range(live)]
    G, P = case["groups"], case["prefix"]
    pre = [P - (g * (P // 3)) // max(1, G - 1) for g in range(G)]
    return seq, pre


def work(case):
    B, T, H, K, D = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
    size = 2 if case["dtype"] == "bf16" else 4
    seq, pre = _lens(case)
    if case["op"] == "append":
        rows = B * T
        kept = 2 * rows * 2 * K * D * size                                  # keys and values in, and into their pages
        turned = 2 * rows * H * D * size if case["rot"] else 0              # queries in and out
        table = len({n - T + t for n in set(seq) for t in range(T)}) * case["rot"] * 4
        return {"bytes": kept + turned + table, "flops": 3 * rows * (H + K) * case["rot"]}
    read = (sum(seq) + sum(pre)) * 2 * K * D * size
    rows = 2 * B * T * H * D * size
    tables = 4 * (B + len(pre) + sum(-(-n // case["page"]) for n in seq + pre))
    # keys seen by the queries of one head; the seed says which group a length falls to, so the mean prefix
    seen = sum(T * (sum(pre) / len(pre) + n) - T * (T - 1) // 2 for n in seq if n)
    return {"bytes": read + rows + tables, "flops": 4 * D * H * int(seen)}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    B, T, H, K, D, page = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "page"))
    seq, pre = _lens(case)
    n_own = -(-max(max(seq), 1) // page)
    n_pre = -(-max(pre) // page) if case["op"] == "attention" else 0
    total = B * n_own + len(pre) * n_pre + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    state = {"case": dict(case)}
    state["k_pages"], state["v_pages"] = normal(total, K, page, D), normal(total, K, page, D)
    state["page_table"] = order[:B * n_own].view(B, n_own).contiguous()
    shuffled = torch.randperm(B, generator=g, device="cuda")
    state["seq_lens"] = torch.tensor(seq, dtype=torch.int32, device="cuda")[shuffled].contiguous()
    state["prefix_table"] = state["prefix_lens"] = None
    if n_pre:
        state["prefix_table"] = order[B * n_own:B * n_own + len(pre) * n_pre].view(len(pre), n_pre).contiguous()
        state["prefix_lens"] = torch.tensor(pre, dtype=torch.int32, device="cuda")
    # queries, keys and values as a fused projection leaves them: [B, T, H + 2 K, D], read in place
    fused = normal(B, T, H + 2 * K, D)
    fused[:, :, :H] *= 2.0                                                  # scores with a spread of 2
    state["fused"] = fused
    state["q"], state["k"], state["v"] = (x.transpose(1, 2) for x in fused.split([H, K, K], dim=2))
    state["cos_sin"] = None
    if case.get("rot"):
        half = case["rot"] // 2
        inv = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(case["context"] + 1, device="cuda", dtype=torch.float64)[:, None] * inv
        state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()
    if own:  # the handle that a server keeps for its cache
        from cutilegpt_b200 import PagedKV
        state["kv"] = PagedKV(state["k_pages"], state["v_pages"], state["page_table"], state["seq_lens"],
                              state["prefix_table"], state["prefix_lens"])
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        import cutilegpt_b200 as cg
        if case["op"] == "append":
            q = cg.cutile_paged_kv_append(state["q"], state["k"], state["v"], state["kv"], state["cos_sin"],
                                          case["interleaved"])
            return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
        return {"out": cg.cutile_shared_prefix_attention(state["q"], state["kv"])}
    return _plain_append(state) if case["op"] == "append" else _plain_attention(state)


def _turned(x, table, rot, interleaved):
    """x [B, H, T, D] in 32 bits, the first `rot` values of each head turned by table [B, T, rot] (cosines, sines)."""
    cos, sin = (y[:, None] for y in table.chunk(2, dim=-1))
    part = x[..., :rot]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = part.chunk(2, dim=-1)
        part = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([part, x[..., rot:]], dim=-1)


def _plain_append(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    T, page = case["tokens"], case["page"]
    at = state["seq_lens"].long()[:, None] - T + torch.arange(T, device=q.device)          # [B, T]
    if case["rot"]:
        table = state["cos_sin"][at]
        q = _turned(q.float(), table, case["rot"], case["interleaved"]).to(q.dtype)
        k = _turned(k.float(), table, case["rot"], case["interleaved"]).to(k.dtype)
    pages = state["page_table"].long().gather(1, at // page)
    state["k_pages"][pages, :, at % page] = k.transpose(1, 2)
    state["v_pages"][pages, :, at % page] = v.transpose(1, 2)
    return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _gathered(pages, table):
    """pages [n, K, page, D] in the order of table [X, m] -> [X, K, m * page, D] in 32 bits."""
    x = pages[table.long()].transpose(1, 2)
    return x.flatten(2, 3).float()


def _plain_attention(state):
    case = state["case"]
    B, G, T, H, K, D = (case[k] for k in ("batch", "groups", "tokens", "heads", "kv_heads", "dim"))
    dev, per, share = state["q"].device, B // G, H // K
    q = state["q"].float().reshape(B, K, share * T, D) / math.sqrt(D)                       # rows: head of the group, token
    index = state["seq_lens"].long()[:, None] - T + torch.arange(T, device=dev)             # [B, T]
    # the prefix: the rows of all sequences of a group against its keys
    k_pre, v_pre = _gathered(state["k_pages"], state["prefix_table"]), _gathered(state["v_pages"], state["prefix_table"])
    n_pre = k_pre.shape[2]
    grouped = q.reshape(G, per, K, share * T, D).transpose(1, 2).reshape(G, K, per * share * T, D)
    pre = grouped @ k_pre.transpose(-1, -2)
    shown = torch.arange(n_pre, device=dev) < state["prefix_lens"][:, None]                 # [G, n_pre]
    pre = pre.masked_fill(~shown[:, None, None], -math.inf)
    pre = pre.reshape(G, K, per, share * T, n_pre).transpose(1, 2).reshape(B, K, share * T, n_pre)
    # the sequence's own keys, causally
    k_own, v_own = _gathered(state["k_pages"], state["page_table"]), _gathered(state["v_pages"], state["page_table"])
    n_own = k_own.shape[2]
    scores = q @ k_own.transpose(-1, -2)
    shown = torch.arange(n_own, device=dev) <= index[..., None]                             # [B, T, n_own]
    scores = scores.reshape(B, K, share, T, n_own).masked_fill(~shown[:, None, None], -math.inf).flatten(2, 3)
    # one softmax over both
    top = torch.maximum(pre.amax(-1, keepdim=True), scores.amax(-1, keepdim=True))
    pre, scores = (pre - top).exp_(), (scores - top).exp_()
    total = pre.sum(-1, keepdim=True) + scores.sum(-1, keepdim=True)
    pre = pre.reshape(G, per, K, share * T, n_pre).transpose(1, 2).reshape(G, K, per * share * T, n_pre)
    out = (pre @ v_pre).reshape(G, K, per, share * T, D).transpose(1, 2).reshape(B, K, share * T, D)
    out = ((out + scores @ v_own) / total).reshape(B, H, T, D)
    out = out.masked_fill((index < 0)[:, None, :, None], 0.0)
    return {"out": out.to(state["q"].dtype)}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)


def _exact_append(case, s):
    T, rot, page = case["tokens"], case["rot"], case["page"]
    half = rot // 2
    q, keys, values = s["q"].double(), s["k_pages"].double(), s["v_pages"].double()
    for b, n in enumerate(s["seq_lens"].tolist()):
        spots = torch.arange(n - T, n, device="cuda")
        new_q, new_k = q[b].clone(), s["k"][b].double().clone()
        if rot:
            first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
            second = first + (1 if case["interleaved"] else half)
            turn = torch.complex(s["cos_sin"][spots, :half].double(), s["cos_sin"][spots, half:].double())
            for x in (new_q, new_k):
                z = torch.complex(x[..., first], x[..., second]) * turn
                x[..., first], x[..., second] = z.real, z.imag
        q[b] = new_q
        where = s["page_table"][b, spots // page].long()
        keys[where, :, spots % page] = new_k.transpose(0, 1)
        values[where, :, spots % page] = s["v"][b].double().transpose(0, 1)
    return {"q": q, "k_pages": keys, "v_pages": values}


def _exact_attention(case, s):
    B, T, H, K, D, page = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "page"))
    per, out = B // case["groups"], torch.zeros(B, H, T, D, dtype=torch.float64, device="cuda")
    last, shared = -1, None
    for b, n in enumerate(s["seq_lens"].tolist()):
        group = b // per
        if group != last:
            m = int(s["prefix_lens"][group])
            at = torch.arange(m, device="cuda")
            pages = s["prefix_table"][group, at // page].long()
            shared = [x[pages, :, at % page].double().permute(1, 2, 0) for x in (s["k_pages"], s["v_pages"])]
            last = group
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        pages = s["page_table"][b, at // page].long()
        k, v = (torch.cat([p, x[pages, :, at % page].double().permute(1, 2, 0)], dim=2)
                for p, x in zip(shared, (s["k_pages"], s["v_pages"])))
        for head in range(K):
            rows = s["q"][b, head * (H // K):(head + 1) * (H // K)].double()                # [share, T, D]
            score = torch.matmul(rows, k[head]) * D ** -0.5
            late = at[None, :] > (n - T + torch.arange(T, device="cuda"))[:, None]
            score[..., m:] += torch.where(late, -math.inf, 0.0).double()
            weight = torch.softmax(score, dim=-1)
            out[b, head * (H // K):(head + 1) * (H // K)] = torch.matmul(weight, v[head].transpose(0, 1))
    return {"out": out}
