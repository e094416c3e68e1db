"""CutileGPT.generate_samples (prompts once, samples over shared pages) against generate on the repeated prompts.

Both run the same model; they differ in the attention kernels only, so fp32 tokens are the same and bf16 greedy
tokens are the fp64 oracle's argmax under teacher forcing up to the model tests' noise floor (2e-2 of the largest logit).
"""
import pytest
import torch

from oracle import ref_gpt as R
from cutilegpt_b200 import CutileGPT, GPTConfig
from cutilegpt_b200 import _lib as L
from cutilegpt_b200.models.init import init_state, randomize_affine

pytestmark = pytest.mark.gpu


def make(cfg, dtype, seed=0):
    w = init_state(cfg, seed)
    randomize_affine(w, cfg, seed + 1)
    m = CutileGPT(cfg, dtype=dtype, device="cuda", seed=0)
    m.load_state(w)
    return m, w


def ids(P, T, V, seed):
    return torch.randint(0, V, (P, T), generator=torch.Generator().manual_seed(seed)).cuda()


CFG = dict(n_layer=2, n_head=3, n_embd=96, vocab_size=211, block_size=200)


@pytest.mark.parametrize("P,n,T0,new", [(1, 1, 5, 4), (2, 3, 70, 80), (3, 2, 64, 9), (1, 5, 1, 12)])
def test_fp32_samples_are_those_of_the_repeated_prompts(P, n, T0, new):
    m, _ = make(GPTConfig(**CFG), torch.float32)
    idx = ids(P, T0, 211, 3)
    rows = idx.repeat_interleave(n, 0)
    got = m.generate_samples(idx, n, new, top_k=1)
    assert got.shape == (P, n, T0 + new)
    assert torch.equal(got.view(P * n, -1), m.generate(rows, new, top_k=1))
    for kw in (dict(temperature=0.9), dict(temperature=1.3, top_k=20)):
        a = m.generate_samples(idx, n, new, generator=torch.Generator().manual_seed(7), **kw)
        b = m.generate(rows, new, generator=torch.Generator().manual_seed(7), **kw)
        assert torch.equal(a.view(P * n, -1), b)
        c = m.generate_samples(idx, n, new, use_cuda_graph=False, generator=torch.Generator().manual_seed(7), **kw)
        assert torch.equal(a, c)
    assert L.device_error() == 0


@pytest.mark.parametrize("C,H", [(256, 4), (256, 2), (96, 3), (80, 4)])
def test_bf16_greedy_samples_follow_the_oracle(C, H):
    cfg = GPTConfig(n_layer=2, n_head=H, n_embd=C, vocab_size=307, block_size=256)
    m, w = make(cfg, torch.bfloat16, 4)
    P, n, T0, new = 2, 4, 90, 40
    idx = ids(P, T0, 307, 5)
    seq = m.generate_samples(idx, n, new, top_k=1)
    assert torch.equal(seq, seq[:, :1].expand_as(seq).contiguous())       # greedy: all samples of a prompt agree
    rows = seq[:, 0].cpu()
    logits = R.gpt_forward(R.cast_weights(w, round_to=torch.bfloat16), cfg.n_layer, cfg.n_head, rows[:, :-1])[:, T0 - 1:]
    gap = logits.amax(-1) - logits.gather(-1, rows[:, T0:, None]).squeeze(-1)
    assert (gap <= 2e-2 * logits.abs().max()).all()
    assert L.device_error() == 0


def test_samples_many_rows_and_refold():
    """More rows than the folded decode step takes, and sampled rows that differ."""
    m, _ = make(GPTConfig(**CFG), torch.bfloat16)
    idx = ids(3, 40, 211, 8)
    seq = m.generate_samples(idx, 50, 20, temperature=1.0, generator=torch.Generator().manual_seed(1))
    assert seq.shape == (3, 50, 60) and (seq[:, :, :40] == idx[:, None]).all()
    assert len({tuple(r) for r in seq[0].tolist()}) > 40
    again = m.generate_samples(idx, 50, 20, temperature=1.0, generator=torch.Generator().manual_seed(1))
    assert torch.equal(seq, again)


def test_samples_past_the_block_and_refusals():
    m, _ = make(GPTConfig(**{**CFG, "block_size": 24}), torch.float32)
    idx = ids(2, 20, 211, 9)
    got = m.generate_samples(idx, 2, 10, top_k=1)
    assert torch.equal(got.view(4, -1), m.generate(idx.repeat_interleave(2, 0), 10, top_k=1))
    assert torch.equal(m.generate_samples(idx, 3, 0), idx[:, None].expand(2, 3, 20))
    with pytest.raises(ValueError):
        m.generate_samples(idx, 0, 3)
    with pytest.raises(ValueError):
        m.generate_samples(idx, 2, 3, temperature=0.0)
