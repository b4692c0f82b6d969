"""Generation through the cache on the GPU: a Decoder's steps (chunks, single
tokens, trees, kept paths) against a float64 restatement that knows no cache,
what a node's logits may depend on, and generate's tokens.
"""
import math

import numpy as np
import pytest
import torch
from scipy.special import erf

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ids(v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


def _status():
    from kansaiml_b200 import quantize as kq
    return kq.device_status()


# ------------------------------------------------------- the model in float64

def _coded(x, axis):
    """x as its int8 codes along that axis stand for it."""
    s = np.abs(x).max(axis, keepdims=True) / 127
    s = np.where(s > 0, s, 1.0)
    return np.clip(np.rint(x / s), -127, 127) * s


def _norm(x):
    return (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + 1e-5)


def _decoder_64(model, tokens):
    """The logits after each of `tokens`: every linear's input quantized row by
    row, keys and values by token and head, all else in float64."""
    f, heads, n = model.fp32, model.heads, len(tokens)
    d = model.d_model // heads
    x = f["tok"][tokens].astype(np.float64) + f["pos"][:n]

    def linear(h, w, b=0.0):
        return _coded(h, -1) @ _coded(w.astype(np.float64), 0) + b

    for w in f["blocks"]:
        h = _norm(x)
        q = linear(h, w["w_q"]).reshape(n, heads, d)
        k, v = (_coded(linear(h, w[name]).reshape(n, heads, d), -1) for name in ("w_k", "w_v"))
        s = np.einsum("ihd,jhd->hij", q, k) / math.sqrt(d)
        s[:, np.triu(np.ones((n, n), bool), 1)] = -np.inf
        e = np.exp(s - s.max(-1, keepdims=True))
        att = np.einsum("hij,jhd->ihd", e / e.sum(-1, keepdims=True), v).reshape(n, -1)
        x = x + linear(att, w["w_o"])
        u = linear(_norm(x), w["fc1"], w["fc1_b"])
        x = x + linear(0.5 * u * (1 + erf(u / math.sqrt(2))), w["fc2"], w["fc2_b"])
    return linear(_norm(x), f["head"], f["head_b"])


# What may differ from float64: 32-bit sums (1e-6 relative, far below what
# follows) and codes that they tip over a rounding border.  A code takes an
# input's largest value / 127: of a normalised row of 256 (largest 3 to 4, norm
# 16) 2e-3 of the row's norm at most, and so of the linear's output.  An input
# is off by up to 1e-3 codes, so 256 inputs have half a code tipped, the 8
# linears before a logit 4, with fc2's 1024 narrower inputs 6: were all 10 to
# point the same way, 2e-2.
REL = 2e-2


def _near(got, want):
    off = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    assert off.max() <= REL, off


@pytest.fixture(scope="module")
def model():
    from kansaiml_b200 import workloads
    return workloads.Decoder(seed=3)


def test_steps_through_the_cache_equal_the_whole_sequence(cuda_device, model):
    """Ragged prompts in two chunks, single tokens, a tree with nodes down to
    depth 3, a path kept that skips nodes, and steps after it: the logits of
    each are those of the token's own sequence, run as one."""
    rs = np.random.RandomState(5)
    batch = 3
    seqs = [[] for _ in range(batch)]
    cache = model.new_cache(batch, capacity=150, page_size=16)

    def chunk(new):
        n = max(len(x) for x in new)
        got = model.extend(_ids([x + [9] * (n - len(x)) for x in new]), cache, _i32([len(x) for x in new])).numpy()
        for s, x, y in zip(seqs, new, got):
            s += x
            if x:
                _near(y[:len(x)], _decoder_64(model, s)[len(s) - len(x):])
        cache.advance(_i32([len(x) for x in new]), max(len(s) for s in seqs))

    def some(*lengths):
        return [rs.randint(0, model.vocab, n).tolist() for n in lengths]

    chunk(some(30, 1, 12))
    chunk(some(17, 0, 40))
    chunk(some(1, 1, 1))
    parents, depths = [-1, 0, 0, 1, 2, 4, 4], [0, 1, 1, 2, 2, 3, 3]
    for paths in ([[0, 2, 4, 6], [0], [0, 1, 3]], [[0, 2], [0, 1], [0, 2, 4, 5]]):
        tree = some(7, 7, 7)
        got = model.extend(_ids(tree), cache, None, _i32([parents] * batch), _ids([depths] * batch)).numpy()
        for s, t, y in zip(seqs, tree, got):
            for node in range(7):
                up, at = [], node
                while at >= 0:
                    up.insert(0, t[at])
                    at = parents[at]
                _near(y[node], _decoder_64(model, s + up)[-1])
        cache.keep(_i32([p + [-1] * (7 - len(p)) for p in paths]), _i32([len(p) for p in paths]))
        for s, t, p in zip(seqs, tree, paths):
            s += [t[j] for j in p]
        cache.advance(_i32([len(p) for p in paths]), max(len(s) for s in seqs))
        chunk(some(1, 1, 1))
    chunk(some(0, 20, 1))
    assert _status() == 0


def test_a_nodes_logits_depend_on_its_own_sequence_only(cuda_device, model):
    """Other ids in padding rows, in the batch's other sequences and in the
    tree's other branches (their activations as large as they may be) leave a
    node's logits as they were, bit for bit."""
    rs = np.random.RandomState(6)
    counts, parents, depths = [40, 7, 23], [-1, 0, 0, 1, 2, 4], [0, 1, 1, 2, 2, 3]

    def run(ids, tree):
        cache = model.new_cache(3)
        first = model.extend(_ids(ids), cache, _i32(counts)).numpy()
        cache.advance(_i32(counts), 40)
        return first, model.extend(_ids(tree), cache, None, _i32(parents), _ids([depths] * 3)).numpy()

    ids, tree = rs.randint(0, 65, (3, 40)), rs.randint(0, 65, (3, 6))
    first, second = run(ids, tree)
    for _ in range(4):
        other, other_tree = rs.randint(0, 65, (3, 40)), rs.randint(0, 65, (3, 6))
        other[1, :7] = ids[1, :7]                       # sequence 1 stays, its padding does not
        other_tree[1, [0, 1, 3]] = tree[1, [0, 1, 3]]   # and one branch of its tree
        a, b = run(other, other_tree)
        np.testing.assert_array_equal(a[1, :7], first[1, :7])
        np.testing.assert_array_equal(b[1, [0, 1, 3]], second[1, [0, 1, 3]])


@pytest.mark.parametrize("drafts", [0, 6])
def test_greedy_tokens_are_the_likeliest(cuda_device, model, drafts, monkeypatch):
    """At temperature 0 every token is the likeliest after its sequence, to what
    two logits may be off (four times their mean share of REL each), whether it
    was a step's own or a draft that stood."""
    from kansaiml_b200.workloads import DecoderCache
    stood, inner = [1], DecoderCache.keep

    def spy(self, path, count):
        stood.append(int(count.max()))
        inner(self, path, count)

    monkeypatch.setattr(DecoderCache, "keep", spy)
    rs = np.random.RandomState(8)
    prompts = [rs.randint(0, 65, n).tolist() for n in (5, 40, 100, 1)]
    prompts[1] = prompts[1][:10] * 4
    out = model.generate(prompts, 40, 0.0, drafts, seed=2)
    assert (max(stood) > 1) == (drafts > 0)
    for p, o in zip(prompts, out):
        want = _decoder_64(model, p + o)[len(p) - 1:-1]
        gap = want.max(-1) - want[np.arange(40), o]
        assert np.all(gap <= 2 * 4 * REL * np.linalg.norm(want, axis=-1) / math.sqrt(65)), gap
    assert _status() == 0


@pytest.mark.parametrize("quantize", [None, dict(per_channel=True), dict(per_channel=False, activations="int8"),
                                      dict(per_channel=True, activations="int8_per_row"), dict(per_channel=False)])
def test_a_blocks_rows_do_not_meet_in_a_step(cuda_device, quantize):
    """Whatever a block's linears quantize, in a step of generation a sequence's
    rows come out the same beside others a hundred times as large."""
    from kansaiml_b200 import nn as knn
    from kansaiml_b200.cache import PagePool, QCache
    from kansaiml_b200.tensor import Tensor
    blk = knn.TransformerBlock(64, 2, 128, seed=2, device="cuda")
    if quantize is not None:
        blk.quantize(**quantize)
    x = torch.randn(2, 5, 64, device="cuda")
    out = []
    for factor in (1.0, 100.0):
        pool, cache = PagePool(4, 2, 2, 16, "cuda"), QCache(4, 2, 32, 16, "cuda")
        pool.reserve(5)
        y = x.clone()
        y[1] *= factor
        step = knn.CacheStep(cache, pool.table, _i32([0, 0]))
        out.append((blk(Tensor(y), step=step).data[0], blk.attn(*[Tensor(y)] * 3, step=step).data[0]))
    if quantize is None:                # products of 32-bit matrices, whose order may depend on the rest
        assert all(torch.allclose(a, b, rtol=0, atol=64 * 2.0**-23 * 8) for a, b in zip(*out))
    else:
        assert all(torch.equal(a, b) for a, b in zip(*out))
    assert _status() == 0


def test_generate_at_the_smallest_temperatures(cuda_device, model):
    """A temperature below what a division by it survives is the limit that it
    stands for: the likeliest token."""
    prompts = [[1, 2, 3], [60]]
    want = model.generate(prompts, 8, 0.0)
    for temperature in (1e-300, 1e-40, 1e-38, 1e-20):
        assert model.generate(prompts, 8, temperature) == want
    assert all(0 <= t < 65 for o in model.generate(prompts, 8, math.inf) for t in o)
    assert _status() == 0


def test_generate_reports_what_the_device_recorded(cuda_device):
    """A model whose logits are not finite raises instead of returning ids, and
    an error recorded before the call is left to whoever caused it."""
    from kansaiml_b200 import _lib, workloads
    model = workloads.Decoder(seed=3, layers=1)
    torch.cuda.synchronize()
    model.pos.weight.data[2] = math.nan
    with pytest.raises(ValueError, match="NaN or Inf"):
        model.generate([[1, 2, 3]], 4)
    assert _status() == 0
    model.generate([[1]], 1)                           # does not reach the row
    broken = torch.full((1, 1, 5), math.nan, device="cuda")
    from kansaiml_b200.cache import verify_tree
    verify_tree(_ids([[0]]), _i32([-1]), broken, None, torch.zeros(1, 1, device="cuda"), torch.zeros(1, device="cuda"))
    model.generate([[1]], 1)
    assert _status() == _lib.KZ_ERR_NONFINITE


@pytest.mark.parametrize("quantized", [False, True])
def test_an_attention_of_a_users_own(cuda_device, quantized):
    """A block whose attention takes query, key, value and mask, as the
    reference's does, runs without a cache as it always has."""
    from kansaiml_b200 import nn as knn
    from kansaiml_b200.tensor import Tensor

    class Own(knn.MultiHeadAttention):
        def forward(self, query, key, value, mask=None):
            return super().forward(query, key, value, mask)

    blk = knn.TransformerBlock(64, 2, 128, seed=1, device="cuda")
    own = knn.TransformerBlock(64, 2, 128, seed=1, device="cuda")
    own.attn = Own(64, 2, seed=1, device="cuda")
    if quantized:
        blk.quantize()
        own.quantize()
    x, mask = Tensor(torch.randn(2, 9, 64, device="cuda")), knn.causal_mask(9, device="cuda")
    assert torch.equal(own(x, mask).data, blk(x, mask).data)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_generate_refuses_logits_that_are_none(cuda_device, temperature):
    """NaN that enters behind the last cached layer, in the logits alone."""
    from kansaiml_b200 import workloads
    model = workloads.Decoder(seed=3, layers=1)
    model.head.bias.data[7] = math.nan
    with pytest.raises(ValueError, match="NaN or Inf"):
        model.generate([[1, 2, 3], [4]], 3, temperature)
    assert _status() == 0
