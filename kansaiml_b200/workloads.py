"""Seeded synthetic models and inputs for the benchmark configurations, shared
by bench.py and the tests (no datasets or checkpoints are involved).

Config 3 is an int8 decoder-only transformer with the layout of the
reference's examples/tinyshakespeare/train_shakespeare.py:79-111 (token +
learned position embeddings, pre-LN TransformerBlocks under one causal mask,
final LayerNorm, Linear head): d_model 256, 4 heads, FFN 1024 with GELU,
vocab 65, context 256, 2 blocks.  Every Linear weight is drawn ~ N(0, 0.02)
from a seeded numpy stream and quantized per output channel; activations are
quantized per tensor on the fly (W8A8 on the int8 tensor cores, bias, GELU
and rescale fused); LayerNorm, attention scores and softmax stay fp32.
"""
import numpy as np
import torch

from . import nn
from ._lib import KZ_ERR_NONFINITE, KZ_TREE_MAX_NODES, KzError
from .cache import PagePool, QCache, verify_tree
from .quantize import QActivation, QLinear, device_status
from .tensor import Tensor, from_numpy


def _param(a, device):
    t = from_numpy(a, device)
    t.requires_grad = True
    return t


class DecoderCache:
    """What a Decoder keeps of a batch of sequences: one QCache a layer, their
    common pages, and how many tokens each sequence has (``lengths``, on the
    device).  ``most`` bounds them on the host: pages are reserved by it."""

    def __init__(self, layers, batch, kv_heads, head_dim, capacity, page_size, device):
        columns = -(-capacity // page_size)
        self.capacity, self.most = capacity, 0
        self.pool = PagePool(batch * columns, batch, columns, page_size, device)
        self.layers = [QCache(batch * columns, kv_heads, head_dim, page_size, device) for _ in range(layers)]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.pool.table.device)

    def room(self, tokens):
        """Pages for `tokens` more tokens of every sequence; raises past the capacity."""
        if self.most + tokens > self.capacity:
            raise ValueError(f"DecoderCache: {self.most} + {tokens} tokens, the capacity is {self.capacity}")
        self.pool.reserve(self.most + tokens)

    def advance(self, counts, most):
        """The last step's first counts[b] tokens stay (an int, or int32 [batch]); most: no sequence has more."""
        self.lengths += counts
        self.most = most

    def keep(self, path, count):
        """An accepted path's tokens to the front, in every layer."""
        for layer in self.layers:
            layer.keep(self.pool.table, self.lengths, path, count)


class Decoder(nn.Module):
    """Config 3 decoder.  ``fp32`` keeps the unquantized weights (numpy) so a
    CPU restatement can rebuild the same model."""

    def __init__(self, vocab=65, d_model=256, heads=4, d_ff=1024, layers=2, ctx=256, seed=0, device="cuda"):
        rs = np.random.RandomState(seed)

        def normal(*shape):
            return (rs.standard_normal(shape) * 0.02).astype(np.float32)

        self.vocab, self.d_model, self.heads, self.ctx = vocab, d_model, heads, ctx
        self.tok = nn.Embedding(vocab, d_model, seed=seed, device=device)
        self.pos = nn.Embedding(ctx, d_model, seed=seed + 1, device=device)
        self.fp32 = {"tok": self.tok.weight.numpy(), "pos": self.pos.weight.numpy(), "blocks": []}
        self.blocks = []
        for i in range(layers):
            blk = nn.TransformerBlock(d_model, heads, d_ff, seed=seed + 10 + i, device=device)
            w = {name: normal(d_model, d_model) for name in ("w_q", "w_k", "w_v", "w_o")}
            for name, value in w.items():
                setattr(blk.attn, name, _param(value, device))
            w["fc1"], w["fc2"] = normal(d_model, d_ff), normal(d_ff, d_model)
            blk.fc1.weight = _param(w["fc1"], device)
            blk.fc2.weight = _param(w["fc2"], device)
            w["fc1_b"], w["fc2_b"] = blk.fc1.bias.numpy(), blk.fc2.bias.numpy()
            blk.quantize(per_channel=True, activations="int8")
            self.blocks.append(blk)
            self.fp32["blocks"].append(w)
        self.ln = nn.LayerNorm(d_model, device=device)
        head = nn.Linear(d_model, vocab, seed=seed + 99, device=device)
        self.fp32["head"], self.fp32["head_b"] = normal(d_model, vocab), head.bias.numpy()
        head.weight = _param(self.fp32["head"], device)
        self.head = QLinear(head, per_channel=True, activations="int8")
        self.mask = nn.causal_mask(ctx, device=device)

    def forward(self, ids):
        """ids: int64 [B, S] (S <= ctx) on the model's device -> logits [B, S, vocab]."""
        s = ids.shape[1]
        x = Tensor(self.tok.weight.data[ids] + self.pos.weight.data[:s])
        mask = self.mask if s == self.ctx else nn.CausalMask(self.mask.data[:, :, :s, :s].contiguous())
        # each block's feed-forward residual is added inside the next LayerNorm
        pending = None
        for blk in self.blocks:
            if blk._w8a8():
                x, pending = blk._forward_w8a8(x, mask, pending)
            else:
                x = blk(x if pending is None else x.add(pending), mask=mask)
                pending = None
        return self._logits(x, pending)

    def _logits(self, x, pending, rows=False):
        ln = self.ln
        if pending is None:
            qa = QActivation.layernorm(x, ln.weight, ln.bias, ln.eps, rows)
        else:
            _, qa = QActivation.add_layernorm(x, pending, ln.weight, ln.bias, ln.eps, rows)
        return self.head(qa)

    # ------------------------------------------------------------ generation
    def new_cache(self, batch, capacity=None, page_size=64):
        """An empty cache for `batch` sequences of at most `capacity` (default: the context) tokens."""
        capacity = self.ctx if capacity is None else capacity
        if not 0 < capacity <= self.ctx:
            raise ValueError(f"Decoder: the capacity must be 1 to the context's {self.ctx} (got {capacity})")
        return DecoderCache(len(self.blocks), batch, self.heads, self.d_model // self.heads, capacity, page_size,
                            self.tok.weight.device)

    def extend(self, ids, cache, counts=None, parents=None, depths=None):
        """The logits [B, T, vocab] of new tokens ids int64 [B, T] over what the
        cache holds; their keys and values enter it behind that (cache.advance
        then makes them part of it).  counts: rows that are tokens (None: all);
        parents (with depths int64 [B, T], a node's distance from the root): the
        tokens form a tree.  Activations are quantized row by row, so that a
        token's logits follow from its own sequence (with forward's one scale
        for all rows they would shift with padding, neighbours and drafts)."""
        if parents is not None and depths is None:
            raise ValueError("Decoder.extend: parents need the nodes' depths, from which their positions follow")
        cache.room(ids.shape[1])
        where = torch.arange(ids.shape[1], device=ids.device) if depths is None else depths
        where = (cache.lengths[:, None] + where).clamp(max=self.ctx - 1)
        x = Tensor(self.tok.weight.data[ids] + self.pos.weight.data[where])
        pending = None
        for blk, layer in zip(self.blocks, cache.layers):
            step = nn.CacheStep(layer, cache.pool.table, cache.lengths, counts, parents)
            if blk._w8a8():
                x, pending = blk._forward_w8a8(x, None, pending, step)
            else:
                x = blk(x if pending is None else x.add(pending), step=step)
                pending = None
        return self._logits(x, pending, rows=True)

    def generate(self, prompts, new_tokens, temperature=1.0, drafts=0, seed=0):
        """`new_tokens` more tokens for each prompt (lists of ids), drawn at
        `temperature` (0: the likeliest).  With drafts > 0, each step verifies
        up to that many tokens looked up in the sequence itself -- what followed
        earlier occurrences of its last token, as a tree -- and keeps those that
        the model's own probabilities accept.  These follow from a token's own
        sequence, so the tokens are distributed as without drafts and as in
        another batch, but for what the order of the attention's 32-bit sums
        moves.  Returns one list of new ids per prompt; raises ValueError where
        something on the way was NaN or Inf (a model whose weights are), and
        KzError for any other error that the device recorded."""
        device = self.tok.weight.device
        seen = [list(p) for p in prompts]
        batch, longest = len(seen), max((len(p) for p in seen), default=0)
        if not seen or min(len(p) for p in seen) < 1 or not all(0 <= t < self.vocab for p in seen for t in p):
            raise ValueError(f"Decoder.generate: a prompt is one or more ids below {self.vocab}")
        if not 0 <= drafts < KZ_TREE_MAX_NODES:
            raise ValueError(f"Decoder.generate: drafts must be 0 to {KZ_TREE_MAX_NODES - 1} (got {drafts})")
        if not temperature >= 0:
            raise ValueError(f"Decoder.generate: temperature must be 0 or above (got {temperature})")
        if new_tokens < 1 or longest + new_tokens > self.ctx:
            raise ValueError(f"Decoder.generate: {longest} + {new_tokens} tokens, the context is {self.ctx}")
        cache = self.new_cache(batch)
        earlier = device_status(device, clear=False)         # an error of another call's stays for its caller
        random = torch.Generator(device=device).manual_seed(seed)

        def step(ids, counts, parents=None, depths=None):
            logits = self.extend(ids, cache, counts, parents, depths).data
            top = logits.amax(-1, keepdim=True)
            if temperature > 0:
                # from the largest logit, which stays 0 however small the temperature; one below 1e-30 is its
                # limit already (logits that differ do so by more), and its reciprocal might be infinite
                return torch.softmax((logits - top) / max(temperature, 1e-30), -1)
            likeliest = torch.nn.functional.one_hot(logits.argmax(-1), self.vocab)
            return likeliest + (top - top)                   # NaN where a logit is, for the verification to see

        def verified(ids, parents, probs):
            nodes = ids.shape[1]
            return verify_tree(ids, parents, probs, None, torch.rand(batch, nodes, generator=random, device=device),
                               torch.rand(batch, generator=random, device=device))

        counts = torch.tensor([len(p) for p in seen], dtype=torch.int32, device=device)
        ids = torch.tensor([p + [0] * (longest - len(p)) for p in seen], device=device)
        probs = step(ids, counts)
        probs = probs[torch.arange(batch, device=device), counts.long() - 1][:, None]
        root = torch.full((1,), -1, dtype=torch.int32, device=device)
        _, _, token = verified(ids[:, :1], root, probs)
        cache.advance(counts, longest)
        out = [[t] for t in token.tolist()]
        for s, o in zip(seen, out):
            s += o
        while True:
            live = [len(o) < new_tokens for o in out]
            if not any(live):
                break
            room = min(1 + drafts, cache.capacity - cache.most)
            trees = [_drafted(s, room) if on else ([], [], []) for s, on in zip(seen, live)]
            nodes = max(len(t[0]) for t in trees)
            ids = torch.tensor([t[0] + [0] * (nodes - len(t[0])) for t in trees], device=device)
            parents = torch.tensor([t[1] + [-1] * (nodes - len(t[1])) for t in trees], dtype=torch.int32, device=device)
            depths = torch.tensor([t[2] + [0] * (nodes - len(t[2])) for t in trees], device=device)
            counts = torch.tensor([len(t[0]) for t in trees], dtype=torch.int32, device=device)
            path, count, token = verified(ids, parents, step(ids, counts, parents, depths))
            count = torch.minimum(count, counts)             # 0: a sequence that is done
            cache.keep(path, count)
            for s, o, t, p, n, x in zip(seen, out, trees, path.tolist(), count.tolist(), token.tolist()):
                new = [t[0][i] for i in p[1:n]] + [x] if n else []
                s += new
                o += new
            cache.advance(count, max(len(s) - 1 for s, on in zip(seen, live) if on))
        code = 0 if earlier else device_status(device)
        if code:
            if code == KZ_ERR_NONFINITE:
                raise ValueError("Decoder.generate: the logits, or keys and values on the way to them, contain NaN or Inf")
            raise KzError(code, f"Decoder.generate: the device recorded error {code}")
        return [o[:new_tokens] for o in out]


def _drafted(seen, nodes):
    """A tree of at most `nodes` tokens from the sequence itself: the last token
    as the root, then what followed its earlier occurrences, the latest first.
    Returns (tokens, parents, depths)."""
    tokens, parents, depths, below = [seen[-1]], [-1], [0], {}
    for at in range(len(seen) - 2, -1, -1):
        if seen[at] != seen[-1]:
            continue
        node = 0
        for x in seen[at + 1:at + 5]:
            if len(tokens) >= nodes:
                return tokens, parents, depths
            if (node, x) not in below:
                below[node, x] = len(tokens)
                tokens.append(x)
                parents.append(node)
                depths.append(depths[node] + 1)
            node = below[node, x]
    return tokens, parents, depths


def config3_ids(batch=32, ctx=256, vocab=65, seed=0, device="cuda"):
    """Token ids ~ U{0 .. vocab-1}, int64 [batch, ctx]."""
    ids = np.random.RandomState(seed).randint(0, vocab, (batch, ctx))
    return torch.from_numpy(ids.astype(np.int64)).to(device)
