"""An int8 K/V cache for generation: quantized as it is written, read back,
attended over, and the verification of drafted tokens.

The reference recomputes attention over the whole sequence for every token
(MultiHeadAttention.forward, nn.py:410-427) and keeps nothing; here its keys
and values stay on the GPU as int8 codes, quantized by quantize_symmetric's
rule (quantize.py:66-70) with one scale per token and key head:

* ``QCache``: one attention layer's pages.  ``write`` quantizes new tokens into
  it, ``read`` gives tokens back as fp32, ``attention`` attends over it (one new
  token a sequence, a chunk of a prompt, or a tree of drafted tokens, with
  grouped heads), ``keep`` moves the accepted path of a tree to the front.
* ``PagePool``: which pages each sequence has (one pool serves every layer).
* ``verify_tree``: which drafted tokens stand, and the next token, from the
  target's probabilities and given uniform numbers.  A tree of one node draws
  the next token of plain sampling.

Common arguments: ``table`` int32 [batch, columns], the page numbers of each
sequence; ``lengths`` int32 [batch], its tokens in the cache before the call;
``counts`` int32 [batch] or None, how many of its rows are tokens (None: all;
the rest is padding); ``parents`` int32 [batch, tokens] or [tokens], each new
token's parent in its tree (-1: none; a parent comes before its child).  All
are CUDA tensors, read on the device: nothing here waits for the GPU.  A page
number or position that a cache does not have is left out and recorded in the
device status word (quantize.device_status), as NaN/Inf in a written row is.
Sequences may share pages that are only read; a page that is written to must be
in the table once.
"""
import ctypes

import torch

from . import _lib
from .tensor import Tensor, _as_device, ptr, require_cuda


def _raw(t, what):
    """The fp32 CUDA tensor of a Tensor or torch tensor."""
    x = t.data if isinstance(t, Tensor) else t
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} must be a Tensor or a torch tensor, not {type(t).__name__}")
    if not x.is_cuda:
        require_cuda(x, what)
    return x if x.dtype is torch.float32 else x.float()


def _like(x):
    """A new contiguous tensor like x (the cheapest allocation torch has)."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _ints(t, what, shape, index, dtype=torch.int32):
    """t, contiguous, checked to be integers of that shape on GPU `index`."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index:
        return t if t.is_contiguous() else t.contiguous()
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} must be a {str(dtype)[6:]} tensor {list(shape)}, not {type(t).__name__}")
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{what} must be a {str(dtype)[6:]} tensor {list(shape)}, not {list(t.shape)} {str(t.dtype)[6:]}")
    raise ValueError(f"{what} is on {t.device}, not on cuda:{index}")


def _parents(parents, batch, nodes, index):
    """(parents, batch stride): one tree for every sequence, or one each."""
    if isinstance(parents, torch.Tensor) and parents.dim() == 1:
        return _ints(parents, "parents", (nodes,), index), 0
    return _ints(parents, "parents", (batch, nodes), index), nodes


def _on(index, name, *args):
    """Calls libkz with GPU `index` current, on torch's current stream there."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        status = getattr(_lib.load(), name)(*args, stream)
        if status:
            _lib.check(status, name)
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, stream)


class QCache:
    """One attention layer's int8 K/V pages: codes [pages, kv_heads, page_size,
    head_dim] and fp32 scales [pages, kv_heads, page_size], for K and for V."""

    __slots__ = ("k_codes", "k_scale", "v_codes", "v_scale", "pages", "kv_heads", "page_size", "head_dim", "device", "_at", "_c", "_ref",
                 "_scratch")

    def __init__(self, pages, kv_heads, head_dim, page_size=64, device=None):
        dev = _as_device(device)
        shape = (int(pages), int(kv_heads), int(page_size))
        if min(shape) < 0:
            raise ValueError(f"QCache: negative size {shape}")
        self._bind(*(torch.empty(shape + d, dtype=t, device=dev)
                     for _ in range(2) for d, t in (((int(head_dim),), torch.int8), ((), torch.float32))))

    @classmethod
    def wrap(cls, k_codes, k_scale, v_codes, v_scale):
        """A cache over buffers the caller has."""
        obj = cls.__new__(cls)
        obj._bind(k_codes, k_scale, v_codes, v_scale)
        return obj

    def _bind(self, k_codes, k_scale, v_codes, v_scale):
        if k_codes.dim() != 4:
            raise ValueError(f"QCache: codes must be [pages, kv_heads, page_size, head_dim], not {list(k_codes.shape)}")
        self.pages, self.kv_heads, self.page_size, self.head_dim = k_codes.shape
        if self.head_dim not in (32, 64, 128):
            raise ValueError(f"QCache: head_dim must be 32, 64 or 128 (got {self.head_dim})")
        if self.page_size not in (16, 32, 64, 128):
            raise ValueError(f"QCache: page_size must be 16, 32, 64 or 128 (got {self.page_size})")
        if self.kv_heads < 1:
            raise ValueError("QCache: kv_heads must be at least 1")
        for t, dtype, shape in ((k_codes, torch.int8, k_codes.shape), (v_codes, torch.int8, k_codes.shape),
                                (k_scale, torch.float32, k_codes.shape[:3]),
                                (v_scale, torch.float32, k_codes.shape[:3])):
            if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError("QCache: codes are int8 [pages, kv_heads, page_size, head_dim], scales float32 "
                                 "[pages, kv_heads, page_size], contiguous and on one device")
        self.k_codes, self.k_scale, self.v_codes, self.v_scale = k_codes, k_scale, v_codes, v_scale
        self._c = _lib.KzCache(ptr(k_codes), ptr(k_scale), ptr(v_codes), ptr(v_scale), *k_codes.shape)
        self._ref = ctypes.byref(self._c)
        self.device, self._at = k_codes.device, k_codes.get_device()
        self._scratch = {}                      # (tokens, heads, columns) -> bytes of attention's workspace

    def nbytes(self):
        """Bytes held: one per code and four per scale."""
        return 2 * (self.k_codes.numel() + 4 * self.k_scale.numel())

    def __repr__(self):
        return (f"QCache(pages={self.pages}, kv_heads={self.kv_heads}, head_dim={self.head_dim}, "
                f"page_size={self.page_size}, device={self.device})")

    def _sequences(self, table, lengths, counts=None):
        if self._at < 0:
            require_cuda(self.k_codes, "QCache")
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            raise ValueError("table must be an int32 tensor [batch, columns]")
        batch, cols = table.shape
        return (batch, cols, _ints(table, "table", table.shape, self._at),
                _ints(lengths, "lengths", (batch,), self._at),
                None if counts is None else _ints(counts, "counts", (batch,), self._at))

    def _input(self, t, what, heads, batch):
        """(x, tokens, its address, batch stride, row stride) of [batch, tokens,
        heads * head_dim] rows that a kernel can read in 16-byte pieces; others are copied."""
        x = _raw(t, what)
        shape, width = x.shape, heads * self.head_dim
        if len(shape) != 3 or shape[0] != batch or shape[2] != width:
            raise ValueError(f"{what} must be [{batch}, tokens, {width}], not {list(shape)}")
        if x.get_device() != self._at:
            raise ValueError(f"{what} is on {x.device}, the cache on {self.device}")
        bs, rs, fs = x.stride()
        at, tokens = x.data_ptr(), shape[1]
        if (at | bs << 2 | rs << 2) & 15 or fs != 1 or bs < 0 or (rs < width and tokens > 1):
            x = x.contiguous()
            if x.data_ptr() & 15:
                x = x.clone()
            bs, rs = tokens * width, width          # (a single row's own strides may be anything)
            at = x.data_ptr()
        return x, tokens, at, bs, rs

    def write(self, k, v, table, lengths, counts=None, values=False):
        """Quantizes new tokens' k and v [batch, tokens, kv_heads * head_dim]
        (strided rows allowed, e.g. slices of a fused projection) into positions
        lengths + 0, 1, ...  With ``values``, returns what the codes stand for,
        two Tensors like k and v (0 in padding rows): the K/V a later pass sees."""
        batch, cols, table, lengths, counts = self._sequences(table, lengths, counts)
        k, tokens, k_at, kb, kr = self._input(k, "k", self.kv_heads, batch)
        v, v_tokens, v_at, vb, vr = self._input(v, "v", self.kv_heads, batch)
        if v_tokens != tokens:
            raise ValueError(f"k {list(k.shape)} and v {list(v.shape)} do not match")
        if values:
            ko, vo = _like(k), _like(k)
        _on(self._at, "kz_cache_write_f32", self._ref, k_at, v_at, batch, tokens, kb, kr, vb, vr, table.data_ptr(),
            cols, lengths.data_ptr(), None if counts is None else counts.data_ptr(), ko.data_ptr() if values else None, vo.data_ptr() if values else None)
        return (Tensor(ko), Tensor(vo)) if values else None

    def read(self, table, lengths, most):
        """The first ``lengths`` tokens of each sequence, dequantized: two
        Tensors [batch, most, kv_heads * head_dim], 0 past a sequence's length
        (tokens past ``most`` are left out)."""
        batch, cols, table, lengths, _ = self._sequences(table, lengths)
        if most < 0:
            raise ValueError(f"read: most must not be negative (got {most})")
        shape = (batch, int(most), self.kv_heads * self.head_dim)
        k = self.k_scale.new_empty(shape)
        v = _like(k)
        _on(self._at, "kz_cache_read_f32", self._ref, table.data_ptr(), cols, lengths.data_ptr(), batch, shape[1],
            k.data_ptr(), v.data_ptr())
        return Tensor(k), Tensor(v)

    def attention(self, q, heads, table, lengths, counts=None, parents=None, scale=None):
        """softmax(q k^T * scale) v over the cached tokens and the new ones
        (written before): q [batch, tokens, heads * head_dim], heads a multiple
        of kv_heads; scale 1 / sqrt(head_dim) by default.  A new token sees every
        token before the new ones and, of these, its ancestors and itself in the
        tree ``parents`` (at most 256 nodes), or without one all up to itself.
        Returns [batch, tokens, heads * head_dim], 0 in padding rows."""
        batch, cols, table, lengths, counts = self._sequences(table, lengths, counts)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"attention: heads ({heads}) must be a multiple of kv_heads ({self.kv_heads})")
        q, tokens, q_at, qb, qr = self._input(q, "q", heads, batch)
        pb = 0
        if parents is not None:
            if tokens > _lib.KZ_TREE_MAX_NODES:
                raise ValueError(f"attention: a tree has at most {_lib.KZ_TREE_MAX_NODES} nodes (got {tokens})")
            parents, pb = _parents(parents, batch, tokens, self._at)
        out = _like(q)
        need = self._scratch.get((tokens, heads, cols))
        if need is None:
            with torch.cuda.device(self.device):
                need = _lib.load().kz_cache_attention_workspace_bytes(self._ref, tokens, heads, cols)
            self._scratch[tokens, heads, cols] = need
        work = self.k_codes.new_empty(need) if need else None
        _on(self._at, "kz_cache_attention_f32", self._ref, q_at, batch, tokens, heads, qb, qr, table.data_ptr(), cols,
            lengths.data_ptr(), None if counts is None else counts.data_ptr(), None if parents is None else parents.data_ptr(),
            pb, self.head_dim ** -0.5 if scale is None else scale, out.data_ptr(), None if work is None else work.data_ptr(), need)
        return Tensor(out)

    def keep(self, table, lengths, path, count):
        """Moves the new tokens path[b, 0 .. count[b] - 1] (strictly increasing,
        int32 [batch, nodes], as verify_tree returns it) to positions lengths +
        0, 1, ...: the cache then holds lengths + count tokens of each sequence."""
        batch, cols, table, lengths, count = self._sequences(table, lengths, count)
        if not isinstance(path, torch.Tensor) or path.dim() != 2:
            raise ValueError("path must be an int32 tensor [batch, nodes]")
        path = _ints(path, "path", (batch, path.shape[1]), self._at)
        if count is None:
            raise ValueError("count must be an int32 tensor [batch]")
        _on(self._at, "kz_cache_keep", self._ref, table.data_ptr(), cols, lengths.data_ptr(), path.data_ptr(),
            count.data_ptr(), batch, path.shape[1])


class PagePool:
    """Hands out page numbers 0 .. pages - 1 to ``batch`` sequences.  ``table``
    (int32 [batch, columns] on the device, -1 where a sequence has no page) is
    what every layer's QCache takes; a change is one small copy to the device,
    on the current stream, that the host does not wait for."""

    def __init__(self, pages, batch, columns, page_size=64, device=None):
        self.page_size, self.columns = int(page_size), int(columns)
        self._free = list(range(int(pages) - 1, -1, -1))
        self._held = [[] for _ in range(int(batch))]
        self.table = torch.full((int(batch), self.columns), -1, dtype=torch.int32, device=_as_device(device))

    @property
    def free(self):
        return len(self._free)

    def reserve(self, tokens, sequence=None):
        """Pages for ``tokens`` positions of one sequence, or of each; raises,
        and changes nothing, where the pool or the table is too small."""
        need = -(-int(tokens) // self.page_size)
        if need > self.columns:
            raise ValueError(f"PagePool: {tokens} tokens need {need} pages a sequence, the table has {self.columns}")
        which = range(len(self._held))
        which = which if sequence is None else [which[sequence]]
        short = sum(max(0, need - len(self._held[i])) for i in which)
        if short > len(self._free):
            raise RuntimeError(f"PagePool: {short} pages needed, {len(self._free)} free")
        if not short:
            return
        at = [(i, c) for i in which for c in range(len(self._held[i]), need)]
        new = self._free[:-short - 1:-1]
        # from pinned memory, whose owner keeps it until the copy has run
        change = torch.tensor([[i * self.columns + c for i, c in at], new], pin_memory=self.table.is_cuda)
        change = change.to(self.table.device, non_blocking=True)
        self.table.view(-1).scatter_(0, change[0], change[1].int())
        del self._free[-short:]
        for (i, _), page in zip(at, new):
            self._held[i].append(page)

    def release(self, sequence):
        """Gives a sequence's pages back."""
        self._free += reversed(self._held[sequence])
        self._held[sequence] = []
        self.table[sequence] = -1


def verify_tree(tokens, parents, target, draft, accept_u, sample_u):
    """Which nodes of a drafted tree stand (speculative sampling).

    tokens int64 [batch, nodes], node 0 the root (a token already drawn);
    parents int32 [batch, nodes] or [nodes]; target fp32 [batch, nodes, vocab],
    the model's probabilities after each node; draft, the same shape, the
    probabilities each node's children were drawn from, or None where drafts
    have none; accept_u fp32 [batch, nodes] and sample_u [batch] uniform in
    [0, 1).  With r the target's row at the current node, its children x are
    tried in index order: accepted where accept_u * q(x) < r(x), and the walk
    goes on there; else r = (r - q)+ / sum (r - q)+.  Returns path int32
    [batch, nodes] (the accepted nodes from the root on, then -1), count int32
    [batch], and the next token int64 [batch], drawn from r by sample_u: it is
    distributed as the target's own, whatever was drafted.  NaN or Inf in a row
    that this takes a sum of is recorded in the device status word."""
    target = _raw(target, "target")
    shape = target.shape
    if len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        raise ValueError(f"target must be [batch, nodes, vocab], not {list(shape)}")
    batch, nodes, vocab = shape
    if nodes > 1024:
        raise ValueError(f"verify_tree: at most 1024 nodes (got {nodes})")
    at = target.get_device()

    def floats(t, what, shape):
        x = _raw(t, what)
        if x.shape != shape or x.get_device() != at:
            raise ValueError(f"{what} must be {list(shape)} on {target.device}, not {list(x.shape)} on {x.device}")
        return x.contiguous()

    target = target.contiguous()
    draft = None if draft is None else floats(draft, "draft", shape)
    accept_u, sample_u = floats(accept_u, "accept_u", (batch, nodes)), floats(sample_u, "sample_u", (batch,))
    tokens = _ints(tokens, "tokens", (batch, nodes), at, torch.int64)
    parents, pb = _parents(parents, batch, nodes, at)
    path = _like(parents) if pb else parents.new_empty((batch, nodes))
    count, token = parents.new_empty(batch), tokens.new_empty(batch)
    _on(at, "kz_verify_tree_f32", tokens.data_ptr(), parents.data_ptr(), pb, target.data_ptr(),
        None if draft is None else draft.data_ptr(),
        accept_u.data_ptr(), sample_u.data_ptr(), batch, nodes, vocab, path.data_ptr(), count.data_ptr(), token.data_ptr())
    return path, count, token


__all__ = ["QCache", "PagePool", "verify_tree"]
