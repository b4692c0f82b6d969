"""The int8 K/V cache on the GPU against plain implementations in 64 bits:
writing (codes and scales bit for bit), reading back, moving an accepted path,
attention for tokens, chunks and trees, verification of drafted trees, and the
whole of it as a generation loop uses it.
"""
import math

import numpy as np
import pytest
import torch

from oracle import cpu as ocpu

pytestmark = pytest.mark.gpu


def _dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _status():
    from kansaiml_b200 import quantize as kq
    return kq.device_status()


class Book:
    """A cache with the pages of some sequences, in random order, and the same
    tokens' codes and scales kept on the host, position by position."""

    def __init__(self, totals, kv_heads=2, d=64, page=32, seed=0, spare=2):
        from kansaiml_b200.cache import QCache
        rs = self.rs = np.random.RandomState(seed)
        need = [-(-n // page) for n in totals]
        order = rs.permutation(sum(need) + spare)
        table = np.full((len(totals), max(need + [1]) + 1), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        self.table_h, self.table = table, _dev(table)
        self.page, self.d, self.kv, self.batch = page, d, kv_heads, len(totals)
        self.cache = QCache(len(order), kv_heads, d, page, device="cuda")
        for t, fill in ((self.cache.k_codes, 77), (self.cache.v_codes, -77), (self.cache.k_scale, math.nan),
                        (self.cache.v_scale, math.inf)):
            t.fill_(fill)      # what nothing has written: never to be seen

    def fill(self, lengths, seed=1, spread=1.0):
        """Random codes and scales at positions below lengths; returns (k, v) lists of float64 [n, kv, d]."""
        rs = np.random.RandomState(seed)
        out = []
        for codes, scale in ((self.cache.k_codes, self.cache.k_scale), (self.cache.v_codes, self.cache.v_scale)):
            c, s = codes.cpu().numpy(), scale.cpu().numpy()
            vals = []
            for b, n in enumerate(lengths):
                cc = rs.randint(-127, 128, (n, self.kv, self.d)).astype(np.int8)
                ss = (np.exp(rs.uniform(-spread, spread, (n, self.kv))) / 127).astype(np.float32)
                pos = np.arange(n)
                c[self.table_h[b, pos // self.page], :, pos % self.page] = cc
                s[self.table_h[b, pos // self.page], :, pos % self.page] = ss
                vals.append(cc.astype(np.float64) * ss[..., None].astype(np.float64))
            codes.copy_(torch.from_numpy(c))
            scale.copy_(torch.from_numpy(s))
            out.append(vals)
        return out

    def held(self):
        return [t.cpu().numpy().copy() for t in (self.cache.k_codes, self.cache.k_scale, self.cache.v_codes,
                                                 self.cache.v_scale)]


# -------------------------------------------------------------------- write

def _quantized(x):
    """quantize.py:66-70 of each row of x [.., d]: codes, double scales."""
    q, s = ocpu.quantize_rows(np.ascontiguousarray(x.reshape(-1, x.shape[-1])))
    return q.reshape(x.shape), s.reshape(x.shape[:-1])


@pytest.mark.parametrize("d,kv,page,lengths,counts,tokens", [
    (64, 4, 64, [0, 63, 64, 200], None, 1),                # single tokens, first and last slots of pages
    (128, 2, 16, [0, 5, 31], [37, 0, 9], 37),              # ragged, pages that end inside the rows, none at all
    (32, 3, 32, [7], None, 65),                            # an odd number of heads
    (128, 1, 128, [1, 100], [3, 130], 130),
    (64, 8, 64, [0], None, 300),
])
@pytest.mark.parametrize("values", [False, True])
def test_write_is_bit_exact(cuda_device, d, kv, page, lengths, counts, tokens, values):
    """Codes and scales equal the reference's rule row by row; every other slot
    and the rows past a count stay as they were; the values are the codes times
    the kept scale, one fp32 rounding; k and v are strided columns."""
    n = [tokens] * len(lengths) if counts is None else counts
    book = Book([a + b for a, b in zip(lengths, n)], kv, d, page, seed=d + page)
    before = book.held()
    rs = np.random.RandomState(tokens)
    x = rs.standard_normal((len(lengths), tokens, 3 * kv * d)).astype(np.float32)
    x[0, 0, kv * d:kv * d + d] = 0                          # a row of zeros: scale 1
    x[-1, -1, 2 * kv * d:2 * kv * d + d] = np.arange(d) - d / 2 + 0.5   # ties
    x[:, :, kv * d + 1] *= 30
    xd = _dev(x)
    got = book.cache.write(xd[:, :, kv * d:2 * kv * d], xd[:, :, 2 * kv * d:], book.table, _i32(lengths),
                           None if counts is None else _i32(counts), values=values)
    after = book.held()
    for part in range(2):
        rows = x[:, :, (1 + part) * kv * d:(2 + part) * kv * d].reshape(len(lengths), tokens, kv, d)
        codes, scales = _quantized(rows)
        c, s = before[2 * part], before[2 * part + 1]
        stood = np.zeros(rows.shape, np.float32)
        for b, m in enumerate(n):
            pos = lengths[b] + np.arange(m)
            c[book.table_h[b, pos // page], :, pos % page] = codes[b, :m]
            s[book.table_h[b, pos // page], :, pos % page] = scales[b, :m].astype(np.float32)
            stood[b, :m] = codes[b, :m].astype(np.float32) * scales[b, :m, :, None].astype(np.float32)
        np.testing.assert_array_equal(after[2 * part], c)
        assert after[2 * part + 1].tobytes() == s.tobytes()
        if values:
            np.testing.assert_array_equal(got[part].numpy(), stood.reshape(len(lengths), tokens, kv * d))
    assert values or got is None
    assert _status() == 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_write_marks_rows_that_are_not_finite(cuda_device, bad):
    from kansaiml_b200 import _lib
    book = Book([4], 2, 32, 16)
    k = torch.randn(1, 4, 64, device="cuda")
    v = torch.randn(1, 4, 64, device="cuda")
    k[0, 2, 40] = bad
    book.cache.write(k, v, book.table, _i32([0]))
    assert _status() == _lib.KZ_ERR_NONFINITE
    codes, scale = book.cache.k_codes[book.table_h[0, 0]], book.cache.k_scale[book.table_h[0, 0]]
    assert torch.isnan(scale[1, 2]) and not codes[1, 2].any()
    assert torch.isfinite(scale[:, :4]).sum() == 7


@pytest.mark.parametrize("scale", [1e-42, 1e-33, 1e-30, 3e38])
def test_write_at_the_ends_of_the_range(cuda_device, scale):
    """Rows whose absmax is subnormal, below and above the fast path's border, and near the largest float."""
    book = Book([50], 1, 64, 64)
    x = (np.random.RandomState(3).uniform(-1, 1, (1, 50, 64)) * scale).astype(np.float32)
    book.cache.write(_dev(x), _dev(x), book.table, _i32([0]))
    codes, scales = _quantized(x.reshape(50, 64))
    np.testing.assert_array_equal(book.cache.v_codes[book.table_h[0, 0], 0, :50].cpu().numpy(), codes)
    np.testing.assert_array_equal(book.cache.k_scale[book.table_h[0, 0], 0, :50].cpu().numpy(), scales.astype(np.float32))
    assert _status() == 0


def test_write_copies_views_a_kernel_cannot_read(cuda_device):
    """Odd offsets, transposed and broadcast inputs, and another dtype give the same codes."""
    base = torch.randn(2, 5, 131, device="cuda")
    want = Book([5, 5], 2, 64, 16)
    x = base[:, :, 3:131].contiguous()
    want.cache.write(x, x, want.table, _i32([0, 0]))
    for k in (base[:, :, 3:131], x.transpose(1, 2).contiguous().transpose(1, 2), x.double()):
        book = Book([5, 5], 2, 64, 16)
        book.cache.write(k, x, book.table, _i32([0, 0]))
        for a, b in zip(book.held(), want.held()):
            assert a.tobytes() == b.tobytes()
    one = Book([5, 5], 2, 64, 16)
    one.cache.write(x[:, :1].expand(2, 5, 128), x[:1].expand(2, 5, 128), one.table, _i32([0, 0]))
    full = Book([5, 5], 2, 64, 16)
    full.cache.write(x[:, :1].repeat(1, 5, 1), x[:1].repeat(2, 1, 1), full.table, _i32([0, 0]))
    for a, b in zip(one.held(), full.held()):
        assert a.tobytes() == b.tobytes()


def test_a_single_row_with_any_strides(cuda_device):
    """One row of one sequence is contiguous for torch whatever its strides say."""
    x = torch.randn(1, 1, 128, device="cuda")
    odd = torch.as_strided(x.reshape(-1), (1, 1, 128), (129, 7, 1))
    assert odd.stride() == (129, 7, 1) and odd.is_contiguous()
    books = [Book([5], 2, 64, 16) for _ in range(2)]
    outs = []
    for book, y in zip(books, (x, odd)):
        book.cache.write(y, y, book.table, _i32([4]))
        book.cache.write(y, y, book.table, _i32([0]))
        outs.append(book.cache.attention(y, 2, book.table, _i32([0])).numpy())
    for a, b in zip(books[0].held(), books[1].held()):
        assert a.tobytes() == b.tobytes()
    np.testing.assert_array_equal(outs[0], outs[1])
    assert _status() == 0


# --------------------------------------------------------------------- read

@pytest.mark.parametrize("d,kv,page,lengths,most", [
    (64, 4, 32, [33, 0, 64, 1], 64), (128, 1, 128, [300, 129], 300), (32, 3, 16, [5], 200), (128, 8, 64, [70, 65], 66),
    (32, 1, 16, [0, 0], 3), (64, 2, 64, [10], 0),
])
def test_read_back(cuda_device, d, kv, page, lengths, most):
    """fl32(code * scale) of every token, zeros past a length, nothing past `most`."""
    book = Book(lengths, kv, d, page, seed=page)
    vals = book.fill(lengths)
    got = book.cache.read(book.table, _i32(lengths), most)
    for part in range(2):
        want = np.zeros((len(lengths), most, kv * d), np.float32)
        for b, n in enumerate(lengths):
            n = min(n, most)
            want[b, :n] = vals[part][b][:n].reshape(n, kv * d).astype(np.float32)
        np.testing.assert_array_equal(got[part].numpy(), want)
    assert _status() == 0


# --------------------------------------------------------------------- keep

@pytest.mark.parametrize("d,kv,page", [(32, 3, 16), (64, 4, 64), (128, 2, 32)])
def test_keep_moves_paths_in_place(cuda_device, d, kv, page):
    """Long, short, unmoved and empty paths; other slots stay as they were."""
    lengths, nodes = [14, 0, 63, 5, 30], 70
    paths = [[0, 2, 5, 6, 9], [0], [], list(range(0, 70, 2)) + [69], list(range(1, 70))]
    book = Book([n + nodes for n in lengths], kv, d, page, seed=5)
    book.fill([n + nodes for n in lengths])
    want = book.held()
    path = np.full((5, nodes), -1, np.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = p
        for i, j in enumerate(p):
            new, old = lengths[b] + i, lengths[b] + j
            for x in want:
                x[book.table_h[b, new // page], :, new % page] = x[book.table_h[b, old // page], :, old % page].copy()
    book.cache.keep(book.table, _i32(lengths), _dev(path), _i32([len(p) for p in paths]))
    for a, b in zip(book.held(), want):
        assert a.tobytes() == b.tobytes()
    assert _status() == 0


@pytest.mark.parametrize("path,count", [([0, 2, 2, -1], 3), ([0, 4, -1, -1], 2), ([-1, 1, 2, 3], 2), ([1, 0, 2, 3], 4),
                                        ([0, 1, 2, 3], 5), ([0, 1, 2, 3], -1)])
def test_keep_refuses_paths_that_are_none(cuda_device, path, count):
    from kansaiml_b200 import _lib
    book = Book([8, 8], 1, 32, 16)
    book.fill([8, 8])
    before = book.held()
    book.cache.keep(book.table, _i32([4, 4]), _i32([path, [0, 1, 2, 3]]), _i32([count, 4]))
    assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
    for a, b in zip(book.held(), before):
        assert a.tobytes() == b.tobytes()


# ---------------------------------------------------------------- attention

def _sees(parents, tokens, t):
    if parents is None:
        return list(range(t + 1))
    out = []
    while t >= 0:
        out.append(t)
        up = int(parents[t])
        t = up if 0 <= up < t else -1
    return out


def _attention_64(q, kvals, vvals, length, count, heads, parents, scale):
    """One sequence in float64: output [tokens, heads * d] and the bound on a
    32-bit kernel's error.  A product q . k of d terms whose factors are held to
    22 bits or more and summed in 32 bits, each addition off by at most
    2^-23 of the terms' absolute sum, is off by (d + 4) 2^-23 sum |q k|; a
    weight's relative error is twice that (its own and the largest's) plus the
    exponential's and its own 22 bits; the weighted sum of n values adds
    2^-23 for each 16 keys that a partial sum covers, and 32 for the joining.
    The 22 bits are two fp16 values of an operand whose largest is brought to
    [2^13, 2^14): below 2^-14 fp16 has steps of 2^-24 only, so that a factor is
    off by 2^-25 at least, 2^-38 of the largest in its row: max|q| 2^-38 a term
    of a product (doubled, as above), max(w |v|) 2^-38 a term of the sum."""
    tokens, kv, d = q.shape[0], kvals.shape[1], kvals.shape[2]
    out, bound = np.zeros((tokens, heads * d)), np.zeros((tokens, heads * d))
    for t in range(count):
        seen = np.array(list(range(length)) + [length + j for j in _sees(parents, tokens, t)])
        for h in range(heads):
            k, v = kvals[seen, h * kv // heads], vvals[seen, h * kv // heads]
            qq = q[t, h * d:(h + 1) * d].astype(np.float64)
            s = k @ qq * scale
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[t, h * d:(h + 1) * d] = w @ v
            size = abs(scale)
            off = 2 * (d + 4) * (np.abs(k) @ np.abs(qq)).max() * size + 16 + len(seen) / 16 + 32
            small = 2 * size * np.abs(qq).max() * np.abs(k).sum(1).max() * (w @ np.abs(v)) + len(seen) * (w * np.abs(v).max(1)).max()
            bound[t, h * d:(h + 1) * d] = off * 2.0**-23 * (w @ np.abs(v)) + 2.0**-38 * small
    return out, bound


def _check_attention(book, lengths, counts, tokens, heads, parents=None, seed=9, spread=1.0, strong=1.5, view=False,
                     scale=None):
    n = [tokens] * len(lengths) if counts is None else counts
    kvals, vvals = book.fill([a + b for a, b in zip(lengths, n)], seed=seed, spread=spread)
    q = (np.random.RandomState(seed).standard_normal((len(lengths), tokens, heads * book.d)) * strong).astype(np.float32)
    qd = _dev(q)
    if view:     # columns of a fused projection
        wide = torch.full((len(lengths), tokens, heads * book.d + 64), math.nan, device="cuda")
        wide[:, :, 32:-32] = qd
        qd = wide[:, :, 32:-32]
    pd = None if parents is None else _dev(np.asarray(parents, np.int32))
    y = book.cache.attention(qd, heads, book.table, _i32(lengths), None if counts is None else _i32(counts), pd,
                             scale).numpy()
    for b in range(len(lengths)):
        par = None if parents is None else np.asarray(parents) if np.ndim(parents) == 1 else np.asarray(parents)[b]
        want, bound = _attention_64(q[b], kvals[b], vvals[b], lengths[b], n[b], heads, par,
                                    1 / math.sqrt(book.d) if scale is None else scale)
        off = np.abs(y[b] - want)
        assert np.all(off <= bound), (b, (off - bound).max(), (off / np.maximum(bound, 1e-300)).max())
        assert not y[b, n[b]:].any()
    assert _status() == 0
    return y


@pytest.mark.parametrize("d,kv,heads,page", [(64, 4, 4, 64), (128, 2, 8, 16), (128, 1, 32, 128), (32, 3, 9, 32),
                                             (64, 2, 14, 32), (128, 2, 2, 64)])
def test_attention_single_tokens(cuda_device, d, kv, heads, page):
    """One new token a sequence, lengths from none to several tiles and their neighbours."""
    lengths = [0, 1, 15, 16, 31, 63, 64, 127, 128, 255, 300, 1030]
    book = Book([n + 1 for n in lengths], kv, d, page, seed=heads)
    _check_attention(book, lengths, None, 1, heads, view=heads == kv)


@pytest.mark.parametrize("d,kv,heads,page,tokens", [(64, 2, 2, 64, 5), (128, 1, 4, 32, 33), (32, 2, 8, 16, 130),
                                                    (128, 2, 4, 128, 70), (64, 1, 3, 64, 17)])
def test_attention_chunks(cuda_device, d, kv, heads, page, tokens):
    """Several new tokens, causal among themselves, with padding rows, none at all, and no context."""
    lengths, counts = [0, 40, 200, 77], [tokens, 1, 0, tokens - 2]
    book = Book([a + b for a, b in zip(lengths, counts)], kv, d, page, seed=tokens)
    _check_attention(book, lengths, counts, tokens, heads, view=tokens == 33)


def _tree(n, seed, deep=False):
    rs = np.random.RandomState(seed)
    return [-1] + [j - 1 if deep else int(rs.randint(0, j)) for j in range(1, n)]


@pytest.mark.parametrize("d,kv,heads,page,nodes", [(64, 4, 4, 64, 6), (128, 2, 8, 64, 24), (128, 1, 8, 32, 64),
                                                   (32, 2, 2, 16, 256), (64, 2, 6, 128, 100)])
def test_attention_trees(cuda_device, d, kv, heads, page, nodes):
    """A random tree a sequence, one of them a chain, one a star, one of roots only."""
    lengths, counts = [100, 0, 64, 37], [nodes, nodes - 1, nodes, nodes]
    parents = [_tree(nodes, 1), _tree(nodes, 2, deep=True), [-1] + [0] * (nodes - 1), [-1] * nodes]
    book = Book([a + b for a, b in zip(lengths, counts)], kv, d, page, seed=nodes)
    _check_attention(book, lengths, counts, nodes, heads, parents)


def test_attention_one_tree_for_all_and_odd_parents(cuda_device):
    """parents [nodes] serves every sequence; a parent that is not before its child is none."""
    book = Book([60, 61], 2, 64, 16)
    _check_attention(book, [50, 51], None, 10, 4, _tree(10, 3))
    _check_attention(book, [50, 51], None, 10, 4, [[-1, 0, 5, 2, 99, 4, -7, 7, 7, 3], _tree(10, 4)])


def test_attention_chain_is_causal(cuda_device):
    """A tree that is a chain gives what no tree gives, bit for bit."""
    book = Book([90, 133], 2, 64, 32)
    a = _check_attention(book, [57, 100], None, 33, 4, _tree(33, 0, deep=True))
    b = _check_attention(book, [57, 100], None, 33, 4)
    assert a.tobytes() == b.tobytes()


@pytest.mark.parametrize("tokens", [1, 12])
@pytest.mark.parametrize("spread,strong", [(12.0, 1e-4), (0.5, 12.0), (30.0, 1e-12), (1.0, 0.0), (1.0, 1e-30)])
def test_attention_extreme_scales(cuda_device, tokens, spread, strong):
    """Scales over many orders of magnitude, nearly one-hot softmaxes, q of zeros and of tiny values."""
    book = Book([401, 200], 2, 64, 64)
    _check_attention(book, [401 - tokens, 200 - tokens], None, tokens, 4, spread=spread, strong=strong)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("spread,strong", [(12.0, 1e-4), (0.5, 12.0), (30.0, 1e-12), (1.0, 0.0), (1.0, 1e-30)])
def test_attention_extreme_scales_many_rows(cuda_device, d, spread, strong):
    """The same with more rows a key head than the small kernel takes (40 x 2, and 70 x 4 in three row tiles)."""
    book = Book([441, 140], 2, d, 32)
    _check_attention(book, [401, 100], None, 40, 4, spread=spread, strong=strong)
    book = Book([270], 1, d, 64)
    _check_attention(book, [200], None, 70, 4, _tree(70, 3), spread=spread, strong=strong)


@pytest.mark.parametrize("d,kv,heads,tokens,tree", [(64, 3, 3, 4, True), (128, 2, 2, 3, False), (32, 1, 2, 2, True),
                                                    (128, 2, 4, 1, False), (64, 1, 3, 1, False), (32, 2, 2, 4, False)])
@pytest.mark.parametrize("spread,strong", [(1.0, 1.5), (12.0, 1e-4), (0.5, 12.0), (30.0, 1e-12), (1.0, 0.0)])
def test_attention_up_to_four_rows(cuda_device, d, kv, heads, tokens, tree, spread, strong):
    """A key head's rows are one to four: trees, chunks with padding and single
    tokens, whole and in parts, at ordinary and extreme scales."""
    lengths, counts = [0, 33, 500, 1700], [tokens, max(tokens - 1, 1), 0, tokens]
    book = Book([a + b for a, b in zip(lengths, counts)], kv, d, 32, seed=d)
    parents = [_tree(tokens, b) for b in range(4)] if tree else None
    _check_attention(book, lengths, counts, tokens, heads, parents, spread=spread, strong=strong)


def test_attention_scale_argument(cuda_device):
    book = Book([300], 1, 32, 16)
    _check_attention(book, [299], None, 1, 2, scale=0.03)
    _check_attention(book, [299], None, 1, 2, scale=0.9)
    book = Book([340], 1, 32, 16)
    for scale in (0.03, 0.9, -0.2, 0.0):
        _check_attention(book, [300], None, 40, 2, scale=scale)
        _check_attention(book, [330], None, 1, 2, scale=scale)


@pytest.mark.parametrize("lengths,tokens,heads,kv", [([20000], 1, 8, 1), ([9000, 3, 5000], 1, 2, 2), ([7000], 40, 4, 1)])
def test_attention_long(cuda_device, lengths, tokens, heads, kv):
    """Contexts that are split over many blocks and joined."""
    book = Book([n + tokens for n in lengths], kv, 128, 64)
    _check_attention(book, lengths, None, tokens, heads)


@pytest.mark.parametrize("tokens,heads", [(1, 8), (12, 4), (50, 8)])
def test_attention_is_repeatable(cuda_device, tokens, heads):
    """The same call gives the same bits."""
    book = Book([3000, 700], 2, 128, 64)
    lengths = [3000 - tokens, 700 - tokens]
    a = _check_attention(book, lengths, None, tokens, heads)
    for _ in range(3):
        assert _check_attention(book, lengths, None, tokens, heads).tobytes() == a.tobytes()


@pytest.mark.parametrize("d,kv,heads,tokens,spans", [
    (64, 2, 8, 1, [(40, 600)]), (128, 3, 3, 1, [(1, 1500)]), (32, 1, 4, 2, [(5, 5), (1, 900), (30, 140)]),
    (64, 2, 16, 20, [(1, 1200), (1, 50)]), (32, 4, 16, 20, [(40, 300)]), (128, 1, 8, 17, [(3, 2400), (20, 130)]),
    (64, 2, 8, 1, [(600, 9)]), (64, 1, 1, 3, [(7, 0)])])
def test_attention_in_a_table_wider_than_its_sequences(cuda_device, d, kv, heads, tokens, spans):
    """The table has room for far more than the sequences hold, so how the keys
    are dealt out follows from the lengths: few and many sequences, short and
    long ones together, rows without tokens, and no tokens at all."""
    rs = np.random.RandomState(tokens * d)
    most = [n for many, n in spans for _ in range(many)]
    counts = [int(rs.randint(0, tokens + 1)) if n else 0 for n in most]
    counts[0] = tokens if most[0] else 0
    lengths = [int(rs.randint(n // 2, n + 1)) for n in most]
    book = Book([a + b for a, b in zip(lengths, counts)], kv, d, 16)
    wide = torch.full((len(most), 300), -1, dtype=torch.int32, device="cuda")
    wide[:, :book.table.shape[1]] = book.table
    book.table = wide
    _check_attention(book, lengths, counts, tokens, heads)


def test_attention_many_sequences(cuda_device):
    """More sequences than a block has threads, most of them without tokens."""
    rs = np.random.RandomState(2)
    lengths = [int(n) for n in rs.randint(0, 40, 300)]
    counts = [int(n) for n in rs.randint(0, 2, 300)]
    lengths[150], counts[150] = 900, 1
    book = Book([a + b for a, b in zip(lengths, counts)], 1, 32, 16)
    _check_attention(book, lengths, counts, 1, 1)
    counts = [3 * c for c in counts]
    book = Book([a + b for a, b in zip(lengths, counts)], 1, 32, 16)
    _check_attention(book, lengths, counts, 3, 12)


def test_attention_nan_in_a_visible_row_only(cuda_device):
    """A NaN scale in a token's row reaches the rows that see it and no others."""
    book = Book([70], 2, 64, 32)
    book.fill([70])
    q = torch.randn(1, 6, 4 * 64, device="cuda")
    # node 65's V row of head 1: seen by itself and its descendants (nodes 1 and 3 of the tree)
    book.cache.v_scale[book.table_h[0, 65 // 32], 1, 65 % 32] = math.nan
    y = book.cache.attention(q, 4, book.table, _i32([64]), None, _i32([-1, 0, 0, 1, 2, 0])).data.view(6, 4, 64)
    bad = torch.isnan(y).all(-1).cpu()
    want = torch.zeros(6, 4, dtype=torch.bool)
    want[1, 2:] = want[3, 2:] = True
    assert torch.equal(bad, want) and torch.equal(torch.isnan(y).any(-1).cpu(), want)


@pytest.mark.parametrize("part", ["k", "v"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_nan_among_many_rows(cuda_device, part, d):
    """The same in the kernel for many rows: 40 nodes, a NaN or infinite scale
    at one of them, NaN throughout where no token is."""
    book = Book([140], 2, d, 32)
    book.fill([140])
    parents = _tree(40, 5)
    q = torch.randn(1, 40, 4 * d, device="cuda")
    for bad in (math.nan, math.inf):
        at = 100 + 7
        scale = book.cache.k_scale if part == "k" else book.cache.v_scale
        was = scale[book.table_h[0, at // 32], 1, at % 32].clone()
        scale[book.table_h[0, at // 32], 1, at % 32] = bad
        y = book.cache.attention(q, 4, book.table, _i32([100]), None, _i32(parents)).data.view(40, 4, d)
        sees = torch.tensor([7 in _sees(parents, 40, t) for t in range(40)])
        good = torch.isfinite(y).all(-1).cpu()
        assert good[:, :2].all() and good[~sees].all()
        if part == "v" or math.isnan(bad):
            assert not torch.isfinite(y).any(-1).cpu()[sees][:, 2:].any()
        scale[book.table_h[0, at // 32], 1, at % 32] = was
    assert _status() == 0


@pytest.mark.parametrize("tokens,parents", [(20, True), (40, True), (40, False), (9, False)])
def test_bad_pages_among_many_rows(cuda_device, tokens, parents):
    """Two pages of the context and one of the new tokens' that are none."""
    from kansaiml_b200 import _lib
    n = 200 + tokens
    book = Book([n], 1, 64, 16)
    kvals, vvals = book.fill([n])
    table = book.table.clone()
    for i in (0, 7, 13):
        table[0, i] = 10 ** 6 if i else -1
    par = _tree(tokens, 2) if parents else None
    q = np.random.RandomState(4).standard_normal((1, tokens, 4 * 64)).astype(np.float32)
    y = book.cache.attention(_dev(q), 4, table, _i32([200]), None, None if par is None else _i32(par)).numpy()[0]
    assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
    there = np.array([p // 16 not in (0, 7, 13) for p in range(n)])
    for t in range(tokens):
        seen = [p for p in list(range(200)) + [200 + j for j in _sees(par, tokens, t)] if there[p]]
        for h in range(4):
            want, bound = _attention_64(q[0, t:t + 1, h * 64:(h + 1) * 64], kvals[0][seen], vvals[0][seen], len(seen) - 1, 1,
                                        1, None, 1 / 8)
            assert np.all(np.abs(y[t, h * 64:(h + 1) * 64] - want[0]) <= bound[0]), (t, h)


def test_bad_pages_are_left_out_and_reported(cuda_device):
    """A page number outside the pool, or a position past the table, reads and writes nothing."""
    from kansaiml_b200 import _lib
    for wrong in (10 ** 6, -2):
        book = Book([40], 1, 64, 16)
        kvals, vvals = book.fill([40])
        table = book.table.clone()
        table[0, 1] = wrong
        q = torch.randn(1, 1, 64, device="cuda")
        y = book.cache.attention(q, 1, table, _i32([39])).numpy()[0, 0]
        assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
        seen = np.r_[0:16, 32:40]
        want, bound = _attention_64(q.cpu().numpy()[0], kvals[0][seen], vvals[0][seen], len(seen) - 1, 1, 1, None, 1 / 8)
        assert np.all(np.abs(y - want[0]) <= bound[0])
        k, v = book.cache.read(table, _i32([40]), 40)
        assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
        assert not k.data[0, 16:32].any() and not v.data[0, 16:32].any()
        np.testing.assert_array_equal(k.numpy()[0, seen], kvals[0][seen, 0].astype(np.float32))
        before = book.held()
        book.cache.write(torch.randn(1, 3, 64, device="cuda"), torch.randn(1, 3, 64, device="cuda"), table, _i32([20]))
        assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
        book.cache.keep(table, _i32([20]), _i32([[1, 2]]), _i32([2]))
        assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
        for a, b in zip(book.held(), before):
            assert a.tobytes() == b.tobytes()
    # lengths past the table, and below 0
    for length in (10 ** 9, -5):
        book.cache.attention(torch.randn(1, 2, 64, device="cuda"), 1, book.table, _i32([length]))
        book.cache.write(torch.randn(1, 3, 64, device="cuda"), torch.randn(1, 3, 64, device="cuda"), book.table,
                         _i32([length]))
        assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
    for a, b in zip(book.held(), before):
        assert a.tobytes() == b.tobytes()


def test_empty_calls(cuda_device):
    book = Book([4], 2, 32, 16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    z = torch.empty(0, 3, 64, device="cuda")
    assert book.cache.attention(z, 2, book.table[:0], none).shape == [0, 3, 64]
    book.cache.write(z, z, book.table[:0], none)
    assert book.cache.attention(torch.empty(1, 0, 64, device="cuda"), 2, book.table, _i32([4])).shape == [1, 0, 64]
    assert book.cache.read(book.table[:0], none, 5)[0].shape == [0, 5, 64]
    assert _status() == 0


@pytest.mark.parametrize("tokens,parents", [(5, False), (40, True)])
def test_attention_nan_in_q_stays_in_its_row(cuda_device, tokens, parents):
    """A NaN or infinity in one row of q, and a very large row beside ordinary ones."""
    book = Book([150], 1, 64, 16)
    book.fill([150])
    par = _i32(_tree(tokens, 6)) if parents else None
    q = torch.randn(1, tokens, 4 * 64, device="cuda")
    lengths = _i32([150 - tokens])
    want = book.cache.attention(q, 4, book.table, lengths, None, par).data.view(tokens, 4, 64)
    for bad in (math.nan, math.inf, 1e30):
        x = q.clone()
        x[0, 2, 64 + 9] = bad
        y = book.cache.attention(x, 4, book.table, lengths, None, par).data.view(tokens, 4, 64)
        if bad != 1e30:
            assert torch.isnan(y[2, 1]).all()
        y[2, 1] = want[2, 1]
        assert torch.equal(y, want)
    assert _status() == 0


def test_offsets_past_32_bits(cuda_device):
    """A pool of more than 2^31 bytes of codes, its last pages used: written,
    attended over by both kernels, kept and read."""
    from kansaiml_b200.cache import QCache
    pages, kv, page, d = 17000, 8, 128, 128
    cache = QCache(pages, kv, d, page, "cuda")
    assert cache.k_codes.numel() > 2**31
    table, zero = _i32([[pages - 1, pages - 3, pages - 2]]), _i32([0])
    rs = np.random.RandomState(8)
    k, v = (rs.standard_normal((1, 300, kv * d)).astype(np.float32) for _ in range(2))
    cache.write(_dev(k), _dev(v), table, zero)
    stood = []
    for x in (k, v):
        codes, scales = _quantized(x.reshape(300, kv, d))
        stood.append(codes * scales.astype(np.float32).astype(np.float64)[..., None])
    for tokens in (1, 40):
        q = rs.standard_normal((1, tokens, kv * d)).astype(np.float32)
        y = cache.attention(_dev(q), kv, table, _i32([300 - tokens])).numpy()[0]
        want, bound = _attention_64(q[0], stood[0], stood[1], 300 - tokens, tokens, kv, None, d**-0.5)
        assert np.all(np.abs(y - want) <= bound)
    cache.keep(table, _i32([100]), _i32([[0, 50, 199] + [-1] * 197]), _i32([3]))     # a path of a tree of 200
    got = cache.read(table, _i32([103]), 103)
    for part in range(2):
        want = stood[part][[*range(101), 150, 299]].reshape(103, kv * d).astype(np.float32)
        np.testing.assert_array_equal(got[part].numpy()[0], want)
    assert _status() == 0


# ------------------------------------------------------------- verification

def _verify_64(tokens, parents, target, draft, au, su):
    """One sequence, in float64, straight from the definition."""
    n, vocab = target.shape
    node, r, path = 0, target[0].astype(np.float64), [0]
    for j in range(1, n):
        if parents[j] != node or not 0 <= parents[j] < j or not 0 <= tokens[j] < vocab:
            continue
        q = draft[node].astype(np.float64) if draft is not None else np.eye(vocab)[tokens[j]]
        if float(au[j]) * q[tokens[j]] < r[tokens[j]]:
            node, r = j, target[j].astype(np.float64)
            path.append(j)
        else:
            rest = np.maximum(r - q, 0)
            if rest.sum() > 0:
                r = rest / rest.sum()
    below = np.cumsum(r)
    return path, min(int(np.searchsorted(below, float(su) * below[-1], side="right")), vocab - 1)


def _softmax(rs, shape, strength):
    x = rs.standard_normal(shape) * strength
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("batch,nodes,vocab,draft", [
    (40, 8, 65, True), (40, 8, 65, False), (5, 1, 1, False), (9, 1, 50000, False), (7, 24, 2049, True), (3, 40, 100003, True),
    (3, 40, 32768, False), (2, 300, 33, True), (16, 5, 2, True),
])
@pytest.mark.parametrize("shared", [False, True])
def test_verify_tree(cuda_device, batch, nodes, vocab, draft, shared):
    from kansaiml_b200.cache import verify_tree
    rs = np.random.RandomState(batch * nodes + vocab)
    target = _softmax(rs, (batch, nodes, vocab), 2.0)
    q = (0.6 * target + 0.4 * _softmax(rs, (batch, nodes, vocab), 2.0)).astype(np.float32)
    parents = np.array([_tree(nodes, 7 if shared else 100 + b) for b in range(batch)], np.int32)
    tokens = np.zeros((batch, nodes), np.int64)
    for b in range(batch):
        for j in range(1, nodes):
            p = q[b, parents[b, j]].astype(np.float64)
            tokens[b, j] = rs.choice(vocab, p=p / p.sum())
    au, su = rs.uniform(size=(batch, nodes)).astype(np.float32), rs.uniform(size=batch).astype(np.float32)
    path, count, token = verify_tree(_dev(tokens), _dev(parents[0] if shared else parents), _dev(target),
                                     _dev(q) if draft else None, _dev(au), _dev(su))
    path, count, token = path.cpu().numpy(), count.cpu().numpy(), token.cpu().numpy()
    for b in range(batch):
        want, nxt = _verify_64(tokens[b], parents[b], target[b], q[b] if draft else None, au[b], su[b])
        assert path[b].tolist() == want + [-1] * (nodes - len(want)), b
        assert count[b] == len(want) and token[b] == nxt, b
    assert _status() == 0


def test_verify_edges(cuda_device):
    """u = 0 and the largest u below 1, zeros around the mass, a draft that equals
    the target, the same token twice, and rows that are no distribution."""
    from kansaiml_b200.cache import verify_tree
    top = np.nextafter(np.float32(1), np.float32(0))
    v = 3000
    p = np.zeros((6, 3, v), np.float32)
    p[:, :, 1000] = 0.25
    p[:, :, 2500] = 0.75
    q = p.copy()
    q[3:, 0] = 0
    q[3:, 0, 7] = 1                                          # token 7 has no mass in the target
    tokens = np.array([[0, 1000, 2500]] * 3 + [[0, 7, 7]] * 3, np.int64)
    parents = np.array([[-1, 0, 0]] * 6, np.int32)
    au = np.array([[0, 0, 0], [0, top, top], [0, top, 0], [0, 0, 0], [0, top, top], [0, 0.5, 0.5]], np.float32)
    su = np.array([0, top, 0.25, 0, top, 0.2499999], np.float32)
    for draft in (q, None):
        path, count, token = verify_tree(_dev(tokens), _dev(parents), _dev(p), None if draft is None else _dev(draft),
                                         _dev(au), _dev(su))
        for b in range(6):
            want, nxt = _verify_64(tokens[b], parents[b], p[b], None if draft is None else draft[b], au[b], su[b])
            assert path[b].tolist() == want + [-1] * (3 - len(want)) and count[b] == len(want) and token[b] == nxt, b
    # no mass at all, and tokens and parents that are none: an answer inside the vocabulary, nothing read outside
    path, count, token = verify_tree(_dev(np.array([[0, -1, v]])), _i32([[5, 0, 0]]), torch.zeros(1, 3, v, device="cuda"),
                                     None, torch.rand(1, 3, device="cuda"), torch.rand(1, device="cuda"))
    from kansaiml_b200 import _lib
    assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
    assert count.tolist() == [1] and path.tolist() == [[0, -1, -1]] and token.tolist() == [v - 1]


@pytest.mark.parametrize("draft", [True, False])
def test_verified_tokens_follow_the_target(cuda_device, draft):
    """Whatever is drafted, the token after the root is distributed as the
    target's row: 20000 trees of four drafts from a wrong distribution.  Each
    frequency is within 5 standard deviations (a chance of 6e-7 each) of p."""
    from kansaiml_b200.cache import verify_tree
    n, v = 20000, 6
    rs = np.random.RandomState(11)
    p = np.array([0.4, 0.05, 0.25, 0.0, 0.2, 0.1], np.float32)
    q = np.array([0.1, 0.3, 0.2, 0.2, 0.1, 0.1], np.float32)
    target = np.broadcast_to(p, (n, 5, v))
    tokens = np.concatenate([np.zeros((n, 1)), rs.choice(v, (n, 4), p=q.astype(np.float64) / q.astype(np.float64).sum())],
                            1).astype(np.int64)
    path, count, token = verify_tree(_dev(tokens), _i32([-1, 0, 0, 0, 0]), _dev(target),
                                     _dev(np.broadcast_to(q, (n, 5, v))) if draft else None,
                                     _dev(rs.uniform(size=(n, 5)).astype(np.float32)),
                                     _dev(rs.uniform(size=n).astype(np.float32)))
    path, count, token = path.cpu().numpy(), count.cpu().numpy(), token.cpu().numpy()
    first = np.where(count > 1, tokens[np.arange(n), np.maximum(path[:, 1], 0)], token)
    seen = np.bincount(first, minlength=v) / n
    assert np.all(np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-12), seen


# ----------------------------------------------------- together, as a model uses them

def test_speculative_steps_together(cuda_device):
    """Write, attention, verification and keep over several steps of trees, the
    cache then holding exactly the accepted tokens; every step's attention
    equals the 64-bit one over what the host's own books say is cached."""
    from kansaiml_b200.cache import PagePool, QCache, verify_tree
    rs = np.random.RandomState(21)
    batch, kv, heads, d, page, nodes, vocab = 3, 2, 6, 64, 16, 7, 11
    pool = PagePool(40, batch, 8, page, "cuda")
    cache = QCache(40, kv, d, page, "cuda")
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    books = [[np.zeros((0, kv, d)), np.zeros((0, kv, d))] for _ in range(batch)]
    for step in range(6):
        n = 20 if step == 0 else nodes
        parents = None if step == 0 else np.array([_tree(n, 50 * step + b) for b in range(batch)], np.int32)
        kvs = rs.standard_normal((2, batch, n, kv * d)).astype(np.float32)
        q = rs.standard_normal((batch, n, heads * d)).astype(np.float32)
        pool.reserve(max(len(b[0]) for b in books) + n)
        cache.write(_dev(kvs[0]), _dev(kvs[1]), pool.table, lengths)
        y = cache.attention(_dev(q), heads, pool.table, lengths, None, None if parents is None else _dev(parents)).numpy()
        new = []
        for b in range(batch):
            stood = []
            for part in range(2):
                codes, scales = _quantized(kvs[part, b].reshape(n, kv, d))
                stood.append(codes * scales.astype(np.float32).astype(np.float64)[..., None])
            new.append(stood)
            have = len(books[b][0])
            want, bound = _attention_64(q[b], np.concatenate([books[b][0], stood[0]]), np.concatenate([books[b][1], stood[1]]),
                                        have, n, heads, None if parents is None else parents[b], 1 / 8)
            assert np.all(np.abs(y[b] - want) <= bound)
        if parents is None:
            paths = [list(range(n))] * batch
            lengths += n
        else:
            target = _softmax(rs, (batch, n, vocab), 1.0)
            tokens = rs.randint(0, vocab, (batch, n)).astype(np.int64)
            path, count, _ = verify_tree(_dev(tokens), _dev(parents), _dev(target), None,
                                         _dev(rs.uniform(size=(batch, n)).astype(np.float32) * 0.2),
                                         _dev(rs.uniform(size=batch).astype(np.float32)))
            cache.keep(pool.table, lengths, path, count)
            lengths += count
            paths = [p[:c] for p, c in zip(path.tolist(), count.tolist())]
        for b in range(batch):
            books[b] = [np.concatenate([books[b][i], new[b][i][paths[b]]]) for i in range(2)]
        k, v = cache.read(pool.table, lengths, max(len(b[0]) for b in books))
        for b in range(batch):
            for got, book in zip((k, v), books[b]):
                np.testing.assert_array_equal(got.numpy()[b, :len(book)], book.reshape(len(book), kv * d).astype(np.float32))
    assert _status() == 0


@pytest.mark.parametrize("quantized", [True, False])
def test_module_attention_over_a_cache(cuda_device, quantized):
    """MultiHeadAttention with a step: the output projection of the attention
    over the cache of its own projections, for a prompt and a token after it."""
    from kansaiml_b200 import nn as knn
    from kansaiml_b200.cache import PagePool, QCache
    from kansaiml_b200.tensor import Tensor
    mha = knn.MultiHeadAttention(128, 2, seed=4, device="cuda")
    if quantized:
        mha.quantize(per_channel=True)
    pool, cache = PagePool(8, 2, 4, 16, "cuda"), QCache(8, 2, 64, 16, "cuda")
    pool.reserve(60)
    seen = []
    inner = QCache.attention

    def spy(self, q, *args, **kw):
        out = inner(self, q, *args, **kw)
        seen.append((q.cpu().numpy(), out.numpy()))
        return out

    lengths = _i32([0, 0])
    QCache.attention = spy
    try:
        for n in (33, 1, 4):
            x = Tensor(torch.randn(2, n, 128, device="cuda"))
            step = knn.CacheStep(cache, pool.table, lengths)
            y = mha(x, x, x, step=step)
            assert y.shape == [2, n, 128]
            k, v = cache.read(pool.table, lengths + n, int(lengths[0]) + n)
            for b in range(2):
                want, bound = _attention_64(seen[-1][0][b], k.numpy()[b].reshape(-1, 2, 64).astype(np.float64),
                                            v.numpy()[b].reshape(-1, 2, 64).astype(np.float64), int(lengths[0]), n, 2,
                                            None, 1 / 8)
                assert np.all(np.abs(seen[-1][1][b] - want) <= bound)
            lengths += n
    finally:
        QCache.attention = inner
    with pytest.raises(ValueError, match="self-attention"):
        mha(x, Tensor(x.data.clone()), x, step=step)
    assert _status() == 0


def test_decoder_generates_through_the_cache(cuda_device):
    """Decoder.generate: ragged prompts, with and without looked-up drafts; the
    logits of a prompt through the cache are near those of the whole-context
    forward (its K/V are quantized once more: 8 bits of them, so 5% of the
    logits' norm is far beyond what the rounding moves)."""
    from kansaiml_b200 import workloads
    model = workloads.Decoder(seed=3)
    ids = workloads.config3_ids(batch=4, ctx=100, seed=4)
    cache = model.new_cache(4)
    whole = model(ids).data
    got = model.extend(ids, cache).data
    assert (got - whole).norm() <= 0.05 * whole.norm()
    cache.advance(100, 100)
    more = model.extend(ids[:, :1], cache).data
    assert more.shape == (4, 1, 65) and torch.isfinite(more).all()
    prompts = [ids[i, :n].tolist() for i, n in enumerate((5, 40, 100, 1))]
    for temperature in (0.0, 1.0):
        for drafts in (0, 6):
            a = model.generate(prompts, 30, temperature, drafts, seed=7)
            assert [len(o) for o in a] == [30] * 4 and all(0 <= t < 65 for o in a for t in o)
            assert a == model.generate(prompts, 30, temperature, drafts, seed=7)
    with pytest.raises(ValueError, match="context"):
        model.generate(prompts, 157)
    for empty in ([[1], []], []):
        with pytest.raises(ValueError, match="prompt"):
            model.generate(empty, 3)
    for drafts in (-1, 256):
        with pytest.raises(ValueError, match="drafts"):
            model.generate(prompts, 3, 1.0, drafts)
    for temperature in (-1.0, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            model.generate(prompts, 3, temperature)
    with pytest.raises(ValueError, match="capacity"):
        cache.room(200)
    assert _status() == 0


# ----------------------------------------------------- capture, streams, devices, refusals

def test_captured_steps_replay_with_new_lengths(cuda_device):
    """A step captured into a graph reads lengths, pages and inputs anew at
    each replay; two graphs of the same cache do not share scratch."""
    book = Book([1500, 700], 2, 128, 64)
    lengths, q = _i32([0, 0]), torch.zeros(2, 1, 8 * 128, device="cuda")
    q2, l2 = torch.zeros(2, 20, 8 * 128, device="cuda"), _i32([0, 0])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        book.cache.attention(q, 8, book.table, lengths)
        book.cache.attention(q2, 8, book.table, l2)
    stream.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        y1 = book.cache.attention(q, 8, book.table, lengths).data
    with torch.cuda.graph(two):
        y2 = book.cache.attention(q2, 8, book.table, l2).data
    book.fill([1500, 700])
    for at in ([1499, 699], [3, 500], [800, 0]):
        lengths.copy_(_i32(at))
        l2.copy_(_i32([max(0, n - 30) for n in at]))
        q.copy_(torch.randn_like(q))
        q2.copy_(torch.randn_like(q2))
        one.replay()
        two.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, book.cache.attention(q, 8, book.table, lengths).data)
        assert torch.equal(y2, book.cache.attention(q2, 8, book.table, l2).data)
    assert _status() == 0


@pytest.mark.parametrize("nodes,vocab,draft", [(7, 11, False), (40, 9000, True)])
def test_a_captured_run_of_all(cuda_device, nodes, vocab, draft):
    """Write, attention over a tree, verification, keep and the new lengths as
    one graph, with no call before the capture: each replay leaves what the
    same calls leave one by one."""
    from kansaiml_b200.cache import verify_tree
    batch, kv, heads, d = 3, 2, 4, 64
    rs = np.random.RandomState(31)
    books = [Book([700, 650, 900], kv, d, 32) for _ in range(2)]
    for book in books:
        book.fill([300, 20, 511])
    lengths = [_i32([300, 20, 511]) for _ in range(2)]
    k, v, q = (torch.zeros(batch, nodes, n * d, device="cuda") for n in (kv, kv, heads))
    tokens, parents = torch.zeros(batch, nodes, dtype=torch.int64, device="cuda"), _i32([[-1] * nodes] * batch)
    target, other = (torch.zeros(batch, nodes, vocab, device="cuda") for _ in range(2))
    au, su = torch.zeros(batch, nodes, device="cuda"), torch.zeros(batch, device="cuda")

    def step(book, lengths):
        book.cache.write(k, v, book.table, lengths)
        y = book.cache.attention(q, heads, book.table, lengths, None, parents).data
        path, count, token = verify_tree(tokens, parents, target, other if draft else None, au, su)
        book.cache.keep(book.table, lengths, path, count)
        lengths += count
        return y, path, count, token

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(books[0], lengths[0])
    for turn in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        tokens.copy_(_dev(rs.randint(0, vocab, (batch, nodes))))
        parents.copy_(_dev(np.array([_tree(nodes, 10 * turn + b) for b in range(batch)], np.int32)))
        for t in (target, other):
            t.copy_(_dev(_softmax(rs, (batch, nodes, vocab), 1.0)))
        au.copy_(_dev(rs.uniform(size=(batch, nodes)).astype(np.float32) * (1e-4 if turn % 2 else 0.3)))
        su.copy_(_dev(rs.uniform(size=batch).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(books[1], lengths[1])):
            assert torch.equal(a, b)
        assert torch.equal(lengths[0], lengths[1])
    most = int(lengths[0].max())
    for a, b in zip(*(book.cache.read(book.table, n, most) for book, n in zip(books, lengths))):
        assert torch.equal(a.data, b.data)
    assert _status() == 0


def test_two_streams_at_once(cuda_device):
    book = Book([2000, 2000], 2, 64, 64)
    book.fill([2000, 2000])
    q = [torch.randn(2, 1, 8 * 64, device="cuda") for _ in range(2)]
    lengths = _i32([1999, 1500])
    want = [book.cache.attention(x, 8, book.table, lengths).data for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(book.cache.attention(q[i], 8, book.table, lengths).data)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_refusals(cuda_device):
    from kansaiml_b200.cache import QCache, verify_tree
    book = Book([40], 2, 64, 16)
    c, t, n = book.cache, book.table, _i32([3])
    x = torch.zeros(1, 2, 128, device="cuda")
    for bad, match in (((48, 2), "head_dim"), ((64, 0), "kv_heads")):
        with pytest.raises(ValueError, match=match):
            QCache(4, bad[1], bad[0], 16, "cuda")
    with pytest.raises(ValueError, match="page_size"):
        QCache(4, 2, 64, 24, "cuda")
    with pytest.raises(ValueError, match="contiguous"):
        QCache.wrap(c.k_codes, c.k_scale, c.v_codes, c.v_scale.double())
    with pytest.raises(ValueError, match="k must be"):
        c.write(x[:, :, :64], x, t, n)
    with pytest.raises(ValueError, match="do not match"):
        c.write(x, x[:, :1], t, n)
    with pytest.raises(ValueError, match="lengths must be"):
        c.write(x, x, t, n.long())
    with pytest.raises(ValueError, match="lengths must be"):
        c.write(x, x, t, _i32([3, 4]))
    with pytest.raises(ValueError, match="counts"):
        c.write(x, x, t, n, [1])
    with pytest.raises(ValueError, match="on cpu"):
        c.write(x, x, t.cpu(), n)
    with pytest.raises(RuntimeError, match="GPU only"):
        c.write(x.cpu(), x, t, n)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        c.attention(x, 3, t, n)
    with pytest.raises(ValueError, match="q must be"):
        c.attention(x, 4, t, n)
    with pytest.raises(ValueError, match="parents"):
        c.attention(x, 2, t, n, parents=_i32([0, 1, 2]))
    big = torch.zeros(1, 257, 128, device="cuda")
    with pytest.raises(ValueError, match="256"):
        c.attention(big, 2, t, n, parents=_i32([0] * 257))
    with pytest.raises(ValueError, match="most"):
        c.read(t, n, -1)
    with pytest.raises(ValueError, match="path"):
        c.keep(t, n, _i32([0, 1]), n)
    with pytest.raises(ValueError, match="count"):
        c.keep(t, n, _i32([[0, 1]]), None)
    p, u = torch.full((1, 2, 5), 0.2, device="cuda"), torch.zeros(1, 2, device="cuda")
    tok, par, s = torch.zeros(1, 2, dtype=torch.int64, device="cuda"), _i32([-1, 0]), torch.zeros(1, device="cuda")
    with pytest.raises(ValueError, match="tokens"):
        verify_tree(tok.int(), par, p, None, u, s)
    with pytest.raises(ValueError, match="draft"):
        verify_tree(tok, par, p, p[:, :1], u, s)
    with pytest.raises(ValueError, match="accept_u"):
        verify_tree(tok, par, p, None, s, s)
    with pytest.raises(ValueError, match="target"):
        verify_tree(tok, par, p[0], None, u, s)
    with pytest.raises(ValueError, match="1024"):
        verify_tree(tok, par, torch.zeros(1, 1025, 2, device="cuda"), None, u, s)
    assert _status() == 0


# ------------------------------------------- ends of the range, long contexts, waits

# What even weights over values of one sign may be off by, of the result: no
# score has an error, a weight has 22 bits (two halves of 11; 2^-22), and the
# exponential's argument, up to 2^5 where ranges' largest values differ, is off
# by 2^-20, the ranges then weighing differently by 2^-19 ln 2: 2^-18 for all of
# these.  A sum is a chain of at most 64 additions each off by 2^-23: the
# tensor core's 16 keys at a time (2 to 16 in a step), steps of a range (1 to
# 3 tiles where the keys are dealt out over the GPU), four warps, the ranges
# by eight (157 of them: 20 and 8).  Without a weight's smaller half: 2^-12 on
# the mean, twenty times as much.
EVEN = 64 * 2.0**-23 + 2.0**-18


@pytest.mark.parametrize("tokens,heads", [(1, 2), (1, 16), (40, 2)])
@pytest.mark.parametrize("scale", [1e-34, 1e-30, 1.0, 1e30])
@pytest.mark.parametrize("n", [40000, 400])
def test_attention_long_contexts_at_the_ends_of_v(cuda_device, tokens, heads, scale, n):
    """Keys that weigh the same, in ranges joined and in one, V scales from one
    end of their range to the other: the sum of the weights, measured against
    the largest w * vs, stays a number.  q is 0, so the output is the mean."""
    book = Book([n], 1, 64, 64)
    book.fill([n])
    codes = torch.randint(1, 128, book.cache.v_codes.shape, device="cuda").to(torch.int8)
    book.cache.v_codes.copy_(codes)
    book.cache.v_scale.fill_(scale)
    y = book.cache.attention(torch.zeros(1, tokens, heads * 64, device="cuda"), heads, book.table, _i32([n - tokens])).data
    pos = torch.arange(n, device="cuda")
    sums = (codes[book.table[0, pos // 64].long(), 0, pos % 64].double() * float(np.float32(scale))).cumsum(0)
    for t in (0, tokens - 1):
        seen = n - tokens + 1 + t
        want = (sums[seen - 1] / seen).repeat(heads)
        assert ((y[0, t].double() - want).abs() / want).max().item() <= EVEN, t
    assert _status() == 0


@pytest.mark.parametrize("d,kv,heads,tokens,lengths", [
    (128, 1, 2, 1, [20000]), (64, 2, 16, 1, [17000, 300]), (32, 1, 16, 2, [16500]), (128, 1, 8, 12, [20000, 5]),
    (64, 1, 4, 40, [20000])])
def test_attention_keeps_its_halves_over_long_contexts(cuda_device, d, kv, heads, tokens, lengths):
    """Values of one sign, their scales spread over e^2, under even weights:
    nothing cancels, so what is lost of a weight or in a join shows."""
    book = Book([n + tokens for n in lengths], kv, d, 32)
    _, vvals = book.fill([n + tokens for n in lengths], spread=1.0)
    book.cache.v_codes.copy_(book.cache.v_codes.abs())
    y = book.cache.attention(torch.zeros(len(lengths), tokens, heads * d, device="cuda"), heads, book.table,
                             _i32(lengths)).numpy()
    for b, n in enumerate(lengths):
        sums = np.abs(vvals[b]).cumsum(0)
        for t in range(tokens):
            want = (sums[n + t] / (n + t + 1)).repeat(heads // kv, 0).reshape(-1)
            off = np.abs(y[b, t] - want) / want
            assert off.max() <= EVEN, (b, t, off.max())
    assert _status() == 0


@pytest.mark.parametrize("vocab", [65, 3000, 50001])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("draft", [False, True])
def test_verify_reports_rows_that_are_not_finite(cuda_device, vocab, value, draft):
    """NaN or Inf in a row that a token is drawn from or a draft rejected by:
    the status word says so, the token is one of the vocabulary, and the other
    sequences are answered as ever."""
    from kansaiml_b200 import _lib
    from kansaiml_b200.cache import verify_tree
    rs = np.random.RandomState(vocab)
    batch, nodes = 4, 3
    target, q = _softmax(rs, (batch, nodes, vocab), 1.0), _softmax(rs, (batch, nodes, vocab), 1.0)
    parents, tokens = np.array([[-1, 0, 1]] * batch, np.int32), rs.randint(0, vocab, (batch, nodes)).astype(np.int64)
    # accepted down to the leaf: sequences 0 and 1; rejected at once: 2 and 3
    au = np.array([[0, 0, 0]] * 2 + [[0, 0.999, 0]] * 2, np.float32)
    q[2:, 0, tokens[2:, 1]] = 1
    su = rs.uniform(size=batch).astype(np.float32)

    def run(target, q):
        out = verify_tree(_dev(tokens), _dev(parents), _dev(target), _dev(q) if draft else None, _dev(au), _dev(su))
        return [x.cpu().numpy() for x in out]

    want = run(target, q)
    assert _status() == 0 and want[1].tolist() == [3, 3, 1, 1]
    at = int(tokens[2, 1] + 1) % vocab                     # not the drafted token's own
    for rows, b, node in ((target, 0, 2), (target, 2, 0)) + (((q, 2, 0),) if draft else ()):
        bad = rows.copy()
        bad[b, node, at] = value
        if rows is q and value == math.inf:
            continue                                       # (p - inf)+ is 0: a number
        got = run(*((bad, q) if rows is target else (target, bad)))
        assert _status() == _lib.KZ_ERR_NONFINITE
        assert 0 <= got[2][b] < vocab
        for x, y in zip(got, want):
            np.testing.assert_array_equal(np.delete(x, b, 0), np.delete(y, b, 0))
    bad = target.copy()
    bad[1, 0, (tokens[1, 1] + 1) % vocab] = value          # a row that only its child's own value is read of
    got = run(bad, q)
    assert _status() == 0 and all(np.array_equal(x, y) for x, y in zip(got, want))


def test_pages_are_handed_out_without_waiting(cuda_device):
    """PagePool.reserve and release, sequences that cross pages together and
    alone, make no call that waits for the GPU."""
    from kansaiml_b200.cache import PagePool
    pool, host = PagePool(300, 32, 12, 16, "cuda"), PagePool(300, 32, 12, 16, "cpu")
    for p in (host, pool):
        if p is pool:
            torch.cuda.set_sync_debug_mode("error")
        try:
            p.reserve(1)
            p.reserve(33)
            p.reserve(100, 7)
            p.release(3)
            p.reserve(50, -1)
            p.reserve(60)
            p.reserve(60)
            with pytest.raises(IndexError):
                p.reserve(100, 32)
            with pytest.raises(RuntimeError, match="pages needed"):
                p.reserve(12 * 16)
        finally:
            torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(pool.table.cpu(), host.table) and pool.free == host.free
    held = pool.table[pool.table >= 0].tolist()
    assert len(set(held)) == len(held) == 300 - pool.free


def test_attention_of_long_chunks_in_a_wide_table(cuda_device):
    """4096 rows a sequence in a table of 2.5 million positions: 164 million
    units of work, which 31 bits hold with room."""
    d, kv, heads, tokens = 32, 8, 32, 4096
    lengths, counts = [300, 9000, 0, 77, 1, 5000, 0, 128], [4096, 17, 0, 130, 1, 1000, 4000, 0]
    book = Book([a + b for a, b in zip(lengths, counts)], kv, d, 64)
    wide = torch.full((8, 40000), -1, dtype=torch.int32, device="cuda")
    wide[:, :book.table.shape[1]] = book.table
    kvals, vvals = book.fill([a + b for a, b in zip(lengths, counts)])
    q = torch.randn(8, tokens, heads * d, device="cuda")
    y = book.cache.attention(q, heads, wide, _i32(lengths), _i32(counts)).data
    for b, (n, m) in enumerate(zip(lengths, counts)):
        assert not y[b, m:].any()
        hidden = torch.ones(m, n + m, dtype=torch.bool, device="cuda").triu(n + 1)
        for h in range(0, heads, 5):
            k, v = (_dev(x[b][:, h * kv // heads]) for x in (kvals, vvals))
            qq = q[b, :m, h * d:(h + 1) * d].double()
            w = torch.softmax((qq @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            # as in _attention_64, with the largest product of the whole sequence
            size = (qq.abs() @ k.abs().T).max().item() / math.sqrt(d) if m else 0.0
            bound = (2 * (d + 4) * size + 16 + (n + m) / 16 + 32) * 2.0**-23 * (w @ v.abs())
            assert ((y[b, :m, h * d:(h + 1) * d].double() - w @ v).abs() <= bound).all(), (b, h)
    assert _status() == 0


@pytest.mark.parametrize("vocab", [3000, 128000])
def test_verify_draws_nothing_that_was_taken_out(cuda_device, vocab):
    """Without draft rows: two rejected tokens that are all there is of a
    stretch of the row, one far smaller than the other, and the smallest u: what
    rounding leaves of that stretch's sum is no token's."""
    from kansaiml_b200.cache import verify_tree
    batch, y = 64, 2 * vocab // 3
    small = np.random.RandomState(3).uniform(1e-12, 1e-10, batch).astype(np.float32)
    p = np.zeros((batch, 3, vocab), np.float32)
    p[:, 0, 3] = 0.9
    p[:, 0, 5] = small
    p[:, 0, y] = 0.1
    tokens, parents = np.array([[0, 3, 5]] * batch, np.int64), np.array([-1, 0, 0], np.int32)
    au, su = np.array([[0, 0.95, 0.5]] * batch, np.float32), np.zeros(batch, np.float32)
    su[1::2] = np.float32(2.0**-60)
    path, count, token = verify_tree(_dev(tokens), _dev(parents), _dev(p), None, _dev(au), _dev(su))
    assert count.tolist() == [1] * batch and token.tolist() == [y] * batch
    assert _status() == 0


@pytest.mark.parametrize("tokens", [1, 40])
def test_a_negative_length_is_reported(cuda_device, tokens):
    """By every entry point that takes lengths; the other sequences' rows are as ever."""
    from kansaiml_b200 import _lib
    book = Book([100, 100, 300], 1, 64, 32)
    book.fill([100, 100, 300])
    x, q = torch.randn(3, tokens, 64, device="cuda"), torch.randn(3, tokens, 128, device="cuda")
    good, bad = _i32([50, 20, 200]), _i32([50, -3, 200])
    want = book.cache.attention(q, 2, book.table, good).data
    path, count = _i32([[0] + [-1] * 6] * 3), _i32([1, 1, 1])
    for call in (lambda: book.cache.attention(q, 2, book.table, bad).data, lambda: book.cache.read(book.table, bad, 200)[0].data,
                 lambda: book.cache.keep(book.table, bad, path, count), lambda: book.cache.write(x, x, book.table, bad)):
        assert _status() == 0
        got = call()
        assert _status() == _lib.KZ_ERR_INVALID_ARGUMENT
        if got is not None and got.shape == want.shape:
            assert torch.equal(got[::2], want[::2])
