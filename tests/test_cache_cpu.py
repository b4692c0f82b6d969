"""Host side of the K/V cache, without a GPU: the C entry points' argument
checks (nothing is launched), the page pool, refusals of CPU tensors, the
drafts a Decoder looks up."""
import ctypes

import pytest
import torch

from kansaiml_b200 import _lib
from kansaiml_b200.cache import PagePool, QCache, verify_tree

P = ctypes.c_void_p


def _cache(**kw):
    c = _lib.KzCache(P(1 << 20), P(2 << 20), P(3 << 20), P(4 << 20), 8, 2, 64, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _said(status, text):
    assert status == _lib.KZ_ERR_INVALID_ARGUMENT and text in _lib.last_error(), _lib.last_error()


def test_write_checks():
    lib = _lib.load()

    def write(c, k=P(16), v=P(16), batch=1, tokens=2, kb=512, kr=256, vb=512, vr=256, table=P(16), cols=4, lengths=P(16),
              ko=None):
        return lib.kz_cache_write_f32(ctypes.byref(c) if c else None, k, v, batch, tokens, kb, kr, vb, vr, table, cols,
                                      lengths, None, ko, None, None)

    _said(write(None), "cache is NULL")
    _said(write(_cache(head_dim=96)), "head_dim")
    _said(write(_cache(page_size=48)), "page_size")
    _said(write(_cache(kv_heads=0)), "out of range")
    _said(write(_cache(pages=1 << 30)), "out of range")
    _said(write(_cache(k_codes=P(8))), "aligned")
    _said(write(_cache(v_scale=None)), "NULL cache buffer")
    _said(write(_cache(), batch=-1), "batch")
    _said(write(_cache(), lengths=None), "NULL")
    _said(write(_cache(), table=None), "NULL")
    _said(write(_cache(), tokens=-1), "tokens")
    _said(write(_cache(), batch=1 << 20, tokens=1 << 20), "out of range")
    _said(write(_cache(), k=None), "NULL")
    _said(write(_cache(), k=P(4)), "aligned")
    _said(write(_cache(), ko=P(4)), "aligned")
    _said(write(_cache(), kr=258), "strides")
    _said(write(_cache(), vr=128), "shorter")
    _said(write(_cache(), kb=-512), "negative")
    assert write(_cache(), batch=0) == 0 and write(_cache(), tokens=0) == 0


def test_read_keep_and_attention_checks():
    lib = _lib.load()
    c = _cache()
    r = ctypes.byref(c)
    _said(lib.kz_cache_read_f32(r, P(16), 4, P(16), 1, -1, P(16), P(16), None), "most")
    _said(lib.kz_cache_read_f32(r, P(16), 4, P(16), 1, 5, None, P(16), None), "NULL")
    _said(lib.kz_cache_read_f32(r, P(16), 4, P(16), 1, 5, P(16), P(20), None), "aligned")
    _said(lib.kz_cache_read_f32(r, P(16), 4, P(16), 1 << 20, 1 << 30, P(16), P(16), None), "out of range")
    assert lib.kz_cache_read_f32(r, P(16), 4, P(16), 1, 0, None, None, None) == 0
    _said(lib.kz_cache_keep(r, P(16), 4, P(16), None, P(16), 1, 3, None), "NULL")
    _said(lib.kz_cache_keep(r, P(16), 4, P(16), P(16), P(16), 1, -3, None), "nodes")
    assert lib.kz_cache_keep(r, P(16), 4, P(16), P(16), P(16), 1, 0, None) == 0

    def attend(q=P(16), batch=1, tokens=2, heads=4, qb=1024, qr=512, cols=64, parents=None, pb=0, out=P(16), work=P(16),
               size=1 << 40):
        return lib.kz_cache_attention_f32(r, q, batch, tokens, heads, qb, qr, P(16), cols, P(16), None, parents, pb, 1.0,
                                          out, work, size, None)

    _said(attend(heads=3), "multiple of kv_heads")
    _said(attend(heads=0), "multiple of kv_heads")
    _said(attend(batch=65536), "batch")
    _said(attend(tokens=1 << 24), "out of range")
    c.page_size = 128
    _said(attend(cols=(1 << 24) - 1), "table_cols")          # more positions than an int holds
    c.page_size = 64
    _said(attend(q=None), "NULL")
    _said(attend(out=P(24)), "aligned")
    _said(attend(qr=510), "strides")
    _said(attend(qr=256), "shorter")
    _said(attend(tokens=300, parents=P(16)), "256")
    _said(attend(parents=P(16), pb=1), "parents_batch_stride")
    _said(attend(size=64), "workspace")
    _said(attend(work=None), "workspace")
    assert attend(batch=0) == 0 and attend(tokens=0) == 0
    assert lib.kz_cache_attention_workspace_bytes(r, 1, 4, 8) == 0        # 512 positions: one range each
    assert lib.kz_cache_attention_workspace_bytes(r, 1, 4, 9) > 0
    assert lib.kz_cache_attention_workspace_bytes(None, 1, 4, 9) == 0


def test_verify_checks():
    lib = _lib.load()

    def verify(tokens=P(16), pb=0, batch=1, nodes=3, vocab=5, out=P(16)):
        return lib.kz_verify_tree_f32(tokens, P(16), pb, P(16), None, P(16), P(16), batch, nodes, vocab, out, P(16), P(16),
                                      None)

    _said(verify(nodes=0), "nodes")
    _said(verify(nodes=1025), "nodes")
    _said(verify(vocab=0), "vocab")
    _said(verify(vocab=1 << 24), "vocab")
    _said(verify(batch=-1), "batch")
    _said(verify(tokens=None), "NULL")
    _said(verify(out=None), "NULL")
    _said(verify(pb=2), "parents_batch_stride")
    assert verify(batch=0) == 0


def test_page_pool():
    pool = PagePool(6, 3, 4, page_size=16, device="cpu")
    pool.reserve(17, 0)
    assert pool.free == 4 and (pool.table[0] >= 0).tolist() == [True, True, False, False]
    pool.reserve(20, 0)                                   # fits what it has
    assert pool.free == 4
    pool.reserve(16)
    assert pool.free == 2
    held = pool.table[pool.table >= 0].tolist()
    assert len(set(held)) == 4 and all(0 <= p < 6 for p in held)
    before = pool.table.clone()
    with pytest.raises(RuntimeError, match="3 pages needed, 2 free"):
        pool.reserve(64, 1)
    with pytest.raises(ValueError, match="5 pages"):
        pool.reserve(65, 1)
    assert torch.equal(pool.table, before) and pool.free == 2
    pool.release(0)
    assert pool.free == 4 and (pool.table[0] == -1).all()
    pool.reserve(64, 1)
    assert pool.free == 1 and len(set(pool.table[pool.table >= 0].tolist())) == 5


def test_cpu_tensors_are_refused():
    cache = QCache(4, 2, 32, 16, device="cpu")
    assert cache.nbytes() == 2 * 4 * 2 * 16 * (32 + 4) and "page_size=16" in repr(cache)
    t, n, x = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 64)
    for call in (lambda: cache.write(x, x, t, n), lambda: cache.read(t, n, 3), lambda: cache.attention(x, 2, t, n),
                 lambda: cache.keep(t, n, t, n),
                 lambda: verify_tree(torch.zeros(1, 1).long(), t[:, :1], x, None, x[:, :, 0], x[:, 0, 0])):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="negative"):
        QCache(-1, 2, 32, 16, device="cpu")


def test_looked_up_drafts():
    from kansaiml_b200.workloads import _drafted
    tokens, parents, depths = _drafted([1, 2, 3, 1, 2, 4, 1, 2, 3, 5, 1], 8)
    assert tokens == [1, 2, 3, 5, 1, 4, 1, 2] and parents == [-1, 0, 1, 2, 3, 1, 5, 6]
    assert depths == [0, 1, 2, 3, 4, 2, 3, 4]
    assert _drafted([7], 8) == ([7], [-1], [0])
    assert _drafted([1, 1, 1], 1) == ([1], [-1], [0])
    assert all(p < i for i, p in enumerate(parents))


def test_cache_is_importable_under_the_reference_name():
    import kansai
    import kansai.cache
    import kansaiml_b200.cache
    assert kansai.cache is kansaiml_b200.cache


def test_a_step_of_a_tree_needs_its_nodes_depths():
    """Decoder.extend: parents without depths would take node numbers for positions."""
    from kansaiml_b200.workloads import Decoder
    ids, ints = torch.zeros(1, 3, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="depths"):
        Decoder.extend(None, ids, None, parents=ints)


def test_attention_work_is_counted_in_the_kernels_own_tiles():
    """Row tiles of 128 above 32 rows a key head, one tile below: long chunks
    over long tables are refused only where the units of work pass 31 bits."""
    lib = _lib.load()
    c = _cache()

    def attend(batch, tokens, heads, cols):
        return lib.kz_cache_attention_f32(ctypes.byref(c), None, batch, tokens, heads, tokens * heads * 128, heads * 128,
                                          P(16), cols, P(16), None, None, 0, 1.0, P(16), P(16), 1 << 40, None)

    for batch, tokens, heads, cols in ((64, 4096, 4, 40000), (8, 60000, 4, 60000), (60000, 4, 16, 20000)):
        _said(attend(batch, tokens, heads, cols), "q or out is NULL")
    # 64 sequences x 2 heads x 64 row tiles x 300001 tiles of keys
    _said(attend(64, 4096, 4, 600000), "work is out of range")
    _said(attend(60000, 4, 16, 40000), "work is out of range")


def test_stream_handle_takes_what_torch_calls_a_device(monkeypatch):
    """A device, a name, a number or None (the current device)."""
    from kansaiml_b200.tensor import stream_handle
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for device, index in ((torch.device("cuda", 1), 1), ("cuda:2", 2), (2, 2), (None, 3), ("cuda", 3), (torch.device("cuda"), 3)):
        assert stream_handle(device) == 1000 + index
    with pytest.raises(ValueError, match="cuda"):
        stream_handle("cpu")
