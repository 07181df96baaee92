"""Host side of the paged-cache operators, without a GPU: what they refuse, the rotary tables, the cache's bookkeeping."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

BF16 = torch.bfloat16


def _paged():
    from gen_worker_amd import paged

    return paged


def test_rotary_table_scalings():
    p = _paged()
    cos, sin = p.rotary_table(50, 8, device="cpu")
    f = torch.tensor([10000.0 ** (-2 * i / 8) for i in range(4)], dtype=torch.float64)
    a = torch.arange(50, dtype=torch.float64)[:, None] * f
    assert torch.equal(cos, a.cos().float()) and torch.equal(sin, a.sin().float()) and cos.dtype == torch.float32
    cos, _ = p.rotary_table(50, 8, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(cos, (a / 4).cos().float())
    # the slowest pair is stretched by the factor, the fastest kept
    _, sin = p.rotary_table(50, 8, scaling="ntk", factor=4.0, device="cpu")
    assert torch.allclose(sin[:, 0].double(), a[:, 0].sin(), atol=1e-6)
    assert torch.allclose(sin[:, 3].double(), (a[:, 3] / 4).sin(), atol=1e-6)
    # turns over 64 positions: 10.2, 1.02, 0.1, 0.01: between 1 and 8 turns the second pair is nearly stretched
    cos, sin = p.rotary_table(50, 8, scaling="yarn", factor=4.0, original=64, beta_fast=8.0, beta_slow=1.0, device="cpu")
    gain = 0.1 * math.log(4.0) + 1.0
    ramp = (64 * float(f[1]) / (2 * math.pi) - 1.0) / 7.0
    want = torch.stack([a[:, 0], a[:, 1] * ramp + a[:, 1] / 4 * (1 - ramp), a[:, 2] / 4, a[:, 3] / 4], 1)
    assert 0 < ramp < 0.1 and torch.allclose(cos.double(), want.cos() * gain, atol=1e-6)
    assert torch.allclose(sin.double(), want.sin() * gain, atol=1e-6)
    for bad in (dict(scaling="other"), dict(factor=0.5, scaling="linear"), dict(factor=2.0), dict(scaling="yarn", factor=2.0)):
        with pytest.raises(p.PagedError):
            p.rotary_table(8, 8, device="cpu", **bad)
    with pytest.raises(p.PagedError, match="channels"):
        p.rotary_table(8, 7, device="cpu")


def test_cpu_tensors_are_refused():
    p = _paged()
    cos, sin = p.rotary_table(8, 8, device="cpu")
    x = torch.zeros(4, 2, 8, dtype=BF16)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.rotary_embed(x, cos, sin)
    pages = torch.zeros(2, 2, 16, 8, dtype=BF16)
    one = torch.zeros(1, dtype=torch.int32)
    table, start = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_attention(x, pages, pages, table, start, one, 1, 1)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_write(x, x, x, cos, sin, None, pages, pages, table, start, one)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_evict(pages, pages, torch.zeros(2, 2, 16), table, one, 1, table, 4, 1)


class TestEntryPoints:
    """The C entry points refuse before any launch."""

    def args(self, **change):
        from gen_worker_amd import _native as nat

        v = dict(k=4096, v=4096, w=4096, table=4096, q_start=4096, kv_len=4096, page_stride=2 * 16 * 64,
                 head_stride=16 * 64, slot_stride=64, w_page_stride=32, w_head_stride=16, pages=10, table_stride=4,
                 table_width=4, batch=2, page_size=16, kv_heads=2, head_dim=64, dtype=nat.DT_BF16)
        v.update(change)
        return nat.PagedCacheArgs(**v)

    def refused(self, fn, *args, match):
        from gen_worker_amd import _native as nat

        lib = nat.load()
        assert getattr(lib, fn)(*args) == 1
        assert match in lib.gwa_last_error().decode(), lib.gwa_last_error()

    @pytest.mark.parametrize("change,match", [
        (dict(page_size=12), "page_size"), (dict(page_size=4), "page_size"), (dict(page_size=8192), "page_size"),
        (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(dtype=2), "dtype"),
        (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "pages"), (dict(batch=-1), "batch"),
        (dict(table_stride=3), "table"), (dict(table_width=2 ** 27, table_stride=2 ** 27), "table"),
        (dict(slot_stride=56), "strides"), (dict(page_stride=12), "strides"), (dict(k=None), "null pointer"),
        (dict(kv_len=None), "null pointer"), (dict(v=4098), "aligned"), (dict(q_start=None), "q_start"),
        (dict(w=None), "no gathered weights"), (dict(w_head_stride=8), "weight strides")])
    def test_the_cache(self, change, match):
        c = ctypes.byref(self.args(**change))
        self.refused("gwa_paged_attention", c, 4096, 256, 64, 4096, 4096, 4, 4, 1, 1, 0.125, 1, 1, None, 0, None, match=match)

    def test_attention(self):
        c = ctypes.byref(self.args())
        fn = "gwa_paged_attention"
        self.refused(fn, None, 4096, 256, 64, 4096, 4096, 4, 4, 1, 1, 0.125, 1, 0, None, 0, None, match="null cache")
        self.refused(fn, c, 4096, 256, 64, 4096, 4096, 4, 3, 1, 1, 0.125, 1, 0, None, 0, None, match="query heads")
        self.refused(fn, c, 4096, 256, 64, 4096, 4096, 4, 4, 5, 1, 0.125, 1, 0, None, 0, None, match="max_q")
        self.refused(fn, c, 4096, 256, 64, 4096, 4096, 4, 4, 1, 65, 0.125, 1, 0, None, 0, None, match="max_kv")
        self.refused(fn, c, 4096, 256, 64, 4096, 4096, 4, 4, 1, 1, 0.0, 1, 0, None, 0, None, match="scale")
        self.refused(fn, c, 4096, 256, 64, 4096, 4096, 4, 4, 1, 1, float("nan"), 1, 0, None, 0, None, match="scale")
        self.refused(fn, c, 4096, 252, 64, 4096, 4096, 4, 4, 1, 1, 0.125, 1, 0, None, 0, None, match="strides")
        self.refused(fn, c, 4096, 256, 64, None, 4096, 4, 4, 1, 1, 0.125, 1, 0, None, 0, None, match="null pointer")
        self.refused(fn, c, 4104, 256, 64, 4096, 4096, 4, 4, 1, 1, 0.125, 1, 0, None, 0, None, match="aligned")

    def test_rotary_and_write(self):
        fn = "gwa_rotary_embed"
        self.refused(fn, 4096, 8, 8, 4096, 4096, 9, None, 4096, 8, 8, 2, 1, 8, 10, 0, 0, 0, None, match="rotated channels")
        self.refused(fn, 4096, 8, 8, 4096, 4096, 9, None, 4096, 8, 8, 2, 1, 8, 3, 0, 0, 0, None, match="rotated channels")
        self.refused(fn, 4096, 8, 8, 4096, None, 9, None, 4096, 8, 8, 2, 1, 8, 8, 0, 0, 0, None, match="table")
        self.refused(fn, 4096, 8, 8, 4096, 4096, 0, None, 4096, 8, 8, 2, 1, 8, 8, 0, 0, 0, None, match="table")
        self.refused(fn, 4096, 8, 8, 4096, 4096, 9, None, 4096, 8, 8, -1, 1, 8, 8, 0, 0, 0, None, match="tokens")
        self.refused(fn, 4096, 8, 8, 4096, 4096, 9, None, 4096, 8, 8, 2, 1, 7, 6, 0, 0, 0, None, match="head_dim")
        self.refused(fn, 4096, 8, 8, 4096, 4096, 9, None, 4096, 8, 8, 2, 1, 8, 8, 0, 0, 3, None, match="dtype")
        self.refused(fn, None, 8, 8, 4096, 4096, 9, None, 4096, 8, 8, 2, 1, 8, 8, 0, 0, 0, None, match="null pointer")
        c = ctypes.byref(self.args())
        fn = "gwa_paged_write"
        rest = (4096, 64, 64, 4096, 64, 64, 4096, 64, 64, 4096, 4096, 9, None, 4096)
        self.refused(fn, c, *rest, -1, 1, 64, 0, None, match="tokens")
        self.refused(fn, c, *rest, 2, 1, 66, 0, None, match="rotated channels")
        self.refused(fn, c, *rest[:3], None, *rest[4:], 2, 1, 64, 0, None, match="null pointer")
        self.refused(fn, c, *rest[:-1], 4097, 2, 1, 64, 0, None, match="misaligned")

    def test_evict(self):
        c = ctypes.byref(self.args())
        fn = "gwa_paged_evict"
        self.refused(fn, c, 4096, 2, 2, 64, 0, 0, 4096, 4096, None, match="budget")
        self.refused(fn, c, 4096, 2, 2, 64, 8, 9, 4096, 4096, None, match="budget")
        self.refused(fn, c, 4096, 2, 2, 65, 32, 0, 4096, 4096, None, match="max_kv")
        self.refused(fn, c, 4096, 2, 2, 64, 33, 0, 4096, 4096, None, match="new_table")
        self.refused(fn, c, 4096, 1, 2, 64, 32, 0, 4096, 4096, None, match="new_table")
        self.refused(fn, c, None, 2, 2, 64, 32, 0, 4096, 4096, None, match="null pointer")

    def test_nothing_to_do_needs_no_device(self):
        from gen_worker_amd import _native as nat

        lib = nat.load()
        c = ctypes.byref(self.args(batch=0))
        assert lib.gwa_paged_attention(c, None, 256, 64, None, None, 0, 4, 0, 0, 0.125, 1, 0, None, 0, None) == 0
        assert lib.gwa_paged_evict(c, None, 0, 0, 0, 4, 1, None, None, None) == 0
        assert lib.gwa_rotary_embed(None, 8, 8, None, None, 0, None, None, 8, 8, 0, 1, 8, 0, 0, 0, 0, None) == 0


def test_cache_bookkeeping():
    p = _paged()
    with pytest.raises(p.PagedError, match="power of two"):
        p.PagedCache(4, 12, 1, 64, device="cpu")
    with pytest.raises(p.PagedError, match="heads of"):
        p.PagedCache(4, 16, 1, 60, device="cpu")
    c = p.PagedCache(6, 16, 1, 64, device="cpu", weights=True)
    a, b = c.add(), c.add()
    batch = c.extend([b, a], [17, 0])
    assert batch.tokens == 17 and batch.max_q == 17 and batch.max_kv == 17
    assert batch.q_start.tolist() == [0, 17, 17] and batch.kv_len.tolist() == [17, 0]
    assert batch.positions.tolist() == list(range(17)) and c.free_pages == 4
    assert sorted(batch.table[0].tolist()) == [0, 1] and batch.table.shape == (2, 2)
    batch = c.extend([b], [15])
    assert batch.positions.tolist() == list(range(17, 32)) and c.free_pages == 4 and c.length(b) == 32
    with pytest.raises(p.PagedError, match="pages wanted"):
        c.extend([a], [65])
    assert c.free_pages == 4 and c.length(a) == 0
    for seqs, counts in (([a, a], [1, 1]), ([a], [1, 2]), ([], []), ([99], [1]), ([a], [-1])):
        with pytest.raises(p.PagedError):
            c.extend(seqs, counts)
    assert c.evict([a, b], 32, 4) is None          # nothing is longer
    with pytest.raises(p.PagedError, match="budget"):
        c.evict([b], 4, 5)
    with pytest.raises(p.PagedError, match="no weights"):
        p.PagedCache(4, 16, 1, 64, device="cpu").evict([], 4, 1)
    with pytest.raises(p.PagedError, match="twin"):
        c.twin().add()
    c.drop(b)
    assert c.free_pages == 6
    with pytest.raises(KeyError):
        c.length(b)


def test_tables_whose_rows_overlap_are_copied_apart():
    """The row stride that the library gets is one at which every row lies inside the table's own storage."""
    p = _paged()
    wide = torch.arange(40, dtype=torch.int32).view(5, 8)
    for table in (wide[:1].expand(6, 8), wide.view(-1).as_strided((6, 8), (3, 1)), wide[:1, :1].expand(4, 1), wide,
                  wide[:, 2:5], wide[:1], wide[:1].expand(1, 8), wide[:, :0], wide[:0], wide[0:1, 0:3].expand(3, 3)):
        got, row = p._spaced(table)
        rows, width = table.shape
        assert row >= width and torch.equal(got, table)
        if rows and width:
            end = got.storage_offset() + (rows - 1) * row + width
            assert end <= got.untyped_storage().nbytes() // 4
            assert torch.equal(got.as_strided((rows, width), (row, 1)), table)
    # nothing is copied that need not be
    assert p._spaced(wide[:, 2:5])[0].data_ptr() == wide[:, 2:5].data_ptr()


def test_evict_moves_every_pool_under_the_lists(monkeypatch):
    """The first cache's evict cuts its twins and their twins; a twin, which does not reach the others, refuses and
    changes nothing."""
    p = _paged()
    first = p.PagedCache(12, 8, 1, 64, device="cpu", weights=True)
    twin = first.twin()
    other, below = first.twin(), twin.twin()
    pools = [first, twin, other, below]
    seq = first.add()
    first.extend([seq], [40])
    moved = []

    def evict(k, v, w, table, kv_len, max_kv, new, budget, recent):
        moved.append((k.data_ptr(), v.data_ptr(), w.data_ptr(), table.tolist(), new.tolist()))
        return torch.zeros(1, 1, budget, dtype=torch.int32), kv_len.clamp(max=budget)

    monkeypatch.setattr(p, "paged_evict", evict)
    pages, free = list(first._seqs[seq][0]), first.free_pages
    for cache in pools[1:]:
        with pytest.raises(p.PagedError, match="twin"):
            cache.evict([seq], 16, 4)
    assert not moved and first._seqs[seq][0] == pages and first.free_pages == free and first.length(seq) == 40
    assert first.evict([seq], 16, 4).shape == (1, 1, 16)
    assert {m[:3] for m in moved} == {(c.k.data_ptr(), c.v.data_ptr(), c.weights.data_ptr()) for c in pools}
    assert len(moved) == 4 and all(m[3:] == ([pages], [first._seqs[seq][0]]) for m in moved)
    assert first.length(seq) == 16 and not set(pages) & set(first._seqs[seq][0]) and first.free_pages == free + 3


def test_tangents_are_refused_where_no_gradient_is_defined():
    """A dual tensor's tangent, which neither the native calls nor the registered ops would notice."""
    from torch.autograd import forward_ad

    p = _paged()
    cos, sin = p.rotary_table(8, 8, device="cpu")
    x = torch.zeros(4, 2, 8, dtype=BF16)
    pages, w = torch.zeros(2, 2, 16, 8, dtype=BF16), torch.zeros(2, 2, 16)
    one = torch.zeros(1, dtype=torch.int32)
    table, start = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with forward_ad.dual_level():
        dual, dual_pages, dual_w, dual_cos = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, pages, w, cos))
        for call in (lambda: p.rotary_embed(x, dual_cos, sin),
                     lambda: p.paged_attention(dual, pages, pages, table, start, one, 1, 1),
                     lambda: p.paged_attention(x, dual_pages, pages, table, start, one, 1, 1),
                     lambda: p.paged_attention(x, pages, pages, table, start, one, 1, 1, weights=dual_w),
                     lambda: p.paged_write(x, dual, x, cos, sin, None, pages, pages, table, start, one),
                     lambda: p.paged_write(x, x, x, dual_cos, sin, None, pages, pages, table, start, one),
                     lambda: p.paged_evict(pages, dual_pages, w, table, one, 1, table, 4, 1)):
            with pytest.raises(p.PagedError, match="no gradient"):
                call()
        with pytest.raises(p.PagedError, match="CUDA"):   # as without a level
            p.paged_attention(x, pages, pages, table, start, one, 1, 1)


def test_the_registered_rotation_refuses_tables_that_ask_for_a_gradient():
    p = _paged()
    op = torch.ops.cozy_gen_worker.rotary_embed
    x, cos, sin = (torch.empty(s, device="meta") for s in ((4, 2, 8), (4, 4), (4, 4)))
    for a in ((cos.clone().requires_grad_(True), sin), (cos, sin.clone().requires_grad_(True))):
        for x0 in (x, x.clone().requires_grad_(True)):
            with pytest.raises(p.PagedError, match="no gradient"):
                op(x0, *a, None, False, False)
        with torch.no_grad():
            assert op(x, *a, None, False, False).shape == x.shape
    y = op(x.clone().requires_grad_(True), cos, sin, None, False, False)
    assert y.requires_grad and not op(x, cos, sin, None, False, False).requires_grad
