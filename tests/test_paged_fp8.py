"""Host side of the 8-bit paged cache, without a GPU: what it refuses, the cache's pools."""

from __future__ import annotations

import ctypes

import pytest
import torch

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def test_cpu_tensors_are_refused():
    from gen_worker_amd import paged as p

    x = torch.zeros(4, 2, 16, dtype=BF16)
    pages = torch.zeros(2, 2, 16, 16, dtype=torch.uint8).view(FP8)
    scales = torch.zeros(2, 2, 16, dtype=torch.uint8)
    one = torch.zeros(1, dtype=torch.int32)
    table, start = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pool = (pages, pages, scales, scales)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_attention_fp8(x, *pool, table, start, one, 1, 1)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_write_fp8(x, x, x, None, None, None, *pool, table, start, one)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_read_fp8(*pool, table, start, one, 1)
    with pytest.raises(p.PagedError, match="CUDA"):
        p.paged_evict_fp8(*pool, torch.zeros(2, 2, 16), table, one, 1, table, 4, 1)
    with pytest.raises(p.PagedError, match="k_pages must be"):
        p.paged_attention(x, pages, pages, table, start, one, 1, 1)


class TestEntryPoints:
    """The C entry points refuse before any launch."""

    def args(self, **change):
        from gen_worker_amd import _native as nat

        v = dict(k=4096, v=4096, w=4096, table=4096, q_start=4096, kv_len=4096, page_stride=2 * 16 * 64,
                 head_stride=16 * 64, slot_stride=64, w_page_stride=32, w_head_stride=16, pages=10, table_stride=4,
                 table_width=4, batch=2, page_size=16, kv_heads=2, head_dim=64, dtype=nat.DT_BF16)
        v.update(change)
        return ctypes.byref(nat.PagedCacheArgs(**v))

    def scales(self, **change):
        from gen_worker_amd import _native as nat

        v = dict(k=4096, v=4096, page_stride=32, head_stride=16)
        v.update(change)
        return ctypes.byref(nat.PagedScalesArgs(**v))

    def refused(self, fn, *args, match):
        from gen_worker_amd import _native as nat

        lib = nat.load()
        assert getattr(lib, fn)(*args) == 1
        assert match in lib.gwa_last_error().decode(), lib.gwa_last_error()

    ATTEND = (4096, 256, 64, 4096, 4096, 4, 4, 1, 1, 0.125, 1, 1, None, 0, None)
    WRITE = (4096, 64, 64, 4096, 64, 64, 4096, 64, 64, 4096, 4096, 9, None, 4096)

    @pytest.mark.parametrize("change,match", [
        (dict(page_size=12), "page_size"), (dict(head_dim=72), "head_dim"), (dict(head_dim=8), "head_dim"),
        (dict(head_dim=272), "head_dim"), (dict(dtype=2), "dtype"), (dict(slot_stride=72), "strides"),
        (dict(page_stride=2 * 16 * 64 + 8), "strides"), (dict(head_stride=8), "strides"), (dict(k=None), "null pointer"),
        (dict(v=4104), "aligned"), (dict(q_start=None), "q_start"), (dict(w=None), "no gathered weights")])
    def test_the_cache(self, change, match):
        self.refused("gwa_paged_attention_fp8", self.args(**change), self.scales(), *self.ATTEND, match=match)

    @pytest.mark.parametrize("change", [dict(k=None), dict(v=None), dict(page_stride=0), dict(head_stride=15),
                                        dict(head_stride=2 ** 31), dict(page_stride=2 ** 31)])
    def test_the_scales(self, change):
        c, s = self.args(), self.scales(**change)
        self.refused("gwa_paged_attention_fp8", c, s, *self.ATTEND, match="scales")
        self.refused("gwa_paged_write_fp8", c, s, *self.WRITE, 2, 1, 64, 0, None, match="scales")
        self.refused("gwa_paged_read_fp8", c, s, 4096, 4096, 2, None, match="scales")
        self.refused("gwa_paged_evict_fp8", c, s, 4096, 2, 2, 64, 32, 0, 4096, 4096, None, match="scales")

    def test_the_calls(self):
        c, s = self.args(), self.scales()
        self.refused("gwa_paged_attention_fp8", c, None, *self.ATTEND, match="null scales")
        self.refused("gwa_paged_attention_fp8", None, s, *self.ATTEND, match="null cache")
        self.refused("gwa_paged_write_fp8", c, None, *self.WRITE, 2, 1, 64, 0, None, match="null scales")
        self.refused("gwa_paged_write_fp8", c, s, *self.WRITE, -1, 1, 64, 0, None, match="tokens")
        self.refused("gwa_paged_write_fp8", c, s, *self.WRITE, 2 ** 31 - 1, 1, 64, 0, None, match="too many")
        self.refused("gwa_paged_read_fp8", c, s, 4096, 4096, 2 ** 31 - 1, None, match="too many")
        self.refused("gwa_paged_write_fp8", c, s, *self.WRITE, 2, 1, 66, 0, None, match="rotated channels")
        self.refused("gwa_paged_write_fp8", c, s, *self.WRITE[:-1], 4097, 2, 1, 64, 0, None, match="misaligned")
        self.refused("gwa_paged_write_fp8", c, s, *self.WRITE[:3], None, *self.WRITE[4:], 2, 1, 64, 0, None,
                     match="null pointer")
        self.refused("gwa_paged_read_fp8", c, None, 4096, 4096, 2, None, match="null scales")
        self.refused("gwa_paged_read_fp8", c, s, 4096, 4096, -2, None, match="tokens")
        self.refused("gwa_paged_read_fp8", c, s, None, 4096, 2, None, match="outputs")
        self.refused("gwa_paged_read_fp8", c, s, 4096, 4104, 2, None, match="outputs")
        self.refused("gwa_paged_evict_fp8", c, None, 4096, 2, 2, 64, 32, 0, 4096, 4096, None, match="null scales")
        self.refused("gwa_paged_evict_fp8", c, s, 4096, 2, 2, 64, 8, 9, 4096, 4096, None, match="budget")

    def test_nothing_to_do_needs_no_device(self):
        from gen_worker_amd import _native as nat

        lib = nat.load()
        c, s = self.args(batch=0), self.scales()
        assert lib.gwa_paged_attention_fp8(c, s, None, 256, 64, None, None, 0, 4, 0, 0, 0.125, 1, 0, None, 0, None) == 0
        assert lib.gwa_paged_read_fp8(c, s, None, None, 0, None) == 0
        assert lib.gwa_paged_write_fp8(c, s, *self.WRITE, 0, 1, 64, 0, None) == 0
        assert lib.gwa_paged_evict_fp8(c, s, None, 0, 0, 0, 4, 1, None, None, None) == 0


def test_cache_pools():
    from gen_worker_amd.paged import PagedCache, PagedError

    c = PagedCache(4, 16, 3, 64, dtype=FP8, device="cpu", weights=True)
    assert c.k.dtype == c.v.dtype == FP8 and [t.shape for t in c.scales] == [(4, 3, 16)] * 2
    t = c.twin()
    assert t.scales is not None and t.scales[0].data_ptr() != c.scales[0].data_ptr() and t.k.dtype == FP8
    assert PagedCache(4, 16, 3, 64, device="cpu").scales is None
    with pytest.raises(PagedError, match="heads of"):
        PagedCache(4, 16, 3, 72, dtype=FP8, device="cpu")
    with pytest.raises(PagedError, match="heads of"):
        PagedCache(4, 16, 3, 64, dtype=torch.float8_e5m2, device="cpu")
    with pytest.raises(PagedError, match="sequences"):
        c.read([0])
