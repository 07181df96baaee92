"""The 8-bit paged cache on the GPU (``gen_worker_amd.paged``: ``paged_write_fp8``, ``paged_read_fp8``,
``paged_attention_fp8``, ``paged_evict_fp8``, ``PagedCache`` of float8_e4m3fn) against plain 64-bit implementations.

What a row stands for is a whole number of code steps: reads are equal to the definition. A written row is held to its
definition with the tolerance of what decides it, its rotation in fp32: an unrotated row is equal, code for code. Attention
is held to the bounds that ``test_gpu_paged`` derives, since its keys and values are exact values of the 16-bit type."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged import BF16, DEV, E, F16, F32, LONG_RUNS, SHAPES, Ragged, _check_turned, _gen, _ints, _turn

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def value_of(codes, scales, dtype=torch.float64):
    """By the definition: sign, exponent and fraction of e4m3 times 2^(scale - 127), rounded to the type."""
    c = codes.view(torch.uint8).long()
    sign, exp, frac = 1.0 - 2.0 * (c >> 7).double(), (c >> 3) & 15, (c & 7).double()
    x = torch.where(exp > 0, (1.0 + frac / 8.0) * torch.exp2(exp.double() - 7.0), frac * 2.0 ** -9)
    x = torch.where((c & 127) == 127, math.nan, x)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127.0))
    return (sign * x * s[..., None]).to(dtype)


def held(x, dtype):
    """(codes as values, scale bytes) of rows in 64 bits: the smallest 2^e, e >= -126, with 448 * 2^e >= amax; the nearest
    code, ties to even, inside the type's range; what is not finite NaN."""
    x = x.double()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 448.0)).clamp(min=-126.0)
    e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e).clamp(min=-126.0)   # where log2 was rounded up
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    most = torch.where(256.0 * torch.exp2(e) > torch.finfo(dtype).max, 240.0, 448.0)
    y = torch.minimum(torch.maximum(torch.round(y / step) * step, -most), most)
    return torch.where(x.isfinite(), y, math.nan), (e[..., 0] + 127).to(torch.uint8)


class Ragged8(Ragged):
    """A ragged cache whose rows are held in 8 bits; what no sequence owns holds NaN codes under NaN scales. ``k`` and ``v``
    are what the rows stand for, for the checks."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.pools = {}
        for name in ("k", "v"):
            x = getattr(self, name)
            code, scale = held(x.nan_to_num(), self.dtype)
            stale = x.isnan().any(-1)
            codes = torch.where(stale[..., None], torch.tensor(127, dtype=torch.uint8, device=DEV),
                                code.to(F32).to(FP8).view(torch.uint8))
            self.pools[name] = codes.contiguous().view(FP8)
            self.pools[name + "s"] = torch.where(stale, 255, scale).to(torch.uint8).contiguous()
            setattr(self, name, value_of(self.pools[name], self.pools[name + "s"], self.dtype))

    def pool(self):
        p = self.pools
        return p["k"], p["v"], p["ks"], p["vs"]

    def attend(self, q=None, causal=True, gather=False, scale=None, max_q=None, max_kv=None):
        from gen_worker_amd.paged import paged_attention_fp8

        return paged_attention_fp8(self.q if q is None else q, *self.pool(), self.table, self.q_start, self.kv_len,
                                   max(self.q_len) if max_q is None else max_q,
                                   max(self.kv) if max_kv is None else max_kv, causal=causal, scale=scale,
                                   weights=self.w if gather else None)


# ---------------------------------------------------------------------------
# reading
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
def test_every_code_under_every_scale(dtype):
    """256 codes in rows of 16, under all 256 scale bytes: the definition's value, rounded to the type."""
    from gen_worker_amd.paged import paged_read_fp8

    codes = torch.arange(256, device=DEV, dtype=torch.uint8).view(1, 1, 16, 16)
    codes = codes.expand(256, 1, 16, 16).contiguous()                               # page s: scale byte s
    scales = torch.arange(256, device=DEV, dtype=torch.uint8).view(256, 1, 1).expand(256, 1, 16).contiguous()
    table = torch.arange(256, device=DEV, dtype=torch.int32).view(1, 256)
    k, v = paged_read_fp8(codes.view(FP8), codes.flip(3).contiguous().view(FP8), scales, scales, table, _ints([0, 4096]),
                          _ints([4096]), 4096, dtype=dtype)
    want = value_of(codes, scales, dtype).view(4096, 1, 16)
    assert torch.equal(k.isnan(), want.isnan()) and torch.equal(k.nan_to_num(), want.nan_to_num())
    assert torch.equal(v.nan_to_num(), want.flip(2).nan_to_num())


@pytest.mark.parametrize("q,kv,hk,dim,page", [
    ([1], [1], 1, 16, 8), ([700], [700], 8, 128, 16), ([3, 0, 1, 8], [3, 9, 77, 300], 2, 64, 16),
    ([40, 33], [40, 100], 3, 96, 32), ([5, 1], [50, 1], 2, 256, 64), ([1] * 70, [1 + i for i in range(70)], 1, 80, 8)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_read_gives_each_sequences_last_rows(q, kv, hk, dim, page, dtype):
    from gen_worker_amd.paged import paged_read_fp8

    r = Ragged8(q, kv, hk, hk, dim, page, dtype, seed=dim)
    k, v = paged_read_fp8(*r.pool(), r.table, r.q_start, r.kv_len, r.tokens, dtype=dtype)
    assert k.dtype == v.dtype == dtype and k.shape == (r.tokens, hk, dim)
    for b, n in enumerate(q):
        p, s = r.places(b)
        p, s, t0 = p[kv[b] - n:], s[kv[b] - n:], r.starts[b]
        assert torch.equal(k[t0:t0 + n], r.k[p, :, s]) and torch.equal(v[t0:t0 + n], r.v[p, :, s])


def test_read_leaves_rows_without_a_slot(monkeypatch):
    """Rows before q_start[0], behind the last sequence, and for slots before a sequence's first."""
    from gen_worker_amd import paged

    r = Ragged8([4, 2], [2, 5], 1, 1, 64, 16, BF16, seed=1)
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: real(*a, **k).fill_(9.0) if k.get("dtype") == BF16 else real(*a, **k))
    monkeypatch.setattr(torch, "empty_like", lambda t, **k: torch.full_like(t, 9.0))
    start = _ints([1, 5, 7])
    k, v = paged._read_fp8_body(*r.pool(), r.table, start, r.kv_len, 9, BF16)
    for x, own in ((k, r.k), (v, r.v)):
        assert bool((x[[0, 1, 2, 7, 8]] == 9).all())     # of four rows over two keys the first two have no slot
        p, s = r.places(0)
        assert torch.equal(x[3:5], own[p, :, s])
        p, s = r.places(1)
        assert torch.equal(x[5:7], own[p[3:], :, s[3:]])


# ---------------------------------------------------------------------------
# the write
# ---------------------------------------------------------------------------



@pytest.mark.parametrize("q,kv,heads,hk,dim,rot,page,interleaved,dtype", [
    ([1] * 70, [1 + 13 * i for i in range(70)], 8, 2, 128, 128, 16, False, BF16),
    ([5, 0, 17, 1], [5, 3, 40, 16], 6, 3, 64, 32, 8, True, F16),
    ([33, 2], [100, 2], 4, 4, 80, 20, 32, False, BF16),
    ([9, 4], [30, 4], 3, 1, 96, 96, 16, False, F16),
    ([3, 1], [3, 70], 20, 1, 256, 64, 64, True, BF16),
    ([2, 3], [2, 70], 60, 2, 256, 256, 16, False, BF16),
    ([7], [9], 2, 2, 16, 6, 8, False, F16),
    ([6], [6], 2, 1, 64, 0, 16, False, F16)])
@pytest.mark.parametrize("odd", [False, True])
def test_write_quantises_every_row(q, kv, heads, hk, dim, rot, page, interleaved, dtype, odd):
    """Rotated queries; values (not rotated) code for code and scale for scale; keys within the rotation's rounding of
    their definition; weights 0; everything else as it was. ``odd``: operands off 16-byte alignment."""
    from gen_worker_amd.paged import paged_write_fp8, rotary_table

    r = Ragged8(q, kv, heads, hk, dim, page, dtype, seed=dim + rot)
    row = torch.randn(r.tokens, (heads + 2 * hk) * dim + 8, generator=r.g, device=DEV)
    row *= torch.exp2(torch.randint(-12, 5, (r.tokens, 1), generator=r.g, device=DEV).float())   # rows of any size
    row = row.to(dtype)[:, 1 if odd else 0:]
    nq, nk = heads * dim, hk * dim
    x, k, v = (t.unflatten(1, (-1, dim)) for t in (row[:, :nq], row[:, nq:nq + nk], row[:, nq + nk:nq + 2 * nk]))
    at = torch.tensor([b - a + i for a, b in zip(q, kv) for i in range(a)], device=DEV)
    cos, sin = rotary_table(4096, rot, device=DEV) if rot else (None, None)
    before = {n: t.clone() for n, t in r.pools.items()}
    w0 = r.w.clone()
    got = paged_write_fp8(x, k, v, cos, sin, at.int(), *r.pool(), r.table, r.q_start, r.kv_len, weights=r.w,
                          interleaved=interleaved)
    if rot:
        _check_turned(got, *_turn(x, cos, sin, at, interleaved))
    else:
        assert torch.equal(got, x)
    new = torch.zeros(r.w.shape, dtype=torch.bool, device=DEV)
    for b, n in enumerate(q):
        if not n:
            continue
        p, s = r.places(b)
        p, s, t0 = p[kv[b] - n:], s[kv[b] - n:], r.starts[b]
        new[p, :, s] = True
        codes, scales = held(v[t0:t0 + n], dtype)
        assert torch.equal(r.pools["vs"][p, :, s], scales)
        assert torch.equal(r.pools["v"].view(torch.uint8)[p, :, s].view(FP8).double(), codes)
        turned, tol = _turn(k[t0:t0 + n], cos, sin, at[t0:t0 + n], interleaved) if rot else (k[t0:t0 + n].double(), 0.0)
        # between what the rows' ends of the rotation's tolerance are held as: the nearest code never falls with the value
        (lo, ls), (hi, hs) = held(turned - tol, dtype), held(turned + tol, dtype)
        scale = r.pools["ks"][p, :, s]
        got_k = value_of(r.pools["k"].view(torch.uint8)[p, :, s], scale)
        unit = torch.exp2(scale.double() - 127.0)[..., None]
        # (a scale decided by a value on its border may be either; then the values are a step of the coarser off at most)
        same = ((ls == hs) & (scale == ls))[..., None]
        lo, hi = lo * torch.exp2(ls.double() - 127.0)[..., None], hi * torch.exp2(hs.double() - 127.0)[..., None]
        step = torch.exp2(torch.floor(torch.log2((turned.abs() / unit).clamp(min=2.0 ** -6))) - 3.0) * unit
        assert bool(((got_k >= lo) & (got_k <= hi) | ~same & ((got_k - turned).abs() <= 2 * step)).all())
        assert bool((same.double().mean() > 0.95)) or n * hk < 20
    for n, t in r.pools.items():
        mask = new[..., None] if t.dim() == 4 else new
        assert torch.equal(torch.where(mask, 0, t.view(torch.uint8)), torch.where(mask, 0, before[n].view(torch.uint8)))
    assert bool((r.w[new] == 0).all()) and torch.equal(r.w[~new].nan_to_num(), w0[~new].nan_to_num())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_write_of_ends_of_the_range(dtype):
    """Rows of zeros, of subnormals, on the border between two scales, of the type's largest value, with infinities and
    NaN, of rounding ties: code for code."""
    from gen_worker_amd.paged import paged_write_fp8

    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    ends = [0.0, -0.0, tiny, tiny / 64, big, -big, 448.0, 449.0 if dtype == F16 else 450.0, 1.75, 1.7578125, 2.0 ** -20 if
            dtype == BF16 else 2.0 ** -14, math.inf, -math.inf, math.nan, 17.0, 18.0, 19.0, 25.0, 0.0048828125]
    rows = torch.zeros(len(ends) + 40, 1, 64, device=DEV)
    for i, x in enumerate(ends):
        rows[i, 0, i % 64] = x
        rows[i, 0, (i + 1) % 64] = -x / 3 if math.isfinite(x) else 1.0
        rows[i, 0, (i + 2) % 64] = x / 240 if math.isfinite(x) else -5.0
    rows[len(ends):] = torch.randn(40, 1, 64, generator=_gen(3), device=DEV).mul_(9).round_().div_(16)   # many ties
    rows = rows.to(dtype)
    n = rows.shape[0]
    codes = [torch.zeros(8, 1, 16, 64, dtype=torch.uint8, device=DEV).view(FP8) for _ in range(2)]
    scales = [torch.zeros(8, 1, 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
    table = _ints([[6, 0, 3, 5]])
    for view in (rows, torch.cat([rows.flatten(1), rows.flatten(1)], 1)[:, 1:65].unsqueeze(1)):
        paged_write_fp8(view, view, view, None, None, None, *codes, *scales, table, _ints([0, n]), _ints([n]))
        want, byte = held(view, dtype)
        j = torch.arange(n, device=DEV)
        for c, s in zip(codes, scales):
            got = c.view(torch.uint8)[table[0].long()[j // 16], :, j % 16].view(FP8).double()
            assert torch.equal(s[table[0].long()[j // 16], :, j % 16], byte)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_write_skips_tokens_without_a_slot():
    """Fewer keys than new tokens, a length past the table, rows behind the last sequence."""
    from gen_worker_amd.paged import paged_write_fp8

    x = torch.randn(9, 2, 64, generator=_gen(2), device=DEV).to(BF16)
    codes = [torch.full((3, 2, 8, 64), 5, dtype=torch.uint8, device=DEV).view(FP8) for _ in range(2)]
    scales = [torch.full((3, 2, 8), 5, dtype=torch.uint8, device=DEV) for _ in range(2)]
    got = paged_write_fp8(x, x, x, None, None, None, *codes, *scales, _ints([[0], [2]]), _ints([0, 4, 7]), _ints([2, 10]))
    assert torch.equal(got, x)
    want, byte = held(x, BF16)
    full = torch.full((3, 2, 8), 5, dtype=torch.uint8, device=DEV)
    full[0, :, :2] = byte[2:4].t()        # of four tokens over two keys the last two
    full[2, :, 7:] = byte[4:5].t()        # of slots 7, 8, 9 the one that the table holds
    for c, s in zip(codes, scales):
        assert torch.equal(s, full)
        assert torch.equal(c[0, :, :2].transpose(0, 1).double(), want[2:4])
        assert bool((c.view(torch.uint8)[1] == 5).all()) and bool((c.view(torch.uint8)[2, :, :7] == 5).all())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

SHAPES8 = [s for s in SHAPES if s[4] % 16 == 0] + [([2, 66], [7, 66], 3, 3, 16, 8, BF16), ([4], [700], 4, 2, 80, 8, F16)]


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", SHAPES8)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("gather", [False, True])
def test_attention_matches_64_bits(q, kv, heads, hk, dim, page, dtype, causal, gather):
    """Junk table entries, NaN codes and NaN scales in every slot no sequence owns must not matter."""
    r = Ragged8(q, kv, heads, hk, dim, page, dtype, seed=sum(kv) + dim)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(causal=causal, gather=gather)
    r.check(o, lse, causal, w0=w0)
    o2, lse2 = r.attend(causal=causal)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", LONG_RUNS)
@pytest.mark.parametrize("gather", [False, True])
def test_few_rows_over_more_pages_than_are_staged_at_once(q, kv, heads, hk, dim, page, dtype, gather):
    r = Ragged8(q, kv, heads, hk, dim, page, dtype, seed=dim)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(gather=gather)
    r.check(o, lse, w0=w0, heads=range(0, heads, 3))


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", [
    ([1] * 130, [(37 * i) % 400 + 1 for i in range(130)], 4, 2, 128, 16, BF16),
    ([3, 1], [200, 90], 80, 1, 64, 16, F16), ([2, 1], [70, 40], 260, 1, 64, 16, BF16),
    ([200] + [30] * 6, [7000] + [30] * 6, 2, 2, 128, 64, BF16)])
@pytest.mark.parametrize("gather", [False, True])
def test_many_sequences_heads_and_uneven_lengths(q, kv, heads, hk, dim, page, dtype, gather):
    r = Ragged8(q, kv, heads, hk, dim, page, dtype, seed=heads)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(gather=gather)
    r.check(o, lse, w0=w0, heads=range(0, heads, 13))


@pytest.mark.parametrize("dim,page", [(128, 16), (64, 32), (48, 16)])
@pytest.mark.parametrize("gather", [False, True])
def test_rows_that_see_nothing(dim, page, gather):
    r = Ragged8([5, 4, 0, 300], [3, 0, 0, 100], 4, 2, dim, page, BF16, seed=dim)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(gather=gather)
    r.check(o, lse, w0=w0)
    assert bool((lse[:2] == -math.inf).all()) and bool((lse[5:9] == -math.inf).all())


@pytest.mark.parametrize("dim", [128, 64, 48])
@pytest.mark.parametrize("by", ["code", "scale"])
@pytest.mark.parametrize("n,L", [(6, 40), (300, 500), (4, 5000)])
def test_nan_behind_the_mask_stays_there(dim, by, n, L):
    """The keys and values of a chunk's last tokens are NaN, by a code or by their row's scale: rows that do not see them
    are as if they were finite, rows that do are NaN."""
    r = Ragged8([n], [L], 4, 2, dim, 16, BF16, seed=5)
    o0, lse0 = r.attend()
    p, s = r.places(0)
    if by == "code":
        r.pools["k"].view(torch.uint8)[p[L - 2:], :, s[L - 2:], 3] = 127
        r.pools["v"].view(torch.uint8)[p[L - 2:], :, s[L - 2:], 1] = 255
    else:
        r.pools["ks"][p[L - 2:], :, s[L - 2:]] = 255
        r.pools["vs"][p[L - 2:], :, s[L - 2:]] = 255
    o, lse = r.attend()
    assert torch.equal(o[:n - 2], o0[:n - 2]) and torch.equal(lse[:n - 2], lse0[:n - 2])
    assert bool(o[n - 2:].isnan().all()) and bool(lse[n - 2:].isnan().all())
    # NaN values alone: their channel in the rows that see them
    r = Ragged8([n], [L], 4, 2, dim, 16, BF16, seed=5)
    r.pools["v"].view(torch.uint8)[p[L - 2:], :, s[L - 2:], 1] = 127
    o, lse = r.attend()
    assert torch.equal(lse, lse0) and torch.equal(o[:n - 2], o0[:n - 2])
    assert bool(o[n - 2:, :, 1].isnan().all())
    rest = [i for i in range(dim) if i != 1]
    assert torch.equal(o[n - 2:, :, rest], o0[n - 2:, :, rest])


def test_layouts_of_pages_scales_and_queries():
    """Pages that keep a slot's heads together, codes and scales as slices of wider pools, queries off alignment: the
    contiguous result bit for bit."""
    from gen_worker_amd.paged import paged_attention_fp8

    for q, kv in (([1, 1], [300, 1200]), ([70, 9], [300, 1200])):
        r = Ragged8(q, kv, 8, 2, 128, 16, BF16, seed=11)
        o, lse = r.attend(gather=False)
        u8 = {n: t.view(torch.uint8) for n, t in r.pools.items()}
        major = {n: t.transpose(1, 2).contiguous().transpose(1, 2).view(FP8) for n, t in u8.items() if len(n) == 1}
        wide = torch.full((2, u8["ks"].shape[0], 2, 24), 255, dtype=torch.uint8, device=DEV)
        wide[0, :, :, 5:21], wide[1, :, :, 5:21] = u8["ks"], u8["vs"]
        rest = (r.table, r.q_start, r.kv_len, max(q), max(kv))
        got = paged_attention_fp8(r.q, major["k"], major["v"], wide[0, :, :, 5:21], wide[1, :, :, 5:21], *rest)
        assert torch.equal(got[0], o) and torch.equal(got[1], lse)
        both = torch.stack((u8["k"], u8["v"]), dim=2).contiguous().view(FP8)
        row = torch.zeros(r.tokens, 8 * 128 + 64, dtype=BF16, device=DEV)
        row[:, 3:3 + 1024] = r.q.flatten(1)
        got = paged_attention_fp8(row[:, 3:3 + 1024].view(r.tokens, 8, 128), both[:, :, 0], both[:, :, 1],
                                  r.pools["ks"], r.pools["vs"], *rest)
        assert torch.equal(got[0], o) and torch.equal(got[1], lse)


def test_a_pool_past_32_bits():
    """Codes whose offsets pass 2^32, only the last pages in use."""
    pages = 9 * 2 ** 29 // (2 * 64 * 128)
    k, v = (torch.empty(pages, 2, 64, 128, dtype=torch.uint8, device=DEV).view(FP8) for _ in range(2))
    ks, vs = (torch.empty(pages, 2, 64, dtype=torch.uint8, device=DEV) for _ in range(2))
    assert (pages - 40) * k.stride(0) > 2 ** 32
    for q, kv in (([1, 1], [1000, 70]), ([100, 1], [1000, 70])):
        r = Ragged8(q, kv, 4, 2, 128, 64, BF16, seed=2, extra_pages=0)
        n = r.k.shape[0]
        o, lse = r.attend()
        for big, small in ((k, "k"), (v, "v"), (ks, "ks"), (vs, "vs")):
            big.view(torch.uint8)[pages - n:] = r.pools[small].view(torch.uint8)
        r.table = torch.where((r.table >= 0) & (r.table < 10 ** 6), r.table + (pages - n), r.table)
        r.pools = {"k": k, "v": v, "ks": ks, "vs": vs}
        got = r.attend()
        assert torch.equal(got[0], o) and torch.equal(got[1], lse)


def test_operands_past_32_bits():
    """New rows whose offsets pass 2^31 elements, and rows read back past them."""
    from gen_worker_amd.paged import paged_read_fp8, paged_write_fp8

    stride, n, dim = 2 ** 31 + 128, 2, 64
    pool = torch.empty(stride + n * 3 * dim, dtype=BF16, device=DEV)
    x = pool.as_strided((2, 3 * n, dim), (stride, dim, 1))
    x.copy_(torch.randn(2, 3 * n, dim, generator=_gen(9), device=DEV))
    q, k, v = x[:, :n], x[:, n:2 * n], x[:, 2 * n:]
    got = []
    for a in ((q, k, v), tuple(t.contiguous() for t in (q, k, v))):
        codes = [torch.zeros(1, n, 8, dim, dtype=torch.uint8, device=DEV).view(FP8) for _ in range(2)]
        scales = [torch.zeros(1, n, 8, dtype=torch.uint8, device=DEV) for _ in range(2)]
        out = paged_write_fp8(*a, None, None, None, *codes, *scales, _ints([[0]]), _ints([0, 2]), _ints([2]))
        got.append([out] + [t.view(torch.uint8) for t in codes + scales])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and torch.equal(got[0][0], q)
    del pool, x
    # many sequences that hold the same row: 2^31 elements and more of it
    rows = 2 ** 31 // (n * dim) + 1000
    batch = 60000
    each = rows // batch + 1
    width = -(-each // 8)
    codes = [t.view(FP8) for t in got[0][1:3]]
    table = torch.zeros(batch, width, dtype=torch.int32, device=DEV)
    q_start = (torch.arange(batch + 1, device=DEV) * each).int()
    kv_len = torch.full((batch,), each, dtype=torch.int32, device=DEV)
    k, v = paged_read_fp8(*codes, *got[0][3:], table, q_start, kv_len, batch * each)
    assert k.numel() > 2 ** 31
    first = paged_read_fp8(*codes, *got[0][3:], table[:1], q_start[:2], kv_len[:1], each)
    assert torch.equal(k[-each:], first[0]) and torch.equal(v[-each:], first[1])


def test_large_scores_and_small_rows():
    """One key takes all; all scores equal; a scale of one; rows whose scales differ by 2^40."""
    for mul, scale in ((40.0, None), (0.0, None), (1.0, 1.0)):
        r = Ragged8([1, 70], [900, 333], 8, 2, 128, 32, BF16, seed=3)
        r.q = (r.q.float() * mul).to(BF16)
        o, lse = r.attend(scale=scale)
        r.check(o, lse, scale=scale)
    r = Ragged8([1, 70], [900, 333], 8, 2, 128, 32, BF16, seed=3)
    for name in ("k", "v"):
        less = torch.randint(0, 40, r.pools[name + "s"].shape, generator=r.g, device=DEV)
        s = r.pools[name + "s"]
        s.copy_(torch.where(s == 255, 255, s.long() - less).to(torch.uint8))
        setattr(r, name, value_of(r.pools[name], s, BF16))
    o, lse = r.attend()
    r.check(o, lse)


def test_sizes_the_host_states_too_small_are_still_served():
    r = Ragged8([1, 40, 300], [900, 40, 700], 8, 2, 128, 16, BF16, seed=4)
    for mq, mk in ((1, 1), (0, 0), (2, 900), (300, 10)):
        w0 = r.w.clone()
        o, lse = r.attend(max_q=mq, max_kv=mk, gather=True)
        r.check(o, lse, w0=w0)


def test_write_and_attention_on_another_stream_and_in_a_graph():
    """Captured together once and replayed between eager work, with device lengths that change between replays."""
    from gen_worker_amd.paged import paged_attention_fp8, paged_write_fp8, rotary_table

    cos, sin = rotary_table(4096, 64, device=DEV)
    for q, kv in (([1, 1, 1], [500, 3000, 77]), ([200, 30], [900, 30])):
        r = Ragged8(q, kv, 8, 2, 128, 16, BF16, seed=9)
        k, v = (torch.randn(r.tokens, 2, 128, generator=r.g, device=DEV).to(BF16) for _ in range(2))
        at = torch.arange(r.tokens, device=DEV).int()
        pools = {n: t.clone() for n, t in r.pools.items()}
        lens = r.kv_len.clone()

        def step():
            x = paged_write_fp8(r.q, k, v, cos, sin, at, *r.pool(), r.table, r.q_start, r.kv_len, interleaved=True)
            return paged_attention_fp8(x, *r.pool(), r.table, r.q_start, r.kv_len, max(q), max(kv))

        def fresh(less):
            for n, t in r.pools.items():
                t.view(torch.uint8).copy_(pools[n].view(torch.uint8))
            r.kv_len.copy_(lens - less)

        want = {}
        for less in (0, 1, 5):
            fresh(less)
            want[less] = [t.clone() for t in step()]
        fresh(0)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step()
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
            got = step()
        torch.cuda.synchronize()
        for less in (0, 1, 0, 5, 1):
            fresh(less)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want[less]))
            step()


# ---------------------------------------------------------------------------
# eviction, the cache, the ways of calling
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv,hk,dim,page,budget,recent", [
    ([5, 40, 41, 700], 2, 128, 16, 40, 7), ([3000, 12], 1, 64, 8, 257, 0), ([90], 3, 48, 32, 64, 64)])
def test_evict_copies_codes_and_scales(kv, hk, dim, page, budget, recent):
    """The kept slots of the 16-bit eviction under the same weights, rows copied as they are."""
    from gen_worker_amd.paged import paged_evict, paged_evict_fp8

    r = Ragged8([0] * len(kv), kv, hk, hk, dim, page, BF16, seed=sum(kv))
    old, width = r.w.shape[0], -(-budget // page)
    new = torch.randperm(width * len(kv), generator=r.g, device=DEV).view(len(kv), width).int() + old
    grown = {n: torch.cat([t.view(torch.uint8), torch.zeros_like(t.view(torch.uint8)[:1]).expand(
        width * len(kv), *t.shape[1:])]) for n, t in r.pools.items()}
    w = torch.cat([r.w, torch.zeros(width * len(kv), hk, page, device=DEV)])
    wide = [torch.zeros(w.shape + (dim,), dtype=BF16, device=DEV) for _ in range(2)]
    want, want_len = paged_evict(*wide, w.clone(), r.table, r.kv_len, max(kv), new, budget, recent)
    kept, got_len = paged_evict_fp8(grown["k"].view(FP8), grown["v"].view(FP8), grown["ks"], grown["vs"], w, r.table,
                                    r.kv_len, max(kv), new, budget, recent)
    assert torch.equal(kept, want) and torch.equal(got_len, want_len)
    for b, n in enumerate(kv):
        m = min(n, budget)
        i = torch.arange(m, device=DEV)
        to, slot = new[b].long()[i // page], i % page
        for h in range(hk):
            j = kept[b, h, :m].long()
            p = r.table[b].long()[j // page]
            for name, t in grown.items():
                assert torch.equal(t[to, h, slot], t[p, h, j % page]), name
            assert torch.equal(w[to, h, slot], w[p, h, j % page])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cache_steps_like_one_long_sequence(dtype):
    """A ``PagedCache`` in 8 bits: prompts in chunks, then token by token, two layers; every step's attention equals plain
    attention over what the rows written so far are held as; after an eviction, over the kept ones."""
    from gen_worker_amd.paged import PagedCache, rotary_embed, rotary_table

    g = _gen(21)
    cache = PagedCache(64, 16, 2, 64, dtype=FP8, weights=True, device=DEV)
    layers = [cache, cache.twin()]
    cos, sin = rotary_table(512, 64, device=DEV)
    a, b = cache.add(), cache.add()
    for seqs, counts in (([a], [37]), ([a, b], [20, 90]), ([b, a], [1, 1]), ([a, b], [0, 1]), ([a, b], [1, 5])):
        batch = cache.extend(seqs, counts)
        for layer in layers:
            q, k, v = (torch.randn(batch.tokens, h, 64, generator=g, device=DEV).to(dtype) for h in (6, 2, 2))
            qr = layer.write(batch, q, k, v, cos, sin)
            assert qr.dtype == dtype and torch.equal(qr, rotary_embed(q, cos, sin, batch.positions))
            o, lse = layer.attend(batch, qr)
            first = layer is cache
            rows = cache.read(seqs, dtype=dtype) if first else None
            t = 0
            for i, (s, n) in enumerate(zip(seqs, counts)):
                if not first or not n:
                    t += n
                    continue
                kk, vv = rows[i]
                L = cache.length(s)
                assert kk.shape == (L, 2, 64) and kk.dtype == dtype
                code, byte = held(v[t:t + n], dtype)      # the last rows are this call's values, as they are held
                assert torch.equal(vv[L - n:].double(), code * torch.exp2(byte.double() - 127.0)[..., None])
                kk, vv = (x.double().repeat_interleave(3, dim=1) for x in (kk, vv))
                z = torch.einsum("thd,shd->hts", qr[t:t + n].double(), kk) / 8.0
                j = torch.arange(L, device=DEV)
                z = torch.where(j <= (L - n + torch.arange(n, device=DEV))[:, None], z, -math.inf)
                ref = torch.einsum("hts,shd->thd", torch.softmax(z, -1), vv)
                # p and o each rounded once, |v| < 6
                assert bool(((o[t:t + n].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 6.0) + 1e-4).all())
                t += n
    kept = cache.evict([a, b], 64, 8)
    before = None
    batch = cache.extend([b], [1])
    assert batch.max_kv == 65 and kept.shape == (1, 2, 64)
    q, k, v = (torch.randn(1, h, 64, generator=g, device=DEV).to(dtype) for h in (6, 2, 2))
    qr = cache.write(batch, q, k, v, cos, sin)
    o, _ = cache.attend(batch, qr)
    ((kk, vv),) = cache.read([b], dtype=dtype)
    assert before is None and kk.shape == (65, 2, 64)
    for x in range(6):
        kx, vx = kk[:, x // 3].double(), vv[:, x // 3].double()
        ref = torch.softmax((kx @ qr[0, x].double()) / 8.0, -1) @ vx
        assert bool(((o[0, x].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 6.0) + 1e-4).all())


def test_a_sixteen_bit_cache_reads_what_it_holds():
    from gen_worker_amd.paged import PagedCache, PagedError

    cache = PagedCache(16, 8, 2, 64, device=DEV)
    a, b = cache.add(), cache.add()
    batch = cache.extend([a, b], [19, 3])
    q, k, v = (torch.randn(22, 2, 64, generator=_gen(1), device=DEV).to(BF16) for _ in range(3))
    cache.write(batch, q, k, v)
    for (kk, vv), rows in zip(cache.read([b, a]), (slice(19, 22), slice(0, 19))):
        assert torch.equal(kk, k[rows]) and torch.equal(vv, v[rows])
    with pytest.raises(PagedError):
        cache.read([a], dtype=F16)


def test_native_host_calls_ops_and_python_bodies_agree(monkeypatch):
    """Every function with the native host calls, without them, and through the dispatcher: the same bits; refusals are
    Python's either way, and what a call writes has its version raised."""
    from gen_worker_amd import ops, paged

    assert ops._host is not None
    library = torch.ops.cozy_gen_worker
    r = Ragged8([3, 1], [50, 700], 4, 2, 64, 16, BF16, seed=8)
    cos, sin = paged.rotary_table(64, 32, device=DEV)
    at = torch.arange(r.tokens, device=DEV).int()
    new = _ints([[0, 1], [2, 3]])
    pools0, w0 = {n: t.clone() for n, t in r.pools.items()}, r.w.clone()
    k, v = r.q[:, :2], r.q[:, 2:]

    def everything(through_ops=False):
        r.w.copy_(w0)
        for n, t in r.pools.items():
            t.view(torch.uint8).copy_(pools0[n].view(torch.uint8))
        versions = [t._version for t in (*r.pool(), r.w)]
        a = (r.q, k, v, cos, sin, at, *r.pool(), r.table, r.q_start, r.kv_len)
        if through_ops:
            out = [library.paged_write_fp8(*a, r.w, True)]
        else:
            out = [paged.paged_write_fp8(*a, weights=r.w, interleaved=True)]
        assert all(t._version > n for t, n in zip((*r.pool(), r.w), versions))
        back = (*r.pool(), r.table, r.q_start, r.kv_len, r.tokens)
        out += library.paged_read_fp8(*back, F16) if through_ops else paged.paged_read_fp8(*back, dtype=F16)
        if through_ops:
            out += library.paged_attention_fp8(r.q, *r.pool(), r.table, r.q_start, r.kv_len, 3, 700, 0.125, True, r.w)
        else:
            out += r.attend(gather=True)
        grown = [torch.cat([t.view(torch.uint8), torch.zeros_like(t.view(torch.uint8)[:4])]) for t in r.pool()]
        w = torch.cat([r.w, torch.zeros_like(r.w[:4])])
        e = (grown[0].view(FP8), grown[1].view(FP8), grown[2], grown[3], w, r.table, r.kv_len, 700,
             new + r.w.shape[0], 32, 5)
        out += library.paged_evict_fp8(*e) if through_ops else paged.paged_evict_fp8(*e)
        out += [t.view(torch.uint8).clone() for t in r.pools.values()] + [r.w.clone(), w] + grown
        return out

    def refused():
        p = r.pool()
        for bad in (lambda: r.attend(q=r.q.float()), lambda: r.attend(q=r.q[:, :3]),
                    lambda: paged.paged_attention_fp8(r.q, p[0].view(torch.uint8), *p[1:], r.table, r.q_start, r.kv_len, 3, 700),
                    lambda: paged.paged_attention_fp8(r.q, *p[:2], p[2].int(), p[3], r.table, r.q_start, r.kv_len, 3, 700),
                    lambda: paged.paged_attention_fp8(r.q, *p[:2], p[2][:, :1], p[3], r.table, r.q_start, r.kv_len, 3, 700),
                    lambda: paged.paged_attention(r.q, *p[:2], r.table, r.q_start, r.kv_len, 3, 700),
                    lambda: paged.paged_write_fp8(r.q, k, v.to(F16), cos, sin, at, *p, r.table, r.q_start, r.kv_len),
                    lambda: paged.paged_write_fp8(r.q, r.q, r.q, cos, sin, at, *p, r.table, r.q_start, r.kv_len),
                    lambda: paged.paged_read_fp8(*p, r.table, r.q_start, r.kv_len, -1),
                    lambda: paged.paged_read_fp8(*p, r.table, r.q_start, r.kv_len, 4, dtype=F32),
                    lambda: paged.paged_evict_fp8(*p, None, r.table, r.kv_len, 700, new, 32, 5)):
            with pytest.raises(ValueError):
                bad()

    # (opcheck's schema test multiplies its arguments, which torch does not do in float8)
    for op, args in ((library.paged_attention_fp8, (r.q, *r.pool(), r.table, r.q_start, r.kv_len, 3, 700, 0.125, True, None)),
                     (library.paged_read_fp8, (*r.pool(), r.table, r.q_start, r.kv_len, r.tokens, F16))):
        torch.library.opcheck(op, args, test_utils=("test_faketensor",))
    with_host = everything()
    refused()
    by_ops = everything(through_ops=True)
    monkeypatch.setattr(ops, "_host", None)
    without = everything()
    refused()
    for a, b, c in zip(with_host, without, by_ops):
        assert torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(a.nan_to_num(), c.nan_to_num())
    q = r.q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        r.attend(q=q)[0].sum().backward()


def test_sequences_that_share_a_row_of_the_table():
    """Rows made with expand: what the contiguous copy gives."""
    from gen_worker_amd import ops
    from gen_worker_amd.paged import paged_attention_fp8, paged_read_fp8

    r = Ragged8([1], [300], 4, 2, 64, 16, BF16, seed=3)
    q = torch.randn(3, 4, 64, generator=r.g, device=DEV).to(BF16)
    start, lens = _ints([0, 1, 2, 3]), _ints([300, 100, 7])
    for host in (ops._host, None):
        keep, ops._host = ops._host, host
        try:
            one, many = r.table.expand(3, -1), r.table.expand(3, -1).contiguous()
            for a, b in zip(paged_attention_fp8(q, *r.pool(), one, start, lens, 1, 300),
                            paged_attention_fp8(q, *r.pool(), many, start, lens, 1, 300)):
                assert torch.equal(a, b)
            for a, b in zip(paged_read_fp8(*r.pool(), one, start, lens, 3), paged_read_fp8(*r.pool(), many, start, lens, 3)):
                assert torch.equal(a, b)
        finally:
            ops._host = keep


def test_nothing_to_do():
    from gen_worker_amd.paged import paged_attention_fp8, paged_read_fp8, paged_write_fp8

    r = Ragged8([0, 0], [5, 0], 4, 2, 64, 16, BF16, seed=3)
    before = {n: t.clone() for n, t in r.pools.items()}
    none = torch.empty(0, 4, 64, dtype=BF16, device=DEV)
    assert paged_write_fp8(none, none[:, :2], none[:, :2], None, None, None, *r.pool(), r.table, r.q_start,
                           r.kv_len).shape == (0, 4, 64)
    k, v = paged_read_fp8(*r.pool(), r.table, r.q_start, r.kv_len, 0)
    assert k.shape == v.shape == (0, 2, 64)
    o, lse = paged_attention_fp8(none, *r.pool(), r.table, r.q_start, r.kv_len, 0, 5)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    for n, t in r.pools.items():
        assert torch.equal(t.view(torch.uint8), before[n].view(torch.uint8))


def test_tangents_are_refused():
    """No call here has a forward-mode rule."""
    import torch.autograd.forward_ad as fwad

    from gen_worker_amd.paged import PagedError, paged_write_fp8
    from gen_worker_amd.sampling import SamplingError, sample_tokens

    r = Ragged8([3], [50], 4, 2, 64, 16, BF16, seed=3)
    with fwad.dual_level():
        q = fwad.make_dual(r.q, torch.ones_like(r.q))
        with pytest.raises(PagedError, match="tangent"):
            r.attend(q=q)
        with pytest.raises(PagedError, match="tangent"):
            paged_write_fp8(q, r.q[:, :2], r.q[:, :2], None, None, None, *r.pool(), r.table, r.q_start, r.kv_len)
        x = torch.randn(2, 9, device=DEV)
        with pytest.raises(SamplingError, match="tangent"):
            sample_tokens(fwad.make_dual(x, x), torch.rand(2, device=DEV))
