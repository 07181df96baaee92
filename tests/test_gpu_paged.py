"""The paged-cache operators on the GPU (``gen_worker_amd.paged``) against plain 64-bit implementations.

Tolerances are bounds derived from the operators' stated roundings, element by element (u: the unit roundoff of the
tensors' type, e = 2^-24 that of fp32):

* scores: a dot of d products in fp32 is off by at most (d + 4) e sum|q||k|, so a probability by that on each side of
  the softmax, relatively, plus 2^-20 for the exponential, sums and reciprocal;
* o: p is rounded to the type (u relatively; fp16 also by 2^-25 of a key's largest share where it is subnormal), the
  output once more;
* lse: the scores' bound plus fp32 rounding of the value itself and the logarithm's;
* gathered weights: the probabilities' bound, and fp32 sums over the rows.

Rotations are held to one rounding of the type plus fp32 rounding of the two products; whole numbers and moved
values are equal."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def _turn(x, cos, sin, at, interleaved, inverse=False):
    """64-bit rotation, pair by pair, and the bound on its fp32 evaluation."""
    x, c, s = x.double(), cos.double()[at][:, None], sin.double()[at][:, None]
    if inverse:
        s = -s
    r = cos.shape[1]
    y, tol = x.clone(), torch.zeros_like(x)
    if not r:
        return y, tol
    i0 = torch.arange(r, device=DEV) * (2 if interleaved else 1)
    i1 = i0 + (1 if interleaved else r)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    tol[..., i0] = tol[..., i1] = 4 * E * (a.abs() + b.abs()) * max(1.0, float(c.abs().max()))
    return y, tol


def _check_turned(got, ref, tol):
    u = U[got.dtype]
    err = (got.double() - ref).abs()
    # one rounding of the type (fp16 subnormals: half their spacing)
    assert bool((err <= tol * (1 + u) + u * ref.abs() + (2.0 ** -25 if got.dtype == F16 else 0)).all()), float(err.max())


@pytest.mark.parametrize("tokens,heads,dim,rot,interleaved,dtype", [
    (1, 32, 128, 128, False, BF16), (1, 1, 64, 64, True, F16), (77, 24, 128, 64, True, BF16),
    (1029, 3, 64, 32, False, F16), (33, 5, 80, 20, False, BF16), (17, 7, 96, 6, True, F32), (65, 2, 256, 256, True, F32),
    (40, 4, 6, 2, False, BF16), (300, 8, 128, 128, True, F16), (9, 4, 128, 0, False, BF16)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_matches_the_rotation(tokens, heads, dim, rot, interleaved, dtype, inverse):
    from gen_worker_amd.paged import rotary_embed, rotary_table

    g = _gen(tokens + dim)
    x = torch.randn(tokens, heads, dim, generator=g, device=DEV).to(dtype)
    if rot:
        cos, sin = rotary_table(2048, rot, device=DEV)
    else:
        cos = sin = torch.empty(2048, 0, device=DEV)
    at = torch.randint(0, 2048, (tokens,), generator=g, device=DEV)
    got = rotary_embed(x, cos, sin, at.int(), interleaved=interleaved, inverse=inverse)
    ref, tol = _turn(x, cos, sin, at, interleaved, inverse)
    _check_turned(got, ref, tol)
    assert torch.equal(got[..., rot:], x[..., rot:])


def test_rotary_strides_alignment_and_default_positions():
    """A column slice of a fused projection, a view off 16-byte alignment, heads before tokens, and token indices as
    positions; positions outside the table read its ends."""
    from gen_worker_amd.paged import rotary_embed, rotary_table

    cos, sin = rotary_table(600, 64, device=DEV)
    fused = torch.randn(500, 3 * 6 * 64 + 8, generator=_gen(1), device=DEV).to(BF16)
    at = torch.arange(500, device=DEV)
    for x in (fused[:, 384:768].view(500, 6, 64), fused[:, 1:385].view(500, 6, 64),
              fused[:, :384].reshape(6, 500, 64).transpose(0, 1),
              fused[:, :768].view(500, 6, 128)[..., ::2], fused[:, :64].view(500, 1, 64).expand(500, 6, 64)):
        got = rotary_embed(x, cos, sin)
        _check_turned(got, *_turn(x, cos, sin, at, False))
        assert torch.equal(got, rotary_embed(x.contiguous(), cos, sin, at.int()))
    x = fused[:3, :384].view(3, 6, 64)
    assert torch.equal(rotary_embed(x, cos, sin, _ints([-5, 599, 10 ** 6])), rotary_embed(x, cos, sin, _ints([0, 599, 599])))
    assert rotary_embed(x[:0], cos, sin).shape == (0, 6, 64)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    """Against the formula's gradient (the rotation back), against differences of the fp32 operator, and through an
    expanded upstream gradient."""
    from gen_worker_amd.paged import rotary_embed, rotary_table

    g = _gen(7)
    cos, sin = rotary_table(64, 32, device=DEV)
    at = torch.randint(0, 64, (19,), generator=g, device=DEV)
    x = torch.randn(19, 3, 48, generator=g, device=DEV, requires_grad=True)
    dy = torch.randn(19, 3, 48, generator=g, device=DEV)
    y = rotary_embed(x, cos, sin, at.int(), interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, dy)
    _check_turned(dx, *_turn(dy, cos, sin, at, interleaved, inverse=True))
    # <dy, R(x + h v) - R(x - h v)> / 2h = <dx, v>: the map is linear, so only rounding separates them: outputs of
    # size ~4 h each off by ~8 e |x| over 2 h, summed over 2736 values with |dy| ~ 1
    v = torch.randn(x.shape, generator=g, device=DEV)
    with torch.no_grad():
        up, down = (rotary_embed(x + s * 4.0 * v, cos, sin, at.int(), interleaved=interleaved) for s in (1, -1))
        slope = float((dy.double() * (up.double() - down.double())).sum()) / 8.0
    want = float((dx.double() * v.double()).sum())
    assert abs(slope - want) <= 16 * E * float((dy.abs().double() * (x.detach().abs().mean() + 4 * v.abs()).double()).sum())
    (de,) = torch.autograd.grad(rotary_embed(x, cos, sin, at.int(), interleaved=interleaved).sum(), x)
    _check_turned(de, *_turn(torch.ones_like(x), cos, sin, at, interleaved, inverse=True))


# ---------------------------------------------------------------------------
# a ragged cache
# ---------------------------------------------------------------------------

class Ragged:
    """Sequences of q[i] new tokens and kv[i] keys in shuffled pages. ``stale`` fills what no sequence owns."""

    def __init__(self, q, kv, heads, kv_heads, dim, page, dtype, seed, stale=float("nan"), slot_major=False,
                 extra_pages=3):
        self.q_len, self.kv, self.heads, self.hk, self.dim, self.page, self.dtype = q, kv, heads, kv_heads, dim, page, dtype
        g = self.g = _gen(seed)
        counts = [-(-n // page) for n in kv]
        pages = sum(counts) + extra_pages
        order = torch.randperm(pages, generator=g, device=DEV).tolist()
        width = max(max(counts), 1)
        rows, at = [], 0
        for c in counts:
            rows.append(order[at:at + c] + [2 ** 31 - 1, -7][c % 2:c % 2 + 1] * (width - c))   # junk past the end
            at += c
        self.table, self.kv_len = _ints(rows).view(len(kv), width), _ints(kv)
        starts = [0]
        for n in q:
            starts.append(starts[-1] + n)
        self.starts, self.tokens, self.q_start = starts, starts[-1], _ints(starts)
        shape = (pages, page, kv_heads, dim) if slot_major else (pages, kv_heads, page, dim)
        self.k, self.v = (torch.full(shape, stale, dtype=dtype, device=DEV) for _ in range(2))
        if slot_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.w = torch.full((pages, kv_heads, page), stale, device=DEV)
        for b, n in enumerate(kv):
            p, s = self.places(b)
            self.k[p, :, s] = (torch.randn(n, kv_heads, dim, generator=g, device=DEV) + 0.3).to(dtype)
            self.v[p, :, s] = torch.randn(n, kv_heads, dim, generator=g, device=DEV).to(dtype)
            self.w[p, :, s] = torch.rand(n, kv_heads, generator=g, device=DEV)
        self.q = (torch.randn(self.tokens, heads, dim, generator=g, device=DEV) * 1.5).to(dtype)

    def places(self, b, n=None):
        j = torch.arange(self.kv[b] if n is None else n, device=DEV)
        return self.table[b].long()[j // self.page], j % self.page

    def attend(self, q=None, causal=True, gather=False, scale=None, max_q=None, max_kv=None):
        from gen_worker_amd.paged import paged_attention

        return paged_attention(self.q if q is None else q, self.k, self.v, self.table, self.q_start, self.kv_len,
                               max(self.q_len) if max_q is None else max_q, max(self.kv) if max_kv is None else max_kv,
                               causal=causal, scale=scale, weights=self.w if gather else None)

    def check(self, o, lse, causal=True, scale=None, w0=None, heads=None):
        """o and lse (and the weights gathered on top of w0) against 64 bits."""
        scale = self.dim ** -0.5 if scale is None else scale
        u, g = U[self.dtype], self.heads // self.hk
        assert o.dtype == self.dtype and lse.dtype == F32
        for b, n in enumerate(self.q_len):
            L, t0 = self.kv[b], self.starts[b]
            p, s = self.places(b)
            i = torch.arange(n, device=DEV)
            seen = torch.arange(L, device=DEV) <= (L - n + i if causal else torch.full_like(i, L))[:, None]
            dw = torch.zeros(self.hk, L, dtype=torch.float64, device=DEV)
            dw_tol = torch.zeros_like(dw)
            for x in (range(self.heads) if heads is None or w0 is not None else heads):
                q, k, v = self.q[t0:t0 + n, x].double(), self.k[p, x // g, s].double(), self.v[p, x // g, s].double()
                z = torch.where(seen, (q @ k.t().contiguous()) * scale, -math.inf)
                mag = torch.where(seen, (q.abs() @ k.abs().t().contiguous()) * scale, 0.0)
                top = mag.amax(-1) if L else torch.zeros(n, dtype=torch.float64, device=DEV)
                ds = (self.dim + 4) * E * top                                 # a score's error, by row
                empty = ~seen.any(-1)
                ref_lse = torch.logsumexp(z, -1) if L else torch.full((n,), -math.inf, device=DEV, dtype=torch.float64)
                prob = torch.where(empty[:, None], 0.0, torch.softmax(z, -1)) if L else z.new_zeros(n, 0)
                prob = torch.nan_to_num(prob) if bool(empty.any()) else prob
                vz = v
                ref, spread = prob @ vz, prob @ vz.abs()
                rel = 2 * ds[:, None] + 2.0 ** -20
                tol = (u + rel) * spread + u * ref.abs() + E
                if self.dtype == F16:
                    tol = tol + 2.0 ** -25 * (prob.amax(-1, keepdim=True) if L else 0.0) * vz.abs().sum(0)
                got, glse = o[t0:t0 + n, x].double(), lse[t0:t0 + n, x].double()
                assert bool(((got - ref).abs() <= tol).all()), (b, x, float(((got - ref).abs() - tol).max()))
                assert bool((got[empty] == 0).all()) and bool((glse[empty] == -math.inf).all())
                lt = ds + 4 * E * (top + ref_lse.abs()) + 2.0 ** -20
                assert bool(((glse - ref_lse).abs() <= lt)[~empty].all()), (b, x)
                dw[x // g] += prob.sum(0)
                dw_tol[x // g] += (prob * rel).sum(0)
            if w0 is not None:
                want = w0[p, :, s].double().t() + dw
                err = (self.w[p, :, s].double().t() - want).abs()
                assert bool((err <= dw_tol + (n * g + 4) * E * want).all()), (b, float(err.max()))


SHAPES = [
    # q lens, kv lens, heads, kv heads, dim, page, dtype: one token; ragged ones; groups of 1, 3, 7 and 8; chunks across page
    # and tile ends; idle, new and empty sequences; head dims the matrix cores serve and others
    ([1], [1], 4, 4, 128, 16, BF16),
    ([1], [701], 32, 8, 128, 16, BF16),
    ([1, 1, 1], [17, 1, 2050], 8, 1, 64, 64, F16),
    ([1] * 5, [1, 63, 64, 65, 4097], 6, 2, 128, 8, BF16),
    ([3, 0, 1, 8], [3, 9, 77, 300], 14, 2, 64, 16, BF16),
    ([5, 2], [5000, 1030], 16, 2, 128, 128, F16),
    ([130, 1, 33], [130, 500, 290], 3, 1, 128, 32, BF16),
    ([257, 64, 0, 255], [513, 64, 40, 1000], 4, 4, 64, 16, F16),
    ([600], [1500], 8, 8, 128, 64, BF16),
    ([40, 7], [40, 1024], 16, 2, 64, 4096, BF16),
    ([9, 1], [300, 70], 4, 2, 96, 16, BF16),
    ([20, 1], [90, 129], 2, 1, 256, 16, F16),
    ([2, 66], [7, 66], 3, 3, 8, 8, BF16),
]


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("gather", [False, True])
def test_attention_matches_64_bits(q, kv, heads, hk, dim, page, dtype, causal, gather):
    """Junk table entries and NaN in every slot no sequence owns must not matter."""
    r = Ragged(q, kv, heads, hk, dim, page, dtype, seed=sum(kv) + dim)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(causal=causal, gather=gather)
    r.check(o, lse, causal, w0=w0)
    o2, lse2 = r.attend(causal=causal)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    if gather:
        untouched = torch.ones_like(r.w, dtype=torch.bool)
        for b in range(len(kv)):
            p, s = r.places(b)
            untouched[p, :, s] = False
        assert bool(torch.isnan(r.w[untouched]).all())


def _many(n, lo, hi, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", [
    # more than 64 sequences (one token each; chunks), more than 64 kv heads, groups past 64 and past 256 query heads, one
    # sequence with nearly all of the keys among many short ones
    ([1] * 130, _many(130, 0, 400, 1), 4, 2, 128, 16, BF16),
    (_many(70, 0, 20, 2), [3000] + _many(69, 20, 90, 3), 4, 1, 64, 16, F16),
    ([1, 2, 1], [600, 31, 257], 70, 70, 64, 16, BF16),
    ([3, 1], [200, 90], 80, 1, 64, 16, F16), ([2, 1], [70, 40], 260, 1, 64, 16, BF16),
    ([2] + [1] * 40, [9000] + [5] * 40, 8, 8, 64, 64, BF16), ([200] + [30] * 6, [7000] + [30] * 6, 2, 2, 128, 64, BF16)])
@pytest.mark.parametrize("gather", [False, True])
def test_many_sequences_heads_and_uneven_lengths(q, kv, heads, hk, dim, page, dtype, gather):
    kv = [max(a, b) for a, b in zip(q, kv)]
    r = Ragged(q, kv, heads, hk, dim, page, dtype, seed=heads)
    w0 = r.w.clone() if gather else None
    for causal in (True, False):
        if gather:
            r.w.copy_(w0)
        o, lse = r.attend(causal=causal, gather=gather)
        r.check(o, lse, causal, w0=w0, heads=range(0, heads, 13))


def test_gather_without_room_for_the_scores():
    """A table that could address so many keys that few-row scores are not kept: recomputed, the same sums."""
    r = Ragged([1, 3], [700, 90], 8, 2, 64, 4096, BF16, seed=6)
    w0 = r.w.clone()
    r.attend(gather=True)
    kept = r.w.clone()
    r.w.copy_(w0)
    r.table = torch.cat([r.table, torch.full((2, 4000), -1, dtype=torch.int32, device=DEV)], 1)
    o, lse = r.attend(gather=True)
    r.check(o, lse, w0=w0)
    p, s = r.places(0)
    # both are sums of 8 probabilities of a key, each within its own bound of the exact ones
    assert bool(((r.w - kept)[p, :, s].abs() <= 1e-4 * kept[p, :, s] + 1e-6).all())


@pytest.mark.parametrize("dim,page", [(128, 16), (64, 32), (40, 16)])
@pytest.mark.parametrize("gather", [False, True])
def test_rows_that_see_nothing(dim, page, gather):
    """More new tokens than keys (the first rows see none), no keys at all, no new tokens at all."""
    r = Ragged([5, 4, 0, 300], [3, 0, 0, 100], 4, 2, dim, page, BF16, seed=dim)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(gather=gather)
    r.check(o, lse, w0=w0)
    assert bool((lse[:2] == -math.inf).all()) and bool((lse[5:9] == -math.inf).all())
    o, lse = r.attend(causal=False)
    r.check(o, lse, causal=False)


@pytest.mark.parametrize("dim", [128, 64, 48])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n,L", [(6, 40), (300, 500)])
def test_nonfinite_values_behind_the_mask_stay_there(dim, bad, n, L):
    """The keys and values of a chunk's last tokens hold NaN or infinities: rows that do not see them are as if they were
    finite, and rows that do see them are not finite."""
    r = Ragged([n], [L], 4, 2, dim, 16, BF16, seed=5)
    o0, lse0 = r.attend()
    p, s = r.places(0)
    r.k[p[L - 3:], :, s[L - 3:]] = bad
    r.v[p[L - 2:], :, s[L - 2:], 1] = bad
    o, lse = r.attend(gather=True)
    assert torch.equal(o[:n - 3], o0[:n - 3]) and torch.equal(lse[:n - 3], lse0[:n - 3])
    assert not bool(torch.isfinite(o[n - 1, :, 1]).any())


def test_large_scores_and_ties():
    """Scores of thousands (one key takes all), all scores equal, and a scale of one."""
    for mul, scale in ((40.0, None), (0.0, None), (1.0, 1.0)):
        r = Ragged([1, 70], [900, 333], 8, 2, 128, 32, BF16, seed=3)
        r.q = (r.q.float() * mul).to(BF16)
        o, lse = r.attend(scale=scale)
        r.check(o, lse, scale=scale)


@pytest.mark.parametrize("q,kv", [([1, 1], [300, 1200]), ([70, 9], [300, 1200])])
def test_layouts_of_pages_and_queries(q, kv):
    """Pages that keep a slot's heads together, keys and values in one pool, queries as a column slice of a wider row, a
    query view off 16-byte alignment: the contiguous result bit for bit."""
    r = Ragged(q, kv, 8, 2, 128, 16, BF16, seed=11)
    o, lse = r.attend()
    s = Ragged(q, kv, 8, 2, 128, 16, BF16, seed=11, slot_major=True)
    s.k.copy_(r.k), s.v.copy_(r.v)
    for got in (s.attend(),):
        assert torch.equal(got[0], o) and torch.equal(got[1], lse)
    both = torch.stack((r.k, r.v), dim=2).contiguous()
    r.k, r.v = both[:, :, 0], both[:, :, 1]
    wide = torch.zeros(r.tokens, 8 * 128 + 64, dtype=BF16, device=DEV)
    wide[:, 8:8 + 1024] = r.q.flatten(1)
    for qv in (wide[:, 8:8 + 1024].view(r.tokens, 8, 128), r.q.transpose(0, 1).contiguous().transpose(0, 1)):
        got = r.attend(q=qv)
        assert torch.equal(got[0], o) and torch.equal(got[1], lse)
    wide[:, 3:3 + 1024] = r.q.flatten(1)
    got = r.attend(q=wide[:, 3:3 + 1024].view(r.tokens, 8, 128))
    assert torch.equal(got[0], o) and torch.equal(got[1], lse)


def test_a_pool_past_32_bits():
    """Pages whose byte and element offsets pass 2^32: a pool of 9 GiB of keys, only its last pages in use."""
    pages = 9 * 2 ** 30 // (2 * 64 * 128 * 2)
    k, v = (torch.empty(pages, 2, 64, 128, dtype=BF16, device=DEV) for _ in range(2))
    assert (pages - 40) * k.stride(0) > 2 ** 32
    for q, kv in (([1, 1], [1000, 70]), ([100, 1], [1000, 70])):
        r = Ragged(q, kv, 4, 2, 128, 64, BF16, seed=2, extra_pages=0)
        k[pages - r.k.shape[0]:], v[pages - r.k.shape[0]:] = r.k, r.v
        o, lse = r.attend()
        r.table = torch.where((r.table >= 0) & (r.table < 10 ** 6), r.table + (pages - r.k.shape[0]), r.table)
        r.k, r.v = k, v
        got = r.attend()
        assert torch.equal(got[0], o) and torch.equal(got[1], lse)


def test_sizes_the_host_states_too_small_are_still_served():
    """max_q and max_kv shape the launch only."""
    r = Ragged([1, 40, 300], [900, 40, 700], 8, 2, 128, 16, BF16, seed=4)
    for mq, mk in ((1, 1), (0, 0), (2, 900), (300, 10)):
        w0 = r.w.clone()
        o, lse = r.attend(max_q=mq, max_kv=mk, gather=True)
        r.check(o, lse, w0=w0)


def test_attention_on_another_stream_and_in_a_graph():
    """Decode and chunk with weights, captured once and replayed between eager work; each replay adds its weights."""
    for q, kv in (([1, 1, 1], [500, 3000, 77]), ([200, 30], [900, 30])):
        r = Ragged(q, kv, 8, 2, 128, 16, BF16, seed=9)
        w0 = r.w.clone()
        o, lse = r.attend(gather=True)
        step = r.w.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            o2, lse2 = r.attend()
        s.synchronize()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
        r.w.copy_(w0)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
            og, lg = r.attend(gather=True)
        torch.cuda.synchronize()
        for _ in range(4):
            r.w.copy_(w0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(og, o) and torch.equal(lg, lse)
            assert torch.equal(r.w.nan_to_num(), step.nan_to_num())
            r.attend()


# ---------------------------------------------------------------------------
# the write
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("q,kv,heads,hk,dim,rot,page,interleaved,dtype", [
    ([1] * 70, [1 + 13 * i for i in range(70)], 8, 2, 128, 128, 16, False, BF16),
    ([5, 0, 17, 1], [5, 3, 40, 16], 6, 3, 64, 32, 8, True, F16),
    ([33, 2], [100, 2], 4, 4, 80, 20, 32, False, BF16),
    ([6], [6], 2, 1, 64, 0, 16, False, F16)])
def test_write_places_every_token(q, kv, heads, hk, dim, rot, page, interleaved, dtype):
    """Rotated queries, each key and value in its slot, its weight 0, everything else as it was; operands as slices of
    a fused row."""
    from gen_worker_amd.paged import paged_write, rotary_table

    r = Ragged(q, kv, heads, hk, dim, page, dtype, seed=dim + rot, stale=7.0)
    row = torch.randn(r.tokens, (heads + 2 * hk) * dim, generator=r.g, device=DEV).to(dtype)
    nq, nk = heads * dim, hk * dim
    x, k, v = (t.view(r.tokens, -1, dim) for t in (row[:, :nq], row[:, nq:nq + nk], row[:, nq + nk:]))
    at = torch.tensor([b - a + i for a, b in zip(q, kv) for i in range(a)], device=DEV)
    cos, sin = rotary_table(4096, rot, device=DEV) if rot else (None, None)
    wk, wv, ww = r.k.clone(), r.v.clone(), r.w.clone()
    got = paged_write(x, k, v, cos, sin, at.int(), r.k, r.v, r.table, r.q_start, r.kv_len, weights=r.w,
                      interleaved=interleaved)
    tk = k
    if rot:
        _check_turned(got, *_turn(x, cos, sin, at, interleaved))
        from gen_worker_amd.paged import rotary_embed
        assert torch.equal(got, rotary_embed(x, cos, sin, at.int(), interleaved=interleaved))
        tk = rotary_embed(k, cos, sin, at.int(), interleaved=interleaved)
    else:
        assert torch.equal(got, x)
    for b, n in enumerate(q):
        p, s = r.places(b)
        p, s, t0 = p[kv[b] - n:], s[kv[b] - n:], r.starts[b]
        wk[p, :, s], wv[p, :, s], ww[p, :, s] = tk[t0:t0 + n], v[t0:t0 + n], 0.0
    assert torch.equal(r.k, wk) and torch.equal(r.v, wv) and torch.equal(r.w, ww)


def test_write_skips_tokens_without_a_slot():
    """Fewer keys than new tokens, and a length past the table: the tokens without a slot are rotated, not stored."""
    from gen_worker_amd.paged import paged_write

    r = Ragged([4, 3], [16, 16], 2, 1, 64, 16, BF16, seed=1, stale=7.0)
    k = torch.randn(7, 1, 64, generator=r.g, device=DEV).to(BF16)
    k0, v0 = r.k.clone(), r.v.clone()
    got = paged_write(r.q, k, k, None, None, None, r.k, r.v, r.table, r.q_start, _ints([2, 18]))
    assert torch.equal(got, r.q)
    p0, p1 = int(r.table[0, 0]), int(r.table[1, 0])
    k0[p0, :, 0:2] = v0[p0, :, 0:2] = k[2:4].transpose(0, 1)
    k0[p1, :, 15] = v0[p1, :, 15] = k[4]
    assert torch.equal(r.k, k0) and torch.equal(r.v, v0)


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------

def _evict_reference(w, n, budget, recent):
    """Kept slots of one head, from a sort of (weight, slot) pairs."""
    if n <= budget:
        return list(range(n))
    first = n - recent
    key = lambda j: (0 if math.isnan(w[j]) else 1, -w[j] if not math.isnan(w[j]) else 0.0, j)  # noqa: E731
    return sorted(sorted(range(first), key=key)[:budget - recent]) + list(range(first, n))


@pytest.mark.parametrize("kv,hk,dim,page,budget,recent,dtype", [
    ([640, 259, 512, 513, 0, 1], 3, 128, 16, 512, 64, BF16),
    ([3000, 100], 2, 64, 64, 1, 0, F16), ([3000, 1025], 1, 64, 8, 1024, 1024, BF16),
    ([70, 64, 3], 2, 8, 8, 5, 2, F16), ([33000], 2, 128, 128, 20000, 1, BF16)])
@pytest.mark.parametrize("weights", ["spread", "ties", "odd"])
def test_evict_keeps_the_heaviest(kv, hk, dim, page, budget, recent, dtype, weights):
    from gen_worker_amd.paged import paged_evict

    r = Ragged([0] * len(kv), kv, hk, hk, dim, page, dtype, seed=len(kv) + budget, extra_pages=0)
    g = _gen(budget)
    if weights == "spread":
        w = torch.exp(3 * torch.randn(r.w.shape, generator=g, device=DEV))
    elif weights == "ties":
        w = torch.randint(0, 3, r.w.shape, generator=g, device=DEV).float()
    else:
        pick = torch.tensor([0.0, -0.0, float("nan"), float("inf"), 1e-42, -2.5, 3.0, 3.0000002], device=DEV)
        w = pick[torch.randint(0, 8, r.w.shape, generator=g, device=DEV)]
    r.w.copy_(w)
    # fresh pages behind the old ones
    m = [min(n, budget) for n in kv]
    counts = [-(-n // page) for n in m]
    width, old, rows, at = max(counts), r.k.shape[0], [], r.k.shape[0]
    for c in counts:
        rows.append(list(range(at, at + c)) + [10 ** 9] * (width - c))
        at += c
    grow = lambda t: torch.cat([t, torch.full((at - old,) + t.shape[1:], 7.0, dtype=t.dtype, device=DEV)])  # noqa: E731
    k, v, w = grow(r.k), grow(r.v), grow(r.w)
    wk, wv, ww = k.clone(), v.clone(), w.clone()
    new = _ints(rows)
    # the host's idea of the largest kv_len shapes the launch only
    stated = max(kv) if weights != "ties" else min(max(kv), budget, width * page) // 3
    kept, new_len = paged_evict(k, v, w, r.table, r.kv_len, stated, new, budget, recent)
    assert new_len.tolist() == m
    for b, n in enumerate(kv):
        p, s = r.places(b)
        i = torch.arange(m[b], device=DEV)
        for h in range(hk):
            want = _evict_reference(r.w[p, h, s].tolist(), n, budget, recent)
            assert kept[b, h].tolist() == want + [-1] * (budget - m[b]), (b, h)
            at = torch.tensor(want, dtype=torch.long, device=DEV)
            for dst in (wk, wv, ww):
                dst[new[b].long()[i // page], h, i % page] = dst[p[at], h, s[at]]
    same = lambda a, b: torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0))  # noqa: E731
    assert same(k, wk) and same(v, wv) and same(w, ww)


@pytest.mark.parametrize("n,recent", [(41, 0), (41, 3), (5003, 70)])
def test_evict_reads_weights_of_any_stride(n, recent):
    """Heads and pages of the weights an odd number of elements apart, from an odd one on."""
    from gen_worker_amd.paged import paged_evict

    page, budget, hk = 8, 20 + recent, 3
    r = Ragged([0], [n], hk, hk, 64, page, BF16, seed=n, extra_pages=0)
    pages, m = r.k.shape[0], min(n, budget)
    count = -(-m // page)
    grow = lambda t: torch.cat([t, torch.zeros((count,) + t.shape[1:], dtype=t.dtype, device=DEV)])  # noqa: E731
    w = torch.full((pages + count, hk, page + 1), float("inf"), device=DEV)[:, :, 1:]
    w.copy_(torch.rand(w.shape, generator=_gen(n), device=DEV))
    before = w.clone()
    new = _ints([list(range(pages, pages + count))])
    kept, _ = paged_evict(grow(r.k), grow(r.v), w, r.table, r.kv_len, n, new, budget, recent)
    p, s = r.places(0)
    for h in range(hk):
        assert kept[0, h].tolist() == _evict_reference(before[p, h, s].tolist(), n, budget, recent), h


# ---------------------------------------------------------------------------
# the ops, and the cache that ties them together
# ---------------------------------------------------------------------------

def test_ops_give_what_the_functions_give():
    """The dispatcher's way (taken under compilation, tracing and autograd) runs the same calls."""
    from gen_worker_amd.paged import rotary_table

    ops = torch.ops.cozy_gen_worker
    r = Ragged([3, 1], [50, 9], 4, 2, 64, 16, BF16, seed=8)
    cos, sin = rotary_table(64, 64, device=DEV)
    w0 = r.w.clone()
    o, lse = r.attend(gather=True)
    w1 = r.w.clone()
    r.w.copy_(w0)
    a = (r.q, r.k, r.v, r.table, r.q_start, r.kv_len)
    o2, lse2 = ops.paged_attention(*a, 3, 50, 64 ** -0.5, True, r.w)
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and torch.equal(r.w.nan_to_num(), w1.nan_to_num())
    torch.library.opcheck(ops.rotary_embed, (r.q, cos, sin, None, True, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.paged_attention, (*a, 3, 50, 0.125, True, None), test_utils=("test_schema", "test_faketensor"))
    q = r.q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        r.attend(q=q)[0].sum().backward()


def test_cache_steps_like_one_long_sequence():
    """Prompts in chunks, then token by token, two layers' pools under one bookkeeping: every step's attention equals
    plain attention over all of the sequence's keys; after an eviction, over the kept ones."""
    from gen_worker_amd.paged import PagedCache, rotary_embed, rotary_table

    g = _gen(21)
    cache = PagedCache(64, 16, 2, 64, weights=True, device=DEV)
    layers = [cache, cache.twin()]
    cos, sin = rotary_table(512, 64, device=DEV)
    a, b = cache.add(), cache.add()
    seen = {(s, i): [[], []] for s in (a, b) for i in (0, 1)}
    for seqs, counts in (([a], [37]), ([a, b], [20, 90]), ([b, a], [1, 1]), ([a, b], [0, 1]), ([a, b], [1, 5])):
        batch = cache.extend(seqs, counts)
        assert batch.tokens == sum(counts)
        for i, layer in enumerate(layers):
            q, k, v = (torch.randn(batch.tokens, h, 64, generator=g, device=DEV).to(BF16) for h in (6, 2, 2))
            qr = layer.write(batch, q, k, v, cos, sin)
            assert torch.equal(qr, rotary_embed(q, cos, sin, batch.positions))
            kr = rotary_embed(k, cos, sin, batch.positions)
            o, lse = layer.attend(batch, qr)
            t = 0
            for s, n in zip(seqs, counts):
                seen[s, i][0].append(kr[t:t + n]), seen[s, i][1].append(v[t:t + n])
                kk, vv = (torch.cat(x).double().repeat_interleave(3, dim=1) for x in seen[s, i])
                L = kk.shape[0]
                z = torch.einsum("thd,shd->hts", qr[t:t + n].double(), kk) / 8.0
                j = torch.arange(L, device=DEV)
                z = torch.where(j <= (L - n + torch.arange(n, device=DEV))[:, None], z, -math.inf)
                ref = torch.einsum("hts,shd->thd", torch.softmax(z, -1), vv)
                # p and o each rounded once, |v| < 6
                assert bool(((o[t:t + n].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 6.0) + 1e-4).all())
                t += n
    total = [float(layer.weights[cache._seqs[s][0]].sum()) for layer in layers for s in (a, b)]
    # a row's probabilities sum to 1: every token of every query head has given 1 in all
    want = [6.0 * n for _ in layers for n in (59, 97)]
    assert all(abs(x - y) <= 1e-4 * y for x, y in zip(total, want)), (total, want)
    free = cache.free_pages
    kept = cache.evict([a, b], 64, 8)
    assert cache.length(a) == 59 and cache.length(b) == 64 and kept.shape == (1, 2, 64)
    assert cache.free_pages == free + 7 - 4
    batch = cache.extend([b], [1])
    assert int(batch.positions[0]) == 97 and batch.max_kv == 65
    q, k, v = (torch.randn(1, h, 64, generator=g, device=DEV).to(BF16) for h in (6, 2, 2))
    qr = cache.write(batch, q, k, v, cos, sin)
    o, _ = cache.attend(batch, qr)
    kk, vv = (torch.cat(x)[:97] for x in seen[b, 0])
    kr = rotary_embed(k, cos, sin, batch.positions)
    for x in range(6):
        rows = kept[0, x // 3].long()
        kx, vx = torch.cat([kk[rows, x // 3], kr[:, x // 3]]).double(), torch.cat([vv[rows, x // 3], v[:, x // 3]]).double()
        ref = torch.softmax((kx @ qr[0, x].double()) / 8.0, -1) @ vx
        assert bool(((o[0, x].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 6.0) + 1e-4).all())
    cache.drop(a)
    cache.drop(b)
    assert cache.free_pages == 64


def test_native_host_calls_and_python_bodies_agree(monkeypatch):
    """Every function with the native host calls and without them: the same bits; what the native ones do not take
    (operands of another type, a missing table, autograd through attention) is decided by Python either way."""
    from gen_worker_amd import ops, paged

    assert ops._host is not None
    r = Ragged([3, 1], [50, 700], 4, 2, 64, 16, BF16, seed=8)
    w0, k0 = r.w.clone(), r.k.clone()
    cos, sin = paged.rotary_table(64, 32, device=DEV)
    at = torch.arange(r.tokens, device=DEV).int()
    new = _ints([[0, 1], [2, 3]])
    x = torch.randn(5, 3, 48, generator=r.g, device=DEV, requires_grad=True)

    def everything():
        r.w.copy_(w0), r.k.copy_(k0)
        out = [paged.rotary_embed(r.q, cos, sin, at, interleaved=True), paged.rotary_embed(r.q, cos, sin, inverse=True)]
        y = paged.rotary_embed(x, cos, sin)
        (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        assert dx.requires_grad and y.requires_grad
        out += [y.detach(), dx.detach(), torch.autograd.grad(dx.square().sum(), x)[0]]
        out.append(paged.paged_write(r.q, r.q[:, :2], r.q[:, 2:], cos, sin, at, r.k, r.v, r.table, r.q_start, r.kv_len,
                                     weights=r.w))
        out += [*r.attend(gather=True), r.w.clone()]
        dst_k, dst_v, dst_w = (torch.cat([t, torch.zeros_like(t[:4])]) for t in (r.k, r.v, r.w))
        out += [*paged.paged_evict(dst_k, dst_v, dst_w, r.table, r.kv_len, 700, new + r.k.shape[0], 32, 5), dst_k, dst_v]
        for bad in (lambda: r.attend(q=r.q.to(F16)), lambda: paged.rotary_embed(r.q, cos, sin.double()),
                    lambda: paged.rotary_embed(r.q, cos, sin, at.long()), lambda: r.attend(q=r.q[:, :3]),
                    lambda: paged.paged_write(r.q, r.q, r.q, cos, sin, at, r.k, r.v, r.table, r.q_start, r.kv_len),
                    lambda: paged.paged_evict(r.k, r.v, r.w, r.table, r.kv_len, 700, new, 4, 5),
                    lambda: paged.rotary_embed(r.q, None, None),
                    lambda: paged.rotary_embed(r.q, cos.clone().requires_grad_(True), sin)):
            with pytest.raises(ValueError):
                bad()
        return out

    with_host = everything()
    monkeypatch.setattr(ops, "_host", None)
    without = everything()
    for a, b in zip(with_host, without):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    (dx,) = torch.autograd.grad(paged.rotary_embed(x, cos, sin).square().sum(), x)
    # the rotation keeps lengths: d |y|^2 / dx = 2 x, to rounding of two rotations of values below 6
    assert bool(((dx - 2 * x).abs() <= 64 * E * 6).all())


@pytest.mark.parametrize("native", [True, False])
def test_sequences_that_share_a_row_of_the_table(native, monkeypatch):
    """A table made with expand, all of whose rows are one (and a strided one whose rows overlap): what its contiguous copy
    gives, bit for bit; an expanded target of an eviction is refused."""
    from gen_worker_amd import ops
    from gen_worker_amd.paged import PagedError, paged_attention, paged_evict, paged_write

    if not native:
        monkeypatch.setattr(ops, "_host", None)
    r = Ragged([40], [700], 4, 2, 64, 16, BF16, seed=31)
    for n_seq, each in ((8, 1), (3, 40)):
        tokens = n_seq * each
        q = torch.randn(tokens, 4, 64, generator=r.g, device=DEV).to(BF16)
        start = torch.arange(0, tokens + 1, each, device=DEV, dtype=torch.int32)
        lens = _ints([700 - 3 * i for i in range(n_seq)])
        shared = r.table[:1].expand(n_seq, r.table.shape[1])
        sliding = torch.cat([r.table[0]] * 2).as_strided((n_seq, r.table.shape[1]), (1, 1))
        for table in (shared, sliding):
            got = paged_attention(q, r.k, r.v, table, start, lens, each, 700)
            want = paged_attention(q, r.k, r.v, table.contiguous(), start, lens, each, 700)
            # (shifted rows show slots behind the history's end, which hold NaN)
            assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(got, want))
            assert table is sliding or bool(torch.isfinite(got[0]).all())
    # two sequences of one history; the second alone takes new tokens
    k = torch.randn(3, 2, 64, generator=r.g, device=DEV).to(BF16)
    q = torch.randn(3, 4, 64, generator=r.g, device=DEV).to(BF16)
    table, pools = r.table[:1].expand(2, r.table.shape[1]), []
    for t in (table, table.contiguous()):
        kp, vp = r.k.clone(), r.v.clone()
        paged_write(q, k, k, None, None, None, kp, vp, t, _ints([0, 0, 3]), _ints([600, 700]))
        pools.append((kp, vp))
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(*pools))
    p, s = r.places(0)
    assert torch.equal(pools[0][0][p[697:], :, s[697:]], k)
    w = torch.rand(r.w.shape, generator=r.g, device=DEV)
    outs, new = [], _ints([[0, 1, 2], [3, 4, 5]]) + r.k.shape[0]
    for t in (table, table.contiguous()):
        pool = [torch.cat([x, torch.zeros_like(x[:6])]) for x in (r.k, r.v, w)]
        outs.append([*paged_evict(*pool, t, _ints([700, 650]), 700, new, 40, 4), *pool])
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(*outs))
    with pytest.raises(PagedError, match="overlap"):
        paged_evict(*pool, table, _ints([700, 650]), 700, new[:1].expand(2, 3), 40, 4)


@pytest.mark.parametrize("q,kv,dim,page,max_kv,gather", [
    # two runs of one sequence, the second from key 256 of 512-slot pages on; 32 shares of 137 thousand keys, most of which
    # start inside their page
    ([1], [270003], 128, 512, 512, False), ([2], [270003], 64, 512, 512, True), ([1], [4400001], 64, 256, None, False)])
def test_runs_that_start_inside_a_page_and_pass_the_staged_ids(q, kv, dim, page, max_kv, gather):
    """More pages to a run of keys than the kernel stages at a time, from the middle of a page on."""
    r = Ragged(q, kv, 2, 1, dim, page, BF16, seed=17)
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(max_kv=max_kv, gather=gather)
    r.check(o, lse, w0=w0)


# one run of all of a sequence's keys (the host states one key), longer than the page ids staged at a time
LONG_RUNS = [([1], [5003], 4, 1, 128, 8, BF16), ([6, 3], [8197, 5003], 4, 2, 64, 8, F16), ([8], [8197], 4, 2, 128, 8, BF16),
             ([5], [16400], 6, 1, 64, 16, BF16), ([4, 0, 7], [8193, 70, 4097], 4, 1, 128, 8, F16)]


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", LONG_RUNS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("gather", [False, True])
def test_few_rows_over_more_pages_than_are_staged_at_once(q, kv, heads, hk, dim, page, dtype, causal, gather):
    r = Ragged(q, kv, heads, hk, dim, page, dtype, seed=sum(kv))
    w0 = r.w.clone() if gather else None
    o, lse = r.attend(causal=causal, gather=gather, max_q=max(q), max_kv=1)
    r.check(o, lse, causal, w0=w0)


@pytest.mark.parametrize("q,kv,heads,hk,dim,page,dtype", LONG_RUNS[1:])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_values_behind_the_mask_of_a_late_segment(q, kv, heads, hk, dim, page, dtype, bad):
    """NaN or infinities in the last two tokens' values, in the second or third segment of staged pages: rows that do not
    see them are as if they were finite, rows that do are not finite in their channel and unchanged in the others."""
    r = Ragged(q, kv, heads, hk, dim, page, dtype, seed=sum(kv) + 1)
    o0, lse0 = r.attend(max_kv=1)
    r.check(o0, lse0)
    for b, n in enumerate(q):
        if n:
            p, s = r.places(b)
            r.v[p[-2:], :, s[-2:], 1] = bad
    o, lse = r.attend(max_kv=1)
    assert torch.equal(lse, lse0)
    for b, n in enumerate(q):
        t0 = r.starts[b]
        assert torch.equal(o[t0:t0 + max(n - 2, 0)], o0[t0:t0 + max(n - 2, 0)])
        last = slice(t0 + max(n - 2, 0), t0 + n)
        assert not bool(torch.isfinite(o[last][..., 1]).any())
        other = torch.arange(dim, device=DEV) != 1
        assert torch.equal(o[last][..., other], o0[last][..., other])


@pytest.mark.parametrize("n,L,dim", [(1, 200, 64), (1, 257, 128), (1, 700, 64), (4, 700, 128), (1, 5000, 128), (4, 5000, 64),
                                     (70, 257, 128), (70, 700, 64), (70, 5000, 128), (300, 5000, 64), (3, 257, 48),
                                     (3, 700, 48), (3, 5000, 48)])
@pytest.mark.parametrize("where", ["query", "key"])
@pytest.mark.parametrize("gather", [False, True])
def test_nan_that_a_row_sees_is_in_its_answer(n, L, dim, where, gather):
    """A NaN query, and a NaN last key (the last new token's own): o and lse of the rows that see it are NaN, in every
    form (one run, splits, shares, row tiles, one wave a row); all other rows are as before, bit for bit. Every key
    such a row sees has drawn NaN from it."""
    heads, hk = 4, 2
    r = Ragged([n], [L], heads, hk, dim, 16, BF16, seed=n + L)
    w0 = r.w.clone()
    o0, lse0 = r.attend(gather=gather)
    clean = r.w.clone()
    r.w.copy_(w0)
    p, s = r.places(0)
    hit = torch.zeros(n, heads, dtype=torch.bool, device=DEV)
    drawn = torch.zeros(L, hk, dtype=torch.bool, device=DEV)
    if where == "query":
        t = n // 2
        r.q[t, 1, 5] = float("nan")
        hit[t, 1] = True
        drawn[:L - n + t + 1, 0] = True
    else:
        r.k[p[-1], 1, s[-1], 3] = float("nan")
        hit[n - 1, 2:] = True
        drawn[:, 1] = True
    o, lse = r.attend(gather=gather)
    assert bool(torch.isnan(o[hit]).all()) and bool(torch.isnan(lse[hit]).all())
    assert torch.equal(o[~hit], o0[~hit]) and torch.equal(lse[~hit], lse0[~hit])
    if gather:
        got, want = r.w[p, :, s], clean[p, :, s]
        assert bool(torch.isnan(got[drawn]).all()) and torch.equal(got[~drawn], want[~drawn])


MINUS_INF_FORMS = [(1, 200, 64), (1, 700, 128), (4, 700, 64), (1, 5000, 128), (4, 5000, 64), (70, 700, 128), (300, 5000, 64),
                   (3, 700, 48)]


@pytest.mark.parametrize("n,L,dim", MINUS_INF_FORMS)
@pytest.mark.parametrize("gather", [False, True])
def test_keys_whose_scores_are_minus_infinity(n, L, dim, gather):
    """The first keys (whole tiles that every row sees) score -inf: they draw nothing, and the answer is the softmax over
    the others. A row all of whose scores are -inf is one without keys."""
    heads, hk, lost = 4, 2, 150
    r = Ragged([n], [L], heads, hk, dim, 16, BF16, seed=n + L)
    r.q[..., 0] = 1.0
    p, s = r.places(0)
    w0 = r.w.clone()
    r.k[p[:lost], :, s[:lost], 0] = -math.inf
    o, lse = r.attend(gather=gather)
    u, dw = U[BF16], torch.zeros(L, hk, dtype=torch.float64, device=DEV)
    dw_tol = torch.zeros_like(dw)
    j, i = torch.arange(lost, L, device=DEV), torch.arange(n, device=DEV)
    seen = j <= (L - n + i)[:, None]
    for x in range(heads):
        h = x // (heads // hk)
        q, k, v = r.q[:, x].double(), r.k[p[lost:], h, s[lost:]].double(), r.v[p[lost:], h, s[lost:]].double()
        z = torch.where(seen, (q @ k.t().contiguous()) * dim ** -0.5, -math.inf)
        top = ((q.abs() @ k.abs().t().contiguous()) * dim ** -0.5).amax(-1)
        prob, ref_lse = torch.softmax(z, -1), torch.logsumexp(z, -1)
        ds = (dim + 4) * E * top
        rel = 2 * ds[:, None] + 2.0 ** -20
        ref, spread = prob @ v, prob @ v.abs()
        assert bool(((o[:, x].double() - ref).abs() <= (u + rel) * spread + u * ref.abs() + E).all())
        assert bool(((lse[:, x].double() - ref_lse).abs() <= ds + 4 * E * (top + ref_lse.abs()) + 2.0 ** -20).all())
        dw[lost:, h] += prob.sum(0)
        dw_tol[lost:, h] += (prob * rel).sum(0)
    if gather:
        want = w0[p, :, s].double() + dw
        assert bool(((r.w[p, :, s].double() - want).abs() <= dw_tol + (n * heads // hk + 4) * E * want).all())
        assert torch.equal(r.w[p[:lost], :, s[:lost]], w0[p[:lost], :, s[:lost]])
    r.k[p, 1, s, 0] = -math.inf
    r.w.copy_(w0)
    o, lse = r.attend(gather=gather)
    assert bool((o[:, 2:] == 0).all()) and bool((lse[:, 2:] == -math.inf).all()) and bool(torch.isfinite(lse[:, :2]).all())
    assert not gather or torch.equal(r.w[p, 1, s], w0[p, 1, s])


@pytest.mark.parametrize("dim", [128, 48])
def test_no_stated_keys_with_many_tokens_still_gather(dim):
    """max_kv = 0 with chunks: keys that the host did not know of are attended and their weights gathered, and a batch
    that has none keeps its weights."""
    r = Ragged([300, 40], [700, 40], 8, 2, dim, 16, BF16, seed=13)
    w0 = r.w.clone()
    o, lse = r.attend(max_q=300, max_kv=0, gather=True)
    r.check(o, lse, w0=w0)
    r.kv, r.kv_len = [0, 0], _ints([0, 0])
    r.w.copy_(w0)
    o, lse = r.attend(max_q=300, max_kv=0, gather=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    assert torch.equal(r.w.nan_to_num(), w0.nan_to_num())


def test_evictions_leave_every_layer_with_its_own_keys():
    """Three pools under one bookkeeping, the third a twin of the second: after an eviction each attends the kept keys
    of its own, in the shared pages."""
    from gen_worker_amd.paged import PagedCache

    g = _gen(5)
    first = PagedCache(32, 16, 1, 64, weights=True, device=DEV)
    second = first.twin()
    pools = [first, second, second.twin()]
    seq = first.add()
    first.drop(first.add())
    batch = first.extend([seq], [90])
    held = []
    for pool in pools:
        q, k, v = (torch.randn(90, 1, 64, generator=g, device=DEV).to(BF16) for _ in range(3))
        pool.write(batch, q, k, v)
        # gathered weights of this test's choosing: the same slots are kept in all layers
        pool.weights[batch.table[0].long()] = torch.arange(96, device=DEV).flip(0).float().view(6, 1, 16)
        held.append((k, v))
    kept = first.evict([seq], 40, 8)
    assert kept.tolist() == [[list(range(32)) + list(range(82, 90))]]
    batch = first.extend([seq], [1])
    for pool, (k, v) in zip(pools, held):
        q, kn, vn = (torch.randn(1, 1, 64, generator=g, device=DEV).to(BF16) for _ in range(3))
        o, _ = pool.attend(batch, pool.write(batch, q, kn, vn))
        kk = torch.cat([k[kept[0, 0].long(), 0], kn[:, 0]]).double()
        vv = torch.cat([v[kept[0, 0].long(), 0], vn[:, 0]]).double()
        p = torch.softmax((kk @ q[0, 0].double()) / 8.0, -1)
        ref, spread = p @ vv, p @ vv.abs()
        # p and o each rounded once, scores of a few units off by a few 2^-24 of their terms
        assert bool(((o[0, 0].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + spread) + 1e-4 * spread).all())


@pytest.mark.parametrize("native", [True, False])
def test_pools_that_a_graph_saved_are_known_to_have_changed(native, monkeypatch):
    """Every call that writes raises the version of what it wrote, as an in-place torch operation does, and of nothing
    else; a backward pass over a pool saved before fails instead of using the new values."""
    from gen_worker_amd import ops
    from gen_worker_amd.paged import paged_evict, paged_write

    if not native:
        monkeypatch.setattr(ops, "_host", None)
    r = Ragged([2], [40], 2, 1, 64, 16, BF16, seed=3)
    new = _ints([sorted(set(range(6)) - set(r.table[0].tolist()))[:2]])
    k = torch.randn(2, 1, 64, generator=r.g, device=DEV).to(BF16)
    calls = [
        (lambda: paged_write(r.q, k, k, None, None, None, r.k, r.v, r.table, r.q_start, r.kv_len), (r.k, r.v)),
        (lambda: paged_write(r.q, k, k, None, None, None, r.k, r.v, r.table, r.q_start, r.kv_len, weights=r.w),
         (r.k, r.v, r.w)),
        (lambda: r.attend(), ()), (lambda: r.attend(gather=True), (r.w,)),
        (lambda: paged_evict(r.k, r.v, r.w, r.table, r.kv_len, 40, new, 20, 4), (r.k, r.v, r.w))]
    tensors = (r.k, r.v, r.w, r.q, k, r.table, r.q_start, r.kv_len, new)
    for call, wrote in calls:
        before = [t._version for t in tensors]
        x = torch.ones((), device=DEV, requires_grad=True)
        graphs = [(x * t).nan_to_num().sum() for t in wrote]
        call()
        for t, v in zip(tensors, before):
            assert (t._version > v) == any(t is w for w in wrote)
        for y in graphs:
            with pytest.raises(RuntimeError, match="inplace operation"):
                y.backward()
    with torch.inference_mode():
        s = Ragged([2], [40], 2, 1, 64, 16, BF16, seed=3)
    s.attend(gather=True)   # tensors of inference mode have no version
    paged_write(s.q, k, k, None, None, None, s.k, s.v, s.table, s.q_start, s.kv_len, weights=s.w)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, True)])
def test_rotary_forward_mode(native, interleaved, inverse, monkeypatch):
    """The tangent turns as x does, with the tensor's own dual numbers, under torch.func.jvp and, vectorised, jacfwd."""
    from torch.autograd import forward_ad

    from gen_worker_amd import ops
    from gen_worker_amd.paged import rotary_embed, rotary_table

    if not native:
        monkeypatch.setattr(ops, "_host", None)
    g = _gen(4)
    cos, sin = rotary_table(64, 32, device=DEV)
    at = torch.randint(0, 64, (5,), generator=g, device=DEV)
    x, v = (torch.randn(5, 2, 40, generator=g, device=DEV) for _ in range(2))

    def f(t):
        return rotary_embed(t, cos, sin, at.int(), interleaved=interleaved, inverse=inverse)

    with forward_ad.dual_level():
        y, dy = forward_ad.unpack_dual(f(forward_ad.make_dual(x, v)))
        assert forward_ad.unpack_dual(f(x)).tangent is None
    for got, t in ((y, x), (dy, v), *zip(torch.func.jvp(f, (x,), (v,)), (x, v))):
        _check_turned(got, *_turn(t, cos, sin, at, interleaved, inverse))
    # the Jacobian's columns are the rotated unit vectors: its product with v is v rotated, to fp32 sums of pairs
    j = torch.func.jacfwd(lambda t: f(t.view(1, 1, -1).expand(5, 2, 40)))(x[0, 0])
    assert bool(((j.double() @ v[0, 0].double()) - f(v[:1, :1].expand(5, 2, 40)).double()).abs().max() <= 16 * E * 6)


@pytest.mark.parametrize("native", [True, False])
def test_rotary_gradient_of_upstream_gradients_that_are_not_plain(native, monkeypatch):
    """A lazily negated upstream gradient, a batch of them (a vectorised Jacobian), one under a dispatch mode, and a
    strided one: each is the plain gradient's result."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from gen_worker_amd import ops
    from gen_worker_amd.paged import rotary_embed, rotary_table

    if not native:
        monkeypatch.setattr(ops, "_host", None)

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names = getattr(self, "names", []) + [str(func)]
            return func(*args, **(kwargs or {}))

    cos, sin = rotary_table(16, 8, device=DEV)
    g = _gen(12)
    x = torch.randn(5, 2, 8, generator=g, device=DEV, requires_grad=True)
    dy = torch.randn(3, 5, 2, 8, generator=g, device=DEV)
    y = rotary_embed(x, cos, sin)

    def grad(d, **kw):
        return torch.autograd.grad(y, x, d, retain_graph=True, **kw)[0]

    want = torch.stack([grad(d) for d in dy])
    _check_turned(want[0], *_turn(dy[0], cos, sin, torch.arange(5, device=DEV), False, inverse=True))
    assert torch.equal(grad(torch._neg_view(dy[0])), -want[0])
    assert torch.equal(grad(dy, is_grads_batched=True), want)
    assert torch.equal(grad(dy[1].transpose(0, 2).contiguous().transpose(0, 2)), want[1])
    with Seen() as seen:
        assert torch.equal(grad(dy[2]), want[2])
    assert any("rotary_embed" in n for n in seen.names)
