"""``sample_tokens`` on the GPU against its definition in 64 bits, row by row.

Tokens are equal: the random numbers are given, and a weight's rounding to 2^-45 of the largest moves a border between
tokens by less than 2^-27 of the smallest gap that these rows' fp32 numbers can tell apart, unless a test says so. A
logprob is off by fp32 rounding of itself (2^-24) and, absolutely, by the weights' rounding: vocab 2^-46 of a sum of at
least 1."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def of_row(x, u, t, k, p, m):
    """(token, logprob) of one row by the definition. x: float64 numpy."""
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    u, t, p, m = f32(u), f32(t), min(max(f32(p), 0.0), 1.0), min(max(f32(m), 0.0), 1.0)
    real = np.where(np.isnan(x), -np.inf, x)
    top = real.max()
    if top == -np.inf:
        return -1, math.nan
    if not t > 0:
        return int(np.argmax(real == top)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(real == top, 1.0, np.exp(np.where(real == -np.inf, -np.inf, (real - top) / t)))
    w = np.nan_to_num(w)
    order = np.argsort(-real, kind="stable")
    if k > 0:
        order = order[:k]
    if p < 1:
        upto = np.cumsum(w[order])
        order = order[:int((upto < p * upto[-1]).sum()) + 1]
    order = np.concatenate([order[:1], order[1:][w[order[1:]] >= m]])
    kept = np.sort(order)
    upto = np.cumsum(w[kept])
    at = kept[min(int((upto <= min(max(u, 0.0), 1.0) * upto[-1]).sum()), np.flatnonzero(w[kept])[-1])]
    return int(at), float(np.log(w[at] / upto[-1]))


def check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    from gen_worker_amd.sampling import sample_tokens

    tokens, logprobs = sample_tokens(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert tokens.dtype == torch.int64 and logprobs.dtype == F32 and tokens.shape == logprobs.shape == logits.shape[:1]
    x, u = logits.double().cpu().numpy(), uniform.cpu().numpy()
    each = [v.cpu().numpy() if isinstance(v, torch.Tensor) else [v] * len(x) for v in (temperature, top_k, top_p, min_p)]
    for r in range(len(x)):
        want, lp = of_row(x[r], u[r], *(v[r] for v in each))
        got, glp = int(tokens[r]), float(logprobs[r])
        assert got == want, (r, got, want, [v[r] for v in each], u[r])
        assert (math.isnan(lp) and math.isnan(glp)) or abs(glp - lp) <= 2.0 ** -24 * abs(lp) + x.shape[1] * 2.0 ** -46, (r, glp, lp)
    return tokens


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(temperature=40.0), dict(top_k=1), dict(top_k=7),
            dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.1),
            dict(min_p=1.0), dict(min_p=1e-3), dict(min_p=0.3, top_p=0.7), dict(min_p=1e-6, temperature=2.0),
            dict(top_k=100, top_p=0.8), dict(top_k=600, min_p=0.01), dict(temperature=1.5, top_k=300, top_p=0.95, min_p=0.02), dict(top_k=10 ** 6, top_p=0.3)]


@pytest.mark.parametrize("rows,vocab", [(3, 1), (5, 2), (4, 7), (9, 64), (6, 257), (5, 2048), (5, 2049), (3, 5003),
                                        (3, 8192), (3, 8193), (2, 12289), (2, 70001), (40, 20011), (1, 300007)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_tokens_by_the_definition(rows, vocab, dtype):
    """bf16 rows of tens of thousands hold many equal logits: cuts fall among them."""
    g = _gen(rows * vocab)
    logits = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(dtype)
    for s in SETTINGS:
        check(logits, torch.rand(rows, generator=g, device=DEV), **s)


@pytest.mark.parametrize("spread", [0.0, 1e-6, 1e-3, 0.3, 300.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_one_bin_and_of_many(spread, dtype):
    """All logits equal, all within a bin of the histogram (thousands of them, which are ranked digit by digit), and so far
    apart that nearly all weigh nothing."""
    g = _gen(5)
    logits = (torch.randn(3, 9001, generator=g, device=DEV) * spread + 2.0).to(dtype)
    for s in SETTINGS + [dict(top_k=4000), dict(top_k=9000, top_p=0.7), dict(top_k=5000, min_p=0.5)]:
        check(logits, torch.rand(3, generator=g, device=DEV), **s)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("spread", [1.0, 4.0])
def test_cuts_of_every_length(spread, dtype):
    """A few collected tokens, hundreds, thousands, and more than are collected; bf16: ties on every border."""
    g = _gen(21)
    logits = (torch.randn(2, 50021, generator=g, device=DEV) * spread).to(dtype)
    for k in (2, 63, 64, 65, 255, 256, 257, 511, 513, 1000, 1024, 1025, 2048, 4096, 4097):
        for more in (dict(), dict(top_p=0.9), dict(min_p=0.02)):
            check(logits, torch.rand(2, generator=g, device=DEV), top_k=k, **more)
    for p in (0.01, 0.2, 0.6, 0.97, 0.9999):
        for t in (0.6, 1.0, 3.0):
            check(logits, torch.rand(2, generator=g, device=DEV), temperature=t, top_p=p)


def test_rows_past_32_bits():
    """Rows whose offset passes 2^31 elements and 2^32 bytes."""
    from gen_worker_amd.sampling import sample_tokens

    for vocab in (2000, 40001):
        pool = torch.empty(2 ** 31 + 64 + vocab, dtype=BF16, device=DEV)
        logits = pool.as_strided((2, vocab), (2 ** 31 + 64, 1))
        logits.copy_(torch.randn(2, vocab, generator=_gen(vocab), device=DEV) * 3)
        u = torch.rand(2, generator=_gen(3), device=DEV)
        for s in (dict(), dict(temperature=0.0), dict(top_k=50, top_p=0.9)):
            got, want = sample_tokens(logits, u, **s), sample_tokens(logits.contiguous(), u, **s)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            check(logits.contiguous(), u, **s)


def test_two_streams_at_once():
    from gen_worker_amd.sampling import sample_tokens

    g = _gen(13)
    logits = [torch.randn(32, 60000, generator=g, device=DEV) * 3 for _ in range(2)]
    u = torch.rand(32, generator=g, device=DEV)
    want = [sample_tokens(x, u, top_p=0.95) for x in logits]
    streams = [torch.cuda.Stream() for _ in logits]
    torch.cuda.synchronize()
    got = [[] for _ in logits]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sample_tokens(logits[i], u, top_p=0.95))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, w in enumerate(want) for x in got[i] for a, b in zip(x, w))


def test_equal_weights_split_the_unit_interval():
    """Of n equal tokens number i is drawn from u = i / n on: exactly, borders included; cuts keep the lowest indices."""
    from gen_worker_amd.sampling import sample_tokens

    n = 64
    logits = torch.full((2 * n, 200), -math.inf, device=DEV)
    logits[:, 3::3][:, :n] = 1.25
    u = torch.arange(2 * n, device=DEV).float() / (2 * n)
    tokens, lp = sample_tokens(logits, u)
    i = torch.arange(2 * n, device=DEV)
    assert torch.equal(tokens, 3 + 3 * (i // 2)) and bool((lp + math.log(n)).abs().max() < 1e-6)
    tokens, _ = sample_tokens(logits, u, top_k=32)
    assert torch.equal(tokens, 3 + 3 * (i // 4))
    tokens, _ = sample_tokens(logits, u, top_p=0.25)
    assert torch.equal(tokens, 3 + 3 * (i // 8))
    tokens, _ = sample_tokens(logits, u, top_p=0.25, top_k=32)
    assert torch.equal(tokens, 3 + 3 * (i // 16))
    tokens, _ = sample_tokens(logits, torch.tensor([1.0, 2.0, -1.0, math.nan], device=DEV)[i[:4]].repeat(n // 2))
    assert tokens[:4].tolist() == [3 + 3 * (n - 1)] * 2 + [3, 3]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masked_rows(dtype):
    """-inf, the type's lowest value, NaN and +inf among the logits; rows of nothing but them."""
    low = torch.finfo(dtype).min
    g = _gen(3)
    logits = torch.randn(16, 1001, generator=g, device=DEV).to(dtype)
    logits[0, 1:] = -math.inf
    logits[1] = -math.inf
    logits[2] = math.nan
    logits[3, 5:] = math.nan
    logits[4, :900] = low
    logits[5] = low
    logits[6, 3:] = -math.inf
    logits[7, 100] = logits[7, 300] = math.inf
    logits[8] = math.inf
    logits[9] = torch.finfo(dtype).max
    logits[10, ::2] = low
    logits[11, ::2] = -math.inf
    logits[12, 1::2] = math.nan
    logits[13, :] = -math.inf
    logits[13, 1000] = math.nan
    logits[14, :] = -math.inf
    logits[14, 1000] = low
    logits[15, 0] = torch.finfo(dtype).max
    for s in SETTINGS + [dict(top_k=500), dict(top_k=950, top_p=0.99)]:
        tokens = check(logits, torch.rand(16, generator=g, device=DEV), **s)
        assert tokens[[1, 2, 13]].tolist() == [-1, -1, -1] and int(tokens[14]) == 1000


def test_settings_of_each_row():
    """Per-row settings in every combination, those out of range among them, equal each row's own call."""
    from gen_worker_amd.sampling import sample_tokens

    g = _gen(8)
    ts = [0.0, -1.0, math.nan, 0.3, 1.0, 1e30]
    ks = [0, -5, 1, 40, 10 ** 9]
    ps = [1.0, 0.0, 0.6, 0.95, 7.0, math.nan, -1.0]
    ms = [0.0, 0.05, 1.0, 3.0, math.nan]
    combos = [(t, k, p, m) for t in ts for k in ks for p in ps for m in ms]
    n = len(combos)
    logits = (torch.randn(n, 700, generator=g, device=DEV) * 2).to(BF16)
    u = torch.rand(n, generator=g, device=DEV)
    t, p, m = (torch.tensor([c[i] for c in combos], device=DEV) for i in (0, 2, 3))
    k = torch.tensor([c[1] for c in combos], device=DEV, dtype=torch.int32)
    got = sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    held = lambda x: torch.nan_to_num(x, nan=0.0).clamp(0.0, 1.0)  # noqa: E731
    check(logits, u, temperature=torch.nan_to_num(t, nan=0.0).clamp(min=0.0), top_k=k.clamp(min=0), top_p=held(p),
          min_p=held(m))
    again = sample_tokens(logits, u, temperature=torch.nan_to_num(t, nan=0.0).clamp(min=0.0), top_k=k.clamp(min=0),
                          top_p=held(p), min_p=held(m))
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    for i in range(0, n, 37):
        if ts[0] <= combos[i][0] <= 1.0 and combos[i][1] >= 0 and 0 <= combos[i][2] <= 1 and 0 <= combos[i][3] <= 1:
            one = sample_tokens(logits[i:i + 1], u[i:i + 1], temperature=combos[i][0], top_k=min(combos[i][1], 2 ** 31 - 1),
                                top_p=combos[i][2], min_p=combos[i][3])
            assert torch.equal(one[0], got[0][i:i + 1]) and torch.equal(one[1], got[1][i:i + 1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_alignment(dtype):
    """Rows of a wider tensor from any element on, an expanded row, a transposed tensor: the contiguous result."""
    from gen_worker_amd.sampling import sample_tokens

    g = _gen(4)
    wide = (torch.randn(5, 3000, generator=g, device=DEV) * 2).to(dtype)
    u = torch.rand(5, generator=g, device=DEV)
    for first in range(9):
        for size in (1, 6, 1000 - first, 2001):
            x = wide[:, first:first + size]
            for s in (dict(top_k=5, top_p=0.9), dict(top_p=0.8), dict()):
                a, b = sample_tokens(x, u, **s), sample_tokens(x.contiguous(), u, **s)
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    row = wide[:1].expand(5, -1)
    for x in (row, wide.t().contiguous().t()):
        a, b = sample_tokens(x, u, top_p=0.9), sample_tokens(x.contiguous(), u, top_p=0.9)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_draws_follow_the_weights():
    """Many evenly spaced random numbers: every kept token as often as its share, to one draw."""
    from gen_worker_amd.sampling import sample_tokens

    n = 4096
    x = torch.randn(1, 40, generator=_gen(6), device=DEV) * 1.5
    u = (torch.arange(n, device=DEV).float() + 0.5) / n
    tokens, lp = sample_tokens(x.expand(n, -1), u, temperature=0.9, top_k=12, min_p=0.02)
    z = x[0].double() / float(np.float32(0.9))
    w = torch.exp(z - z.max())
    keep = (torch.argsort(torch.argsort(-w)) < 12) & (w >= float(np.float32(0.02)))
    share = torch.where(keep, w, 0.0) / torch.where(keep, w, 0.0).sum()
    assert bool(((torch.bincount(tokens, minlength=40).double() - n * share).abs() <= 1.0).all())
    assert bool((lp.double() - torch.log(share[tokens])).abs().max() < 1e-6)


@pytest.mark.parametrize("vocab", [700, 20011])
def test_fewer_drawable_tokens_than_top_k(vocab):
    """A mask that leaves a few tokens (of 64, of 200, of 3000), under a larger top_k: its cut drops none of them."""
    g = _gen(vocab)
    logits = torch.full((6, vocab), -math.inf, device=DEV)
    for r, n in enumerate((1, 3, 64, 200, 500, 3000)):
        at = torch.randperm(vocab, generator=g, device=DEV)[:n]
        logits[r, at] = torch.randn(len(at), generator=g, device=DEV) * 2
    logits[3, logits[3] == -math.inf] = torch.finfo(F32).min
    for k in (1, 70, 250, 1500):
        for s in (dict(), dict(top_p=0.8), dict(min_p=0.2)):
            check(logits, torch.rand(6, generator=g, device=DEV), top_k=k, **s)


@pytest.mark.parametrize("min_p", [2.0 ** -30, 2.0 ** -28, 2.0 ** -27, 1e-7, 2.0 ** -10])
def test_least_min_p(min_p):
    """Weights down to nothing on either side of a tiny min_p; below 2^-28 all are kept."""
    from gen_worker_amd.sampling import sample_tokens

    x = -torch.arange(20000, device=DEV).float()[None] * (32.0 / 20000)
    u = torch.tensor([1.0], device=DEV)
    token, _ = sample_tokens(x, u, min_p=min_p)
    # of all, those of weight 2^-46 or more are drawn: the others' integers of 2^-45 are 0 (31.88 units below the largest)
    least = min_p if min_p >= 2.0 ** -28 else 2.0 ** -46
    want = int((torch.exp(x.double()) >= least).sum()) - 1
    # the last kept token, to the one whose weight is on the border to fp32 rounding of its logit
    assert abs(int(token) - want) <= 1


def test_another_stream_and_a_graph():
    """Captured once, replayed on new logits, numbers and settings, with eager work between."""
    from gen_worker_amd.sampling import sample_tokens

    g = _gen(7)
    logits, u = torch.empty(6, 30011, device=DEV), torch.empty(6, device=DEV)
    t = torch.empty(6, device=DEV)

    def new():
        logits.copy_(torch.randn(6, 30011, generator=g, device=DEV) * 3)
        u.copy_(torch.rand(6, generator=g, device=DEV))
        t.copy_(torch.rand(6, generator=g, device=DEV) + 0.2)

    def draw():
        return sample_tokens(logits, u, temperature=t, top_k=40, top_p=0.9) + sample_tokens(logits, u, top_p=0.97)

    new()
    want = draw()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = draw()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        got = draw()
    torch.cuda.synchronize()
    for _ in range(4):
        new()
        want = draw()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ways_of_calling_agree(monkeypatch):
    """The native host call, the Python body and the registered op: the same bits, and refusals by either."""
    from gen_worker_amd import ops
    from gen_worker_amd.sampling import SamplingError, sample_tokens

    g = _gen(9)
    x, u = torch.randn(4, 3001, generator=g, device=DEV), torch.rand(4, generator=g, device=DEV)
    t = torch.rand(4, generator=g, device=DEV)
    assert ops._host is not None
    a = sample_tokens(x, u, temperature=t, top_k=9, top_p=0.9, min_p=0.01)
    op = torch.ops.cozy_gen_worker.sample_tokens
    b = op(x, u, t, None, None, None, 1.0, 9, 0.9, 0.01)
    torch.library.opcheck(op, (x, u, t, None, None, None, 1.0, 9, 0.9, 0.01), test_utils=("test_schema", "test_faketensor"))

    def refused():
        for bad in (lambda: sample_tokens(x.double(), u), lambda: sample_tokens(x[0], u), lambda: sample_tokens(x, u[:3]),
                    lambda: sample_tokens(x, u.double()), lambda: sample_tokens(x, u, temperature=t.double()),
                    lambda: sample_tokens(x, u, top_k=t), lambda: sample_tokens(x, u, top_p=t[:2]),
                    lambda: sample_tokens(x[:, :0], u), lambda: sample_tokens(x, u.cpu())):
            with pytest.raises(SamplingError):
                bad()
        assert sample_tokens(x[:0], u[:0])[0].shape == (0,)

    refused()
    monkeypatch.setattr(ops, "_host", None)
    c = sample_tokens(x, u, temperature=t, top_k=9, top_p=0.9, min_p=0.01)
    refused()
    for y in (b, c):
        assert torch.equal(a[0], y[0]) and torch.equal(a[1], y[1])
