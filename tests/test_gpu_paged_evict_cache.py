"""``PagedCache.evict`` over layers that share one bookkeeping, in 16 and in 8 bits: what every layer holds afterwards is what
it held before of the slots that its own weights select, and the next step attends to that."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged import BF16, DEV, F16, _gen
from test_gpu_paged_fp8 import FP8, held

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def slots(cache, seq):
    """(pages, places in them) of the sequence's keys."""
    j = torch.arange(cache.length(seq), device=DEV)
    pages = torch.tensor(cache._seqs[seq][0], device=DEV)
    return pages[j // cache.page_size], j % cache.page_size


def selected(weights, budget, recent):
    """[heads, budget]: the last ``recent`` slots and the ``budget - recent`` of largest weight before them (equal ones: the
    lowest), in slot order. weights: [keys, heads]."""
    n, heads = weights.shape
    out = []
    for h in range(heads):
        old = weights[:n - recent, h].tolist()
        best = sorted(range(len(old)), key=lambda j: (-old[j], j))[:budget - recent]
        out.append(sorted(best) + list(range(n - recent, n)))
    return torch.tensor(out, device=DEV)


@pytest.mark.parametrize("dtype,values", [(BF16, BF16), (F16, F16), (FP8, BF16), (FP8, F16)])
@pytest.mark.parametrize("recent", [0, 8, 64])
def test_every_layer_keeps_its_own_selection(dtype, values, recent):
    from gen_worker_amd.paged import PagedCache

    g, heads, hk, dim, budget = _gen(recent + 1), 6, 2, 64, 64
    cache = PagedCache(64, 16, hk, dim, dtype=dtype, weights=True, device=DEV)
    layers = [cache, cache.twin(), cache.twin().twin()]
    a, b, c = cache.add(), cache.add(), cache.add()
    rows = lambda n, h: torch.randn(n, h, dim, generator=g, device=DEV).to(values)  # noqa: E731
    for seqs, counts in (([a, b, c], [37, 30, 64]), ([a, b], [20, 90]), ([b, a], [1, 1]), ([a, b], [14, 1])):
        batch = cache.extend(seqs, counts)
        for layer in layers:
            q, k, v = rows(batch.tokens, heads), rows(batch.tokens, hk), rows(batch.tokens, hk)
            layer.attend(batch, layer.write(batch, q, k, v))
    seqs = [a, b, c]
    lens = [cache.length(s) for s in seqs]
    assert lens == [72, 122, 64]                     # the last is no longer than the budget
    read = lambda layer: [(x[0].clone(), x[1].clone()) for x in layer.read(seqs)]  # noqa: E731
    before = [read(layer) for layer in layers]
    weights = [[layer.weights[p, :, s].clone() for p, s in (slots(cache, q) for q in seqs)] for layer in layers]
    want = [[selected(w, budget, recent) if len(w) > budget else torch.arange(len(w), device=DEV).expand(hk, -1)
             for w in of_layer] for of_layer in weights]
    free = cache.free_pages
    kept = cache.evict(seqs, budget, recent)
    assert torch.equal(kept.long(), torch.stack(want[0][:2]))
    # (layers select differently: a copy by another layer's selection would show)
    assert recent == budget or not torch.equal(want[0][1], want[1][1])
    assert [cache.length(s) for s in seqs] == [64, 64, 64] and cache.free_pages == free + 5 + 8 - 2 * 4
    pick = lambda x, w: torch.stack([x[w[h], h] for h in range(hk)], 1)  # noqa: E731
    expected = [[(pick(k, w), pick(v, w)) for (k, v), w in zip(of_layer, sel)] for of_layer, sel in zip(before, want)]
    for layer, exp, sel, old in zip(layers, expected, want, weights):
        for s, got, (k, v), w, x in zip(seqs, read(layer), exp, sel, old):
            assert torch.equal(got[0], k) and torch.equal(got[1], v)
            p, place = slots(cache, s)
            assert torch.equal(layer.weights[p, :, place], pick(x[..., None], w)[..., 0])
    # the next step, over the kept rows and its own
    counts = [1, 3, 2]
    batch = cache.extend(seqs, counts)
    for layer, exp in zip(layers, expected):
        q, k, v = rows(batch.tokens, heads), rows(batch.tokens, hk), rows(batch.tokens, hk)
        o, _ = layer.attend(batch, layer.write(batch, q, k, v))
        t = 0
        for n, (ek, ev) in zip(counts, exp):
            new = []
            for x in (k, v):
                if dtype == FP8:
                    code, byte = held(x[t:t + n], values)
                    new.append(code * torch.exp2(byte.double() - 127.0)[..., None])
                else:
                    new.append(x[t:t + n].double())
            kk, vv = torch.cat([ek.double(), new[0]]), torch.cat([ev.double(), new[1]])
            hidden = torch.arange(64 + n, device=DEV) > torch.arange(64, 64 + n, device=DEV)[:, None]
            for h in range(heads):
                z = ((q[t:t + n, h].double() @ kk[:, h // 3].t().contiguous()) / 8.0).masked_fill(hidden, -math.inf)
                ref = torch.softmax(z, -1) @ vv[:, h // 3]
                # p and o each rounded once, |v| < 6
                assert bool(((o[t:t + n, h].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 6.0) + 1e-4).all())
            t += n


def test_a_sequence_left_out_keeps_its_rows():
    """Only the named sequences are cut; the others' rows, scales and weights stay as they are."""
    from gen_worker_amd.paged import PagedCache

    g = _gen(5)
    cache = PagedCache(40, 8, 1, 32, dtype=FP8, weights=True, device=DEV)
    twin = cache.twin()
    a, b = cache.add(), cache.add()
    batch = cache.extend([a, b], [70, 50])
    for layer in (cache, twin):
        x = [torch.randn(120, 1, 32, generator=g, device=DEV).to(BF16) for _ in range(3)]
        layer.attend(batch, layer.write(batch, *x))
    before = [[t.clone() for t in layer.read([b])[0]] for layer in (cache, twin)]
    p, s = slots(cache, b)
    w = [layer.weights[p, :, s].clone() for layer in (cache, twin)]
    cache.evict([a], 16, 4)
    assert cache.length(a) == 16 and cache.length(b) == 50
    for layer, old, x in zip((cache, twin), before, w):
        assert all(torch.equal(m, n) for m, n in zip(layer.read([b])[0], old))
        assert torch.equal(layer.weights[p, :, s], x)
