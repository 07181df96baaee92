"""The example decoder over caches of 8 bits, and with drawn answers: writing, attention, eviction and sampling together."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_decoder import DEV, _config

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


@pytest.mark.parametrize("kind,head_dim", [("bf16", 64), ("w4a4", 128)])
def test_steps_attend_what_the_cache_holds(kind, head_dim, monkeypatch):
    """Ragged prompts in chunks, then single tokens: every layer's attention is the plain one over what the layer's cache
    gives back for the sequence, and what it gives back lies within a code's rounding of the keys and values written."""
    from gen_worker_amd.decoder import PagedDecoder
    from gen_worker_amd.paged import PagedCache, rotary_embed

    steps = []
    write, attend = PagedCache.write, PagedCache.attend

    def write_too(self, batch, q, k, v, cos, sin, *, interleaved):
        out = write(self, batch, q, k, v, cos, sin, interleaved=interleaved)
        steps.append([self, out, rotary_embed(k, cos, sin, batch.positions, interleaved=interleaved), v])
        return out

    def attend_too(self, batch, q, **kw):
        out = attend(self, batch, q, **kw)
        steps[-1].append(out[0])
        return out

    monkeypatch.setattr(PagedCache, "write", write_too)
    monkeypatch.setattr(PagedCache, "attend", attend_too)
    model = PagedDecoder(_config(head_dim=head_dim, heads=512 // head_dim), kind, seed=3)
    g = torch.Generator().manual_seed(2)
    caches = model.caches(64, dtype=FP8)
    seqs = [caches[0].add(), caches[0].add()]
    for counts in ((50, 3), (17, 30), (1, 1), (1, 1), (21, 6)):
        batch = caches[0].extend(seqs, counts)
        tokens = torch.randint(0, 512, (sum(counts),), generator=g).to(DEV)
        assert bool(model(tokens, batch, caches).isfinite().all())
        for cache, q, k, v, o in steps:
            # the twins follow the first cache's lists
            held = [(x[0].double(), x[1].double()) for x in cache.read(seqs)]
            row = 0
            for (kk, vv), n in zip(held, counts):
                rows, L = slice(row, row + n), kk.shape[0]
                row += n
                for got, x in ((kk[L - n:], k[rows].double()), (vv[L - n:], v[rows].double())):
                    # half a step of a code, 2^-4 of the value, or half the smallest step: 2^-10 of a scale, which is at
                    # most amax / 224; k is compared after one more rounding to bf16 and the rotation's own
                    bound = x.abs() * (2.0 ** -4 + 2.0 ** -7) + x.abs().amax(-1, keepdim=True) * (2.0 ** -10 / 224 + 2.0 ** -14)
                    assert bool(((got - x).abs() <= bound).all())
                group = q.shape[1] // kk.shape[1]
                hidden = torch.arange(L, device=DEV) > torch.arange(L - n, L, device=DEV)[:, None]
                for h in range(q.shape[1]):
                    z = (q[rows, h].double() @ kk[:, h // group].t().contiguous()) * head_dim ** -0.5
                    p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
                    ref, spread = p @ vv[:, h // group], p @ vv[:, h // group].abs()
                    # p and o each rounded once, scores of a few units off by a few 2^-24 of their terms
                    assert bool(((o[rows, h].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + spread) + 1e-4 * spread).all())
        steps.clear()


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
def test_drawn_answers(dtype):
    """The same numbers give the same answers, others others; a cut to one token gives the greedy ones, and so does a
    temperature of next to nothing; with a budget the evictions run on the way."""
    from gen_worker_amd.decoder import PagedDecoder

    model = PagedDecoder(_config(), "bf16", seed=5)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (100, 1, 33)]
    greedy = model.generate(prompts, 8, dtype=dtype)
    assert model.generate(prompts, 8, dtype=dtype, temperature=0.9, top_k=1) == greedy
    assert model.generate(prompts, 8, dtype=dtype, temperature=1e-6) == greedy
    drawn = [model.generate(prompts, 20, dtype=dtype, temperature=2.0, top_p=0.95, min_p=0.001, seed=s) for s in (1, 1, 2)]
    assert drawn[0] == drawn[1]
    # (this model's largest logit, that of the token just read, leads by hundreds: only a far higher temperature draws others)
    hot = [model.generate(prompts, 20, dtype=dtype, temperature=300.0, top_p=0.95, seed=s) for s in (1, 1, 2)]
    assert hot[0] == hot[1] != hot[2]
    cut = model.generate(prompts, 40, budget=48, recent=8, chunk=32, dtype=dtype, temperature=1.0, top_k=40)
    assert [len(x) for x in cut] == [40, 40, 40] and all(0 <= t < 512 for x in drawn[0] + hot[2] + cut for t in x)


def test_drawing_refuses():
    from gen_worker_amd.decoder import PagedDecoder
    from gen_worker_amd.paged import PagedError
    from gen_worker_amd.sampling import SamplingError

    model = PagedDecoder(_config(layers=1), "bf16")
    for bad in (dict(temperature=-1.0), dict(temperature=1.0, top_p=1.5), dict(temperature=1.0, top_k=-2), dict(top_k=2.5)):
        with pytest.raises(SamplingError):
            model.generate([[1]], 1, **bad)
    for bad in (dict(temperature=torch.ones(2, device="cuda")), dict(temperature=1.0, top_p=torch.ones(2))):
        with pytest.raises(PagedError, match="numbers"):
            model.generate([[1], [2]], 1, **bad)


def test_the_command_runs(monkeypatch, capsys):
    from gen_worker_amd import decoder

    monkeypatch.setattr("sys.argv", ["decoder", "--prompts", "40,7", "--tokens", "4", "--layers", "1", "--cache", "fp8",
                                     "--temperature", "0.8", "--top-p", "0.9", "--top-k", "50", "--min-p", "0.01",
                                     "--seed", "3"])
    decoder.main()
    assert "2 sequences x 4 tokens" in capsys.readouterr().out
