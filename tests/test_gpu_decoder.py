"""The example decoder (``gen_worker_amd.decoder``): the rotary, write, attention and eviction operators under quantized
and bf16 linears, against the same blocks over plain attention of each whole sequence."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

# bf16 linears, logits of two blocks: each attention output is rounded once more than the plain form's (2^-9 of a value on
# average, less after the sum with the residual), so the logits stay within the linears' own relative gate. Quantized
# linears turn a last-bit difference into a whole code step, so there each layer's attention is checked on its own inputs.
REL = 2e-2


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def _config(**change):
    from gen_worker_amd.decoder import DecoderConfig

    base = dict(vocab=512, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, mlp=1024, rot=32, positions=1024)
    return DecoderConfig(**{**base, **change})


def _plain_logits(model, tokens):
    """The model over one whole sequence, attention in 64 bits."""
    cfg = model.cfg
    x = model.embed[torch.tensor(tokens, device=DEV)]
    n, r = len(tokens), cfg.rot // 2
    cos, sin = model.cos[:n, None].double(), model.sin[:n, None].double()

    def turn(t):
        t = t.double()
        a, b = (t[..., 0:2 * r:2], t[..., 1:2 * r:2]) if cfg.interleaved else (t[..., :r], t[..., r:2 * r])
        u, v = a * cos - b * sin, a * sin + b * cos
        y = torch.stack((u, v), -1).flatten(-2) if cfg.interleaved else torch.cat((u, v), -1)
        return torch.cat((y, t[..., 2 * r:]), -1).to(torch.bfloat16).double()   # the cache holds bf16

    hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
    for block in model.blocks:
        q, k, v = block.heads_of(x)
        q, k, v = turn(q), turn(k).repeat_interleave(cfg.heads // cfg.kv_heads, 1), v.double().repeat_interleave(
            cfg.heads // cfg.kv_heads, 1)
        o = []
        for h in range(cfg.heads):
            z = (q[:, h] @ k[:, h].t().contiguous()) / math.sqrt(cfg.head_dim)
            o.append(torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[:, h])
        x = block.rest(x, torch.stack(o, 1).to(torch.bfloat16))
    from gen_worker_amd.flux_dit import _rms
    return (_rms(x, model.norm) @ model.embed.t()).float()


@pytest.mark.parametrize("kind,interleaved,head_dim", [("bf16", False, 64), ("w4a4", True, 64), ("bf16", True, 128)])
def test_steps_match_the_whole_sequence(kind, interleaved, head_dim, monkeypatch):
    """Ragged prompts in chunks, then single tokens: every layer's attention is the plain one over all the sequence's
    tokens so far, and (bf16 linears) the logits after every call are the whole sequence's."""
    from gen_worker_amd.decoder import PagedDecoder
    from gen_worker_amd.paged import PagedCache, rotary_embed

    steps = []   # of one call, by layer: rotated queries and keys, values, attention
    write, attend = PagedCache.write, PagedCache.attend

    def write_too(self, batch, q, k, v, cos, sin, *, interleaved):
        out = write(self, batch, q, k, v, cos, sin, interleaved=interleaved)
        steps.append([out, rotary_embed(k, cos, sin, batch.positions, interleaved=interleaved), v])
        return out

    def attend_too(self, batch, q, **kw):
        out = attend(self, batch, q, **kw)
        steps[-1].append(out[0])
        return out

    monkeypatch.setattr(PagedCache, "write", write_too)
    monkeypatch.setattr(PagedCache, "attend", attend_too)

    model = PagedDecoder(_config(interleaved=interleaved, head_dim=head_dim, heads=512 // head_dim), kind, seed=3)
    g = torch.Generator().manual_seed(2)
    texts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (90, 41)]
    caches = model.caches(64)
    a, b = caches[0].add(), caches[0].add()
    whole = [_plain_logits(model, t) for t in texts]
    at = [0, 0]
    seen = {}
    for counts in ((50, 3), (17, 30), (1, 1), (1, 1), (21, 6)):
        batch = caches[0].extend([a, b], counts)
        new = [t[i:i + n] for t, i, n in zip(texts, at, counts)]
        got = model(torch.tensor(new[0] + new[1], device=DEV), batch, caches)
        at = [i + n for i, n in zip(at, counts)]
        for layer, (q, k, v, o) in enumerate(steps):
            row = 0
            for s, n in enumerate(counts):
                rows = slice(row, row + n)
                row += n
                ks, vs = seen.setdefault((layer, s), ([], []))
                ks.append(k[rows]), vs.append(v[rows])
                kk, vv = torch.cat(ks).double(), torch.cat(vs).double()
                group = q.shape[1] // kk.shape[1]
                hidden = torch.arange(at[s], device=DEV) > torch.arange(at[s] - n, at[s], device=DEV)[:, None]
                for h in range(q.shape[1]):
                    z = (q[rows, h].double() @ kk[:, h // group].t().contiguous()) * head_dim ** -0.5
                    p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
                    ref, spread = p @ vv[:, h // group], p @ vv[:, h // group].abs()
                    # p and o each rounded once, scores of a few units off by a few 2^-24 of their terms
                    assert bool(((o[rows, h].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + spread) + 1e-4 * spread).all())
        steps.clear()
        for s in (0, 1) if kind == "bf16" else ():
            want = whole[s][at[s] - 1]
            rel = float((got[s] - want).norm() / want.norm())
            assert rel <= REL, (counts, s, rel)


@pytest.mark.parametrize("kind", ["w4a4", "bf16"])
def test_generate(kind):
    """Greedy answers of ragged prompts (bf16: every token is the best one of a plain run, up to near-ties), and answers
    under a budget, whose evictions run on the way."""
    from gen_worker_amd.decoder import PagedDecoder

    model = PagedDecoder(_config(), kind, seed=5)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (100, 1, 33)]
    one = model.generate(prompts, 8)
    assert [len(x) for x in one] == [8, 8, 8]
    for x, p in zip(one, prompts) if kind == "bf16" else ():
        # every token of the answer scores within the logits' tolerance of the best one given the answer so far
        logits = _plain_logits(model, p + x[:-1])[len(p) - 1:]
        for step, token in enumerate(x):
            assert float(logits[step].max() - logits[step][token]) <= 2 * REL * float(logits[step].abs().max())
    cut = model.generate(prompts, 40, budget=48, recent=8, chunk=32)
    assert [len(x) for x in cut] == [40, 40, 40] and all(0 <= t < 512 for x in cut for t in x)


def test_generate_refuses():
    from gen_worker_amd.decoder import PagedDecoder
    from gen_worker_amd.paged import PagedError

    model = PagedDecoder(_config(layers=1), "bf16")
    for prompts, n in (([], 1), ([[1], []], 1), ([[1]], 0), ([[1] * 1020], 8)):
        with pytest.raises(PagedError):
            model.generate(prompts, n)
