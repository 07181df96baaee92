"""``sample_tokens`` on the largest vocabularies, whose parts the last launch searches in several turns and whose weights have
fewer bits than 45.

A weight is an integer of 2^-shift (45 up to 2^17 tokens, 62 less the bits of the vocabulary past them), off by half of that at
most, so sums are off by E = vocab 2^-(shift + 1). Tokens are equal where every weight is exact (equal logits); elsewhere the
random number, times the total, lies within 3 E of the drawn token's part of the sum (the total, and the sums on either side)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
SIZES = [600011, 1 << 20, 5000011, 1 << 24]


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def sums_off(vocab):
    bits = (vocab - 1).bit_length()
    return vocab * 2.0 ** -((45 if bits <= 17 else 62 - bits) + 1)


@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_equal_logits(vocab, dtype):
    """Token floor(u m) of the first m that a cut leaves: draws all over every part, cuts in its second turn and on."""
    from gen_worker_amd.sampling import sample_tokens

    rows = 24 if vocab < 1 << 21 else 6
    logits = torch.full((1, vocab), 1.5, dtype=dtype, device=DEV).expand(rows, -1).contiguous()
    u = torch.rand(rows, generator=_gen(vocab), device=DEV)
    u[0], u[-1] = 0.0, 1.0 - 2.0 ** -24

    def check(kept, **cut):
        tokens, lp = sample_tokens(logits, u, **cut)
        assert torch.equal(tokens, (u.double() * kept).floor().long()), cut
        # a logprob is -ln m, off by a rounding of itself
        assert bool(((lp.double() + math.log(kept)).abs() <= 2.0 ** -24 * math.log(kept) + 1e-12).all()), cut

    check(vocab)
    check(vocab, temperature=0.3)
    for k in (1, 4096, 4097, 9001, vocab - 1, vocab // 3):
        check(k, top_k=k)
    for p in (0.75, 0.03125, 0.984375):
        m = math.ceil(p * vocab)
        check(m, top_p=p)
        check(math.ceil(p * 9001), top_k=9001, top_p=p)
        check(m, top_p=p, min_p=0.5)


@pytest.mark.parametrize("vocab", SIZES)
def test_two_values_take_turns(vocab):
    """Every third token of weight 1, the others of weight 1 / 2 (a logit ln 2 below, off by 2^-25 in fp32): ties
    that span turns on either side of a cut."""
    from gen_worker_amd.sampling import sample_tokens

    rows = 8 if vocab < 1 << 21 else 3
    i = torch.arange(vocab, device=DEV)
    high = i % 3 == 1
    logits = torch.where(high, 0.0, -math.log(2.0)).to(F32)[None].expand(rows, -1).contiguous()
    u = torch.rand(rows, generator=_gen(vocab + 1), device=DEV)
    n = int(high.sum())
    for kept, cut in ((n, dict(top_k=n)), (n, dict(min_p=0.75)), (n // 2, dict(top_k=n // 2)), (n, dict(top_p=0.25, top_k=n)),
                      (n + 5001, dict(top_k=n + 5001))):
        if "top_p" in cut:
            kept = math.ceil(0.25 * n)
        tokens, _ = sample_tokens(logits, u, **cut)
        low_kept = max(kept - n, 0)
        high_rank, low_rank = torch.cumsum(high, 0), torch.cumsum(~high, 0)
        w = torch.where(high & (high_rank <= kept), 1.0, torch.where(~high & (low_rank <= low_kept), 0.5, 0.0)).double()
        upto = torch.cumsum(w, 0)
        if low_kept == 0:
            # all kept weights are exact
            want = torch.searchsorted(upto, torch.floor(u.double() * kept), right=True)
            assert torch.equal(tokens, want), cut
        else:
            # each low one's weight is off by 2^-25 of itself, the same for all, and by its rounding
            off = low_kept * 2.0 ** -26 + 3 * sums_off(vocab)
            at = u.double() * upto[-1]
            assert bool((w[tokens] > 0).all())
            assert bool(((upto[tokens] + off >= at) & (upto[tokens] - w[tokens] - off <= at)).all()), cut


@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_random_rows(vocab, dtype):
    """Normal logits, drawn from by random numbers at both ends and between, uncut and cut."""
    from gen_worker_amd.sampling import sample_tokens

    us = [0.0, 1e-6, 0.3, 0.5, 0.8, 1.0 - 2.0 ** -24]
    rows = len(us)
    g = _gen(vocab)
    logits = torch.empty(rows, vocab, dtype=dtype, device=DEV)
    for r in range(rows):
        logits[r] = torch.randn(vocab, generator=g, device=DEV) * (3.0 if r % 2 else 1.0)
    u = torch.tensor(us, device=DEV)
    e = sums_off(vocab)
    for s in (dict(), dict(temperature=0.5), dict(temperature=4.0), dict(top_p=0.75), dict(top_k=40), dict(top_k=3000),
              dict(top_k=20000), dict(min_p=0.0078125), dict(top_k=100000, top_p=0.5)):
        tokens, lps = sample_tokens(logits, u, **s)
        for r in range(rows):
            x = logits[r].double()
            w = torch.exp((x - x.max()) / s.get("temperature", 1.0))
            order = torch.sort(x, descending=True, stable=True).indices
            border = 0.0              # the weight that a cut may leave or drop where sums are off
            if "top_k" in s:
                order = order[:s["top_k"]]
            if "top_p" in s:
                sums = torch.cumsum(w[order], 0)
                m = int((sums < s["top_p"] * sums[-1]).sum()) + 1
                border = float(w[order[m - 1]])
                order = order[:m]
            if "min_p" in s:
                order = order[w[order] >= s["min_p"]]
                border = s["min_p"]
            kept = torch.zeros_like(w)
            kept[order] = w[order]
            upto = torch.cumsum(kept, 0)
            total, t = float(upto[-1]), int(tokens[r])
            # the kept set may differ by tokens at the cut whose weights the sums' error covers, and by one more
            off = 3 * e + (3 * e + border if border else 0.0) + total * 2.0 ** -44
            at = float(u[r]) * total
            assert float(upto[t]) + off >= at and float(upto[t] - kept[t]) - off <= at, (s, r, t)
            assert float(w[t]) > 0 and (border or float(kept[t]) > 0), (s, r, t)
            lp = float(torch.log(w[t] / total))
            # (a total off by d moves its logarithm by at most d / (total - d))
            d = e + (3 * e + border if border else 0.0) + total * 2.0 ** -44
            assert abs(float(lps[r]) - lp) <= 2.0 ** -24 * abs(lp) + d / (total - d), (s, r, t)


def test_the_registered_op_refuses_a_top_k_past_32_bits():
    """As the function does: 2^32 + 1 is not 1."""
    from gen_worker_amd.sampling import SamplingError, sample_tokens

    x, u = torch.randn(2, 50, generator=_gen(1), device=DEV), torch.tensor([0.1, 0.9], device=DEV)
    op = torch.ops.cozy_gen_worker.sample_tokens
    for k in ((1 << 32) + 1, 1 << 31, -1):
        with pytest.raises(SamplingError, match="top_k"):
            op(x, u, None, None, None, None, 1.0, k, 1.0, 0.0)
        with pytest.raises(SamplingError, match="top_k"):
            sample_tokens(x, u, top_k=k)
    got = op(x, u, None, None, None, None, 1.0, (1 << 31) - 1, 1.0, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(got, sample_tokens(x, u)))
