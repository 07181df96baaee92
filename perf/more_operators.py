"""The 8-bit paged cache's and the sampler's speed: keys and values quantised as they are written, read back, attended;
and the next tokens drawn from a step's logits.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, in 64 for the sampler, whose
borders 32 would move) or, with ``own``, through the package. ``exact`` restates each in 64 bits from the definition. The
models behind the sizes are generic decoders (heads of 64 or 128, query heads sharing key/value heads in groups), the
vocabularies this package's own decoder's and generic ones.

The cache holds e4m3 codes and, for every key slot of every kv head, one power of two: value = code * 2^(scale - 127). A
ragged batch's lengths follow from the case alone, so that ``work`` knows them; the seed makes the values.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False  # False: the plain forms; True: the package's operators

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3 = torch.float8_e4m3fn


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "python-gen-worker_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from gen_worker_amd import paged, sampling

    return paged, sampling


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one new token for each of 48 sequences, as every step of token-by-token serving writes it
        {"name": "write8_48_single", "kind": "write8", "batch": 48, "max_q": 1, "max_kv": 1500, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "interleaved": False, "dtype": "bf16"},
        # prompts of several lengths written whole, interleaved pairs on half of each head, two-byte IEEE inputs
        {"name": "write8_prompts_4096", "kind": "write8", "batch": 6, "max_q": 4096, "max_kv": 4096, "heads": 16,
         "kv_heads": 16, "dim": 64, "rot": 32, "page": 64, "interleaved": True, "dtype": "fp16"},
        # a short sequence's keys and values taken out of the pool, for another one
        {"name": "read8_single_700", "kind": "read8", "batch": 1, "max_kv": 700, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16"},
        # several long ones
        {"name": "read8_6x16384", "kind": "read8", "batch": 6, "max_kv": 16384, "kv_heads": 8, "dim": 128, "page": 32,
         "dtype": "bf16"},
        # one sequence, one token, a short cache: what a single interactive user waits for
        {"name": "attn8_single_701", "kind": "attention8", "batch": 1, "max_q": 1, "max_kv": 701, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "weights": False, "dtype": "bf16"},
        # a full server step: one token each for 32 sequences with long caches of very different lengths
        {"name": "attn8_decode_32x32768", "kind": "attention8", "batch": 32, "max_q": 1, "max_kv": 32768, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "weights": False, "dtype": "bf16"},
        # chunks of a few prompts over what is cached of them, heads of 64 that share nothing, odd lengths, one idle,
        # with the weights
        {"name": "attn8_chunk_5x509", "kind": "attention8", "batch": 5, "max_q": 509, "max_kv": 4001, "heads": 16,
         "kv_heads": 16, "dim": 64, "page": 32, "causal": True, "weights": True, "dtype": "fp16"},
        # a long document's chunk, bound by the matrix cores
        {"name": "attn8_chunk_2048_16500", "kind": "attention8", "batch": 1, "max_q": 2048, "max_kv": 16500,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "weights": False, "dtype": "bf16"},
        # this package's own decoder answering one user
        {"name": "sample_1x2048", "kind": "sample", "rows": 1, "vocab": 2048, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "each": False, "dtype": "fp32"},
        # a few users, a larger vocabulary of an odd size, the usual pair of cuts
        {"name": "sample_12x50021", "kind": "sample", "rows": 12, "vocab": 50021, "top_k": 50, "top_p": 0.95,
         "min_p": 0.0, "each": False, "dtype": "fp32"},
        # a server's step, every sequence with settings of its own
        {"name": "sample_64x131072_each", "kind": "sample", "rows": 64, "vocab": 131072, "top_k": 200, "top_p": 0.9,
         "min_p": 0.05, "each": True, "dtype": "bf16"},
        # many answers at once, nothing cut off but the last twentieth of the probability
        {"name": "sample_256x131072", "kind": "sample", "rows": 256, "vocab": 131072, "top_k": 0, "top_p": 0.95,
         "min_p": 0.0, "each": False, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write8", "read8", "attention8", "attention8", "attention8", "sample", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 257, 131072), "top_k": rng.choice([0, 0, 1, 20, 50, 400]),
                "top_p": rng.choice([1.0, 0.5, 0.8, 0.95]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
                "each": rng.random() < 0.4, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    dim, dtype = rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    if kind == "write8":
        q = _log(rng, 1, 4096)
        return {"kind": kind, "batch": rng.randint(1, 6) if q > 64 else rng.randint(1, 64), "max_q": q,
                "max_kv": q + _log(rng, 1, 1500) - 1, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim // 2, dim]), "page": page, "interleaved": rng.random() < 0.5, "dtype": dtype}
    if kind == "read8":
        return {"kind": kind, "batch": rng.randint(1, 6), "max_kv": _log(rng, 1, 16384), "kv_heads": kv_heads,
                "dim": dim, "page": page, "dtype": dtype}
    q = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 8, 1024)])
    kv = q + _log(rng, 1, 32768 if q <= 8 else 8192) - 1
    return {"kind": kind, "batch": rng.randint(1, 32) if q <= 8 else rng.randint(1, 2), "max_q": q, "max_kv": kv,
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "causal": rng.random() < 0.8,
            "weights": rng.random() < 0.3, "dtype": dtype}


def _lengths(case):
    """New tokens and keys (those of the new tokens among them) of each sequence: the first has the most of both, of
    four or more chunked ones the last has nothing new. What is read back is all a sequence holds."""
    rng = random.Random("%s %s %s" % (case["batch"], case.get("max_q", 0), case["max_kv"]))
    n, max_q, max_kv = case["batch"], case.get("max_q", 0), case["max_kv"]
    q = [max_q] + [_log(rng, max(1, max_q // 8), max_q) if max_q else 0 for _ in range(n - 1)]
    if n >= 4 and max_q > 1:
        q[-1] = 0
    kv = [max_kv] + [max(_log(rng, max(1, max_kv // 16), max_kv), x) for x in q[1:]]
    return (list(kv) if case["kind"] == "read8" else q), kv


def _visible(q, kv, causal):
    return sum(kv - q + i + 1 for i in range(q)) if causal else q * kv


def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        # every logit is read, compared, and turned into a weight and a sum
        return {"bytes": n * e + case["rows"] * 16, "flops": 4 * n}
    q, kv = _lengths(case)
    t, g, d = sum(q), case["kv_heads"], case["dim"]
    stored = 2 * g * (d + 1)  # bytes a slot
    if case["kind"] == "write8":
        # the new rows are read, rotated queries and codes written, the codes read back for the values they stand for
        h = case["heads"]
        return {"bytes": t * ((2 * h + 2 * g) * d * e + 2 * stored + 2 * g * d * e) + t * (case["rot"] * 4 + 4),
                "flops": 3 * t * (h + g) * case["rot"] + 4 * t * g * d}
    if case["kind"] == "read8":
        return {"bytes": t * (stored + 2 * g * d * e), "flops": 2 * t * g * d}
    h = case["heads"]
    seen = sum(_visible(a, b, case["causal"]) for a, b in zip(q, kv))
    read = sum(b for a, b in zip(q, kv) if a)
    return {"bytes": read * stored + 2 * t * h * d * e + t * h * 4 + (8 * read * g if case["weights"] else 0),
            "flops": 4 * seen * h * d + 6 * seen * h}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(dtype)


def _table(rot, positions):
    """cos and sin [positions, rot / 2] of the angles position * 10000^(-2 i / rot)."""
    inv = torch.pow(10000.0, -torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _page_table(kv_lens, page, seed):
    """Each sequence's pages, scattered over the pool in an order of the seed; entries past a sequence's own are 0."""
    counts = [-(-n // page) for n in kv_lens]
    order = list(range(sum(counts)))
    random.Random(seed).shuffle(order)
    width, rows, at = max(max(counts), 1), [], 0
    for c in counts:
        rows.append(order[at:at + c] + [0] * (width - c))
        at += c
    return _ints(rows), sum(counts)


def _quantise(x, dtype):
    """fp32 rows [..., d] as e4m3 codes (their bytes) and one scale byte a row: the smallest power of two under which no
    value passes 448, the largest code. A value is not rounded past the type's own range."""
    amax = x.abs().amax(-1, keepdim=True)
    half, exp = torch.frexp(amax)                       # amax = half * 2^exp, half in [1/2, 1): 448 = 0.875 * 2^9
    exp = (exp - 9 + (half > 0.875)).clamp(min=-126)
    most = torch.where(torch.ldexp(torch.full_like(half, 256.0 * 2.0 ** -32), exp + 32 - 128)
                       > torch.finfo(dtype).max * 2.0 ** -128, 240.0, 448.0)
    code = torch.ldexp(x, -exp)
    code = torch.minimum(torch.maximum(code, -most), most).to(E4M3)
    return code.view(torch.uint8), (exp + 127).to(torch.uint8)[..., 0]


def _stored(g, pool, hk, page, d, dtype, common):
    """A pool as prompts leave it: rows with a common part, as trained projections have them (attention is uneven),
    quantised."""
    shape = (max(pool, 1), hk, page, d)
    x = torch.randn(shape, generator=g, device=DEV)
    x.add_(torch.randn((1, hk, 1, d), generator=g, device=DEV).mul_(common))
    codes, scales = _quantise(x, dtype)
    return codes.view(E4M3), scales


def _prepare_sample(case, seed):
    g, n, v = _generator(seed), case["rows"], case["vocab"]
    s = dict(case)
    # a step's logits: most tokens far below a few candidates, how far from row to row
    z = torch.randn((n, v), generator=g, device=DEV)
    z.mul_(torch.rand((n, 1), generator=g, device=DEV).mul_(2.0).add_(1.5))
    z[:, :v // 8] += 3.0
    s["logits"] = z.to(DTYPES[case["dtype"]])
    s["uniform"] = torch.rand(n, generator=g, device=DEV)
    s["temperature"] = 0.8
    if case["each"]:
        # sequences with settings of their own: some greedy, some without a cut
        s["temperature"] = torch.rand(n, generator=g, device=DEV).mul_(1.2).add_(0.3)
        s["temperature"][::7] = 0.0
        s["top_k"] = torch.randint(1, 2 * max(case["top_k"], 1) + 1, (n,), generator=g, device=DEV).int()
        s["top_k"][::3] = 0
        s["top_p"] = torch.rand(n, generator=g, device=DEV).mul_(1 - case["top_p"] / 2).add_(case["top_p"] / 2)
        s["top_p"][::5] = 1.0
        s["min_p"] = torch.rand(n, generator=g, device=DEV).mul_(case["min_p"])
        s["min_p"][::2] = 0.0
    return s


def prepare(case, seed):
    if case["kind"] == "sample":
        return _prepare_sample(case, seed)
    g, dt, d, hk, page = _generator(seed), DTYPES[case["dtype"]], case["dim"], case["kv_heads"], case["page"]
    s = dict(case, dtype=dt)
    q, kv = _lengths(case)
    s["table"], pool = _page_table(kv, page, seed)
    s["kv_len"], s["max_kv"] = _ints(kv), max(kv)
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    s["q_start"], s["max_q"], s["tokens"] = _ints(starts), max(q), starts[-1]
    t = starts[-1]
    if case["kind"] == "write8":
        # what a fused projection leaves: queries, keys and values side by side in one row a token
        hq = case["heads"]
        row = _randn(g, (t, (hq + 2 * hk) * d), dt)
        s["q"] = row[:, :hq * d].view(t, hq, d)
        s["k"] = row[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["v"] = row[:, (hq + hk) * d:].view(t, hk, d)
        s["positions"] = _ints([b - a + i for a, b in zip(q, kv) for i in range(a)])
        s["cos"], s["sin"] = _table(case["rot"], max(kv))
        for name in ("k", "v"):
            s[name + "_pages"] = torch.zeros((max(pool, 1), hk, page, d), dtype=torch.uint8, device=DEV).view(E4M3)
            s[name + "_scales"] = torch.zeros((max(pool, 1), hk, page), dtype=torch.uint8, device=DEV)
        return s
    s["k_pages"], s["k_scales"] = _stored(g, pool, hk, page, d, dt, 0.5)
    s["v_pages"], s["v_scales"] = _stored(g, pool, hk, page, d, dt, 0.0)
    if case["kind"] == "attention8":
        s["q"] = _randn(g, (t, case["heads"], d), dt, 1.5)
        s["scale"] = 1.0 / math.sqrt(d)
        s["w_pages"] = torch.rand((max(pool, 1), hk, page), generator=g, device=DEV) if case["weights"] else None
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 bits, its first 2 * cos.shape[-1] channels rotated."""
    half = cos.shape[-1]
    head, tail = x[..., :2 * half], x[..., 2 * half:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((turned, tail), dim=-1)


def _token_places(s):
    """Each new token's sequence, its index among the sequence's new ones, its key's page and its place there."""
    start = s["q_start"].long()
    t = torch.arange(s["tokens"], device=DEV)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    i = t - start[b]
    slot = s["kv_len"].long()[b] - (start[1:] - start[:-1])[b] + i
    return b, i, s["table"].long()[b, slot // s["page"]], slot % s["page"]


def _values(codes, scales):
    """fp32 of e4m3 codes under their rows' scale bytes."""
    return torch.ldexp(codes.float(), scales.int()[..., None] - 127)


def _plain_read(s):
    _, _, page, at = _token_places(s)
    out = {}
    for x in ("k", "v"):
        codes = s[x + "_pages"].view(torch.uint8)[page, :, at].view(E4M3)
        out[x] = _values(codes, s[x + "_scales"][page, :, at]).to(s["dtype"])
    return out


def _plain_write(s):
    row = s["positions"].long()
    cos, sin = s["cos"][row][:, None], s["sin"][row][:, None]
    q = _rotate(s["q"].float(), cos, sin, s["interleaved"]).to(s["dtype"])
    k = _rotate(s["k"].float(), cos, sin, s["interleaved"])
    _, _, page, at = _token_places(s)
    for name, x in (("k", k), ("v", s["v"].float())):
        codes, scales = _quantise(x, s["dtype"])
        s[name + "_pages"].view(torch.uint8)[page, :, at] = codes
        s[name + "_scales"][page, :, at] = scales
    return {"q": q, **_plain_read(s)}


def _gathered(s, name, table):
    """[B, H, max_kv, D] in 32 bits."""
    x = _values(s[name + "_pages"].view(torch.uint8)[table].view(E4M3), s[name + "_scales"][table]).transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :s["max_kv"]]


def _plain_attention(s):
    table, kv_len, start = s["table"].long(), s["kv_len"].long(), s["q_start"].long()
    length, max_q, hk, d = s["max_kv"], s["max_q"], s["kv_heads"], s["dim"]
    group, batch = s["heads"] // hk, table.shape[0]
    n = start[1:] - start[:-1]
    i = torch.arange(max_q, device=DEV)
    j = torch.arange(length, device=DEV)
    tok = (start[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][tok].view(batch, max_q, hk, group, d).transpose(1, 2).reshape(batch, hk, max_q * group, d).float()
    p = torch.matmul(q, _gathered(s, "k", table).transpose(-1, -2)).mul_(s["scale"])
    last = (kv_len - n)[:, None] + i if s["causal"] else (kv_len - 1)[:, None].expand(batch, max_q)
    last = torch.where(i < n[:, None], torch.minimum(last, kv_len[:, None] - 1), -1)
    hidden = j > last[..., None]
    p.view(batch, hk, max_q, group, length).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    o = torch.matmul(p, _gathered(s, "v", table)) / torch.where(total == 0, 1.0, total)
    b, index, _, _ = _token_places(s)

    def rows(x):
        x = x.view(batch, hk, max_q, group, -1).transpose(1, 2)
        return x[b, index].reshape(s["tokens"], s["heads"], -1)

    out = {"o": rows(o).to(s["dtype"]), "lse": rows(lse)[..., 0].contiguous()}
    if s["w_pages"] is not None:
        share = p.div_(torch.where(total == 0, 1.0, total)).sum(2)
        page = table[:, j // s["page"]]
        at = (page[:, None] * hk + torch.arange(hk, device=DEV)[:, None]) * s["page"] + j % s["page"]
        # a sequence's entries past its end add 0, wherever they point
        s["w_pages"].view(-1).index_add_(0, at.reshape(-1), share.reshape(-1))
        out["weights"] = s["w_pages"]
    return out


def _column(x, dtype):
    """A setting, of all rows or of each, as a column of the type."""
    if isinstance(x, torch.Tensor):
        return x[:, None].to(dtype)
    return torch.full((1, 1), x, dtype=torch.float32 if dtype == torch.float64 else dtype, device=DEV).to(dtype)


def _plain_sample(s):
    """Sorted, cut, put back in the vocabulary's order, drawn by the sum of the weights up to each."""
    z, n = s["logits"].double(), s["vocab"]
    t, p = _column(s["temperature"], torch.float64), _column(s["top_p"], torch.float64)
    k, low = _column(s["top_k"], torch.int64), _column(s["min_p"], torch.float64)
    ordered, index = torch.sort(z, dim=-1, descending=True, stable=True)
    w = torch.exp((ordered - ordered[:, :1]) / torch.where(t > 0, t, 1.0))
    place = torch.arange(n, device=DEV)
    keep = (place < torch.where(k > 0, k, n)) & (place < torch.where(t > 0, n, 1))
    w = torch.where(keep, w, 0.0)
    upto = torch.cumsum(w, -1)
    # the shortest run of the most probable that reaches p of the sum: what lies before a kept one does not
    keep = keep & (((upto - w) < p * upto[:, -1:]) | (p >= 1) | (place < 1))
    keep = keep & ((w >= low) | (place < 1))
    w = torch.zeros_like(w).scatter_(-1, index, torch.where(keep, w, 0.0))
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    token = (upto > s["uniform"].double()[:, None] * total).to(torch.uint8).argmax(-1)
    logprob = torch.log(w.gather(-1, token[:, None]) / total)[:, 0]
    return {"token": token, "logprob": logprob.float()}


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------

def _own_read(s):
    paged, _ = _package()
    k, v = paged.paged_read_fp8(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["q_start"],
                                s["kv_len"], s["tokens"], dtype=s["dtype"])
    return {"k": k, "v": v}


def _own_write(s):
    paged, _ = _package()
    q = paged.paged_write_fp8(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["k_pages"], s["v_pages"],
                              s["k_scales"], s["v_scales"], s["table"], s["q_start"], s["kv_len"],
                              interleaved=s["interleaved"])
    return {"q": q, **_own_read(s)}


def _own_attention(s):
    paged, _ = _package()
    o, lse = paged.paged_attention_fp8(s["q"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"],
                                       s["q_start"], s["kv_len"], s["max_q"], s["max_kv"], scale=s["scale"],
                                       causal=s["causal"], weights=s["w_pages"])
    out = {"o": o, "lse": lse}
    if s["w_pages"] is not None:
        out["weights"] = s["w_pages"]
    return out


def _own_sample(s):
    _, sampling = _package()
    token, logprob = sampling.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                            top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


_PLAIN = {"write8": _plain_write, "read8": _plain_read, "attention8": _plain_attention, "sample": _plain_sample}
_OWN = {"write8": _own_write, "read8": _own_read, "attention8": _own_attention, "sample": _own_sample}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turned(x, positions, rot, interleaved):
    """Each pair as a complex number times e^(i angle)."""
    freq = torch.exp(-math.log(10000.0) * 2.0 * torch.arange(rot // 2, device=DEV, dtype=torch.float64) / rot)
    angles = positions.double()[:, None] * freq
    x = x.double()
    pairs = x[..., :rot].unflatten(-1, (-1, 2)) if interleaved else x[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angles), angles)[:, None]
    pairs = torch.view_as_real(z)
    turned = pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _exact_held(x, dtype):
    """What rows in 64 bits are held as: the scale's exponent e from 448 * 2^e >= amax, every value rounded to the
    nearest multiple of its binade's eighth (2^-9 at least), ties to the even one, within the type's range."""
    e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448.0)).clamp(min=-126.0)
    unit = torch.exp2(e)
    y = x / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    most = torch.where(256.0 * unit > torch.finfo(dtype).max, 240.0, 448.0)
    return torch.minimum(torch.maximum(torch.round(y / step) * step, -most), most) * unit


def _exact_value(codes, scales):
    """Code bytes by their fields: sign, four bits of exponent, three of fraction."""
    c = codes.view(torch.uint8).long()
    sign, exp, frac = 1.0 - 2.0 * (c >> 7).double(), (c >> 3) & 15, (c & 7).double()
    x = torch.where(exp > 0, (1.0 + frac / 8.0) * torch.exp2(exp.double() - 7.0), frac * 2.0 ** -9)
    return sign * x * torch.exp2(scales.double() - 127.0)[..., None]


def _exact_sample(case, s):
    tokens, logprobs = [], []
    for r in range(case["rows"]):
        def of(x):
            return float(x[r]) if isinstance(x, torch.Tensor) else float(torch.tensor(x, dtype=torch.float32))

        z, t = s["logits"][r].double(), of(s["temperature"])
        if t == 0:
            tokens.append(int((z == z.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        w = torch.exp(z / t - z.max() / t)
        order = torch.argsort(w, descending=True, stable=True)
        if of(s["top_k"]) > 0:
            order = order[:int(of(s["top_k"]))]
        ranked = w[order]
        if of(s["top_p"]) < 1:
            upto = torch.cumsum(ranked, 0)
            order = order[:int((upto < of(s["top_p"]) * upto[-1]).sum()) + 1]
        order = torch.cat((order[:1], order[1:][w[order[1:]] >= of(s["min_p"])]))
        kept = torch.sort(order).values
        upto = torch.cumsum(w[kept], 0)
        at = kept[min(int((upto <= float(s["uniform"][r]) * upto[-1]).sum()), len(kept) - 1)]
        tokens.append(int(at))
        logprobs.append(float(torch.log(w[at] / upto[-1])))
    return {"token": torch.tensor(tokens), "logprob": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(case, s)
    if case["kind"] == "write8":
        turn = (s["positions"], case["rot"], case["interleaved"])
        return {"q": _exact_turned(s["q"], *turn), "k": _exact_held(_exact_turned(s["k"], *turn), s["dtype"]),
                "v": _exact_held(s["v"].double(), s["dtype"])}
    places = []  # per sequence: its first new token, how many, its keys' pages and slots
    starts = s["q_start"].tolist()
    for b, n in enumerate(s["kv_len"].tolist()):
        j = torch.arange(n, device=DEV)
        places.append((starts[b], starts[b + 1] - starts[b], s["table"][b].long()[j // case["page"]], j % case["page"]))
    if case["kind"] == "read8":
        return {x: torch.cat([_exact_value(s[x + "_pages"].view(torch.uint8)[page, :, slot], s[x + "_scales"][page, :, slot])
                              for _, _, page, slot in places]) for x in ("k", "v")}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    g = h // hk
    o = torch.zeros(s["tokens"], h, d, dtype=torch.float64, device=DEV)
    lse = torch.full((s["tokens"], h), -math.inf, dtype=torch.float64, device=DEV)
    w = s["w_pages"].double() if case["weights"] else None
    for t0, n, page, slot in places:
        if not n:
            continue
        length = len(page)
        seen = torch.arange(length, device=DEV) <= (
            torch.arange(length - n, length, device=DEV)[:, None] if case["causal"] else length)
        for y in range(hk):
            k, v = (_exact_value(s[x + "_pages"].view(torch.uint8)[page, y, slot], s[x + "_scales"][page, y, slot])
                    for x in ("k", "v"))
            k = k.t().contiguous()
            for x in range(y * g, (y + 1) * g):
                z = s["q"][t0:t0 + n, x].double() @ k
                z = torch.where(seen, z / math.sqrt(d), -math.inf)
                lse[t0:t0 + n, x] = torch.logsumexp(z, -1)
                z = torch.softmax(z, -1)
                o[t0:t0 + n, x] = z @ v
                if w is not None:
                    w[page, y, slot] += z.sum(0)
    out = {"o": o, "lse": lse}
    if w is not None:
        out["weights"] = w
    return out
