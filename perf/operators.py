"""The paged-cache operators' speed: rotary positions, the write into a paged key/value cache, attention over it, and
eviction from it.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, with ``own``, through
the package. ``exact`` restates each in 64 bits from the definition. The models behind the sizes are generic
decoders (heads of 64 or 128, query heads sharing key/value heads in groups) and this package's denoiser blocks
(24 heads of 128); lengths go from one new token to prompts of thousands, caches to tens of thousands of keys.

A ragged batch's lengths follow from the case alone, so that ``work`` knows them; the seed makes the values.
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


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "python-gen-worker_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from gen_worker_amd import paged

    return paged


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the queries of one token of one sequence: the smallest call, all latency
        {"name": "rotary_one_token", "kind": "rotary", "tokens": 1, "heads": 32, "dim": 128, "rot": 128,
         "interleaved": False, "grad": False, "dtype": "bf16"},
        # a training pass over the queries of a batch of images, interleaved pairs on half of each head, forward and
        # gradient
        {"name": "rotary_train_16411", "kind": "rotary", "tokens": 16411, "heads": 24, "dim": 128, "rot": 64,
         "interleaved": True, "grad": True, "dtype": "bf16"},
        # one new token for each of 48 sequences, as every step of token-by-token serving writes it
        {"name": "write_48_single", "kind": "write", "batch": 48, "max_q": 1, "max_kv": 1500, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "page": 16, "interleaved": False, "dtype": "bf16"},
        # prompts of several lengths written whole, interleaved pairs on half of each head, two-byte IEEE values
        {"name": "write_prompts_4096", "kind": "write", "batch": 6, "max_q": 4096, "max_kv": 4096, "heads": 16,
         "kv_heads": 16, "dim": 64, "rot": 32, "page": 64, "interleaved": True, "dtype": "fp16"},
        # one sequence, one token, a short cache: what a single interactive user waits for
        {"name": "attn_single_701", "kind": "attention", "batch": 1, "max_q": 1, "max_kv": 701, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "weights": False, "dtype": "bf16"},
        # a full server step: one token each for 32 sequences with long caches of very different lengths
        {"name": "attn_decode_32x32768", "kind": "attention", "batch": 32, "max_q": 1, "max_kv": 32768, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "causal": True, "weights": False, "dtype": "bf16"},
        # chunks of a few prompts over what is cached of them, heads of 64 that share nothing, odd lengths, one idle
        {"name": "attn_chunk_5x509", "kind": "attention", "batch": 5, "max_q": 509, "max_kv": 4001, "heads": 16,
         "kv_heads": 16, "dim": 64, "page": 32, "causal": True, "weights": False, "dtype": "fp16"},
        # a long document's chunk: the largest, bound by the matrix cores
        {"name": "attn_chunk_4096_16500", "kind": "attention", "batch": 1, "max_q": 4096, "max_kv": 16500, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "weights": False, "dtype": "bf16"},
        # a server step that also gathers every key's attention weight, for the eviction to come
        {"name": "gather_decode_16x8192", "kind": "attention", "batch": 16, "max_q": 1, "max_kv": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "causal": True, "weights": True, "dtype": "bf16"},
        # prompt chunks that gather weights
        {"name": "gather_chunk_2x1021", "kind": "attention", "batch": 2, "max_q": 1021, "max_kv": 6007, "heads": 24,
         "kv_heads": 4, "dim": 128, "page": 64, "causal": True, "weights": True, "dtype": "bf16"},
        # a few short caches cut back to their budget
        {"name": "evict_4x640", "kind": "evict", "batch": 4, "max_kv": 640, "kv_heads": 8, "dim": 128, "page": 16,
         "budget": 512, "recent": 64, "dtype": "bf16"},
        # long prompts' caches reduced to an eighth
        {"name": "evict_8x32768", "kind": "evict", "batch": 8, "max_kv": 32768, "kv_heads": 8, "dim": 128, "page": 64,
         "budget": 4096, "recent": 256, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "write", "attention", "attention", "attention", "evict"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    if kind == "rotary":
        return {"kind": kind, "tokens": _log(rng, 1, 16411), "heads": rng.choice([1, 8, 20, 24, 32]), "dim": dim,
                "rot": rng.choice([dim // 4, dim // 2, dim]), "interleaved": rng.random() < 0.5,
                "grad": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "write":
        q = _log(rng, 1, 4096)
        return {"kind": kind, "batch": rng.randint(1, 6) if q > 64 else rng.randint(1, 64), "max_q": q,
                "max_kv": q + _log(rng, 1, 1500) - 1, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim // 2, dim]), "page": page, "interleaved": rng.random() < 0.5, "dtype": dtype}
    if kind == "attention":
        q = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 8, 1024)])
        kv = q + _log(rng, 1, 32768 if q <= 8 else 8192) - 1
        return {"kind": kind, "batch": rng.randint(1, 32) if q <= 8 else rng.randint(1, 2), "max_q": q, "max_kv": kv,
                "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page,
                "causal": rng.random() < 0.8, "weights": rng.random() < 0.3, "dtype": dtype}
    kv = _log(rng, 64, 32768)
    budget = max(2, int(kv * rng.uniform(0.05, 0.9)))
    return {"kind": kind, "batch": rng.randint(1, 8), "max_kv": kv, "kv_heads": kv_heads, "dim": dim, "page": page,
            "budget": budget, "recent": rng.randint(0, budget // 2), "dtype": dtype}


def _lengths(case):
    """New tokens and keys (those of the new tokens among them) of each sequence: the first has the most of both, of
    four or more chunked ones the last has nothing new."""
    rng = random.Random("%s %s %s" % (case["batch"], case.get("max_q", 0), case["max_kv"]))
    n, max_q, max_kv = case["batch"], case.get("max_q", 0), case["max_kv"]
    q = [max_q] + [_log(rng, max(1, max_q // 8), max_q) if max_q else 0 for _ in range(n - 1)]
    if n >= 4 and max_q > 1:
        q[-1] = 0
    kv = [max_kv] + [max(_log(rng, max(1, max_kv // 16), max_kv), x) for x in q[1:]]
    return q, kv


def _pages(kv_lens, page):
    return [-(-n // page) for n in kv_lens]


def _visible(q, kv, causal):
    return sum(kv - q + i + 1 for i in range(q)) if causal else q * kv


def work(case):
    e, d = BYTES[case["dtype"]], case["dim"]
    if case["kind"] == "rotary":
        n = case["tokens"] * case["heads"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * d * e) + case["tokens"] * (case["rot"] * 4 + 4),
                "flops": passes * 3 * n * case["rot"]}
    q, kv = _lengths(case)
    if case["kind"] == "write":
        t, h, g = sum(q), case["heads"], case["kv_heads"]
        return {"bytes": 2 * t * (h + 2 * g) * d * e + t * (case["rot"] * 4 + 4), "flops": 3 * t * (h + g) * case["rot"]}
    g = case["kv_heads"]
    if case["kind"] == "attention":
        t, h = sum(q), case["heads"]
        seen = sum(_visible(a, b, case["causal"]) for a, b in zip(q, kv))
        read = sum(b for a, b in zip(q, kv) if a)
        more = case["weights"]
        return {"bytes": 2 * read * g * d * e + 2 * t * h * d * e + t * h * 4 + (8 * read * g if more else 0),
                "flops": 4 * seen * h * d + 6 * seen * h}
    kept = sum(min(n, case["budget"]) for n in kv)
    return {"bytes": sum(kv) * g * 4 + kept * g * (4 * d * e + 4 + 4), "flops": sum(kv) * g}


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


def _page_table(kv_lens, page, seed, first=0):
    """Each sequence's pages, scattered over the pool in an order of the seed; entries past a sequence's own are 0."""
    counts = _pages(kv_lens, page)
    order = list(range(first, first + sum(counts)))
    random.Random(seed).shuffle(order)
    width, rows, at = max(max(counts), 1), [], 0
    for c in counts:
        rows.append(order[at:at + c] + [0] * (width - c))
        at += c
    return _ints(rows), sum(counts)


def prepare(case, seed):
    g = _generator(seed)
    dt, d = DTYPES[case["dtype"]], case["dim"]
    s = dict(case, dtype=dt)
    if case["kind"] == "rotary":
        t, h = case["tokens"], case["heads"]
        s["cos"], s["sin"] = _table(case["rot"], t + 4096)
        s["positions"] = (torch.arange(t, device=DEV) + torch.randint(0, 4096, (1,), generator=g, device=DEV)).int()
        s["x"] = _randn(g, (t, h, d), dt)
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dy"] = _randn(g, (t, h, d), dt)
        return s
    q, kv = _lengths(case)
    hk, page = case["kv_heads"], case["page"]
    s["table"], pool = _page_table(kv, page, seed)
    s["kv_len"] = _ints(kv)
    s["max_kv"] = max(kv)
    if case["kind"] in ("write", "attention"):
        starts = [0]
        for n in q:
            starts.append(starts[-1] + n)
        s["q_start"], s["max_q"], t = _ints(starts), max(q), starts[-1]
        s["tokens"] = t
    shape = (max(pool, 1), hk, page, d)
    if case["kind"] == "write":
        # what a fused projection leaves: queries, keys and values side by side in one row a token
        row = _randn(g, (t, (case["heads"] + 2 * hk) * d), dt)
        hq = case["heads"]
        s["q"] = row[:, :hq * d].view(t, hq, d)
        s["k"] = row[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["v"] = row[:, (hq + hk) * d:].view(t, hk, d)
        s["positions"] = _ints([b - a + i for a, b in zip(q, kv) for i in range(a)])
        s["cos"], s["sin"] = _table(case["rot"], max(kv))
        s["k_pages"], s["v_pages"] = torch.zeros(shape, dtype=dt, device=DEV), torch.zeros(shape, dtype=dt, device=DEV)
        return s
    # keys with a common part, as trained projections have: attention is uneven, some keys draw much of it
    s["k_pages"] = _randn(g, shape, dt, 1.0).add_(_randn(g, (1, hk, 1, d), dt, 0.5))
    s["v_pages"] = _randn(g, shape, dt, 1.0)
    if case["kind"] == "attention":
        s["q"] = _randn(g, (t, case["heads"], d), dt, 1.5)
        s["scale"] = 1.0 / math.sqrt(d)
        if case["weights"]:
            s["w_pages"] = torch.rand((shape[0], hk, page), generator=g, device=DEV)
        else:
            s["w_pages"] = None
        return s
    # gathered weights: a few keys hold most, many hold next to nothing, some (never seen) exactly nothing
    w = torch.exp(2.0 * torch.randn((shape[0], hk, page), generator=g, device=DEV))
    s["w_pages"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.05, torch.zeros_like(w), w)
    kept = [min(n, case["budget"]) for n in kv]
    s["new_table"], new_pool = _page_table(kept, page, seed + 1, first=shape[0])
    # the pool's free pages, which the kept rows go to
    for name in ("k_pages", "v_pages", "w_pages"):
        old = s[name]
        s[name] = torch.cat([old, torch.zeros((new_pool,) + old.shape[1:], dtype=old.dtype, device=DEV)])
    s["old_pool"] = shape[0]
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


def _plain_rotary(s):
    x = s["x"].detach()
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    y = _rotate(x.float(), cos, sin, s["interleaved"]).to(x.dtype)
    if not s["grad"]:
        return {"y": y}
    return {"y": y, "dx": _rotate(s["dy"].float(), cos, -sin, s["interleaved"]).to(x.dtype)}


def _token_places(s):
    """Each new token's sequence, its index among the sequence's new ones, and its key's slot."""
    start = s["q_start"].long()
    t = torch.arange(s["tokens"], device=DEV)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    i = t - start[b]
    n = start[1:] - start[:-1]
    return b, i, s["kv_len"].long()[b] - n[b] + i


def _plain_write(s):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = _rotate(s["q"].float(), cos, sin, s["interleaved"]).to(s["dtype"])
    k = _rotate(s["k"].float(), cos, sin, s["interleaved"]).to(s["dtype"])
    b, _, slot = _token_places(s)
    page = s["table"].long()[b, slot // s["page"]]
    s["k_pages"][page, :, slot % s["page"]] = k
    s["v_pages"][page, :, slot % s["page"]] = s["v"]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _gathered(pages, table, length):
    """[B, H, length, D] in 32 bits."""
    x = pages[table].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :length].float()


def _plain_attention(s):
    table, kv_len, start = s["table"].long(), s["kv_len"].long(), s["q_start"].long()
    length, max_q, hk, d = s["max_kv"], s["max_q"], s["kv_heads"], s["dim"]
    group, batch = s["heads"] // hk, table.shape[0]
    n = start[1:] - start[:-1]
    i = torch.arange(max_q, device=DEV)
    j = torch.arange(length, device=DEV)
    tok = (start[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][tok].view(batch, max_q, hk, group, d).transpose(1, 2).reshape(batch, hk, max_q * group, d).float()
    k = _gathered(s["k_pages"], table, length)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"])
    last = (kv_len - n)[:, None] + i if s["causal"] else (kv_len - 1)[:, None].expand(batch, max_q)
    last = torch.where(i < n[:, None], torch.minimum(last, kv_len[:, None] - 1), -1)
    hidden = j > last[..., None]
    p.view(batch, hk, max_q, group, length).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    o = torch.matmul(p, _gathered(s["v_pages"], table, length)) / torch.where(total == 0, 1.0, total)
    b, index, _ = _token_places(s)

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


def _plain_evict(s):
    table, kv_len, page = s["table"].long(), s["kv_len"].long(), s["page"]
    length, budget, recent, hk = s["max_kv"], s["budget"], s["recent"], s["kv_heads"]
    batch = table.shape[0]
    w = s["w_pages"][table].transpose(1, 2).reshape(batch, hk, -1)[..., :length]
    j = torch.arange(length, device=DEV)
    n = kv_len[:, None]
    rank = torch.where(j >= n - recent, math.inf, w.transpose(0, 1)).transpose(0, 1)
    rank = torch.where((j < n)[:, None], rank, -math.inf)
    if length < budget:
        rank = torch.nn.functional.pad(rank, (0, budget - length), value=-math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    new_len = kv_len.clamp(max=budget)
    past = torch.arange(budget, device=DEV) >= new_len[:, None, None]
    kept = torch.sort(order.masked_fill(past.expand_as(order), length + budget), dim=-1).values
    kept = kept.masked_fill(past, -1)
    i = torch.arange(budget, device=DEV)
    # rows past a sequence's own go where its last kept one does, with its values
    i = torch.minimum(i, (new_len - 1).clamp(min=0)[:, None])
    src = kept.gather(-1, i[:, None].expand_as(kept))
    heads = torch.arange(hk, device=DEV)[:, None]
    from_page = table[torch.arange(batch, device=DEV)[:, None, None], src // page]
    to_page = s["new_table"].long().gather(1, i // page)[:, None]
    to_slot = (i % page)[:, None]
    out = {"kept": kept.int(), "kv_len": new_len.int()}
    s["k_pages"][to_page, heads, to_slot] = s["k_pages"][from_page, heads, src % page]
    s["v_pages"][to_page, heads, to_slot] = s["v_pages"][from_page, heads, src % page]
    s["w_pages"][to_page, heads, to_slot] = s["w_pages"][from_page, heads, src % page]
    out["k_pages"], out["v_pages"], out["weights"] = (s[x][s["old_pool"]:] for x in ("k_pages", "v_pages", "w_pages"))
    return out


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------

def _own_rotary(s, paged):
    y = paged.rotary_embed(s["x"], s["cos"], s["sin"], s["positions"], interleaved=s["interleaved"])
    if not s["grad"]:
        return {"y": y}
    return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def _own_write(s, paged):
    q = paged.paged_write(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["k_pages"], s["v_pages"],
                          s["table"], s["q_start"], s["kv_len"], interleaved=s["interleaved"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attention(s, paged):
    o, lse = paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["q_start"], s["kv_len"],
                                   s["max_q"], s["max_kv"], scale=s["scale"], causal=s["causal"],
                                   weights=s["w_pages"])
    out = {"o": o, "lse": lse}
    if s["w_pages"] is not None:
        out["weights"] = s["w_pages"]
    return out


def _own_evict(s, paged):
    kept, kv_len = paged.paged_evict(s["k_pages"], s["v_pages"], s["w_pages"], s["table"], s["kv_len"], s["max_kv"],
                                     s["new_table"], s["budget"], s["recent"])
    out = {"kept": kept, "kv_len": kv_len}
    out["k_pages"], out["v_pages"], out["weights"] = (s[x][s["old_pool"]:] for x in ("k_pages", "v_pages", "w_pages"))
    return out


_PLAIN = {"rotary": _plain_rotary, "write": _plain_write, "attention": _plain_attention, "evict": _plain_evict}
_OWN = {"rotary": _own_rotary, "write": _own_write, "attention": _own_attention, "evict": _own_evict}


def run(state):
    if own:
        return _OWN[state["kind"]](state, _package())
    return _PLAIN[state["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turned(x, angles, interleaved):
    """Each pair as a complex number times e^(i angle)."""
    r = 2 * angles.shape[1]
    x = x.double()
    pairs = x[..., :r].unflatten(-1, (-1, 2)) if interleaved else x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angles), angles)[:, None]
    pairs = torch.view_as_real(z)
    turned = pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def _exact_angles(positions, rot):
    freq = torch.exp(-math.log(10000.0) * 2.0 * torch.arange(rot // 2, device=DEV, dtype=torch.float64) / rot)
    return positions.double()[:, None] * freq


def _sequences(case, s):
    """Per sequence: its first new token, how many, its keys' count, their pages and slots."""
    starts = s["q_start"].tolist() if "q_start" in s else [0] * (case["batch"] + 1)
    for b, n in enumerate(s["kv_len"].tolist()):
        j = torch.arange(n, device=DEV)
        yield b, starts[b], starts[b + 1] - starts[b], n, s["table"][b].long()[j // case["page"]], j % case["page"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        a = _exact_angles(s["positions"], case["rot"])
        out = {"y": _exact_turned(s["x"].detach(), a, case["interleaved"])}
        if case["grad"]:
            out["dx"] = _exact_turned(s["dy"], -a, case["interleaved"])
        return out
    if case["kind"] == "write":
        a = _exact_angles(s["positions"], case["rot"])
        k = _exact_turned(s["k"], a, case["interleaved"])
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for b, t0, n, length, page, slot in _sequences(case, s):
            page, slot = page[length - n:], slot[length - n:]
            kp[page, :, slot], vp[page, :, slot] = k[t0:t0 + n], s["v"][t0:t0 + n].double()
        return {"q": _exact_turned(s["q"], a, case["interleaved"]), "k_pages": kp, "v_pages": vp}
    if case["kind"] == "attention":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        g = h // hk
        o = torch.zeros(s["tokens"], h, d, dtype=torch.float64, device=DEV)
        lse = torch.full((s["tokens"], h), -math.inf, dtype=torch.float64, device=DEV)
        w = s["w_pages"].double() if case["weights"] else None
        for b, t0, n, length, page, slot in _sequences(case, s):
            if not n:
                continue
            seen = torch.arange(length, device=DEV) <= (
                torch.arange(length - n, length, device=DEV)[:, None] if case["causal"] else length)
            for x in range(h):
                z = s["q"][t0:t0 + n, x].double() @ s["k_pages"][page, x // g, slot].double().t().contiguous()
                z = torch.where(seen, z / math.sqrt(d), -math.inf)
                lse[t0:t0 + n, x] = torch.logsumexp(z, -1)
                z = torch.softmax(z, -1)
                o[t0:t0 + n, x] = z @ s["v_pages"][page, x // g, slot].double()
                if w is not None:
                    w[page, x // g, slot] += z.sum(0)
        out = {"o": o, "lse": lse}
        if w is not None:
            out["weights"] = w
        return out
    budget, old = case["budget"], s["old_pool"]
    kept = torch.full((case["batch"], case["kv_heads"], budget), -1, dtype=torch.int32)
    new = {x: s[x].double() for x in ("k_pages", "v_pages", "w_pages")}
    for b, _, _, length, page, slot in _sequences(case, s):
        m = min(length, budget)
        i = torch.arange(m, device=DEV)
        to_page, to_slot = s["new_table"][b].long()[i // case["page"]], i % case["page"]
        for x in range(case["kv_heads"]):
            w = s["w_pages"][page, x, slot].tolist()
            first = 0 if length <= budget else length - case["recent"]
            best = sorted(range(first), key=lambda j: (-w[j], j))[:budget - case["recent"]]
            ids = torch.tensor(sorted(best) + list(range(first, length)), dtype=torch.long)
            kept[b, x, :m] = ids.int()
            ids = ids.to(DEV)
            for pages in new.values():
                pages[to_page, x, to_slot] = pages[page[ids], x, slot[ids]]
    return {"kept": kept, "kv_len": s["kv_len"].clamp(max=budget), "k_pages": new["k_pages"][old:],
            "v_pages": new["v_pages"][old:], "weights": new["w_pages"][old:]}
