"""Rotary positions and a paged key/value cache: what a decoder on this package's quantized linears needs beside them.

The reference serves denoisers, whose attention sees every token at once; a model that answers token by token keeps
the keys and values of what it has seen. Here they live in a pool of pages (``page_size`` key slots of every kv
head), a sequence in the pages its row of a table lists, and new tokens of several sequences come packed
([tokens, heads, head_dim], sequence b's rows ``q_start[b]`` to ``q_start[b + 1] - 1``). Four operators
(``csrc/paged_cache.hip``, ``csrc/paged_attention.hip``), each a function here and a ``cozy_gen_worker::*`` op:

* ``rotary_embed``: rotary positions, half or interleaved pairs, on all or part of a head; differentiable.
  ``rotary_table`` makes the tables, scaled for long contexts on request.
* ``paged_write``: new tokens' queries and keys rotated, keys and values stored.
* ``paged_attention``: the new tokens' attention over their sequences' keys, one token a sequence or long chunks;
  with ``weights`` it also adds up the attention each key draws.
* ``paged_evict``: the keys that drew least dropped, the others copied to fresh pages.

``PagedCache`` keeps the pool, the page lists and the lengths on the host and calls them. Everything runs on the current
stream; the functions do not synchronise and may be captured in a HIP graph (outputs come from torch's allocator).
The cache's values are bf16 or fp16; scores, softmax statistics, sums and gathered weights are fp32. CPU tensors
are refused: there is no CPU implementation.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Iterator, Optional, Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _native as nat
from . import ops

_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16, torch.float32: nat.DT_F32}


class PagedError(ValueError):
    """An argument the paged-cache operators do not take."""


def _require(ok: bool, name: str, message: str) -> None:
    if not ok:
        raise PagedError(f"{name}: {message}")


def _ints(name: str, what: str, t: Tensor, shape: tuple, device: torch.device) -> None:
    _require(t.dtype == torch.int32 and t.device == device and tuple(t.shape) == shape
             and (t.dim() == 0 or t.numel() == 0 or t.stride(-1) == 1), name,
             f"{what} must be int32 {list(shape)} on {device} with unit last stride, got {t.dtype} {list(t.shape)} "
             f"strides {t.stride()} on {t.device}")


def _heads(name: str, what: str, t: Tensor, dtype: torch.dtype, device: torch.device, tokens: int, heads: int,
           dim: int) -> None:
    _require(t.dtype == dtype and t.device == device and tuple(t.shape) == (tokens, heads, dim)
             and (t.numel() == 0 or t.stride(2) == 1), name,
             f"{what} must be {dtype} {[tokens, heads, dim]} on {device} with unit last stride, got {t.dtype} "
             f"{list(t.shape)} strides {t.stride()} on {t.device}")


def _tables(name: str, cos: Optional[Tensor], sin: Optional[Tensor], positions: Optional[Tensor], tokens: int, dim: int,
            device: torch.device) -> tuple[int, int]:
    """(rotated channels, table rows) of checked tables."""
    _require((cos is None) == (sin is None), name, "cos and sin go together")
    if positions is not None:
        _ints(name, "positions", positions, (tokens,), device)
    if cos is None:
        return 0, 0
    for what, t in (("cos", cos), ("sin", sin)):
        _require(t.dtype == torch.float32 and t.device == device and t.dim() == 2 and t.shape == cos.shape
                 and t.is_contiguous(), name,
                 f"{what} must be a contiguous float32 [positions, rotated / 2] table on {device}, got {t.dtype} "
                 f"{list(t.shape)} on {t.device}")
    rows, half = int(cos.shape[0]), int(cos.shape[1])
    _require(2 * half <= dim, name, f"tables for {2 * half} channels of {dim}")
    _require(rows > 0 or tokens == 0 or half == 0, name, "tables without positions")
    _require(positions is not None or rows >= tokens or half == 0, name,
             f"{tokens} tokens without positions over a table of {rows}")
    return 2 * half, rows


def _spaced(table: Tensor) -> tuple[Tensor, int]:
    """A table of page ids and its row stride as the library takes them. Rows that overlap (``expand``: sequences that read
    the same pages) are copied apart; of a single row the stride is not read."""
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        table = table.contiguous()
    return table, max(table.stride(0), table.shape[1])


def _host():
    """The native host calls, which make these calls in a few microseconds; None while the library is not loaded,
    without them, and under compilation. Theirs return None for whatever the Python way has to decide or refuse."""
    host = ops._host
    return None if host is None or torch.compiler.is_compiling() else host


def _plain(*tensors: Optional[Tensor]) -> bool:
    """Whether a call may skip the dispatcher: plain CUDA tensors in plain eager mode, nothing for autograd to
    record (see ``ops.eager_call_ok``, whose conditions these are for every operand)."""
    if (torch.compiler.is_compiling() or torch._C._is_tracing() or torch._C._is_torch_function_mode_enabled()
            or torch._C._len_torch_dispatch_stack() != 0):
        return False
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (type(t) is not Tensor or (grad and t.requires_grad) or t.is_neg()
                              or torch._C._functorch.is_functorch_wrapped_tensor(t)):
            return False
    return True


def _tangent(t: Optional[Tensor]) -> Optional[Tensor]:
    """The tangent of a dual tensor (forward-mode differentiation), None of any other."""
    return forward_ad.unpack_dual(t).tangent if t is not None and forward_ad._current_level >= 0 else None


def _no_tangents(name: str, *tensors: Optional[Tensor]) -> None:
    if forward_ad._current_level >= 0:   # neither the native calls nor the registered ops would notice
        _require(all(_tangent(t) is None for t in tensors), name, "no gradient is defined for a dual tensor's tangent")


def _written(out, *tensors: Optional[Tensor]):
    """``out`` of a call that wrote into these tensors past the dispatcher: as the registered op does for its
    ``mutates_args``, their version counters are raised, by which autograd knows what changed behind a graph."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])
    return out


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_table(positions: int, rot: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device="cuda") -> tuple[Tensor, Tensor]:
    """fp32 cos and sin [positions, rot / 2] of the angles ``position * f_i``, ``f_i = base^(-2 i / rot)``, for heads
    whose first ``rot`` channels turn; angles are formed in 64 bits. ``scaling`` stretches a model trained on shorter
    contexts by ``factor`` >= 1:

    * ``linear``: f_i / factor (position interpolation);
    * ``ntk``: base * factor^(rot / (rot - 2)), which keeps the fastest pair and stretches the slowest by factor;
    * ``yarn`` (Peng et al., 2023): with r_i = original * f_i / (2 pi) turns over the trained length ``original``,
      pairs of r_i >= beta_fast keep f_i, those of r_i <= beta_slow take f_i / factor, a ramp linear in r_i between;
      cos and sin are multiplied by 0.1 ln(factor) + 1."""
    name = "rotary_table"
    _require(positions > 0 and rot > 0 and rot % 2 == 0, name, f"{positions} positions of {rot} channels")
    _require(scaling in SCALINGS, name, f"scaling {scaling!r} not in {SCALINGS}")
    _require(factor >= 1.0 and base > 1.0, name, f"factor {factor} (at least 1), base {base}")
    _require(scaling != "none" or factor == 1.0, name, "a factor needs a scaling")
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot
    if scaling == "ntk":
        _require(rot > 2, name, "ntk needs more than one pair")
        base = base * factor ** (rot / (rot - 2))
    f = torch.pow(torch.tensor(base, dtype=torch.float64, device=device), -i)
    gain = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        _require(original > 0 and beta_fast > beta_slow, name, f"yarn over an original length of {original}, between "
                 f"{beta_slow} and {beta_fast} turns")
        keep = ((original * f / (2 * math.pi) - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / factor
        gain = 0.1 * math.log(factor) + 1.0
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return (a.cos() * gain).float(), (a.sin() * gain).float()


def _rotary_body(x: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor], interleaved: bool,
                 inverse: bool) -> Tensor:
    name = "rotary_embed"
    _require(x.dim() == 3 and x.dtype in _DTYPES and x.is_cuda, name,
             f"x must be a bf16, fp16 or fp32 CUDA tensor [tokens, heads, head_dim], got {x.dtype} {list(x.shape)} on "
             f"{x.device}")
    _require(cos is not None and sin is not None, name, "cos and sin are needed")
    t, h, d = x.shape
    rot, rows = _tables(name, cos, sin, positions, t, d, x.device)
    _require(d % 2 == 0 and 2 <= d <= 1024, name, f"head_dim {d} (an even number up to 1024)")
    if x.stride(2) != 1:
        x = x.contiguous()
    y = torch.empty((t, h, d), dtype=x.dtype, device=x.device)
    if y.numel():
        nat.call("gwa_rotary_embed", x.data_ptr(), x.stride(0), x.stride(1), cos.data_ptr(), sin.data_ptr(), rows,
                 nat.ptr(positions), y.data_ptr(), h * d, d, t, h, d, rot, int(interleaved), int(inverse),
                 _DTYPES[x.dtype], nat.stream_of(x))
    return y


@torch.library.custom_op("cozy_gen_worker::rotary_embed", mutates_args=())
def _rotary_op(x: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor], interleaved: bool,
               inverse: bool) -> Tensor:
    return _rotary_body(x, cos, sin, positions, interleaved, inverse)


@_rotary_op.register_fake
def _(x, cos, sin, positions, interleaved, inverse):
    return x.new_empty(x.shape)


def _rotary_setup(ctx, inputs, output):
    _require(not any(ctx.needs_input_grad[1:3]), "rotary_embed", "the tables have no gradient")
    _, cos, sin, positions, ctx.interleaved, ctx.inverse = inputs
    ctx.save_for_backward(cos, sin, positions)


def _rotary_backward(ctx, dy):
    # a rotation's transpose is the rotation back
    cos, sin, positions = ctx.saved_tensors
    return _rotary_op(dy, cos, sin, positions, ctx.interleaved, not ctx.inverse), None, None, None, None, None


_rotary_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)


def rotary_embed(x: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor] = None, *,
                 interleaved: bool = False, inverse: bool = False) -> Tensor:
    """x [tokens, heads, head_dim] (bf16, fp16 or fp32; token and head strides free) with the first
    ``2 * cos.shape[1]`` channels of every head rotated by their token's position, the others copied. Pairs are
    (2i, 2i + 1) with ``interleaved``, else (i, i + half). ``positions``: int32 [tokens] rows of the tables (held inside
    them), or None for 0, 1, 2, ... ``inverse`` rotates back. Computed in fp32, rounded once; differentiable in x, in
    reverse and forward mode."""
    _require(not torch.is_grad_enabled() or not (cos is not None and cos.requires_grad or sin is not None
                                                 and sin.requires_grad), "rotary_embed", "the tables have no gradient")
    if forward_ad._current_level >= 0:
        _no_tangents("rotary_embed", cos, sin)
        primal, tangent = forward_ad.unpack_dual(x)
        if tangent is not None:   # the map is linear: a tangent turns as x does
            return forward_ad.make_dual(*(rotary_embed(t, cos, sin, positions, interleaved=interleaved, inverse=inverse)
                                          for t in (primal, tangent)))
    host = _host()
    if host is not None:
        y = host.rotary_embed(x, cos, sin, positions, interleaved, inverse)
        if y is not None:
            return y
    if _plain(x, cos, sin, positions):
        return _rotary_body(x, cos, sin, positions, interleaved, inverse)
    return _rotary_op(x, cos, sin, positions, interleaved, inverse)


# ---------------------------------------------------------------------------
# the cache operators
# ---------------------------------------------------------------------------

def _cache_args(name: str, k_pages: Tensor, v_pages: Tensor, weights: Optional[Tensor], table: Tensor,
                q_start: Optional[Tensor], kv_len: Tensor) -> nat.PagedCacheArgs:
    dev = k_pages.device
    _require(k_pages.is_cuda and k_pages.dtype in (torch.bfloat16, torch.float16) and k_pages.dim() == 4
             and k_pages.stride(3) == 1, name,
             f"k_pages must be a bf16 or fp16 CUDA tensor [pages, kv_heads, page_size, head_dim] with unit last stride, "
             f"got {k_pages.dtype} {list(k_pages.shape)} strides {k_pages.stride()} on {k_pages.device}")
    _require(v_pages.dtype == k_pages.dtype and v_pages.device == dev and v_pages.shape == k_pages.shape
             and v_pages.stride() == k_pages.stride(), name,
             f"v_pages must have k_pages' type, shape and strides, got {v_pages.dtype} {list(v_pages.shape)} strides "
             f"{v_pages.stride()} on {v_pages.device}")
    pages, heads, size, dim = k_pages.shape
    batch = kv_len.shape[0] if kv_len.dim() == 1 else -1
    _ints(name, "kv_len", kv_len, (batch,), dev)
    _ints(name, "table", table, (batch, table.shape[-1] if table.dim() == 2 else -1), dev)
    if q_start is not None:
        _ints(name, "q_start", q_start, (batch + 1,), dev)
    ws = (0, 0)
    if weights is not None:
        _require(weights.dtype == torch.float32 and weights.device == dev and tuple(weights.shape) == (pages, heads, size)
                 and (size == 1 or weights.stride(2) == 1), name,
                 f"weights must be float32 {[pages, heads, size]} on {dev} with unit last stride, got {weights.dtype} "
                 f"{list(weights.shape)} strides {weights.stride()} on {weights.device}")
        ws = weights.stride()
    table, row = _spaced(table)
    args = nat.PagedCacheArgs(k_pages.data_ptr(), v_pages.data_ptr(), nat.ptr(weights), table.data_ptr(),
                              nat.ptr(q_start), kv_len.data_ptr(), k_pages.stride(0), k_pages.stride(1),
                              k_pages.stride(2), ws[0], ws[1], pages, row, table.shape[1], batch, size, heads, dim,
                              _DTYPES[k_pages.dtype])
    args.table_kept = table  # a copy lives until the call has been made
    return args


def _write_body(q: Tensor, k: Tensor, v: Tensor, cos: Optional[Tensor], sin: Optional[Tensor],
                positions: Optional[Tensor], k_pages: Tensor, v_pages: Tensor, table: Tensor, q_start: Tensor,
                kv_len: Tensor, weights: Optional[Tensor], interleaved: bool) -> Tensor:
    name = "paged_write"
    args = _cache_args(name, k_pages, v_pages, weights, table, q_start, kv_len)
    dev, dt, d = k_pages.device, k_pages.dtype, args.head_dim
    _require(q.dim() == 3, name, f"q must be [tokens, heads, {d}], got {list(q.shape)}")
    t, h = int(q.shape[0]), int(q.shape[1])
    _heads(name, "q", q, dt, dev, t, h, d)
    _heads(name, "k", k, dt, dev, t, args.kv_heads, d)
    _heads(name, "v", v, dt, dev, t, args.kv_heads, d)
    rot, rows = _tables(name, cos, sin, positions, t, d, dev)
    out = torch.empty((t, h, d), dtype=dt, device=dev)
    nat.call("gwa_paged_write", ctypes.byref(args), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
             k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), nat.ptr(cos), nat.ptr(sin), rows, nat.ptr(positions),
             out.data_ptr(), t, h, rot, int(interleaved), nat.stream_of(k_pages))
    return out


@torch.library.custom_op("cozy_gen_worker::paged_write", mutates_args=("k_pages", "v_pages", "weights"))
def _write_op(q: Tensor, k: Tensor, v: Tensor, cos: Optional[Tensor], sin: Optional[Tensor],
              positions: Optional[Tensor], k_pages: Tensor, v_pages: Tensor, table: Tensor, q_start: Tensor,
              kv_len: Tensor, weights: Optional[Tensor], interleaved: bool) -> Tensor:
    return _write_body(q, k, v, cos, sin, positions, k_pages, v_pages, table, q_start, kv_len, weights, interleaved)


@_write_op.register_fake
def _(q, k, v, cos, sin, positions, k_pages, v_pages, table, q_start, kv_len, weights, interleaved):
    return q.new_empty(q.shape)


def paged_write(q: Tensor, k: Tensor, v: Tensor, cos: Optional[Tensor], sin: Optional[Tensor],
                positions: Optional[Tensor], k_pages: Tensor, v_pages: Tensor, table: Tensor, q_start: Tensor,
                kv_len: Tensor, *, weights: Optional[Tensor] = None, interleaved: bool = False) -> Tensor:
    """Stores new tokens and returns their rotated queries [tokens, heads, head_dim].

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim] (strides free: column slices of a fused
    projection), k_pages and v_pages [pages, kv_heads, page_size, head_dim] (any page order and strides with unit last
    stride; page_size a power of two), table int32 [batch, width] of page ids, q_start int32 [batch + 1], kv_len
    int32 [batch] (keys with the new ones: a sequence's n new tokens take its slots kv_len - n to kv_len - 1). Queries
    and keys are rotated as ``rotary_embed`` does (cos = sin = None: not at all); the new slots' gathered ``weights``
    [pages, kv_heads, page_size] start at 0. No two sequences may write one page."""
    a = (q, k, v, cos, sin, positions, k_pages, v_pages, table, q_start, kv_len, weights)
    _no_tangents("paged_write", q, k, v, cos, sin, k_pages, v_pages, weights)
    host = _host()
    if host is not None:
        out = host.paged_write(*a, interleaved)
        if out is not None:
            return out
    if _plain(*a):
        return _written(_write_body(*a, interleaved), k_pages, v_pages, weights)
    return _write_op(*a, interleaved)


def _attention_body(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, q_start: Tensor, kv_len: Tensor,
                    max_q: int, max_kv: int, scale: float, causal: bool,
                    weights: Optional[Tensor]) -> tuple[Tensor, Tensor]:
    name = "paged_attention"
    args = _cache_args(name, k_pages, v_pages, weights, table, q_start, kv_len)
    d, hk = args.head_dim, args.kv_heads
    _require(q.dim() == 3, name, f"q must be [tokens, heads, {d}], got {list(q.shape)}")
    t, h = int(q.shape[0]), int(q.shape[1])
    _heads(name, "q", q, k_pages.dtype, k_pages.device, t, h, d)
    _require(h > 0 and hk > 0 and h % hk == 0, name, f"{h} query heads over {hk} kv heads")
    if t and (q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16 or q.stride(0) == 0 or q.stride(1) == 0):
        q = q.contiguous() if not q.is_contiguous() else q.clone()
    o = torch.empty((t, h, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((t, h), dtype=torch.float32, device=q.device)
    lib = nat.load()
    gather = int(weights is not None)
    n = int(lib.gwa_paged_attention_workspace(args.batch, t, h, hk, d, max_q, max_kv,
                                              args.table_width * args.page_size, gather))
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    nat.call("gwa_paged_attention", ctypes.byref(args), q.data_ptr(), q.stride(0), q.stride(1), o.data_ptr(),
             lse.data_ptr(), t, h, max_q, max_kv, scale, int(causal), gather, nat.ptr(ws), n, nat.stream_of(q))
    return o, lse


@torch.library.custom_op("cozy_gen_worker::paged_attention", mutates_args=("weights",))
def _attention_op(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, q_start: Tensor, kv_len: Tensor,
                  max_q: int, max_kv: int, scale: float, causal: bool,
                  weights: Optional[Tensor]) -> tuple[Tensor, Tensor]:
    return _attention_body(q, k_pages, v_pages, table, q_start, kv_len, max_q, max_kv, scale, causal, weights)


@_attention_op.register_fake
def _(q, k_pages, v_pages, table, q_start, kv_len, max_q, max_kv, scale, causal, weights):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, q_start: Tensor, kv_len: Tensor,
                    max_q: int, max_kv: int, *, scale: Optional[float] = None, causal: bool = True,
                    weights: Optional[Tensor] = None) -> tuple[Tensor, Tensor]:
    """Attention of the new tokens over their sequences' cached keys (their own among them, see ``paged_write``):
    (o [tokens, heads, head_dim] in q's type, lse fp32 [tokens, heads], the natural log of the sum of exponentials).

    Query head x reads kv head x // (heads / kv_heads). With ``causal`` token i of n in a sequence of L keys sees the
    first L - n + i + 1, else all L; a row that sees none, or scores of -inf alone, gives o = 0 and lse = -inf, one that
    sees a NaN score NaN. ``scale`` defaults to head_dim^-0.5. ``max_q`` and ``max_kv``: the batch's largest new-token count and kv_len, which choose the launch.
    ``weights`` fp32 [pages, kv_heads, page_size]: every key's slot gets, added, the probability it drew from the
    sequence's new tokens over the kv head's query heads, in an order that does not depend on timing; sequences may
    share pages only without it. head_dim: a multiple of 8 up to 256 (the matrix cores serve 64 and 128, up to 256 query
    heads to a kv head). Rows of q that belong to no sequence (before q_start[0], behind q_start[batch]) are not written. No
    gradient is defined."""
    if scale is None:
        scale = float(q.shape[-1]) ** -0.5
    _no_tangents("paged_attention", q, k_pages, v_pages, weights)
    host = _host()
    if host is not None:
        out = host.paged_attention(q, k_pages, v_pages, table, q_start, kv_len, weights, max_q, max_kv, scale, causal)
        if out is not None:
            return out
    if _plain(q, k_pages, v_pages, table, q_start, kv_len, weights):
        return _written(_attention_body(q, k_pages, v_pages, table, q_start, kv_len, max_q, max_kv, scale, causal,
                                        weights), weights)
    return _attention_op(q, k_pages, v_pages, table, q_start, kv_len, max_q, max_kv, scale, causal, weights)


def _evict_body(k_pages: Tensor, v_pages: Tensor, weights: Tensor, table: Tensor, kv_len: Tensor, max_kv: int,
                new_table: Tensor, budget: int, recent: int) -> tuple[Tensor, Tensor]:
    name = "paged_evict"
    _require(weights is not None, name, "weights are needed")
    args = _cache_args(name, k_pages, v_pages, weights, table, None, kv_len)
    dev = k_pages.device
    _require(budget > 0 and 0 <= recent <= budget, name, f"a budget of {budget} keys, {recent} of them recent")
    _ints(name, "new_table", new_table, (args.batch, new_table.shape[-1] if new_table.dim() == 2 else -1), dev)
    _require(args.batch < 2 or new_table.stride(0) >= new_table.shape[1], name,
             f"new_table's rows overlap (row stride {new_table.stride(0)}): sequences would be copied into one page")
    kept = torch.empty((args.batch, args.kv_heads, budget), dtype=torch.int32, device=dev)
    new_len = torch.empty(args.batch, dtype=torch.int32, device=dev)
    nat.call("gwa_paged_evict", ctypes.byref(args), new_table.data_ptr(), max(new_table.stride(0), new_table.shape[1]),
             new_table.shape[1], max_kv, budget, recent, kept.data_ptr(), new_len.data_ptr(), nat.stream_of(k_pages))
    return kept, new_len


@torch.library.custom_op("cozy_gen_worker::paged_evict", mutates_args=("k_pages", "v_pages", "weights"))
def _evict_op(k_pages: Tensor, v_pages: Tensor, weights: Tensor, table: Tensor, kv_len: Tensor, max_kv: int,
              new_table: Tensor, budget: int, recent: int) -> tuple[Tensor, Tensor]:
    return _evict_body(k_pages, v_pages, weights, table, kv_len, max_kv, new_table, budget, recent)


@_evict_op.register_fake
def _(k_pages, v_pages, weights, table, kv_len, max_kv, new_table, budget, recent):
    b = kv_len.shape[0]
    return kv_len.new_empty((b, k_pages.shape[1], budget)), kv_len.new_empty((b,))


def paged_evict(k_pages: Tensor, v_pages: Tensor, weights: Tensor, table: Tensor, kv_len: Tensor, max_kv: int,
                new_table: Tensor, budget: int, recent: int) -> tuple[Tensor, Tensor]:
    """Cuts every sequence with more than ``budget`` keys back to it, for each kv head on its own: the last
    ``recent`` keys stay, and of the others the ``budget - recent`` of largest gathered weight (equal ones: the lowest
    slots; NaN ranks highest). What stays (k, v and weights, in slot order; all of a shorter sequence) is copied into
    the pages of ``new_table`` int32 [batch, width], which must be pages that ``table`` does not use and hold
    min(budget, the largest kv_len) keys a row; ``max_kv``: the largest kv_len, which shapes the launch. Returns (kept int32
    [batch, kv_heads, budget]: the old slots, -1 past the end; the new kv_len)."""
    a = (k_pages, v_pages, weights, table, kv_len)
    _no_tangents("paged_evict", k_pages, v_pages, weights)
    host = _host()
    if host is not None:
        out = host.paged_evict(*a, new_table, max_kv, budget, recent)
        if out is not None:
            return out
    if _plain(*a, new_table):
        return _written(_evict_body(*a, max_kv, new_table, budget, recent), k_pages, v_pages, weights)
    return _evict_op(*a, max_kv, new_table, budget, recent)


# ---------------------------------------------------------------------------
# the cache and its batches
# ---------------------------------------------------------------------------

@dataclass
class PagedBatch:
    """The new tokens of one call: device arrays for the operators, and the host's sizes. ``positions``: each new
    token's place in its sequence, counted over everything the sequence has seen (evicted keys too)."""

    table: Tensor
    q_start: Tensor
    kv_len: Tensor
    positions: Tensor
    tokens: int
    max_q: int
    max_kv: int


class PagedCache:
    """A pool of ``pages`` pages for the keys and values of one layer's kv heads, and the sequences in it.

    Page lists, lengths and the free list are host state; device work is enqueued on the current stream in call order, so
    use one stream for one cache (or order the streams). ``weights=True`` keeps each key's gathered attention
    weight, which ``evict`` needs. Several layers that always hold the same tokens can share one bookkeeping: ``twin``
    gives another pool under this cache's page lists."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", weights: bool = False) -> None:
        name = "PagedCache"
        _require(pages > 0 and kv_heads > 0 and 8 <= page_size <= 4096 and page_size & (page_size - 1) == 0, name,
                 f"{pages} pages of {page_size} slots (a power of two, 8 to 4096), {kv_heads} kv heads")
        _require(dtype in (torch.bfloat16, torch.float16) and head_dim % 8 == 0 and 8 <= head_dim <= 256, name,
                 f"{dtype} heads of {head_dim} (bf16 or fp16, a multiple of 8 up to 256)")
        self.page_size = page_size
        self.k = torch.zeros((pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.weights = (torch.zeros((pages, kv_heads, page_size), dtype=torch.float32, device=device)
                        if weights else None)
        self._free = list(range(pages - 1, -1, -1))
        self._seqs: dict[int, list] = {}   # id -> [page ids, keys held, tokens seen]
        self._next = 0
        self._twins: list["PagedCache"] = []

    def twin(self) -> "PagedCache":
        """A pool of the same shape whose pages follow this cache's lists: another layer's keys and values. Write and
        attend with this cache's batches. Sequences are added to and cut by the first cache alone, whose ``evict`` serves
        its twins and theirs."""
        other = PagedCache.__new__(PagedCache)
        other.page_size, other._free, other._seqs = self.page_size, self._free, self._seqs
        other.k, other.v = torch.zeros_like(self.k), torch.zeros_like(self.v)
        other.weights = None if self.weights is None else torch.zeros_like(self.weights)
        other._next, other._twins = -1, []
        self._twins.append(other)
        return other

    def _pools(self) -> Iterator["PagedCache"]:
        """Every pool under this cache's lists."""
        yield self
        for twin in self._twins:
            yield from twin._pools()

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        """Keys the sequence holds."""
        return self._seqs[seq][1]

    def add(self) -> int:
        """A new, empty sequence's id."""
        _require(self._next >= 0, "PagedCache.add", "sequences belong to the cache this is a twin of")
        self._next += 1
        self._seqs[self._next - 1] = [[], 0, 0]
        return self._next - 1

    def drop(self, seq: int) -> None:
        """Gives the sequence's pages back."""
        self._free.extend(reversed(self._seqs.pop(seq)[0]))

    def _take(self, name: str, wanted: int) -> list[int]:
        _require(wanted <= len(self._free), name, f"{wanted} pages wanted, {len(self._free)} free")
        return [self._free.pop() for _ in range(wanted)]

    def _device_rows(self, rows: Sequence[Sequence[int]]) -> list[Tensor]:
        """int32 device tensors of several lists, in one copy."""
        flat = torch.tensor([x for r in rows for x in r], dtype=torch.int32).to(self.k.device)
        out, at = [], 0
        for r in rows:
            out.append(flat[at:at + len(r)])
            at += len(r)
        return out

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> PagedBatch:
        """Room for ``counts[i]`` new tokens of sequence ``seqs[i]``, and the batch that writes and attends them."""
        name = "PagedCache.extend"
        _require(len(seqs) == len(counts) and len(set(seqs)) == len(seqs) and len(seqs) > 0, name,
                 "one count for each of at least one sequence, each named once")
        _require(all(s in self._seqs for s in seqs) and all(c >= 0 for c in counts), name,
                 f"sequences {list(seqs)} with {list(counts)} new tokens")
        need = [max(0, -(-(self._seqs[s][1] + c) // self.page_size) - len(self._seqs[s][0]))
                for s, c in zip(seqs, counts)]
        fresh = self._take(name, sum(need))
        starts, positions, lens = [0], [], []
        for s, c, n in zip(seqs, counts, need):
            e = self._seqs[s]
            e[0].extend(fresh[:n])
            del fresh[:n]
            positions.extend(range(e[2], e[2] + c))
            e[1] += c
            e[2] += c
            starts.append(starts[-1] + c)
            lens.append(e[1])
        table, width = self._table_rows(seqs)
        q_start, kv_len, pos, flat = self._device_rows([starts, lens, positions, table])
        return PagedBatch(flat.view(len(seqs), width), q_start, kv_len, pos, starts[-1], max(counts), max(lens))

    def _table_rows(self, seqs: Sequence[int]) -> tuple[list[int], int]:
        width = max(max(len(self._seqs[s][0]) for s in seqs), 1)
        return [x for s in seqs for x in self._seqs[s][0] + [0] * (width - len(self._seqs[s][0]))], width

    def write(self, batch: PagedBatch, q: Tensor, k: Tensor, v: Tensor, cos: Optional[Tensor] = None,
              sin: Optional[Tensor] = None, *, interleaved: bool = False) -> Tensor:
        """``paged_write`` of the batch's tokens at its positions; the rotated queries."""
        return paged_write(q, k, v, cos, sin, batch.positions, self.k, self.v, batch.table, batch.q_start, batch.kv_len,
                           weights=self.weights, interleaved=interleaved)

    def attend(self, batch: PagedBatch, q: Tensor, *, scale: Optional[float] = None, causal: bool = True,
               gather: Optional[bool] = None) -> tuple[Tensor, Tensor]:
        """``paged_attention`` of the batch's (rotated) queries: (o, lse). Weights are gathered where the cache keeps
        them, unless ``gather`` is False."""
        gather = self.weights is not None if gather is None else gather
        _require(not gather or self.weights is not None, "PagedCache.attend", "the cache keeps no weights")
        return paged_attention(q, self.k, self.v, batch.table, batch.q_start, batch.kv_len, batch.max_q, batch.max_kv,
                               scale=scale, causal=causal, weights=self.weights if gather else None)

    def evict(self, seqs: Sequence[int], budget: int, recent: int) -> Optional[Tensor]:
        """Cuts those of ``seqs`` that hold more than ``budget`` keys back to it (``paged_evict``), here and in all
        twins (a twin itself refuses: it does not reach the others); their old pages are free afterwards. Returns this cache's kept slots [cut sequences, kv_heads, budget], or
        None if no sequence was longer. Needs budget / page_size free pages a cut sequence."""
        name = "PagedCache.evict"
        _require(self._next >= 0, name, "sequences belong to the cache this is a twin of")
        _require(all(s in self._seqs for s in seqs) and len(set(seqs)) == len(seqs), name, f"sequences {list(seqs)}")
        _require(self.weights is not None, name, "the cache keeps no weights")
        _require(budget > 0 and 0 <= recent <= budget, name, f"a budget of {budget} keys, {recent} of them recent")
        cut = [s for s in seqs if self._seqs[s][1] > budget]
        if not cut:
            return None
        width = -(-budget // self.page_size)
        fresh = self._take(name, width * len(cut))
        table, old_width = self._table_rows(cut)
        lens = [self._seqs[s][1] for s in cut]
        kv_len, flat, new = self._device_rows([lens, table, fresh])
        flat, new = flat.view(len(cut), old_width), new.view(len(cut), width)
        kept = None
        try:
            for cache in self._pools():
                got = paged_evict(cache.k, cache.v, cache.weights, flat, kv_len, max(lens), new, budget, recent)[0]
                kept = got if kept is None else kept
        except Exception:
            self._free.extend(fresh)   # nothing has moved: the sequences keep their pages
            raise
        for i, s in enumerate(cut):
            e = self._seqs[s]
            self._free.extend(reversed(e[0]))
            e[0], e[1] = fresh[i * width:(i + 1) * width], budget
        return kept
