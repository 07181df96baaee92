"""Drawing the next tokens from a step's logits (``csrc/sampling.hip``): temperature, top-k, top-p and min-p, each row by a
random number that the caller gives, so that an answer can be drawn again.

``sample_tokens`` runs on the current stream, does not synchronise and may be captured in a HIP graph. CPU tensors are
refused: there is no CPU implementation.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch
from torch import Tensor

from . import _native as nat
from . import paged

_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16, torch.float32: nat.DT_F32}
MAX_VOCAB = 1 << 24
MAX_TOP_K = (1 << 31) - 1


class SamplingError(ValueError):
    """An argument the sampler does not take."""


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise SamplingError(f"sample_tokens: {message}")


def _column(what: str, t: Optional[Tensor], dtype: torch.dtype, rows: int, device: torch.device) -> None:
    _require(t is None or (t.dtype == dtype and t.device == device and tuple(t.shape) == (rows,)
                           and (rows < 2 or t.stride(0) == 1)),
             f"{what} must be a contiguous {dtype} [{rows}] on {device}" + (
                 "" if t is None else f", got {t.dtype} {list(t.shape)} strides {t.stride()} on {t.device}"))


def _sample_body(logits: Tensor, uniform: Tensor, temperature: Optional[Tensor], top_k: Optional[Tensor],
                 top_p: Optional[Tensor], min_p: Optional[Tensor], all_temperature: float, all_top_k: int,
                 all_top_p: float, all_min_p: float) -> tuple[Tensor, Tensor]:
    _require(logits.is_cuda and logits.dim() == 2 and logits.dtype in _DTYPES,
             f"logits must be a bf16, fp16 or fp32 CUDA tensor [rows, vocab], got {logits.dtype} {list(logits.shape)} on "
             f"{logits.device}")
    rows, vocab = int(logits.shape[0]), int(logits.shape[1])
    dev = logits.device
    _require(0 < vocab <= MAX_VOCAB, f"a vocabulary of {vocab} (1 to {MAX_VOCAB})")
    _require(uniform is not None, "a random number a row is needed")
    for what, t, dtype in (("uniform", uniform, torch.float32), ("temperature", temperature, torch.float32),
                           ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        _column(what, t, dtype, rows, dev)
    _require(0 <= all_top_k <= MAX_TOP_K, f"top_k must be 0 to {MAX_TOP_K}, got {all_top_k}")
    if vocab > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    args = nat.SamplingArgs(nat.ptr(temperature), nat.ptr(top_k), nat.ptr(top_p), nat.ptr(min_p), all_temperature, all_top_k,
                            all_top_p, all_min_p)
    n = int(nat.load().gwa_sample_tokens_workspace(rows, vocab))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    with nat.on_device_of(logits):
        nat.call("gwa_sample_tokens", logits.data_ptr(), max(logits.stride(0), vocab), _DTYPES[logits.dtype],
                 uniform.data_ptr(), ctypes.byref(args), tokens.data_ptr(), logprobs.data_ptr(), rows, vocab, nat.ptr(ws),
                 n, nat.stream_of(logits))
    return tokens, logprobs


@torch.library.custom_op("cozy_gen_worker::sample_tokens", mutates_args=())
def _sample_op(logits: Tensor, uniform: Tensor, temperature: Optional[Tensor], top_k: Optional[Tensor],
               top_p: Optional[Tensor], min_p: Optional[Tensor], all_temperature: float, all_top_k: int,
               all_top_p: float, all_min_p: float) -> tuple[Tensor, Tensor]:
    return _sample_body(logits, uniform, temperature, top_k, top_p, min_p, all_temperature, all_top_k, all_top_p,
                        all_min_p)


@_sample_op.register_fake
def _(logits, uniform, temperature, top_k, top_p, min_p, all_temperature, all_top_k, all_top_p, all_min_p):
    rows = logits.shape[0]
    return logits.new_empty((rows,), dtype=torch.int64), logits.new_empty((rows,), dtype=torch.float32)


def _setting(value, plain, what: str, low, high):
    """(tensor, 0) or (None, number) of a setting."""
    if isinstance(value, Tensor):
        return value, plain
    kinds = int if isinstance(plain, int) else (int, float)
    _require(isinstance(value, kinds) and not isinstance(value, bool) and low <= value <= high,
             f"{what} must be {low} to {high} or a tensor, got {value!r}")
    return None, type(plain)(value)


def settings(temperature, top_k, top_p, min_p) -> tuple[tuple, tuple]:
    """``sample_tokens``' settings, checked: (tensors, None for numbers; numbers, a default for tensors)."""
    pairs = (_setting(temperature, 1.0, "temperature", 0.0, 3.0e38), _setting(top_k, 0, "top_k", 0, MAX_TOP_K),
             _setting(top_p, 1.0, "top_p", 0.0, 1.0), _setting(min_p, 0.0, "min_p", 0.0, 1.0))
    return tuple(t for t, _ in pairs), tuple(n for _, n in pairs)


def sample_tokens(logits: Tensor, uniform: Tensor, *, temperature: Union[float, Tensor] = 1.0,
                  top_k: Union[int, Tensor] = 0, top_p: Union[float, Tensor] = 1.0,
                  min_p: Union[float, Tensor] = 0.0) -> tuple[Tensor, Tensor]:
    """A token of each row of logits [rows, vocab] (bf16, fp16 or fp32): (tokens int64 [rows], logprobs fp32 [rows]).

    Weights are w_i = exp((x_i - max x) / temperature). In falling order of the logits (equal ones: the lowest index first)
    the tokens are cut to the first ``top_k`` (0: all), then to the shortest run whose weight reaches ``top_p`` of what is
    left (1: all), then to those with w_i >= ``min_p``; the first always stays. The token is the first, in the vocabulary's
    order, at which the kept weights up to and with its own pass ``uniform[row]`` (fp32 [rows], in [0, 1)) times their sum;
    its logprob is log(w_i / sum), of the distribution that was drawn from. Temperature 0 takes the largest, logprob 0.

    A setting is a number, or a tensor [rows] (top_k int32, the others fp32) with one for each row, whose values out of
    range count as the nearest in it (a NaN as 0). Settings are fp32. -inf and NaN are never drawn; a row with nothing else
    gives token -1 and logprob NaN. Weights and sums are integers in 64 bits, of 2^-45 of the largest weight (2^-38 at
    2^24 tokens; half of that or less is never drawn), so the result does not depend on how the work is split. No gradient is
    defined."""
    each, numbers = settings(temperature, top_k, top_p, min_p)
    a = (logits, uniform, *each)
    _require(all(paged._tangent(x) is None for x in a), "no gradient is defined for a dual tensor's tangent")
    host = paged._host()
    if host is not None:
        out = host.sample_tokens(*a, *numbers)
        if out is not None:
            return out
    if paged._plain(*a):
        return _sample_body(*a, *numbers)
    return _sample_op(*a, *numbers)
