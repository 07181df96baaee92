"""Host side of the sampler, without a GPU: what it refuses."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch


def test_refusals_without_a_gpu():
    from gen_worker_amd.sampling import SamplingError, sample_tokens

    x, u = torch.zeros(2, 5), torch.zeros(2)
    with pytest.raises(SamplingError, match="CUDA"):
        sample_tokens(x, u)
    for bad in (dict(temperature=-0.1), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_k=-1),
                dict(top_k=2 ** 31), dict(top_p=1.01), dict(top_p=-0.5), dict(top_p=math.nan), dict(min_p=2.0),
                dict(min_p="0.5"), dict(temperature=None), dict(top_k=True)):
        with pytest.raises(SamplingError, match="must be"):
            sample_tokens(x, u, **bad)


class TestEntryPoint:
    """The C entry point refuses before any launch."""

    def call(self, logits=4096, ld=100, dtype=2, uniform=4096, tokens=4096, logprobs=4096, rows=2, vocab=100, settings=True,
             workspace=None, nbytes=0, **change):
        from gen_worker_amd import _native as nat

        v = dict(all_temperature=1.0, all_top_k=0, all_top_p=1.0, all_min_p=0.0)
        v.update(change)
        s = ctypes.byref(nat.SamplingArgs(**v)) if settings else None
        lib = nat.load()
        rc = lib.gwa_sample_tokens(logits, ld, dtype, uniform, s, tokens, logprobs, rows, vocab, workspace, nbytes, None)
        return rc, lib.gwa_last_error().decode()

    @pytest.mark.parametrize("change,match", [
        (dict(settings=False), "settings"), (dict(dtype=3), "dtype"), (dict(vocab=0), "tokens"),
        (dict(vocab=2 ** 24 + 1, ld=2 ** 25), "tokens"), (dict(rows=-1), "rows"), (dict(ld=99), "stride"),
        (dict(logits=None), "null pointer"), (dict(uniform=None), "null pointer"), (dict(tokens=None), "null pointer"),
        (dict(logprobs=None), "null pointer"), (dict(logits=4098), "misaligned"), (dict(tokens=4100), "misaligned"),
        (dict(temperature=4098), "misaligned"), (dict(all_temperature=-1.0), "temperature"),
        (dict(all_temperature=math.nan), "temperature"), (dict(all_temperature=math.inf), "temperature"),
        (dict(all_top_k=-1), "top_k"), (dict(all_top_p=1.5), "top_p"), (dict(all_top_p=math.nan), "top_p"),
        (dict(all_min_p=-0.1), "min_p"), (dict(vocab=50000, ld=50000), "workspace"),
        (dict(vocab=50000, ld=50000, workspace=4096, nbytes=1000), "workspace"),
        (dict(vocab=50000, ld=50000, workspace=4104, nbytes=1 << 30), "workspace"),
        (dict(rows=2 ** 30, vocab=50000, ld=50000, workspace=4096, nbytes=1 << 60), "too many"),
        (dict(rows=2 ** 22), "too many"),
        (dict(rows=2 ** 22 - 1, vocab=50000, ld=50000, workspace=4096, nbytes=1 << 60), "too many")])
    def test_refuses(self, change, match):
        rc, said = self.call(**change)
        assert rc == 1 and match in said, said

    def test_no_rows_need_no_device(self):
        assert self.call(rows=0, logits=None)[0] == 0

    def test_workspace(self):
        from gen_worker_amd import _native as nat

        of = nat.load().gwa_sample_tokens_workspace
        assert of(5, 8192) == of(0, 10 ** 6) == of(3, 0) == of(-1, 50000) == 0
        assert 0 < of(1, 8193) < of(2, 8193) < of(2, 2 ** 24) < 2 ** 20
