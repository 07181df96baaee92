"""The 8-bit paged cache where its format ends: keys that the rotation takes past their type's range, and
which values a read gives back exactly. Tables of 2 and 0 turn nothing and scale exactly, so rows are equal to their definition,
code for code."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged import BF16, DEV, F16, _gen, _ints
from test_gpu_paged_fp8 import FP8, held, value_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import gen_worker_amd  # noqa: F401
    from gen_worker_amd import _native

    _native.load()
    yield


def _pools(pages, heads, size, dim):
    codes = [torch.zeros(pages, heads, size, dim, dtype=torch.uint8, device=DEV).view(FP8) for _ in range(2)]
    return (*codes, *(torch.zeros(pages, heads, size, dtype=torch.uint8, device=DEV) for _ in range(2)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rot,interleaved,odd", [(64, False, False), (64, True, False), (32, False, False), (64, False, True),
                                                 (20, True, False)])
def test_keys_that_the_rotation_takes_past_the_type(dtype, rot, interleaved, odd):
    """Tables longer than 1 (as scaled rotations have): a finite value past the type's largest counts as that one, so no row
    reads as infinite. ``odd``: operands off 16-byte alignment."""
    from gen_worker_amd.paged import paged_attention_fp8, paged_read_fp8, paged_write_fp8

    big, gain, g = torch.finfo(dtype).max, 2.0, _gen(rot)
    n = 90
    k = torch.randn(n, 2, 64, generator=g, device=DEV)
    k *= torch.exp2(torch.randint(-6, 3, (n, 2, 1), generator=g, device=DEV).float())
    top = torch.arange(n // 2, device=DEV)           # rows that end in the type's last binades, at every channel
    k[top, :, top % 64] = big * (0.2 + 0.8 * torch.rand(n // 2, 2, generator=g, device=DEV)) * (1.0 - 2.0 * (top % 2))[:, None]
    k = k.to(dtype)
    k[0, 0, 3], k[1, 0, 5], k[2, 0, :] = big, -big, big
    q, v = torch.randn(n, 4, 64, generator=g, device=DEV).to(dtype), torch.randn(n, 2, 64, generator=g, device=DEV).to(dtype)
    if odd:
        q, k, v = (torch.cat([x.flatten(1), x.flatten(1)], 1)[:, 1:1 + x[0].numel()].unflatten(1, (-1, 64))
                   for x in (q, k, v))
    cos, sin = (torch.full((n, rot // 2), c, device=DEV) for c in (gain, 0.0))
    pool = _pools(8, 2, 16, 64)
    table, start, length = _ints([[5, 2, 7, 0, 3, 6]]), _ints([0, n]), _ints([n])
    paged_write_fp8(q, k, v, cos, sin, torch.arange(n, device=DEV).int(), *pool, table, start, length, interleaved=interleaved)
    turned = k.float()
    turned[..., :rot] = turned[..., :rot] * gain      # exact, but where it overflows fp32
    want, byte = held(torch.where(turned.isfinite(), turned.clamp(-big, big), turned), dtype)
    j = torch.arange(n, device=DEV)
    at = table[0].long()[j // 16]
    assert torch.equal(pool[2][at, :, j % 16], byte)
    got = pool[0].view(torch.uint8)[at, :, j % 16].view(FP8).double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    kk, vv = paged_read_fp8(*pool, table, start, length, n, dtype=dtype)
    assert torch.equal(kk.isfinite(), turned.isfinite()) and bool(vv.isfinite().all())
    if dtype == F16:                                  # (bf16's products with such keys pass fp32)
        o, lse = paged_attention_fp8((q * 2.0 ** -9).to(dtype), *pool, table, start, length, n, n)
        assert bool(o.isfinite().all()) and bool(lse.isfinite().all())


def test_bf16_reads_exactly_what_it_can_hold():
    """Every finite code under the scale bytes 3 to 246 is a bf16 number, and read as it is; past them the nearest one, or
    infinity."""
    from gen_worker_amd.paged import paged_read_fp8

    codes = torch.arange(256, device=DEV, dtype=torch.uint8).view(1, 1, 16, 16).expand(256, 1, 16, 16).contiguous()
    scales = torch.arange(256, device=DEV, dtype=torch.uint8).view(256, 1, 1).expand(256, 1, 16).contiguous()
    table = torch.arange(256, device=DEV, dtype=torch.int32).view(1, 256)
    k, _ = paged_read_fp8(codes.view(FP8), codes.view(FP8), scales, scales, table, _ints([0, 4096]), _ints([4096]), 4096)
    got, want = k.view(256, 16, 16).double(), value_of(codes, scales)[:, 0]
    assert torch.equal(got[3:247].nan_to_num(), want[3:247].nan_to_num())
    assert not torch.equal(got[2].nan_to_num(), want[2].nan_to_num()) and bool(got[247].isinf().any())
    assert torch.equal(got.nan_to_num(), want.to(BF16).double().nan_to_num())
