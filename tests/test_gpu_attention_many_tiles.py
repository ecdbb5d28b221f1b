"""Packed batches whose grid has far more tiles than there is work: the number of sequences bounds it, and most are empty."""
import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"


def _run(q, k, v, do, cu):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cp.causal_attention(*leaves, cu)
    return [o.detach(), *torch.autograd.grad(o, leaves, do)]


@gpu
def test_the_most_sequences_and_many_heads():
    """2^20 offsets of which 1024 are of sequences, 128 heads: 1.3e8 tiles of dq that there are none of, more than a second of
    looking for work while the other warps of a CTA wait for it.  Some heads against the same call without the empty ones."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    n, length, real, hq, d = 1 << 20, 1024, 1024, 128, 8
    rows = real * length
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, do = (torch.randn(rows, hq, d, device=DEV, generator=gen, dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(rows, 1, d, device=DEV, generator=gen, dtype=torch.bfloat16) for _ in range(2))
    cu = torch.full((n + 1,), rows, device=DEV, dtype=torch.int32)
    cu[:real + 1] = torch.arange(real + 1, device=DEV) * length
    got = _run(q, k, v, do, cu)
    cp.check_device_status()
    want = _run(q, k, v, do, cu[:real + 1].clone())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("rows", [1, 3, 130, 1000])
def test_more_sequences_than_rows(rows):
    """The rows bound the tiles too: sequences of one row or none, a long one, rows of none in front and behind."""
    gen = torch.Generator(device=DEV).manual_seed(rows)
    q, do = (torch.randn(rows, 4, 64, device=DEV, generator=gen).bfloat16() for _ in range(2))
    k, v = (torch.randn(rows, 2, 64, device=DEV, generator=gen).bfloat16() for _ in range(2))
    steps = torch.randint(0, 2, (5000,), device=DEV, generator=gen)
    steps[2500] = rows // 2
    cu = (torch.cat([steps.new_zeros(1), steps.cumsum(0)]) + rows // 8).clamp(max=rows - rows // 8).to(torch.int32)
    few = torch.unique(cu)
    if few.numel() == 1:
        few = few.repeat(2)
    for a, b in zip(_run(q, k, v, do, cu), _run(q, k, v, do, few)):
        assert torch.equal(a, b)
    cp.check_device_status()
