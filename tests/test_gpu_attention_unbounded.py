"""Infinities and NaN among the values of causal attention: they reach the rows that see them, as what they are, and nothing else;
and a piece of work that has some does not slow down the pieces behind it."""
import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"


@gpu
@pytest.mark.parametrize("heads", [(4, 2, 64), (3, 3, 64), (8, 2, 128), (3, 1, 80)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_scattered_over_many_pieces_of_work(heads, dt):
    """Every CTA has several pieces of work, some with such values in the first block of their own rows, the second, both or
    neither: the sum of the infinities and NaN that a row sees where there are any, the bits of a call without them elsewhere."""
    hq, hkv, d = heads
    B, n = 60, 700
    gen = torch.Generator(device=DEV).manual_seed(hq + d)
    q, k, v = (torch.randn(B, n, h, d, device=DEV, generator=gen).to(dt) for h in (hq, hkv, hkv))
    spoilt = torch.rand(B, n, hkv, d, device=DEV, generator=gen) < 2e-5 * torch.randint(0, 3, (B, 1, 1, 1), device=DEV, generator=gen)
    what = torch.tensor([float("inf"), float("-inf"), float("nan")], device=DEV)
    bad = torch.where(spoilt, what[torch.randint(0, 3, spoilt.shape, device=DEV, generator=gen)], 0.0)
    clean = cp.causal_attention(q, k, torch.where(spoilt, 0, v))
    got = cp.causal_attention(q, k, torch.where(spoilt, bad.to(dt), v))
    cp.check_device_status()
    seen = bad.cumsum(1).repeat_interleave(hq // hkv, 2)     # (finite parts are zeros)
    touched = spoilt.cumsum(1).repeat_interleave(hq // hkv, 2) > 0
    assert 0 < int(touched.sum()) < touched.numel() // 2
    assert torch.equal(got[~touched], clean[~touched])
    assert torch.allclose(got[touched].float(), seen[touched], equal_nan=True)


@gpu
def test_padding_of_nan_and_training():
    """A batch padded with NaN: rows in front of the padding have the bits of a batch padded with zeros, with and without what
    the backward keeps."""
    B, n, lens = 6, 400, (1, 128, 129, 255, 300, 400)
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(B, n, 4, 64, device=DEV, generator=gen).bfloat16() for _ in range(3))
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        for b, m in enumerate(lens):
            q[b, m:], k[b, m:], v[b, m:] = fill, fill, fill
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        outs += [cp.causal_attention(q, k, v), cp.causal_attention(*leaves).detach()]
    cp.check_device_status()
    for b, m in enumerate(lens):
        assert all(torch.equal(o[b, :m], outs[0][b, :m]) for o in outs)
        assert all(torch.isnan(o[b, m:]).all() for o in outs[2:])


@gpu
def test_one_nan_costs_the_pieces_that_see_it_only():
    """One value of 12.6 million: the call takes less than 8 times as long (67 us and 2.5 times as long when this was written, the
    longest chain of a CTA's pieces being what is measured; 64 times with a mark that outlived its piece)."""
    q, k, v = (torch.randn(16, 1024, 12, 64, device=DEV).bfloat16() for _ in range(3))
    spoilt = v.clone()
    spoilt[0, 3, 0, 1] = float("nan")

    def best(values):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(3):
                cp.causal_attention(q, k, values)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert best(spoilt) < 8 * best(v)
