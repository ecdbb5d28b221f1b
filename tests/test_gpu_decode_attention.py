"""decode_attention against a float64 restatement, with an element-wise error bound.

|o - o64| <= (u + e) sum_j P_j |v_j| + u |o|: the probabilities are rounded to the inputs' type once (u: half a step), the
result once, and e is what fp32 leaves of an exponent (see the bound of the prompt's attention).  In fp16 probabilities
below 2^-14 of the largest are off by up to 2^-25 of it, each with its value's weight."""
import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"


def _inputs(b, room, hq, hkv, d, dt, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen).to(dt)
    return r(b, hq, d), r(b, room, hkv, d), r(b, room, hkv, d)


def _check(o, q, k, v, lens, scale):
    u = torch.finfo(q.dtype).eps / 2
    g, d = q.shape[1] // k.shape[2], q.shape[2]
    for i, n in enumerate(lens):
        if n == 0:
            assert torch.count_nonzero(o[i]) == 0
            continue
        Q = q[i].double().unflatten(0, (-1, g))
        K, V = k[i, :n].double().transpose(0, 1), v[i, :n].double().transpose(0, 1)
        P = torch.softmax(Q @ K.transpose(1, 2) * scale, -1)
        e = 2 * (d + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().transpose(1, 2)).max() + 2.0 ** -20
        O = (P @ V).flatten(0, 1)
        tol = (u + e) * (P @ V.abs()).flatten(0, 1) + u * O.abs()
        if q.dtype == torch.float16:
            tol = tol + 2.0 ** -25 * (P.amax(-1, keepdim=True) * V.abs().sum(1, keepdim=True)).flatten(0, 1) + 2.0 ** -24
        bad = ~((o[i].double() - O).abs() <= tol)
        assert not bad.any(), (i, n, int(bad.sum()), float((o[i].double() - O).abs().max()))


@gpu
@pytest.mark.parametrize("lens", [(1,), (63, 64, 65), (0, 5, 0, 1000, 128, 0), (2000,), (17,) * 70])
@pytest.mark.parametrize("heads", [(1, 1, 64), (12, 12, 64), (8, 2, 128), (6, 2, 72), (40, 2, 32), (16, 1, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_lengths_and_heads(lens, heads, dt):
    hq, hkv, d = heads
    q, k, v = _inputs(len(lens), max(lens) + 9, hq, hkv, d, dt, seed=sum(lens) + d)
    for i, n in enumerate(lens):   # what is behind the length does not matter
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    o = cp.decode_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32))
    _check(o, q, k, v, lens, d ** -0.5)


@gpu
@pytest.mark.parametrize("heads", [(6, 2, 64), (34, 1, 128)])
def test_more_sequences_than_ctas(heads):
    """Many short sequences, empty ones among them, and a long one that several CTAs share."""
    hq, hkv, d = heads
    gen = torch.Generator().manual_seed(hq)
    lens = torch.randint(0, 200, (1200,), generator=gen).tolist()
    lens[::17] = [0] * len(lens[::17])
    lens[600] = 3000
    q, k, v = _inputs(len(lens), 3000, hq, hkv, d, torch.bfloat16, seed=d)
    o = cp.decode_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32))
    _check(o, q, k, v, lens, d ** -0.5)
    assert torch.equal(o, cp.decode_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32)))


@gpu
@pytest.mark.parametrize("d", [8, 16, 24, 40, 56, 80, 96, 104, 112, 120])
def test_head_dims(d):
    lens = (300, 33)
    q, k, v = _inputs(2, 310, 4, 2, d, torch.bfloat16, seed=d)
    o = cp.decode_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32), scale=0.2)
    _check(o, q, k, v, lens, 0.2)


@gpu
def test_caches_in_place_and_lengths_out_of_range():
    lens = (100, 37, 256)
    q, k, v = _inputs(3, 256, 8, 4, 64, torch.bfloat16)
    n = torch.tensor(lens, device=DEV, dtype=torch.int32)
    want = cp.decode_attention(q, k, v, n)
    # heads before rows; a slice of a larger cache; one cache of keys and values side by side; q as a column range
    heads = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(cp.decode_attention(q, heads(k), heads(v), n), want)
    big = torch.full((5, 300, 4, 128), float("nan"), device=DEV, dtype=torch.bfloat16)
    big[1:4, 20:276, :, :64], big[1:4, 20:276, :, 64:] = k, v
    assert torch.equal(cp.decode_attention(q, big[1:4, 20:276, :, :64], big[1:4, 20:276, :, 64:], n), want)
    wide = torch.cat([q.flatten(1), q.flatten(1)], 1)[:, :512].unflatten(1, (8, 64))
    assert torch.equal(cp.decode_attention(wide, k, v, n), want)
    one = k[:1].expand(3, 256, 4, 64)
    assert torch.equal(cp.decode_attention(q, one, one, n), cp.decode_attention(q, one.contiguous(), one.contiguous(), n))
    got = cp.decode_attention(q, k, v, torch.tensor([-5, 1000, 37], device=DEV, dtype=torch.int32))
    assert torch.count_nonzero(got[0]) == 0 and torch.equal(
        got[1:], cp.decode_attention(q, k, v, torch.tensor([0, 256, 37], device=DEV, dtype=torch.int32))[1:])
    assert torch.count_nonzero(cp.decode_attention(q, k[:, :0], v[:, :0], n)) == 0
    assert cp.decode_attention(q[:0], k[:0], v[:0], n[:0]).shape == (0, 8, 64)
    with pytest.raises(ValueError, match="16-byte"):
        off = torch.empty(k.numel() + 1, device=DEV, dtype=k.dtype)[1:].view(k.shape)
        cp.decode_attention(q, off, v, n)


@gpu
@pytest.mark.parametrize("heads", [(12, 12, 64), (8, 2, 128)])
def test_same_bits_streams_and_graphs_with_growing_lengths(heads):
    hq, hkv, d = heads
    q, k, v = _inputs(5, 700, hq, hkv, d, torch.bfloat16)
    n = torch.tensor((1, 690, 300, 0, 64), device=DEV, dtype=torch.int32)
    first = cp.decode_attention(q, k, v, n)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(cp.decode_attention(q, k, v, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = cp.decode_attention(q, k, v, n)
    for lens in ((1, 690, 300, 0, 64), (2, 691, 301, 1, 65), (700, 700, 700, 700, 700)):
        n.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        _check(o, q, k, v, lens, d ** -0.5)


@gpu
def test_long_caches_and_offsets_past_32_bits():
    room, hkv, d = 600000, 16, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    k = torch.empty(2, room, hkv, d, device=DEV, dtype=torch.bfloat16)     # 2.5e9 elements
    lens = (50, room)
    k[0, :50].normal_()
    for i in range(0, room, 100000):
        k[1, i:i + 100000].normal_()
    q = torch.randn(2, hkv, d, device=DEV).bfloat16()
    n = torch.tensor(lens, device=DEV, dtype=torch.int32)
    o = cp.decode_attention(q, k, k, n)
    for h in (0, hkv - 1):   # (two of the heads: the rest only takes time)
        _check(o[:, h:h + 1], q[:, h:h + 1], k[:, :, h:h + 1], k[:, :, h:h + 1], lens, d ** -0.5)
    del k


@gpu
def test_traced_calls_agree_with_eager_ones():
    q, k, v = _inputs(3, 90, 4, 2, 64, torch.float16)
    n = torch.tensor((90, 1, 33), device=DEV, dtype=torch.int32)
    assert torch.equal(torch.ops.prism_b200.decode_attention(q, k, v, n, 0.125), cp.decode_attention(q, k, v, n))
