"""The decoder's operators together, as a model uses them: norm -> QKV -> attention -> projection -> residual and norm -> MLP,
trained on packed sequences, and the next token served from the keys and values of the prompt."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as TF

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"
D, HEADS, KV, DH = 256, 4, 2, 64


class Block(nn.Module):
    def __init__(self):
        super().__init__()
        lin = lambda i, o: cp.PrismLinear(i, o, group_size=64, reconn_sz=16, activation="silu_gate")
        self.ln1, self.ln2 = cp.LayerNorm(D), cp.LayerNorm(D)
        self.qkv, self.proj = lin(D, (HEADS + 2 * KV) * DH), lin(HEADS * DH, D)
        self.up, self.down = lin(D, 4 * D), lin(4 * D, D)

    def split(self, h):
        return self.qkv(h).unflatten(-1, (HEADS + 2 * KV, DH)).split([HEADS, KV, KV], -2)

    def rest(self, o, x):
        h, x = self.ln2(self.proj(o.flatten(-2)), x)
        return x + self.down(TF.gelu(self.up(h)))

    def forward(self, x, cu):
        q, k, v = self.split(self.ln1(x))
        return self.rest(cp.causal_attention(q, k, v, cu), x), k, v


class Plain(nn.Module):
    """The same in elementary operations, 64 bits, with the block's parameters.  ``step`` > 0: every intermediate value, and
    every gradient on its way back through it, is off by a random relative error of up to that."""

    def __init__(self, block, step=0.0):
        super().__init__()
        self.p = nn.ParameterDict({k.replace(".", "_"): nn.Parameter(t.detach().double()) for k, t in block.named_parameters()})
        self.step, self.gen = step, torch.Generator(device=DEV).manual_seed(77)

    def off(self, x):
        if not self.step:
            return x
        noise = lambda t: 1 + self.step * (2 * torch.rand(t.shape, device=DEV, generator=self.gen, dtype=torch.float64) - 1)
        y = x * noise(x)
        y.register_hook(lambda g: g * noise(g))
        return y

    def norm(self, x, name):
        mean, var = x.mean(-1, keepdim=True), x.var(-1, unbiased=False, keepdim=True)
        return self.off((x - mean) / torch.sqrt(var + 1e-5) * self.p[name + "_weight"] + self.p[name + "_bias"])

    def lin(self, x, name, gs=64, rs=16):
        B, R, bias = (self.p[f"{name}_{n}"] for n in ("weight", "reconn", "bias"))
        n, k = B.shape
        out = []
        for g in range(n // gs):
            r = R[g * rs:(g + 1) * rs].view(rs, k // rs, rs)                       # [i, block, j]
            s = self.off(torch.einsum("mbj,ibj->mbi", x.view(-1, k // rs, rs), r).flatten(1))
            out.append(self.off(x * self.off(s * self.off(torch.sigmoid(s)))) @ B[g * gs:(g + 1) * gs].T)
        return self.off(torch.cat(out, 1) + bias)

    def forward(self, x, lens):
        q, k, v = self.lin(self.norm(x, "ln1"), "qkv").unflatten(-1, (HEADS + 2 * KV, DH)).split([HEADS, KV, KV], -2)
        o, at = [], 0
        for n in lens:
            s = torch.einsum("ihd,jhd->hij", q[at:at + n], k[at:at + n].repeat_interleave(HEADS // KV, 1)) * DH ** -0.5
            s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=x.device).tril(), float("-inf"))
            o.append(torch.einsum("hij,jhd->ihd", self.off(torch.softmax(s, -1)), v[at:at + n].repeat_interleave(HEADS // KV, 1)))
            at += n
        x = self.off(x + self.lin(self.off(torch.cat(o).flatten(1)), "proj"))
        return self.off(x + self.lin(self.off(TF.gelu(self.lin(self.norm(x, "ln2"), "up"))), "down"))


def _block(dt):
    torch.manual_seed(0)
    return Block().to(DEV).to(dt)


@gpu
def test_training_step_on_packed_sequences():
    """Outputs and gradients against the 64-bit block.  Tolerance: four times what one rounding of fp16 (2^-11) at every
    intermediate, forward and backward, does to that block itself; the gate's approximate tanh and its several roundings
    (each of the same size) are what the factor is for."""
    lens = (70, 1, 129, 56)
    block = _block(torch.float16)
    # (the gated layer scales its backward by a constant that a plain derivative does not have)
    for m in block.modules():
        if isinstance(m, cp.PrismLinear):
            m._bwd_scale = 1.0
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(sum(lens), D, device=DEV, generator=gen).half()
    do = torch.randn(sum(lens), D, device=DEV, generator=gen).half()
    cu = torch.tensor([0] + list(lens), device=DEV).cumsum(0).to(torch.int32)
    xa = x.clone().requires_grad_()
    y, _, _ = block(xa, cu)
    y.backward(do)
    cp.check_device_status()
    exact, noisy = Plain(block), Plain(block, 2.0 ** -11)
    results = []
    for plain in (exact, noisy):
        xb = x.double().requires_grad_()
        z = plain(xb, lens)
        z.backward(do.double())
        results.append({"y": z.detach(), "x": xb.grad, **{n: p.grad for n, p in plain.p.items()}})
    got = {"y": y.detach(), "x": xa.grad, **{n.replace(".", "_"): p.grad for n, p in block.named_parameters()}}
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())
    for name, t in results[0].items():
        assert rel(got[name], t) < 4 * rel(results[1][name], t), (name, rel(got[name], t), rel(results[1][name], t))


@gpu
@torch.no_grad()
def test_next_token_from_the_prompts_cache():
    """One token more through decode_attention gives what the prompt with that token gives, to the roundings of its attention
    (P in 16 bits: 2^-8 a value at most on each side, through the rest of the block)."""
    lens = (40, 1, 129)
    block = _block(torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(3)
    xs = [torch.randn(n + 1, D, device=DEV, generator=gen).bfloat16() for n in lens]
    cu = torch.tensor([0] + [n + 1 for n in lens], device=DEV).cumsum(0).to(torch.int32)
    whole, _, _ = block(torch.cat(xs), cu)
    want = whole[(cu[1:] - 1).long()]
    cu = torch.tensor([0] + list(lens), device=DEV).cumsum(0).to(torch.int32)
    _, k, v = block(torch.cat([x[:-1] for x in xs]), cu)
    room = 160
    cache = torch.empty(2, len(lens), room, KV, DH, device=DEV, dtype=torch.bfloat16).fill_(float("nan"))
    for i, n in enumerate(lens):
        cache[0, i, :n], cache[1, i, :n] = k[cu[i]:cu[i + 1]], v[cu[i]:cu[i + 1]]
    x = torch.stack([t[-1] for t in xs])
    q, k1, v1 = block.split(block.ln1(x))
    at = torch.tensor(lens, device=DEV)
    rows = torch.arange(len(lens), device=DEV)
    cache[0, rows, at], cache[1, rows, at] = k1, v1
    got = block.rest(cp.decode_attention(q, cache[0], cache[1], (at + 1).to(torch.int32)), x)
    cp.check_device_status()
    err = (got.float() - want.float()).norm() / want.float().norm()
    assert err < 2 * 2.0 ** -8, float(err)
