"""The operators that a decoder made of Prism layers needs around its linears, as measurable cases.

Three operators: layer norm (with or without the residual sum before it; forward, and forward + backward),
causal attention over whole prompts (packed sequences or a dense batch, grouped heads; forward, and
forward + backward), and attention of single tokens over their sequences' keys and values.  ``run`` with
``own`` false computes them from elementary torch operations in 32 bits; with ``own`` true it makes the calls
of the package.
"""
import math
import random

import torch

own = False   # set by whoever measures: False = elementary torch operations, True = the package's operators

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one generated token on its way through a block of the 768-wide decoder: latency alone
        {"name": "norm_one_token", "op": "norm", "rows": 1, "cols": 768, "dtype": "bf16", "weight": "bf16",
         "residual": True, "train": False},
        # a prompt batch of the 4096-wide layer, forward only
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "weight": "bf16",
         "residual": True, "train": False},
        # the norm before the MLP of the 768-wide decoder in training: 16 sequences of 1024
        {"name": "norm_train_decoder", "op": "norm", "rows": 16384, "cols": 768, "dtype": "bf16", "weight": "bf16",
         "residual": True, "train": True},
        # an odd width, fewer rows than a full batch, parameters kept in 32 bits
        {"name": "norm_train_odd", "op": "norm", "rows": 5003, "cols": 1537, "dtype": "fp16", "weight": "fp32",
         "residual": False, "train": True},
        # a chat turn: one short prompt through the 12 heads of the decoder
        {"name": "attention_short_prompt", "op": "attention", "sequences": 1, "longest": 77, "ragged": False, "mix": 0,
         "kv_heads": 12, "group": 1, "dim": 64, "dtype": "bf16", "train": False},
        # the decoder's training micro-batch: 16 sequences of 1024, 12 heads of 64
        {"name": "attention_train_decoder", "op": "attention", "sequences": 16, "longest": 1024, "ragged": False, "mix": 0,
         "kv_heads": 12, "group": 1, "dim": 64, "dtype": "bf16", "train": True},
        # packed documents of very different lengths, grouped heads of 128, in training
        {"name": "attention_train_packed", "op": "attention", "sequences": 24, "longest": 4096, "ragged": True, "mix": 5,
         "kv_heads": 8, "group": 4, "dim": 128, "dtype": "bf16", "train": True},
        # odd everything: 37 short prompts, heads of 80, groups of 3, fp16
        {"name": "attention_prompt_odd", "op": "attention", "sequences": 37, "longest": 701, "ragged": True, "mix": 3,
         "kv_heads": 5, "group": 3, "dim": 80, "dtype": "fp16", "train": False},
        # one long document
        {"name": "attention_long_prompt", "op": "attention", "sequences": 1, "longest": 16384, "ragged": False, "mix": 0,
         "kv_heads": 8, "group": 4, "dim": 128, "dtype": "bf16", "train": False},
        # one conversation of the decoder, one token: latency alone
        {"name": "decode_one", "op": "decode", "sequences": 1, "longest": 1000, "room": 1024, "ragged": False, "mix": 0,
         "kv_heads": 12, "group": 1, "dim": 64, "dtype": "bf16"},
        # a full serving batch at different positions, grouped heads
        {"name": "decode_batch", "op": "decode", "sequences": 64, "longest": 8000, "room": 8192, "ragged": True, "mix": 1,
         "kv_heads": 8, "group": 4, "dim": 128, "dtype": "bf16"},
        # two conversations over a very long text: few rows, the keys have to be split
        {"name": "decode_long", "op": "decode", "sequences": 2, "longest": 100003, "room": 100352, "ragged": True, "mix": 2,
         "kv_heads": 4, "group": 8, "dim": 96, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "attention", "decode"])
        case = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
        if op == "norm":
            case.update(rows=_log(rng, 1, 65536), cols=_log(rng, 64, 8192), weight=rng.choice([case["dtype"], "fp32"]),
                        residual=rng.random() < 0.5, train=rng.random() < 0.5)
            if rng.random() < 0.5:
                case["cols"] = max(64, case["cols"] // 64 * 64)
        else:
            case.update(kv_heads=rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), group=rng.choice([1, 1, 2, 3, 4, 5, 8]),
                        dim=rng.choice([32, 64, 64, 72, 80, 96, 128, 128]), ragged=rng.random() < 0.6, mix=rng.randrange(1 << 20))
            if op == "attention":
                case.update(sequences=_log(rng, 1, 48), longest=_log(rng, 1, 16384), train=rng.random() < 0.5)
            else:
                case.update(sequences=_log(rng, 1, 128), longest=_log(rng, 1, 100000))
                case["room"] = case["longest"] + rng.randrange(0, 1 + case["longest"] // 4)
        w, limit = work(case), _limit(op)
        if w["bytes"] <= limit["bytes"] and w["flops"] <= limit["flops"] and _held(case) <= 4 << 30:
            return case


def _limit(op):
    ws = [work(c) for c in listed() if c["op"] == op]
    return {k: max(w[k] for w in ws) for k in ("bytes", "flops")}


def _held(case):
    """Bytes of the inputs."""
    if case["op"] == "decode":
        return case["sequences"] * case["room"] * case["kv_heads"] * case["dim"] * 4
    return work(case)["bytes"]


def _lengths(case):
    """The sequences' lengths, the same for every seed: the longest, and the others spread down to one token (to
    an empty row of the batch for single tokens)."""
    n, top = case["sequences"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    rng = random.Random(case["mix"])
    out = [top] + [_log(rng, max(1, top // 64), top) for _ in range(n - 1)]
    rng.shuffle(out)
    return out


def work(case):
    size = 2
    if case["op"] == "norm":
        m, n = case["rows"], case["cols"]
        wsize = 4 if case["weight"] == "fp32" else 2
        tensors = (4 if case["residual"] else 2)                           # x (, residual) in, y (, sum) out
        if case["train"]:
            tensors += 3 if case["residual"] else 2                        # dy (, dsum) in, dx out
        return {"bytes": m * n * size * tensors + n * wsize * (4 if case["train"] else 2),
                "flops": m * n * (8 + (12 if case["train"] else 0))}
    lens, hkv, hq, d = _lengths(case), case["kv_heads"], case["kv_heads"] * case["group"], case["dim"]
    if case["op"] == "attention":
        pairs = sum(x * (x + 1) // 2 for x in lens)
        rows = sum(lens)
        tensors = rows * d * (2 * hq + 2 * hkv)                            # q, k, v in, o out
        if case["train"]:
            tensors += rows * d * (2 * hq + 2 * hkv)                       # do in, dq, dk, dv out
        # two products forward; four more backward (dP, dQ, dK, dV)
        return {"bytes": tensors * size, "flops": pairs * hq * d * 2 * (6 if case["train"] else 2)}
    keys = sum(lens)
    return {"bytes": (keys * hkv * d * 2 + case["sequences"] * hq * d * 2) * size, "flops": keys * hq * d * 4}


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 11)
    dt = _TYPES[case["dtype"]]
    st = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen, dtype=torch.float32)

    if case["op"] == "norm":
        m, n, train = case["rows"], case["cols"], case["train"]
        # a residual stream: rows of different size and offset, a few loud features
        loud = 1.0 + 6.0 * (torch.rand(n, device=dev, generator=gen) < 0.01).float()
        x = randn(m, n).mul_(loud).mul_(0.5 + torch.rand(m, 1, device=dev, generator=gen)).add_(0.3 * randn(m, 1))
        st["x"] = x.to(dt)
        st["weight"] = (1.0 + 0.1 * randn(n)).to(_TYPES[case["weight"]])
        st["bias"] = (0.1 * randn(n)).to(_TYPES[case["weight"]])
        st["residual"] = randn(m, n).to(dt) if case["residual"] else None
        if train:
            st["dy"] = randn(m, n).to(dt)
            st["dsum"] = randn(m, n).to(dt) if case["residual"] else None
            for name in ("x", "weight", "bias", "residual"):
                if st[name] is not None:
                    st[name].requires_grad_()
        return st
    hkv, hq, d = case["kv_heads"], case["kv_heads"] * case["group"], case["dim"]
    lens = _lengths(case)
    if case["op"] == "attention":
        rows = sum(lens)
        # queries, keys and values as they leave one linear layer: column ranges of one matrix
        qkv = randn(rows, (hq + 2 * hkv) * d).to(dt)
        q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=1)
        st["q"], st["k"], st["v"] = q.unflatten(1, (hq, d)), k.unflatten(1, (hkv, d)), v.unflatten(1, (hkv, d))
        st["lens"] = lens
        st["cu_seqlens"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        if not case["ragged"]:   # a dense batch is handed over as one
            shape = (len(lens), lens[0])
            for name in ("q", "k", "v"):
                st[name] = st[name].unflatten(0, shape)
            st["cu_seqlens"] = None
        if case["train"]:
            st["do"] = randn(*st["q"].shape).to(dt)
            for name in ("q", "k", "v"):
                st[name] = st[name].detach().requires_grad_()
        return st
    b, room = case["sequences"], case["room"]
    st["q"] = randn(b, hq, d).to(dt)
    st["k"] = torch.empty(b, room, hkv, d, device=dev, dtype=dt)
    st["v"] = torch.empty(b, room, hkv, d, device=dev, dtype=dt)
    for i in range(b):
        st["k"][i], st["v"][i] = randn(room, hkv, d), randn(room, hkv, d)
    st["lens"] = lens
    st["lengths"] = torch.tensor(lens, device=dev, dtype=torch.int32)
    return st


# --------------------------------------------------------------------------- the package's calls
def _run_own(st):
    import cute_mma_b200 as cp
    case = st["case"]
    if case["op"] == "norm":
        if not case["train"]:
            return cp.layer_norm(st["x"], st["weight"], st["bias"], eps=_EPS, residual=st["residual"])
        out = cp.layer_norm(st["x"], st["weight"], st["bias"], eps=_EPS, residual=st["residual"])
        if case["residual"]:
            y, s = out
            dx, dw, db = torch.autograd.grad([y, s], [st["x"], st["weight"], st["bias"]], [st["dy"], st["dsum"]])
            return y.detach(), s.detach(), dx, dw, db
        dx, dw, db = torch.autograd.grad(out, [st["x"], st["weight"], st["bias"]], st["dy"])
        return out.detach(), dx, dw, db
    if case["op"] == "attention":
        o = cp.causal_attention(st["q"], st["k"], st["v"], st["cu_seqlens"])
        if not case["train"]:
            return o
        return (o.detach(), *torch.autograd.grad(o, [st["q"], st["k"], st["v"]], st["do"]))
    return cp.decode_attention(st["q"], st["k"], st["v"], st["lengths"])


# --------------------------------------------------------------------------- the plain form
def _plain_norm(st):
    case = st["case"]
    dt = st["x"].dtype
    w, b = st["weight"].float(), st["bias"].float()
    s = st["x"].float()
    if case["residual"]:
        s = (s + st["residual"].float()).to(dt).float()     # the sum is an output; what is normalised is that output
    mean = s.mean(1, keepdim=True)
    c = s - mean
    rstd = (c * c).mean(1, keepdim=True).add(_EPS).rsqrt()
    xhat = c * rstd
    y = (xhat * w + b).to(dt)
    out = (y, s.to(dt)) if case["residual"] else (y,)
    if not case["train"]:
        return out if case["residual"] else y
    dy = st["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if case["residual"]:
        dx = dx + st["dsum"].float()
    wt = st["weight"].dtype
    return (*out, dx.to(dt), (dy * xhat).sum(0).to(wt), dy.sum(0).to(wt))


def _plain_attention(st):
    case = st["case"]
    hkv, g, d = case["kv_heads"], case["group"], case["dim"]
    dt = st["q"].dtype
    scale = d ** -0.5
    q, k, v = [st[n].reshape(-1, *st[n].shape[-2:]) for n in ("q", "k", "v")]
    outs = [torch.empty(q.shape, device=q.device, dtype=dt)]
    if case["train"]:
        do = st["do"].reshape(q.shape)
        outs += [torch.empty(t.shape, device=q.device, dtype=dt) for t in (q, k, v)]
    at = 0
    for n in st["lens"]:
        sl = slice(at, at + n)
        at += n
        step = max(1, min(hkv, (1 << 28) // (n * n * g)))
        keep = torch.ones(n, n, device=q.device, dtype=torch.bool).tril()
        for h in range(0, hkv, step):
            he = min(hkv, h + step)
            qh = q[sl, h * g:he * g].float().unflatten(1, (he - h, g)).permute(1, 2, 0, 3)   # heads, group, rows, dim
            kh = k[sl, h:he].float().permute(1, 0, 2).unsqueeze(1)
            vh = v[sl, h:he].float().permute(1, 0, 2).unsqueeze(1)
            p = torch.matmul(qh, kh.transpose(-1, -2)).mul_(scale).masked_fill_(~keep, float("-inf"))
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True))
            o = torch.matmul(p, vh)
            outs[0][sl, h * g:he * g] = o.permute(2, 0, 1, 3).flatten(1, 2).to(dt)
            if not case["train"]:
                continue
            doh = do[sl, h * g:he * g].float().unflatten(1, (he - h, g)).permute(1, 2, 0, 3)
            outs[3][sl, h:he] = torch.matmul(p.transpose(-1, -2), doh).sum(1).permute(1, 0, 2).to(dt)
            ds = torch.matmul(doh, vh.transpose(-1, -2)).sub_((doh * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            outs[1][sl, h * g:he * g] = torch.matmul(ds, kh).permute(2, 0, 1, 3).flatten(1, 2).to(dt)
            outs[2][sl, h:he] = torch.matmul(ds.transpose(-1, -2), qh).sum(1).permute(1, 0, 2).to(dt)
    outs[0] = outs[0].view(st["q"].shape)
    if not case["train"]:
        return outs[0]
    return (outs[0], outs[1].view(st["q"].shape), outs[2].view(st["k"].shape), outs[3].view(st["v"].shape))


def _plain_decode(st):
    case = st["case"]
    g, d = case["group"], case["dim"]
    out = torch.empty_like(st["q"])
    for i, n in enumerate(st["lens"]):
        qi = st["q"][i].float().unflatten(0, (-1, g))                       # kv heads, group, dim
        ki, vi = st["k"][i, :n].float().permute(1, 0, 2), st["v"][i, :n].float().permute(1, 0, 2)
        s = torch.matmul(qi, ki.transpose(1, 2)) * d ** -0.5
        p = (s - s.amax(-1, keepdim=True)).exp()
        out[i] = (torch.matmul(p, vi) / p.sum(-1, keepdim=True)).flatten(0, 1).to(out.dtype)
    return out


_PLAIN = {"norm": _plain_norm, "attention": _plain_attention, "decode": _plain_decode}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------------------- 64 bits, from the definitions
def _exact_norm(st):
    case = st["case"]
    dt = st["x"].dtype
    with torch.no_grad():
        s = st["x"].double()
        total = s
        if case["residual"]:
            total = s + st["residual"].double()
            s = (st["x"].float() + st["residual"].float()).to(dt).double()   # what is normalised is the rounded sum
    w, b = st["weight"].detach().double(), st["bias"].detach().double()
    if case["train"]:
        s.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    var, mean = torch.var_mean(s, dim=1, unbiased=False, keepdim=True)
    y = (s - mean) / torch.sqrt(var + _EPS) * w + b
    out = (y.detach(), total) if case["residual"] else (y.detach(),)
    if not case["train"]:
        return out if case["residual"] else out[0]
    dx, dw, db = torch.autograd.grad(y, [s, w, b], st["dy"].double())
    if case["residual"]:
        dx = dx + st["dsum"].double()
    return (*out, dx, dw, db)


def _exact_attention(st):
    """One head at a time, a band of query rows at a time, the gradients by automatic differentiation."""
    case = st["case"]
    g, d = case["group"], case["dim"]
    q, k, v = [st[n].detach().reshape(-1, *st[n].shape[-2:]) for n in ("q", "k", "v")]
    out = torch.zeros(q.shape, device=q.device, dtype=torch.float64)
    grads = [torch.zeros(t.shape, device=q.device, dtype=torch.float64) for t in (q, k, v)] if case["train"] else []
    do = st["do"].reshape(q.shape) if case["train"] else None
    start = 0
    for n in st["lens"]:
        end = start + n
        for h in range(q.shape[1]):
            kh, vh = k[start:end, h // g].double(), v[start:end, h // g].double()
            for r in range(0, n, 2048):
                re = min(n, r + 2048)
                leaves = [q[start + r:start + re, h].double(), kh[:re].clone(), vh[:re].clone()]
                if case["train"]:
                    leaves = [t.requires_grad_() for t in leaves]
                logits = torch.einsum("id,jd->ij", leaves[0], leaves[1]) / math.sqrt(d)
                later = torch.arange(re, device=q.device)[None, :] > torch.arange(r, re, device=q.device)[:, None]
                probs = torch.softmax(logits.masked_fill(later, float("-inf")), dim=1)
                o = torch.einsum("ij,jd->id", probs, leaves[2])
                out[start + r:start + re, h] = o.detach()
                if case["train"]:
                    dq, dk, dv = torch.autograd.grad(o, leaves, do[start + r:start + re, h].double())
                    grads[0][start + r:start + re, h] = dq
                    grads[1][start:start + re, h // g] += dk
                    grads[2][start:start + re, h // g] += dv
        start = end
    out = out.view(st["q"].shape)
    if not case["train"]:
        return out
    return (out, *[t.view(st[n].shape) for t, n in zip(grads, ("q", "k", "v"))])


def _exact_decode(st):
    case = st["case"]
    out = torch.zeros(st["q"].shape, device=st["q"].device, dtype=torch.float64)
    for i, n in enumerate(st["lens"]):
        for h in range(case["kv_heads"]):
            heads = slice(h * case["group"], (h + 1) * case["group"])
            logits = torch.einsum("gd,jd->gj", st["q"][i, heads].double(), st["k"][i, :n, h].double()) / math.sqrt(case["dim"])
            out[i, heads] = torch.einsum("gj,jd->gd", torch.softmax(logits, dim=1), st["v"][i, :n, h].double())
    return out


_EXACT = {"norm": _exact_norm, "attention": _exact_attention, "decode": _exact_decode}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
