"""The language-model operators of this library as measured cases.

Three families, one for each kind of contraction the library has in float64:

* ``linear`` / ``train``: the product of 8-bit floating-point matrices with a
  scale for each block of 128 (dense contraction).  ``linear`` is the serving
  form: 16- or 32-bit activations against stored 8-bit weights.  ``train`` is
  a training step of the layer: the output and both gradients.
* ``experts``: a whole mixture-of-experts layer for a few tokens (block-sparse
  contraction whose blocks the data choose).
* ``lookup`` / ``embed``: embedding rows with scaling (contraction with a
  one-hot tensor); ``embed`` adds the gradient of the table.

``run`` computes a case in its plain form from elementary torch operations in
32 bits, or, where ``own`` is true, with the library's calls.
"""

import math
import os
import sys

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
TINY = 2.0 ** -100
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _library():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ndtensors-rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import ndtensors_b200

    return ndtensors_b200


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one user's next token through one layer whose weights are read once: latency and bandwidth
        {"name": "linear 1 token", "op": "linear", "tokens": 1, "n": 10240, "k": 8192, "x": "bf16", "out": "bf16"},
        # a small decoding batch, nothing a multiple of a tile
        {"name": "linear 27 tokens, odd", "op": "linear", "tokens": 27, "n": 5003, "k": 2056, "x": "f16", "out": "f16"},
        # a prompt of ordinary length
        {"name": "linear 2048 tokens", "op": "linear", "tokens": 2048, "n": 8192, "k": 4096, "x": "bf16", "out": "bf16"},
        # the largest: a batch of prompts through a wide layer, results kept in 32 bits
        {"name": "linear 8192 tokens, wide", "op": "linear", "tokens": 8192, "n": 8192, "k": 8192, "x": "bf16", "out": "f32"},
        # a training step on a ragged micro-batch, weights in 32 bits
        {"name": "train 1000 tokens, odd", "op": "train", "tokens": 1000, "n": 1544, "k": 1111, "x": "bf16", "w": "f32"},
        # a training step of ordinary size
        {"name": "train 4096 tokens", "op": "train", "tokens": 4096, "n": 4096, "k": 4096, "x": "bf16", "w": "bf16"},
        # one token through a layer of small experts
        {"name": "experts 1 token", "op": "experts", "tokens": 1, "experts": 64, "top": 8, "h": 2048, "i": 1024,
         "w": "bf16", "renorm": True},
        # a handful of tokens, two experts each, odd sizes, weights of the full softmax
        {"name": "experts 5 tokens, odd", "op": "experts", "tokens": 5, "experts": 13, "top": 2, "h": 1000, "i": 1208,
         "w": "f16", "renorm": False},
        # a decoding batch that touches nearly every expert, 8-bit expert weights
        {"name": "experts 64 tokens, 8-bit", "op": "experts", "tokens": 64, "experts": 64, "top": 4, "h": 4096, "i": 1280,
         "w": "f8", "renorm": True},
        # the ids of one decoding step
        {"name": "lookup 16 tokens", "op": "lookup", "tokens": 16, "v": 50000, "d": 2048, "t": "bf16", "scale": 45.25},
        # a training batch: rows and the dense gradient of the table, ids by their frequency
        {"name": "embed 16384 tokens", "op": "embed", "tokens": 16384, "v": 65536, "d": 2048, "t": "bf16", "scale": 1.0},
        # a small ragged batch over a 32-bit table
        {"name": "embed 3001 tokens, odd", "op": "embed", "tokens": 3001, "v": 5003, "d": 771, "t": "f32", "scale": 27.75},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over the logarithm of [lo, hi]: a power of two, an odd multiple of 128 or of 8, or odd."""
    n = _log(rng, lo, hi)
    step = rng.choice((0, 128, 8, 1))
    if step == 0:
        n = 2 ** round(math.log2(n))
    elif n >= step:
        n = (n // (2 * step) * 2 + 1) * step
    return max(lo, min(n, hi))


def draw(rng):
    op = rng.choice(("linear", "linear", "train", "experts", "experts", "lookup", "embed"))
    if op == "linear":
        return {"op": op, "tokens": _size(rng, 1, 8192), "n": _size(rng, 128, 8192), "k": _size(rng, 128, 8192),
                "x": rng.choice(("bf16", "f16", "f32")), "out": rng.choice(("bf16", "f16", "f32"))}
    if op == "train":
        return {"op": op, "tokens": _size(rng, 64, 4096), "n": _size(rng, 128, 4096), "k": _size(rng, 128, 4096),
                "x": rng.choice(("bf16", "f16", "f32")), "w": rng.choice(("bf16", "f32"))}
    if op == "experts":
        w = rng.choice(("bf16", "f16", "f8"))
        return {"op": op, "tokens": _size(rng, 1, 64), "experts": rng.choice((8, 13, 32, 64)), "top": rng.choice((1, 2, 4, 8)),
                "h": _size(rng, 512, 4096), "i": _size(rng, 128, 1280 if w == "f8" else 640), "w": w,
                "renorm": rng.choice((True, False))}
    return {"op": op, "tokens": _size(rng, 1, 16384), "v": _size(rng, 1000, 65536), "d": _size(rng, 64, 2048),
            "t": rng.choice(("bf16", "f16", "f32")), "scale": rng.choice((1.0, 45.25))}


# ------------------------------------------------------------------ inputs


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, t, k, dtype):
    """Normal values of which a few channels are large, as hidden states are."""
    x = _normal(g, t, k)
    x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return x.to(dtype)


def _stored(w):
    """8-bit weights and the scales of their 128 x 128 blocks, as a checkpoint holds them (w: [..., rows, columns])."""
    r, c = w.shape[-2:]
    rb, cb = -(-r // 128), -(-c // 128)
    p = torch.nn.functional.pad(w, (0, cb * 128 - c, 0, rb * 128 - r)).unflatten(-1, (cb, 128)).unflatten(-3, (rb, 128))
    s = p.abs().amax((-3, -1)).clamp(min=TINY) / F8_MAX
    q = (p / s[..., :, None, :, None]).to(F8)
    return q.flatten(-2).flatten(-3, -2)[..., :r, :c].contiguous(), s


def _frequent(g, n, v):
    """Ids by rank of frequency (about 1 / rank), the ranks spread over the vocabulary."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp(0, v - 1)
    return torch.randperm(v, generator=g, device="cuda")[rank]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op == "linear":
        s["act"] = _activations(g, case["tokens"], case["k"], DTYPES[case["x"]])
        s["wq"], s["ws"] = _stored(_normal(g, case["n"], case["k"]) * case["k"] ** -0.5)
    elif op == "train":
        s["act"] = _activations(g, case["tokens"], case["k"], DTYPES[case["x"]]).requires_grad_()
        s["weight"] = (_normal(g, case["n"], case["k"]) * case["k"] ** -0.5).to(DTYPES[case["w"]]).requires_grad_()
        s["grad"] = (_normal(g, case["tokens"], case["n"]) * 1e-3).to(DTYPES[case["x"]])
    elif op == "experts":
        t, e, h, i = case["tokens"], case["experts"], case["h"], case["i"]
        dt = DTYPES["bf16" if case["w"] == "f8" else case["w"]]
        s["act"] = _normal(g, t, h).to(dt)
        s["router"] = (_normal(g, e, h) * h ** -0.5).to(dt)
        w_in, w_out = _normal(g, e, 2 * i, h) * h ** -0.5, _normal(g, e, h, i) * i ** -0.5
        s["in_scales"] = s["out_scales"] = None
        if case["w"] == "f8":
            s["w_in"], s["in_scales"] = _stored(w_in)
            s["w_out"], s["out_scales"] = _stored(w_out)
        else:
            s["w_in"], s["w_out"] = w_in.to(dt), w_out.to(dt)
    else:
        s["table"] = (_normal(g, case["v"], case["d"]) * 0.02).to(DTYPES[case["t"]])
        s["ids"] = _frequent(g, case["tokens"], case["v"])
        if op == "embed":
            s["table"].requires_grad_()
            s["grad"] = _normal(g, case["tokens"], case["d"]).to(DTYPES[case["t"]])
    return s


# ------------------------------------------------------------------ the plain forms


def _blocks(x, rows):
    """8-bit values (in 32 bits) of x [r, c] and the scales of its blocks of rows x 128, padded with zeros to whole blocks."""
    r, c = x.shape
    rb, cb = -(-r // rows), -(-c // 128)
    p = torch.nn.functional.pad(x.float(), (0, cb * 128 - c, 0, rb * rows - r)).view(rb, rows, cb, 128)
    s = p.abs().amax((1, 3)).clamp(min=TINY)
    s = s / torch.full_like(s, F8_MAX)  # a quotient: by a plain number torch multiplies with the reciprocal
    return (p / s[:, None, :, None]).to(F8).float(), s


def _rounded(x, rows):
    """What the block-scaled 8-bit form of x stands for, in 32 bits."""
    q, s = _blocks(x, rows)
    return (q * s[:, None, :, None]).flatten(2).flatten(0, 1)[: x.shape[0], : x.shape[1]]


def _stands_for(q, s):
    """The values of stored 8-bit weights [..., r, c] in 32 bits."""
    r, c = q.shape[-2:]
    return q.float() * s.repeat_interleave(128, -2)[..., :r, :].repeat_interleave(128, -1)[..., :c]


def _plain_linear(s):
    return (_rounded(s["act"], 1) @ _stands_for(s["wq"], s["ws"]).T).to(DTYPES[s["out"]])


def _plain_train(s):
    x, w, dy = s["act"].detach(), s["weight"].detach(), s["grad"]
    w8 = _rounded(w, 128)
    y = _rounded(x, 1) @ w8.T
    dx = _rounded(dy, 1) @ w8
    dw = _rounded(dy.T, 1) @ _rounded(x.T, 1).T
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(w.dtype)}


def _plain_experts(s):
    x = s["act"].float()
    t, k, e, i = x.shape[0], min(s["top"], s["experts"]), s["experts"], s["i"]
    logits = x @ s["router"].float().T
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
    weights = torch.gather(p, 1, ids)
    if s["renorm"]:
        weights = weights / weights.sum(1, keepdim=True)

    def values(w, scales, at):
        w, scales = (w, scales) if at is None else (w[at], None if scales is None else scales[at])
        return w.float() if scales is None else _stands_for(w, scales)

    if t * k <= e:  # few experts are touched: theirs alone are read
        at = ids.reshape(-1)
        a = torch.bmm(values(s["w_in"], s["in_scales"], at), x.repeat_interleave(k, 0)[:, :, None])[:, :, 0]
        g, u = a[:, :i], a[:, i:]
        o = torch.bmm(values(s["w_out"], s["out_scales"], at), (g / (1 + torch.exp(-g)) * u)[:, :, None])
        y = (o.view(t, k, -1) * weights[:, :, None]).sum(1)
    else:  # every expert on every token, the unchosen at weight zero
        a = torch.matmul(x, values(s["w_in"], s["in_scales"], None).transpose(1, 2))
        g, u = a[:, :, :i], a[:, :, i:]
        o = torch.matmul(g / (1 + torch.exp(-g)) * u, values(s["w_out"], s["out_scales"], None).transpose(1, 2))
        dense = torch.zeros(t, e, device=x.device).scatter_(1, ids, weights)
        y = (o * dense.T[:, :, None]).sum(0)
    return {"y": y.to(s["act"].dtype), "ids": ids.to(torch.int32), "weights": weights}


def _plain_lookup(s):
    table = s["table"].detach()
    return (table[s["ids"]].float() * s["scale"]).to(table.dtype)


def _plain_embed(s):
    table = s["table"].detach()
    g = torch.zeros(table.shape, device=table.device).index_add_(0, s["ids"], s["grad"].float())
    return {"out": _plain_lookup(s), "dtable": (g * s["scale"]).to(table.dtype)}


PLAIN = {"linear": _plain_linear, "train": _plain_train, "experts": _plain_experts, "lookup": _plain_lookup, "embed": _plain_embed}


# ------------------------------------------------------------------ the library's calls


def _own(s):
    ndt, op = _library(), s["op"]
    if op == "linear":
        return ndt.scaled_linear(s["act"], s["wq"], s["ws"], out_dtype=DTYPES[s["out"]])
    if op == "train":
        y = ndt.torch_scaled_linear(s["act"], s["weight"])
        dx, dw = torch.autograd.grad(y, (s["act"], s["weight"]), s["grad"])
        return {"y": y, "dx": dx, "dw": dw}
    if op == "experts":
        y, ids, weights = ndt.expert_layer(s["act"], s["router"], s["w_in"], s["w_out"], min(s["top"], s["experts"]),
                                           in_scales=s["in_scales"], out_scales=s["out_scales"], renormalize=s["renorm"])
        return {"y": y, "ids": ids, "weights": weights}
    if op == "lookup":
        return ndt.embedding(s["table"], s["ids"], scale=s["scale"])
    out = ndt.torch_embedding(s["table"], s["ids"], scale=s["scale"])
    return {"out": out, "dtable": torch.autograd.grad(out, s["table"], s["grad"])[0]}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ------------------------------------------------------------------ work


def work(case):
    op, t = case["op"], case["tokens"]
    size = {"bf16": 2, "f16": 2, "f32": 4, "f8": 1}
    if op == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": t * k * size[case["x"]] + n * k + 4 * -(-n // 128) * -(-k // 128) + t * n * size[case["out"]],
                "flops": 2 * t * n * k}
    if op == "train":
        n, k = case["n"], case["k"]
        return {"bytes": size[case["x"]] * 2 * (t * k + t * n) + size[case["w"]] * 2 * n * k, "flops": 6 * t * n * k}
    if op == "experts":
        e, k, h, i = case["experts"], min(case["top"], case["experts"]), case["h"], case["i"]
        touched = e * (1 - (1 - k / e) ** t)  # the mean number of experts that t tokens choose among
        act = 2
        return {"bytes": act * (e * h + 2 * t * h) + touched * 3 * h * i * size[case["w"]] + 8 * t * k,
                "flops": 2 * t * h * e + 6 * t * k * h * i}
    b, v, d = size[case["t"]], case["v"], case["d"]
    rows = min(t, v)
    bytes_ = 8 * t + rows * d * b + t * d * b
    return {"bytes": bytes_ if op == "lookup" else bytes_ + t * d * b + v * d * b, "flops": t * d * (1 if op == "lookup" else 2)}


# ------------------------------------------------------------------ in 64 bits


def _round8(v):
    """float64 values to the nearest e4m3 value, ties to even, in float64."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20)))
    e = torch.where(torch.ldexp(torch.ones_like(v), e) > v.abs(), e - 1, e)
    step = torch.ldexp(torch.ones_like(v), e.clamp(min=-6.0) - 3)
    return (torch.round(v / step) * step).clamp(-F8_MAX, F8_MAX)


def _exact8(x, rows):
    """x [r, c] in its block-scaled 8-bit form, block by block of columns; scales and quotients are 32-bit numbers by definition."""
    x = x.double()
    out = torch.empty_like(x)
    r = x.shape[0]
    for c in range(0, x.shape[1], 128):
        part = x[:, c : c + 128]
        top = part.abs().amax(1)
        if rows > 1:
            n = -(-r // rows)
            top = torch.nn.functional.pad(top, (0, n * rows - r)).view(n, rows).amax(1).repeat_interleave(rows)[:r]
        scale = (top.clamp(min=TINY) / F8_MAX).float().double()[:, None]
        out[:, c : c + 128] = _round8((part / scale).float().double()) * scale
    return out


def _exact_stored(q, s):
    r, c = q.shape
    out = q.float().double()
    for i in range(0, r, 128):
        out[i : i + 128] *= s[i // 128].double().repeat_interleave(128)[:c]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact8(s["act"], 1) @ _exact_stored(s["wq"], s["ws"]).T
    if op == "train":
        x, w, dy = s["act"].detach(), s["weight"].detach(), s["grad"]
        w8 = _exact8(w, 128)
        return {"y": _exact8(x, 1) @ w8.T, "dx": _exact8(dy, 1) @ w8,
                "dw": _exact8(dy.T, 1) @ _exact8(x.T, 1).T}
    if op == "experts":
        x = s["act"].double()
        k, i = min(case["top"], case["experts"]), case["i"]
        p = torch.softmax(x @ s["router"].double().T, 1)
        weights, ids = torch.topk(p, k, dim=1)
        if case["renorm"]:
            weights = weights / weights.sum(1, keepdim=True)
        y = torch.zeros_like(x)
        for e in range(case["experts"]):
            t, j = torch.nonzero(ids == e, as_tuple=True)
            if not len(t):
                continue
            w_in, w_out = ((_exact_stored(s[w][e], s[c][e]) if s[c] is not None else s[w][e].double())
                           for w, c in (("w_in", "in_scales"), ("w_out", "out_scales")))
            a = x[t] @ w_in.T
            y.index_add_(0, t, weights[t, j][:, None] * ((torch.nn.functional.silu(a[:, :i]) * a[:, i:]) @ w_out.T))
        return {"y": y, "ids": None, "weights": weights}
    table = s["table"].detach().double()
    out = table[s["ids"]] * case["scale"]
    if op == "lookup":
        return out
    grad = torch.zeros_like(table)
    grad.index_put_((s["ids"],), s["grad"].double() * case["scale"], accumulate=True)
    return {"out": out, "dtable": grad}
