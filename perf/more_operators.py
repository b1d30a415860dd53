"""What the 8-bit operators and the loss of this library are measured on: conversion to 8-bit floating point with a scale
for each block of 128, products of such matrices, plain and grouped by expert, a gated activation that keeps its input in 8
bits for the backward pass, and softmax cross entropy over a large vocabulary with its gradient.

A case is a dict of plain values; `op` names the operator.  `own` chooses between the library's entry points and the
operators' plain form in elementary torch operations, in 32 bits, rounded once at the end.

    listed()              the cases that stand for the ranges
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   inputs and output buffers, on the GPU
    run(state)            one pass; returns the outputs
    work(case)            bytes and operations that one pass cannot do without
    exact(case, seed)     the outputs from the definitions in 64 bits
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}
# Of each format: bits of mantissa, exponent of the smallest normal value, largest value.
_FORMATS = {"e4m3": (3, -6, 448.0), "e5m2": (2, -14, 57344.0)}
LARGEST_FLOPS = 8.0 * 4096 * 32768 * 4096
LARGEST_BYTES = 1.5e9

_module = None


def _package():
    global _module
    if _module is None:
        from __graft_entry__ import load_package
        _module = load_package()
        _module.init(0)
    return _module


def listed():
    return [
        # Activations of a short prefill on their way into 8 bits (and back, which is how what was kept is looked at).  Latency.
        dict(name="fp8_activations", op="convert", rows=128, k=4096, type="bf16", format="e4m3", square=False, turned=False),
        # A whole layer's weights, one scale for 128 x 128.
        dict(name="fp8_weights", op="convert", rows=8192, k=8192, type="f16", format="e4m3", square=True, turned=False),
        # A projection of a short prompt, odd sizes throughout, Float32 results.
        dict(name="fp8_ragged", op="product", m=509, n=656, k=720, out="f32", format="e4m3"),
        # A projection over a prefill.
        dict(name="fp8_forward", op="product", m=4096, n=4096, k=8192, out="bf16", format="e4m3"),
        # The experts' first projection in a decoding step of 32 sequences, weights kept in 8 bits.
        dict(name="fp8_grouped_decode", op="grouped", tokens=32, experts=64, top=4, n=2048, k=2048, out="f16", format="e4m3", skew=0.0, gated=False),
        # The same over a training batch with uneven loads, the activation with it.
        dict(name="fp8_grouped_train", op="grouped", tokens=8192, experts=8, top=2, n=4096, k=4096, out="bf16", format="e4m3", skew=0.5, gated=True),
        # The activation of a short sequence, its input kept in 8 bits, and its gradient.
        dict(name="kept_small", op="kept", rows=61, n=2048, type="f16"),
        # The same over the rows of a training batch.
        dict(name="kept_train", op="kept", rows=16381, n=8192, type="bf16"),
        # How likely a few tokens are: sixteen rows against the vocabulary.  Bound by reading the vocabulary's vectors.
        dict(name="loss_few", op="loss", tokens=16, vocabulary=32768, width=4096, type="bf16", grad=False, ignored=0.0),
        # Scores of a validation batch.
        dict(name="loss_scores", op="loss", tokens=8192, vocabulary=32003, width=2048, type="bf16", grad=False, ignored=0.1),
        # A short sequence's step, odd sizes, with both gradients.
        dict(name="loss_ragged", op="loss", tokens=509, vocabulary=4999, width=720, type="f16", grad=True, ignored=0.3),
        # A training batch's loss with both gradients.  The largest.
        dict(name="loss_train", op="loss", tokens=4096, vocabulary=32768, width=4096, type="bf16", grad=True, ignored=0.05),
    ]


def _size(rng, low, high, step=1):
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def _width(rng, low, high):
    """An extent of a matrix: half of them multiples of 64, the others of 16 or of 8."""
    return _size(rng, low, high, rng.choice((64, 64, 16, 8)))


def _draw(rng):
    op = rng.choice(("convert", "product", "product", "grouped", "grouped", "kept", "loss", "loss", "loss"))
    kind = rng.choice(("f16", "bf16"))
    form = rng.choice(("e4m3", "e4m3", "e5m2"))
    if op == "convert":
        return dict(op=op, rows=_size(rng, 1, 8192), k=_size(rng, 64, 8192, rng.choice((128, 32, 1))), type=rng.choice(("f16", "bf16", "f32")), format=form,
                    square=rng.random() < 0.4, turned=rng.random() < 0.3)
    if op == "product":
        return dict(op=op, m=_size(rng, 1, 4096), n=_width(rng, 256, 8192), k=_size(rng, 256, 8192, rng.choice((128, 16, 1))), out=rng.choice((kind, "f32")), format=form)
    if op == "grouped":
        experts = _size(rng, 4, 64)
        return dict(op=op, tokens=_size(rng, 1, 8192), experts=experts, top=rng.randint(1, min(8, experts)), n=_width(rng, 256, 4096), k=_size(rng, 256, 4096, rng.choice((128, 16, 1))),
                    out=rng.choice((kind, "f32")), format=form, skew=rng.choice((0.0, 0.5, 1.5)), gated=rng.random() < 0.4)
    if op == "kept":
        return dict(op=op, rows=_size(rng, 1, 16384), n=_size(rng, 256, 8192, rng.choice((128, 16, 2))), type=kind)
    return dict(op=op, tokens=_size(rng, 1, 8192), vocabulary=_size(rng, 512, 65536, rng.choice((256, 8, 1))), width=_width(rng, 256, 4096), type=kind, grad=rng.random() < 0.6,
                ignored=rng.choice((0.0, 0.1, 0.6)))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= LARGEST_FLOPS and w["bytes"] <= LARGEST_BYTES:
            return case


def _used(case):
    """Experts that some row goes to, as many as there are on average with even loads."""
    rows, experts = case["tokens"] * case["top"], case["experts"]
    return experts * (1 - (1 - 1 / experts) ** rows)


def work(case):
    op = case["op"]
    code = 1 + 1 / 128  # bytes of a value in 8 bits
    if op == "convert":
        return {"bytes": case["rows"] * case["k"] * (_SIZE[case["type"]] + 2 * code + 2), "flops": 2.0 * case["rows"] * case["k"]}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + n * k) * code + _SIZE[case["out"]] * m * n, "flops": 2.0 * m * n * k}
    if op == "grouped":
        rows, n, k = case["tokens"] * case["top"], case["n"], case["k"]
        return {"bytes": (case["tokens"] * k + _used(case) * n * k) * code + _SIZE[case["out"]] * rows * n / (2 if case["gated"] else 1), "flops": 2.0 * rows * n * k}
    if op == "kept":
        # forward: Z read, A and what is kept written; back: what was kept and dA read, dZ and A written
        return {"bytes": case["rows"] * case["n"] * (2 + 1 + code + code + 1 + 2 + 1), "flops": 12.0 * case["rows"] * case["n"]}
    t, v, d, s = case["tokens"], case["vocabulary"], case["width"], _SIZE[case["type"]]
    both = s * (t + v) * d
    return {"bytes": both + 12.0 * t + case["grad"] * (2 * both + 8.0 * t), "flops": (8.0 if case["grad"] else 2.0) * t * v * d}


def _assignments(gen, case):
    """`top` different experts for every token, some likelier than others by `skew`; sorted by expert: where each expert's
    positions start, and the token at each position."""
    t, e, top = case["tokens"], case["experts"], case["top"]
    score = torch.rand((t, e), device="cuda", generator=gen) + case["skew"] * torch.rand((e,), device="cuda", generator=gen)
    chosen = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :top].reshape(-1)
    group, order = torch.sort(chosen, stable=True)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum((group[:, None] == torch.arange(e, device="cuda")).sum(0), 0)
    return offsets, (order // top).to(torch.int32)


# ---- 8-bit matrices: codes, rows of 128 ceil(k / 128) bytes, and scales, in panels of four blocks (512 values of k) the rows of
# which lie one after the other, four bytes each, rows rounded up to a multiple of four.

def _panels(rows, k):
    return -(-k // 512), -(-rows // 4) * 4, 4


def _padded(x):
    rows, k = x.shape
    p = torch.zeros((rows, -(-k // 128) * 128), dtype=x.dtype, device=x.device)
    p[:, :k] = x
    return p.view(rows, -1, 128)


def _exponents(top, form):
    """The smallest e with top <= largest 2^e, kept in -127 .. 127; and the scales' bytes."""
    mantissa, exponent = torch.frexp(top)  # top = mantissa 2^exponent, 0.5 <= mantissa < 1; both formats' largest is 0.875 2^n
    largest = {"e4m3": 9, "e5m2": 16}[form]
    e = torch.where(top > 0, exponent - largest + (mantissa > 0.875).to(exponent.dtype), -127).clamp(-127, 127)
    return e, torch.where(torch.isfinite(top), e + 127, 255).to(torch.uint8)


def _quantize(x, form, square=False):
    """(rounded values over their block's scale, exponents of the scales) of a Float32 matrix, rows x blocks x 128."""
    v = _padded(x)
    top = v.abs().amax(-1)
    if square:
        rows, blocks = top.shape
        tall = torch.zeros((-(-rows // 128) * 128, blocks), dtype=top.dtype, device=top.device)
        tall[:rows] = top
        top = tall.view(-1, 128, blocks).amax(1).repeat_interleave(128, 0)[:rows]
    e, _ = _exponents(top, form)
    scaled = torch.ldexp(v, -e[..., None])
    bits, lowest, _ = _FORMATS[form]
    step = torch.ldexp(torch.ones_like(scaled), (torch.frexp(scaled)[1] - 1).clamp(min=lowest) - bits)
    return torch.round(scaled / step) * step, e


def _codes(gen, rows, k, scale, form, square=False):
    """Codes and scales as converting a normal matrix of that standard deviation leaves them."""
    q, e = _quantize(torch.empty((rows, k), device="cuda").normal_(0.0, scale, generator=gen), form, square)
    kind = torch.float8_e4m3fn if form == "e4m3" else torch.float8_e5m2
    panels = torch.zeros(_panels(rows, k), dtype=torch.uint8, device="cuda")
    flat = torch.zeros((panels.shape[1], panels.shape[0] * 4), dtype=torch.uint8, device="cuda")
    flat[:rows, :e.shape[1]] = (e + 127).to(torch.uint8)
    panels.copy_(flat.view(panels.shape[1], -1, 4).transpose(0, 1))
    return q.view(rows, -1).to(kind).view(torch.uint8), panels


def _row_exponents(codes, panels):
    """One row of scales' exponents for each row of codes."""
    return panels.transpose(0, 1).reshape(panels.shape[1], -1)[:codes.shape[0], :codes.shape[1] // 128].int() - 127


def _values(codes, panels, k, form):
    kind = torch.float8_e4m3fn if form == "e4m3" else torch.float8_e5m2
    q = codes.view(kind).float().view(codes.shape[0], -1, 128)
    return torch.ldexp(q, _row_exponents(codes, panels)[..., None]).view(codes.shape[0], -1)[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    state = dict(case)

    def normal(shape, scale, kind):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen).to(_TORCH[kind])

    def empty(shape, kind):
        return torch.zeros(shape, dtype=_TORCH.get(kind, kind), device="cuda")

    if op == "convert":
        rows, k = case["rows"], case["k"]
        # rows of different size, a few of zeros
        x = torch.empty((rows, k), device="cuda").normal_(0.0, 1.0, generator=gen) * torch.exp(torch.randn((rows, 1), device="cuda", generator=gen))
        x[torch.rand(rows, device="cuda", generator=gen) < 0.01] = 0.0
        x = x.to(_TORCH[case["type"]])
        state.update(x=x.t().contiguous() if case["turned"] else x, codes=empty((rows, -(-k // 128) * 128), torch.uint8), scales=empty(_panels(rows, k), torch.uint8),
                     back=empty((rows, k), "bf16"))
    elif op == "product":
        state.update(a=_codes(gen, case["m"], case["k"], 1.0, case["format"]), b=_codes(gen, case["n"], case["k"], 0.02, "e4m3", True), y=empty((case["m"], case["n"]), case["out"]))
    elif op == "grouped":
        n, k, e, rows = case["n"], case["k"], case["experts"], case["tokens"] * case["top"]
        offsets, gather = _assignments(gen, case)
        codes, scales = zip(*(_codes(gen, n, k, 0.02, "e4m3", True) for _ in range(e)))
        state.update(offsets=offsets, gather=gather, bounds=offsets.tolist(), a=_codes(gen, case["tokens"], k, 1.0, case["format"]), b=(torch.stack(codes), torch.stack(scales)),
                     y=empty((rows, n // 2 if case["gated"] else n), case["out"]), rows=rows)
    elif op == "kept":
        rows, n, kind = case["rows"], case["n"], case["type"]
        state.update(z=normal((rows, n), 1.5, kind), da=normal((rows, n // 2), 1.0, kind), a=empty((rows, n // 2), kind), again=empty((rows, n // 2), kind), dz=empty((rows, n), kind),
                     codes=empty((rows, -(-n // 128) * 128), torch.uint8), scales=empty(_panels(rows, n), torch.uint8))
    else:
        t, v, d, kind = case["tokens"], case["vocabulary"], case["width"], case["type"]
        # hidden rows of unit size against vectors that make logits of a standard deviation of two; some tokens count nothing
        targets = torch.randint(0, v, (t,), device="cuda", generator=gen).to(torch.int32)
        targets[torch.rand(t, device="cuda", generator=gen) < case["ignored"]] = -1
        state.update(x=normal((t, d), 1.0, kind), w=normal((v, d), 2.0 / math.sqrt(d), kind), targets=targets, losses=empty(t, "f32"), lse=empty(t, "f32"))
        if case["grad"]:  # each token's share of the mean, a few weighted otherwise
            share = torch.rand(t, device="cuda", generator=gen).add_(0.5).div_(t)
            state.update(share=share, dx=empty((t, d), kind), dw=empty((v, d), kind))
    if own:
        pkg = _package()
        kinds = {"f16": pkg.WMMA.Float16, "bf16": pkg.BFloat16, "f32": pkg.WMMA.Float32}
        state.update(pkg=pkg, kind=kinds.get(case.get("type")), out_kind=kinds.get(case.get("out")), address={key: _address(v) for key, v in state.items()})
        if op == "loss":
            need = pkg.LOSS.cross_entropy_workspace(case["tokens"], case["vocabulary"], case["width"], grad=case["grad"])
            state["workspace"] = pkg.DeviceArray.undef(np.uint8, max(16, need))
    return state


def _address(v):
    """Raw addresses of a tensor or of several, as the entry points take them."""
    if isinstance(v, torch.Tensor):
        return v.data_ptr()
    return tuple(map(_address, v)) if isinstance(v, tuple) else None


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    op, at, pkg = s["op"], s["address"], s["pkg"]
    Q, L = pkg.FP8, pkg.LOSS
    form = {"e4m3": Q.E4M3, "e5m2": Q.E5M2}.get(s.get("format"))
    if op == "convert":
        Q.quantize(at["x"], at["codes"], at["scales"], rows=s["rows"], k=s["k"], dtype=s["kind"], format=form, block_rows=128 if s["square"] else 1,
                   x_layout=pkg.WMMA.ColMajor if s["turned"] else pkg.WMMA.RowMajor)
        Q.dequantize(at["codes"], at["scales"], at["back"], rows=s["rows"], k=s["k"], dtype=pkg.BFloat16, format=form)
        return s["back"]
    if op == "product":
        Q.gemm(*at["a"], *at["b"], at["y"], m=s["m"], n=s["n"], k=s["k"], d_type=s["out_kind"], a_format=form)
        return s["y"]
    if op == "grouped":
        Q.grouped_gemm(*at["a"], *at["b"], at["y"], at["offsets"], rows=s["rows"], groups=s["experts"], n=s["n"], k=s["k"], d_type=s["out_kind"], a_format=form,
                       gather=at["gather"], a_rows=s["tokens"], epilogue=pkg.EXPERTS.GATED_SILU if s["gated"] else None)
        return s["y"]
    if op == "kept":
        Q.gated_silu(at["z"], at["a"], at["codes"], at["scales"], rows=s["rows"], n=s["n"], dtype=s["kind"])
        Q.gated_silu_grad(at["codes"], at["scales"], at["da"], at["dz"], A=at["again"], rows=s["rows"], n=s["n"], dtype=s["kind"])
        return [s["a"], s["dz"], s["again"]]
    sizes = dict(tokens=s["tokens"], vocabulary=s["vocabulary"], width=s["width"], dtype=s["kind"], workspace=s["workspace"])
    L.cross_entropy(at["x"], at["w"], at["targets"], at["losses"], at["lse"], **sizes)
    if not s["grad"]:
        return [s["losses"], s["lse"]]
    L.cross_entropy_grad(at["x"], at["w"], at["targets"], at["lse"], at["share"], at["dx"], at["dw"], **sizes)
    return [s["losses"], s["lse"], s["dx"], s["dw"]]


def _gated(y):
    u, v = y[:, 0::2], y[:, 1::2]
    return u / (1 + torch.exp(-u)) * v


def _plain(s):
    op = s["op"]
    if op == "convert":
        q, e = _quantize((s["x"].t() if s["turned"] else s["x"]).float(), s["format"], s["square"])
        return torch.ldexp(q, e[..., None]).view(s["rows"], -1)[:, :s["k"]].to(torch.bfloat16)
    if op == "product":
        return (_values(*s["a"], s["k"], s["format"]) @ _values(*s["b"], s["k"], "e4m3").t()).to(s["y"].dtype)
    if op == "grouped":
        a = _values(*s["a"], s["k"], s["format"])[s["gather"].long()]
        y = torch.cat([a[i:j] @ _values(s["b"][0][g], s["b"][1][g], s["k"], "e4m3").t() for g, (i, j) in enumerate(zip(s["bounds"], s["bounds"][1:]))])
        return (_gated(y) if s["gated"] else y).to(s["y"].dtype)
    if op == "kept":
        z, kind = s["z"].float(), s["z"].dtype
        q, e = _quantize(z, "e4m3")
        kept = torch.ldexp(q, e[..., None]).view(s["rows"], -1)[:, :s["n"]]
        u, v, da = kept[:, 0::2], kept[:, 1::2], s["da"].float()
        gate = 1 / (1 + torch.exp(-u))
        dz = torch.stack((da * v * gate * (1 + u * (1 - gate)), da * u * gate), -1).view(s["rows"], -1)
        return [_gated(z).to(kind), dz.to(kind), _gated(kept).to(kind)]
    x, w, some, target = s["x"].float(), s["w"].float(), s["targets"] >= 0, s["targets"].long().clamp(min=0)
    z = x @ w.t()
    most = z.amax(1)
    lse = torch.log(torch.exp(z - most[:, None]).sum(1)) + most
    losses = torch.where(some, lse - z.gather(1, target[:, None])[:, 0], 0.0)
    if not s["grad"]:
        return [losses, lse]
    share = torch.where(some, s["share"], 0.0)
    p = torch.exp(z - lse[:, None]) * share[:, None]
    p.scatter_add_(1, target[:, None], -share[:, None])
    return [losses, lse, (p @ w).to(s["dx"].dtype), (p.t() @ x).to(s["dw"].dtype)]


# ---- the definitions in 64 bits

def _value64(codes, panels, k, form):
    """What codes and scales stand for, from the formats' fields: sign, exponent, mantissa."""
    bits, lowest, _ = _FORMATS[form]
    code = codes.long()
    sign = torch.where(code >= 128, -1.0, 1.0).double()
    exponent, mantissa = (code % 128) // 2 ** bits, (code % 2 ** bits).double() / 2 ** bits
    value = torch.where(exponent > 0, (1 + mantissa) * torch.exp2((exponent - 1 + lowest).double()), mantissa * 2.0 ** lowest)
    scale = torch.exp2(panels.permute(1, 0, 2).reshape(panels.shape[1], -1).double() - 127)[:codes.shape[0], :codes.shape[1] // 128]
    return (sign * value * scale.repeat_interleave(128, 1))[:, :k]


def _nearest64(x, form, square):
    """Every value of a 64-bit matrix taken to its block's nearest code, ties to the even one, and back."""
    bits, lowest, largest = _FORMATS[form]
    out = torch.zeros_like(x)
    tall = 128 if square else 1
    rows, k = x.shape
    size = torch.zeros((-(-rows // tall) * tall, -(-k // 128) * 128), dtype=torch.float64, device=x.device)
    size[:rows, :k] = x.abs()
    top = size.view(-1, tall, size.shape[1] // 128, 128).amax((1, 3))
    # log2 of the quotient is exact enough to be off by one at most: that is looked at
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, largest) / largest)))
    scale = torch.where(top > largest * scale, 2 * scale, scale)
    scale = torch.where(2 * top <= largest * scale, scale / 2, scale)
    scale = scale.repeat_interleave(tall, 0).repeat_interleave(128, 1)[:rows, :k]
    v = x / scale
    step = torch.exp2(torch.floor(torch.log2(torch.where(v == 0, 1.0, v.abs()))).clamp(min=lowest) - bits)
    down = torch.floor(v / step)
    rest = v / step - down
    up = (rest > 0.5) | ((rest == 0.5) & (down % 2 != 0))
    out = (down + up) * step * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "convert":
        x = (s["x"].t() if case["turned"] else s["x"]).double().contiguous()
        return _nearest64(x, case["format"], case["square"])
    if op == "product":
        return torch.matmul(_value64(*s["a"], case["k"], case["format"]), _value64(*s["b"], case["k"], "e4m3").transpose(0, 1).contiguous())
    if op == "grouped":
        x = _value64(*s["a"], case["k"], case["format"])[s["gather"].long()]
        first = s["offsets"].tolist()
        y = torch.zeros((s["rows"], case["n"]), dtype=torch.float64, device="cuda")
        for g in range(case["experts"]):
            weight = _value64(s["b"][0][g], s["b"][1][g], case["k"], "e4m3")
            y[first[g]:first[g + 1]] = torch.matmul(x[first[g]:first[g + 1]], weight.transpose(0, 1).contiguous())
        return y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2] if case["gated"] else y
    if op == "kept":
        z, da = s["z"].double(), s["da"].double()
        near = _nearest64(z, "e4m3", False)
        u, v = near[:, 0::2], near[:, 1::2]
        gate = torch.sigmoid(u)
        dz = torch.empty_like(z)
        dz[:, 0::2] = da * v * (gate + u * gate * torch.sigmoid(-u))
        dz[:, 1::2] = da * u * gate
        return [z[:, 0::2] * torch.sigmoid(z[:, 0::2]) * z[:, 1::2], dz, u * gate * v]
    x, w = s["x"].double(), s["w"].double()
    counted = (s["targets"] >= 0).nonzero()[:, 0]
    target = s["targets"].long()[counted]
    t = case["tokens"]
    losses, lse = torch.zeros(t, dtype=torch.float64, device="cuda"), torch.zeros(t, dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    columns = w.transpose(0, 1).contiguous()
    for i in range(0, t, 2048):
        lse[i:i + 2048] = torch.logsumexp(torch.matmul(x[i:i + 2048], columns), 1)
    for i in range(0, len(counted), 2048):
        these, goal = counted[i:i + 2048], target[i:i + 2048]
        z = torch.matmul(x[these], columns)
        each = torch.arange(len(these), device="cuda")
        losses[these] = lse[these] - z[each, goal]
        if case["grad"]:
            p = torch.exp(z - lse[these][:, None])
            p[each, goal] -= 1.0
            p *= s["share"].double()[these][:, None]
            dx[these] = torch.matmul(p, w)
            dw += torch.matmul(p.transpose(0, 1).contiguous(), x[these])
    return [losses, lse, dx, dw] if case["grad"] else [losses, lse]
