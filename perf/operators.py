"""What the experts' operators of this library are measured on: routing, products grouped by expert, the join of
the experts' answers, and microscaled 4-bit quantisation and products.

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
LARGEST_FLOPS = 2.0 * 16384 * 4096 * 4096
LARGEST_BYTES = 1.2e9
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)

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
        # One decoding step of sixteen sequences: the router's choice among 64 experts.  Latency alone.
        dict(name="route_decode", op="route", tokens=16, experts=64, top=4, type="f32", over_all=False, masked=False, grad=False),
        # A training batch of packed sequences with experts switched off for some tokens, gradient to the logits included.
        dict(name="route_train", op="route", tokens=16381, experts=128, top=8, type="bf16", over_all=True, masked=True, grad=True),
        # The experts' first projection in that decoding step: 64 assignments over 64 experts, one or two rows each.  Bound
        # by reading the weights of the experts that are used.
        dict(name="grouped_decode", op="grouped", tokens=16, experts=64, top=4, n=1024, k=2048, type="f16", out="f16", skew=0.0),
        # A short prompt with small experts, odd sizes throughout, Float32 results.
        dict(name="grouped_ragged", op="grouped", tokens=509, experts=13, top=2, n=656, k=720, type="f16", out="f32", skew=1.0),
        # The experts' projection over a training batch, uneven loads.  The largest.
        dict(name="grouped_forward", op="grouped", tokens=8192, experts=8, top=2, n=4096, k=4096, type="bf16", out="bf16", skew=0.5),
        # Both gradients of such a projection: to the rows and, in Float32, to the weights.
        dict(name="grouped_backward", op="grouped_grad", tokens=4099, experts=16, top=2, n=2048, k=4096, type="bf16", out="f32", skew=0.5),
        # The experts' answers of a decoding step joined by their gates.
        dict(name="combine_decode", op="combine", tokens=16, top=4, n=4096, type="f16", grad=False),
        # The same for a training batch, with the gradients to the answers and to the gates.
        dict(name="combine_train", op="combine", tokens=8191, top=4, n=4096, type="bf16", grad=True),
        # Activations of a short prefill on their way into 4 bits (and back, which is how what was kept is looked at).
        dict(name="mxfp4_activations", op="quantize", rows=128, k=4096, type="bf16"),
        # A whole layer's weights.
        dict(name="mxfp4_weights", op="quantize", rows=8192, k=8192, type="f16"),
        # A projection over a prefill in 4 bits.
        dict(name="mxfp4_forward", op="mxfp4", m=4096, n=4096, k=8192, out="bf16"),
        # The experts' projection of a decoding step with weights kept in 4 bits.
        dict(name="mxfp4_grouped_decode", op="mxfp4_grouped", tokens=32, experts=64, top=4, n=2048, k=2048, out="f16", skew=0.0),
    ]


def _size(rng, low, high, step=1):
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def _width(rng, low, high):
    """An extent of a matrix: half of them multiples of 64, the others of 16 or of 8."""
    return _size(rng, low, high, rng.choice((64, 64, 16, 8)))


def _draw(rng):
    op = rng.choice(("route", "grouped", "grouped", "grouped", "grouped_grad", "combine", "quantize", "mxfp4", "mxfp4_grouped"))
    kind = rng.choice(("f16", "bf16"))
    if op == "route":
        experts = _size(rng, 8, 256)
        return dict(op=op, tokens=_size(rng, 1, 16384), experts=experts, top=rng.randint(1, min(8, experts)), type=rng.choice(("f32", "f16", "bf16")),
                    over_all=rng.random() < 0.5, masked=rng.random() < 0.3, grad=rng.random() < 0.5)
    if op in ("grouped", "grouped_grad", "mxfp4_grouped"):
        experts = _size(rng, 4, 64)
        case = dict(op=op, tokens=_size(rng, 1 if op != "grouped_grad" else 64, 8192), experts=experts, top=rng.randint(1, min(8, experts)), n=_width(rng, 256, 4096),
                    k=_width(rng, 256, 4096), out=rng.choice((kind, "f32")), skew=rng.choice((0.0, 0.5, 1.5)))
        if op != "mxfp4_grouped":
            case["type"] = kind
        return case
    if op == "combine":
        return dict(op=op, tokens=_size(rng, 1, 8192), top=rng.randint(1, 8), n=_width(rng, 256, 8192), type=kind, grad=rng.random() < 0.5)
    if op == "quantize":
        return dict(op=op, rows=_size(rng, 1, 8192), k=_size(rng, 64, 8192, rng.choice((32, 32, 1))), type=rng.choice(("f16", "bf16", "f32")))
    return dict(op=op, m=_size(rng, 16, 4096), n=_width(rng, 256, 8192), k=_size(rng, 256, 8192, 32), out=rng.choice((kind, "f32")))


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
    if op == "route":
        t, e, k, s = case["tokens"], case["experts"], case["top"], _SIZE[case["type"]]
        return {"bytes": t * e * s + t * k * 16 + 4 * e + case["grad"] * t * (e * s * (2 if case["over_all"] else 1) + 12 * k), "flops": 4.0 * t * e}
    if op in ("grouped", "grouped_grad", "mxfp4_grouped"):
        rows, used = case["tokens"] * case["top"], _used(case)
        n, k = case["n"], case["k"]
        flops = 2.0 * rows * n * k
        if op == "grouped":
            return {"bytes": _SIZE[case["type"]] * (case["tokens"] * k + used * n * k) + _SIZE[case["out"]] * rows * n, "flops": flops}
        if op == "mxfp4_grouped":
            return {"bytes": (case["tokens"] * k + used * n * k) * 17 / 32 + _SIZE[case["out"]] * rows * n, "flops": flops}
        s = _SIZE[case["type"]]
        return {"bytes": s * (rows * n + used * n * k + rows * k + case["tokens"] * k) + _SIZE[case["out"]] * case["experts"] * n * k, "flops": 2 * flops}
    if op == "combine":
        t, k, n, s = case["tokens"], case["top"], case["n"], _SIZE[case["type"]]
        return {"bytes": s * (t * k * n + t * n) + 8 * t * k + case["grad"] * (s * (2 * t * k * n + t * n) + 12 * t * k), "flops": 2.0 * t * k * n * (1 + 2 * case["grad"])}
    if op == "quantize":
        return {"bytes": case["rows"] * case["k"] * (_SIZE[case["type"]] + 17 / 32 + 17 / 32 + 2), "flops": 2.0 * case["rows"] * case["k"]}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": (m * k + n * k) * 17 / 32 + _SIZE[case["out"]] * m * n, "flops": 2.0 * m * n * k}


def _assignments(gen, case):
    """`top` different experts for every token, some likelier than others by `skew`; sorted by expert: the group each
    sorted position belongs to, where each starts, and the token at each position."""
    t, e, top = case["tokens"], case["experts"], case["top"]
    score = torch.rand((t, e), device="cuda", generator=gen) + case["skew"] * torch.rand((e,), device="cuda", generator=gen)
    chosen = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :top].reshape(-1)
    group, order = torch.sort(chosen, stable=True)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum((group[:, None] == torch.arange(e, device="cuda")).sum(0), 0)
    return offsets, (order // top).to(torch.int32)


def _mxfp4_codes(gen, rows, k, scale):
    """Codes and scales as quantising a normal matrix of that standard deviation leaves them."""
    x = torch.empty((rows, k), device="cuda").normal_(0.0, scale, generator=gen)
    return _quantize(x)


def _blocks(x):
    rows, k = x.shape
    blocks = -(-k // 32)
    padded = torch.zeros((rows, blocks * 32), dtype=x.dtype, device=x.device)
    padded[:, :k] = x
    return padded.view(rows, blocks, 32)


def _quantize(x):
    """(codes, scales) of a Float32 matrix: two e2m1 values to a byte, the one of the lower k in the low half, and one
    e8m0 byte for 32 values along k: floor(log2(largest magnitude)) - 2, or 255 where one is not finite.  Scales lie in
    panels of eight blocks (256 values of k), the rows of a panel one after the other, eight bytes each."""
    v = _blocks(x)
    top = v.abs().amax(-1)
    exponent = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)
    scaled = torch.ldexp(v, -exponent[..., None])
    size = scaled.abs()
    code = ((size > 0.25).to(torch.uint8) + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5) + (size > 5.0))
    code = code + 8 * torch.signbit(scaled).to(torch.uint8)
    code = code.view(v.shape[0], -1)
    scales = torch.where(torch.isfinite(top), exponent + 127, 255).to(torch.uint8)
    rows, blocks = scales.shape
    panels = torch.zeros(_panels(rows, x.shape[1]), dtype=torch.uint8, device=x.device)
    padded = torch.zeros((panels.shape[1], panels.shape[0] * 8), dtype=torch.uint8, device=x.device)
    padded[:rows, :blocks] = scales
    panels.copy_(padded.view(panels.shape[1], -1, 8).transpose(0, 1))
    return (code[:, 0::2] + 16 * code[:, 1::2]).contiguous(), panels


def _panels(rows, k):
    return -(-k // 256), rows + rows % 2, 8


def _row_scales(codes, panels):
    """One row of scales for each row of codes."""
    return panels.transpose(0, 1).reshape(panels.shape[1], -1)[:codes.shape[0], :codes.shape[1] // 16]


def _dequantize(codes, panels, k, dtype=torch.float32):
    table, scales = torch.tensor(E2M1, dtype=dtype, device=codes.device), _row_scales(codes, panels)
    values = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).view(codes.shape[0], -1, 32)
    factor = torch.where(scales == 255, math.nan, torch.ldexp(torch.ones((), dtype=dtype, device=codes.device), scales.int() - 127))
    return (values * factor[..., None]).view(codes.shape[0], -1)[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    state = dict(case)

    def normal(shape, scale, kind):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen).to(_TORCH[kind])

    def empty(shape, kind):
        return torch.zeros(shape, dtype=_TORCH.get(kind, kind), device="cuda")

    if op == "route":
        t, e, top = case["tokens"], case["experts"], case["top"]
        z = normal((t, e), 1.5, case["type"])
        if case["masked"]:  # experts switched off, by -inf or by the type's lowest value, and a few tokens without any expert
            off = torch.rand((t, e), device="cuda", generator=gen)
            z[off < 0.25] = -math.inf
            z[off > 0.95] = torch.finfo(z.dtype).min
            z[torch.rand(t, device="cuda", generator=gen) < 0.02] = -math.inf
        state.update(z=z, chosen=empty((t, top), torch.int32), gates=empty((t, top), "f32"), offsets=empty(e + 1, torch.int32),
                     rows=empty(t * top, torch.int32), place=empty((t, top), torch.int32))
        if case["grad"]:
            state.update(dgates=normal((t, top), 1.0, "f32"), dz=empty((t, e), case["type"]))
    elif op in ("grouped", "grouped_grad"):
        n, k, e, rows = case["n"], case["k"], case["experts"], case["tokens"] * case["top"]
        offsets, gather = _assignments(gen, case)
        state.update(offsets=offsets, gather=gather, bounds=offsets.tolist(), x=normal((case["tokens"], k), 1.0, case["type"]),
                     w=normal((e, n, k), 0.02, case["type"]), rows=rows)
        if op == "grouped":
            state.update(y=empty((rows, n), case["out"]))
        else:
            state.update(dy=normal((rows, n), 1.0, case["type"]), dx=empty((rows, k), case["type"]), dw=empty((e, n, k), case["out"]))
    elif op == "combine":
        t, top, n = case["tokens"], case["top"], case["n"]
        gates = torch.rand((t, top), device="cuda", generator=gen)
        place = torch.randperm(t * top, device="cuda", generator=gen).to(torch.int32).view(t, top)
        place[torch.rand((t, top), device="cuda", generator=gen) < 0.02] = -1  # choices that went to no expert
        state.update(h=normal((t * top, n), 1.0, case["type"]), gates=gates / gates.sum(1, keepdim=True), place=place, y=empty((t, n), case["type"]))
        if case["grad"]:
            state.update(dy=normal((t, n), 1.0, case["type"]), dh=empty((t * top, n), case["type"]), dgates=empty((t, top), "f32"))
    elif op == "quantize":
        rows, k = case["rows"], case["k"]
        blocks = -(-k // 32)
        # rows of different size, a few of zeros
        x = torch.empty((rows, k), device="cuda").normal_(0.0, 1.0, generator=gen) * torch.exp(torch.randn((rows, 1), device="cuda", generator=gen))
        x[torch.rand(rows, device="cuda", generator=gen) < 0.01] = 0.0
        state.update(x=x.to(_TORCH[case["type"]]), codes=empty((rows, 16 * blocks), torch.uint8), scales=empty(_panels(rows, k), torch.uint8), back=empty((rows, k), "bf16"))
    elif op == "mxfp4":
        state.update(a=_mxfp4_codes(gen, case["m"], case["k"], 1.0), b=_mxfp4_codes(gen, case["n"], case["k"], 0.02), y=empty((case["m"], case["n"]), case["out"]))
    else:
        n, k, e, rows = case["n"], case["k"], case["experts"], case["tokens"] * case["top"]
        offsets, gather = _assignments(gen, case)
        codes, scales = zip(*(_mxfp4_codes(gen, n, k, 0.02) for _ in range(e)))
        state.update(offsets=offsets, gather=gather, bounds=offsets.tolist(), a=_mxfp4_codes(gen, case["tokens"], k, 1.0), b=(torch.stack(codes), torch.stack(scales)),
                     y=empty((rows, n), case["out"]), rows=rows)
    if own:
        pkg = _package()
        kinds = {"f16": pkg.WMMA.Float16, "bf16": pkg.BFloat16, "f32": pkg.WMMA.Float32}
        state.update(pkg=pkg, kind=kinds.get(case.get("type")), out_kind=kinds.get(case.get("out")), address={key: _address(v) for key, v in state.items()})
        if op == "route":
            state["workspace"] = pkg.DeviceArray.undef(np.uint8, max(16, pkg.EXPERTS.route_workspace(case["tokens"], case["experts"], case["top"])))
    return state


def _address(v):
    """Raw addresses of a tensor or of several, as the entry points take them."""
    if isinstance(v, torch.Tensor):
        return v.data_ptr()
    return tuple(map(_address, v)) if isinstance(v, tuple) else None


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    op, at = s["op"], s["address"]
    E, Q = s["pkg"].EXPERTS, s["pkg"].MXFP4
    if op == "route":
        sizes = dict(tokens=s["tokens"], experts=s["experts"], top=s["top"], dtype=s["kind"], over_all=s["over_all"])
        E.route(at["z"], at["chosen"], at["gates"], at["offsets"], at["rows"], at["place"], workspace=s["workspace"], **sizes)
        out = [s["chosen"], s["gates"], s["offsets"], s["rows"], s["place"]]
        if s["grad"]:
            E.route_grad(at["z"], at["chosen"], at["gates"], at["dgates"], at["dz"], **sizes)
            out.append(s["dz"])
        return out
    if op == "grouped":
        E.grouped_gemm(at["x"], at["w"], at["y"], at["offsets"], rows=s["rows"], groups=s["experts"], n=s["n"], k=s["k"], dtype=s["kind"], d_type=s["out_kind"],
                       gather=at["gather"], a_rows=s["tokens"])
        return s["y"]
    if op == "grouped_grad":
        # (the weights lie N x K for the forward pass: as the right operand of dY W they are row-major)
        E.grouped_gemm(at["dy"], at["w"], at["dx"], at["offsets"], rows=s["rows"], groups=s["experts"], n=s["k"], k=s["n"], dtype=s["kind"], d_type=s["kind"],
                       w_layout=s["pkg"].WMMA.RowMajor)
        E.grouped_wgrad(at["dy"], at["x"], at["dw"], at["offsets"], rows=s["rows"], groups=s["experts"], m=s["n"], n=s["k"], dtype=s["kind"], d_type=s["out_kind"],
                        gather=at["gather"], b_rows=s["tokens"])
        return [s["dx"], s["dw"]]
    if op == "combine":
        sizes = dict(tokens=s["tokens"], top=s["top"], n=s["n"], rows=s["tokens"] * s["top"], dtype=s["kind"])
        E.combine(at["h"], at["place"], at["y"], gates=at["gates"], **sizes)
        if not s["grad"]:
            return s["y"]
        E.combine_grad(at["dy"], at["h"], at["place"], at["dh"], at["dgates"], gates=at["gates"], **sizes)
        return [s["y"], s["dh"], s["dgates"]]
    if op == "quantize":
        Q.quantize(at["x"], at["codes"], at["scales"], rows=s["rows"], k=s["k"], dtype=s["kind"])
        Q.dequantize(at["codes"], at["scales"], at["back"], rows=s["rows"], k=s["k"], dtype=s["pkg"].BFloat16)
        return s["back"]
    if op == "mxfp4":
        Q.gemm(*at["a"], *at["b"], at["y"], m=s["m"], n=s["n"], k=s["k"], d_type=s["out_kind"])
        return s["y"]
    Q.grouped_gemm(*at["a"], *at["b"], at["y"], at["offsets"], rows=s["rows"], groups=s["experts"], n=s["n"], k=s["k"], d_type=s["out_kind"], gather=at["gather"],
                   a_rows=s["tokens"])
    return s["y"]


def _plain(s):
    op = s["op"]
    if op == "route":
        return _plain_route(s)
    if op == "grouped":
        x = s["x"].float()[s["gather"].long()]
        return torch.cat([x[a:b] @ s["w"][e].float().t() for e, (a, b) in enumerate(zip(s["bounds"], s["bounds"][1:]))]).to(s["y"].dtype)
    if op == "grouped_grad":
        parts = list(enumerate(zip(s["bounds"], s["bounds"][1:])))
        dy, x = s["dy"].float(), s["x"].float()[s["gather"].long()]
        dx = torch.cat([dy[a:b] @ s["w"][e].float() for e, (a, b) in parts]).to(s["dx"].dtype)
        return [dx, torch.stack([dy[a:b].t() @ x[a:b] for e, (a, b) in parts]).to(s["dw"].dtype)]
    if op == "combine":
        h, some, at = s["h"].float(), (s["place"] >= 0), s["place"].long().clamp(min=0)
        gates = torch.where(some, s["gates"], 0.0)
        answers = torch.where(some[..., None], h[at], 0.0)
        y = (gates[..., None] * answers).sum(1).to(s["y"].dtype)
        if not s["grad"]:
            return y
        dy = s["dy"].float()
        dh = torch.zeros_like(h)
        dh[at[some]] = (gates[..., None] * dy[:, None])[some]
        return [y, dh.to(s["dh"].dtype), (dy[:, None] * answers).sum(2)]
    if op == "quantize":
        return _dequantize(*_quantize(s["x"].float()), s["k"]).to(torch.bfloat16)
    if op == "mxfp4":
        return (_dequantize(*s["a"], s["k"]) @ _dequantize(*s["b"], s["k"]).t()).to(s["y"].dtype)
    a = _dequantize(*s["a"], s["k"])[s["gather"].long()]
    return torch.cat([a[i:j] @ _dequantize(s["b"][0][e], s["b"][1][e], s["k"]).t() for e, (i, j) in enumerate(zip(s["bounds"], s["bounds"][1:]))]).to(s["y"].dtype)


def _plain_route(s):
    t, e, top = s["tokens"], s["experts"], s["top"]
    z = s["z"].float()
    value, chosen = torch.sort(z, dim=1, descending=True, stable=True)
    value, chosen = value[:, :top], chosen[:, :top]
    none = value == -math.inf
    largest = torch.where(none[:, :1], 0.0, value[:, :1])
    part = torch.exp(value - largest)
    every = torch.exp(z - largest)
    total = (every if s["over_all"] else part).sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    gates = part / total
    chosen = torch.where(none, -1, chosen)
    flat = torch.where(none, e, chosen).reshape(-1)
    group, order = torch.sort(flat, stable=True)
    counts = (group[:, None] == torch.arange(e, device="cuda")).sum(0)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(counts, 0)
    rows = torch.where(group < e, order // top, -1).to(torch.int32)
    place = torch.empty_like(order)
    place[order] = torch.arange(t * top, device="cuda")
    place = torch.where(none, -1, place.view(t, top)).to(torch.int32)
    out = [chosen.to(torch.int32), gates, offsets, rows, place]
    if s["grad"]:
        dg = s["dgates"]
        inner = (gates * dg).sum(1, keepdim=True)
        if s["over_all"]:
            dz = -(every / total) * inner
        else:
            dz = torch.zeros_like(z)
        own_part = gates * dg if s["over_all"] else gates * (dg - inner)
        dz.scatter_add_(1, chosen.clamp(min=0).long(), torch.where(none, 0.0, own_part))
        out.append(dz.to(s["z"].dtype))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(s)
    if op in ("grouped", "grouped_grad", "mxfp4_grouped"):
        e, rows = case["experts"], s["rows"]
        take = s["gather"].long()
        if op == "mxfp4_grouped":
            x, weight = _value64(*s["a"], case["k"])[take], lambda g: _value64(s["b"][0][g], s["b"][1][g], case["k"])
        else:
            x, weight = s["x"].double()[take], lambda g: s["w"][g].double()
        first = s["offsets"].tolist()
        if op != "grouped_grad":
            y = torch.zeros((rows, case["n"]), dtype=torch.float64, device="cuda")
            for g in range(e):
                y[first[g]:first[g + 1]] = torch.matmul(x[first[g]:first[g + 1]], weight(g).transpose(0, 1).contiguous())
            return y
        dy = s["dy"].double()
        dx, dw = torch.zeros((rows, case["k"]), dtype=torch.float64, device="cuda"), torch.zeros((e, case["n"], case["k"]), dtype=torch.float64, device="cuda")
        for g in range(e):
            part = slice(first[g], first[g + 1])
            dx[part] = torch.matmul(dy[part], weight(g))
            dw[g] = torch.matmul(dy[part].transpose(0, 1).contiguous(), x[part])
        return [dx, dw]
    if op == "combine":
        t, top, n = case["tokens"], case["top"], case["n"]
        h, gates, place = s["h"].double(), s["gates"].double(), s["place"].long()
        y = torch.zeros((t, n), dtype=torch.float64, device="cuda")
        dh, dg = torch.zeros_like(h), torch.zeros((t, top), dtype=torch.float64, device="cuda")
        for j in range(top):
            has = (place[:, j] >= 0).nonzero()[:, 0]
            rows = place[has, j]
            y[has] += gates[has, j, None] * h[rows]
            if case["grad"]:
                dy = s["dy"].double()[has]
                dh[rows] = gates[has, j, None] * dy
                dg[has, j] = (dy * h[rows]).sum(1)
        return [y, dh, dg] if case["grad"] else y
    if op == "quantize":
        v = _blocks(s["x"].double())
        top = v.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2)
        # distance to each of the eight magnitudes, ties to the even code
        size, places = (v.abs() / step).unsqueeze(-1), torch.tensor(E2M1[:8], dtype=torch.float64, device="cuda")
        out = torch.empty_like(v)
        for i in range(0, v.shape[0], 256):
            far = (size[i:i + 256] - places).abs()
            nearest = far.amin(-1, keepdim=True)
            code = torch.where(far == nearest, torch.arange(8, device="cuda") + 16 * (torch.arange(8, device="cuda") % 2), 99).amin(-1) % 16
            out[i:i + 256] = torch.sign(v[i:i + 256]) * places[code] * step[i:i + 256]
        return out.view(v.shape[0], -1)[:, :case["k"]]
    return torch.matmul(_value64(*s["a"], case["k"]), _value64(*s["b"], case["k"]).transpose(0, 1).contiguous())


def _value64(codes, panels, k):
    """What codes and scales stand for, from the fields of e2m1: sign, two bits of exponent, one of mantissa."""
    scales = _row_scales(codes, panels)
    nibble = torch.stack((codes % 16, codes // 16), -1).view(codes.shape[0], -1).double()
    sign = torch.where(nibble >= 8, -1.0, 1.0).double()
    nibble = nibble % 8
    exponent, mantissa = torch.floor(nibble / 2), nibble % 2
    value = torch.where(exponent > 0, (1 + mantissa / 2) * torch.exp2(exponent - 1), mantissa / 2)
    return (sign * value * torch.exp2(scales.double() - 127).repeat_interleave(32, 1))[:, :k]


def _exact_route(s):
    t, e, top = s["tokens"], s["experts"], s["top"]
    z = s["z"].double().cpu().numpy()
    order = np.argsort(-z, axis=1, kind="stable")[:, :top]
    value = np.take_along_axis(z, order, 1)
    none = np.isneginf(value)
    shift = np.where(none[:, :1], 0.0, value[:, :1])
    every = np.exp(z - shift)
    total = np.where(none, 0.0, np.exp(value - shift)).sum(1, keepdims=True) if not s["over_all"] else every.sum(1, keepdims=True)
    total[total == 0] = 1.0
    gates = np.where(none, 0.0, np.exp(value - shift) / total)
    chosen = np.where(none, -1, order)
    offsets, rows, place = np.zeros(e + 1, np.int64), np.full(t * top, -1, np.int64), np.full((t, top), -1, np.int64)
    at = 0
    for g in range(e):
        token, slot = np.nonzero(chosen == g)
        place[token, slot] = np.arange(at, at + len(token))
        rows[at:at + len(token)] = token
        at += len(token)
        offsets[g + 1] = at
    out = [chosen, gates, offsets, rows, place]
    if s["grad"]:
        dg = np.where(none, 0.0, s["dgates"].double().cpu().numpy())
        inner = (gates * dg).sum(1, keepdims=True)
        p = every / total if s["over_all"] else np.zeros_like(z)
        direct = np.zeros_like(z)
        token, slot = np.nonzero(~none)
        direct[token, chosen[token, slot]] = (gates * dg)[token, slot]
        if not s["over_all"]:
            p[token, chosen[token, slot]] = gates[token, slot]
        out.append(direct - p * inner)
    return out
