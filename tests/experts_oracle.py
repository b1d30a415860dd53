"""Plain 64-bit implementations that the tests of the experts' operators and of the 4-bit matrices compare with, and the
bfloat16 conversions that numpy lacks."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def to_bf16(x):
    """Bits of the nearest bfloat16 (ties to even) of a Float32 array without NaN."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32)


class Kind:
    """An element type: how it is stored, and its unit roundoff."""

    def __init__(self, name, dtype, roundoff):
        self.name, self.dtype, self.roundoff = name, dtype, roundoff

    def store(self, x):
        return to_bf16(x) if self.name == "bf16" else np.asarray(x, np.float64).astype(self.dtype)

    def load(self, stored):
        return (from_bf16(stored) if self.name == "bf16" else np.asarray(stored)).astype(np.float64)

    def marker(self, miw):
        return miw.BFloat16 if self.name == "bf16" else self.dtype


F16, BF16, F32 = Kind("f16", np.float16, 2.0 ** -11), Kind("bf16", np.uint16, 2.0 ** -8), Kind("f32", np.float32, 2.0 ** -24)
KINDS = {k.name: k for k in (F16, BF16, F32)}


def upload(miw, a):
    """A row-major array as the operators take it."""
    return miw.DeviceArray(np.ascontiguousarray(a).reshape(-1))


def route(z, top, over_all):
    """(chosen, gates, offsets, rows, place) of logits in 64 bits."""
    tokens, experts = z.shape
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max))
    order = np.argsort(-z, axis=1, kind="stable")[:, :top]
    value = np.take_along_axis(z, order, 1)
    none = np.isneginf(value)
    shift = np.where(none[:, :1], 0.0, value[:, :1])
    with np.errstate(over="ignore"):
        part, every = np.where(none, 0.0, np.exp(value - shift)), np.exp(z - shift)
    total = (every if over_all else part).sum(1, keepdims=True)
    gates = part / np.where(total > 0, total, 1.0)
    chosen = np.where(none, -1, order).astype(np.int32)
    rows, place, offsets = np.full(tokens * top, -1, np.int32), np.full((tokens, top), -1, np.int32), np.zeros(experts + 1, np.int32)
    at = 0
    for e in range(experts):
        t, j = np.nonzero(chosen == e)
        place[t, j] = at + np.arange(len(t))
        rows[at:at + len(t)] = t
        at += len(t)
        offsets[e + 1] = at
    return chosen, gates, offsets, rows, place


def route_grad(z, chosen, dgates, over_all):
    """The formula's gradient, in 64 bits."""
    tokens, experts = z.shape
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max))
    dz = np.zeros((tokens, experts))
    for t in range(tokens):
        e = chosen[t][chosen[t] >= 0]
        dg = dgates[t][chosen[t] >= 0]
        if not len(e):
            continue
        with np.errstate(over="ignore"):
            p = np.exp(z[t] - z[t, e[0]])
        if not over_all:
            keep = np.zeros(experts)
            keep[e] = 1
            p = p * keep
        p = p / p.sum()
        full = np.zeros(experts)
        full[e] = dg
        dz[t] = p * (full - (p * full).sum())
    return dz


def grouped(a, w, offsets, gather, out):
    """out[r] = a[gather[r]] w_g, w: groups x k x n; and the sums of magnitudes that bound a Float32 sum's error."""
    size = np.zeros(out.shape)
    for g in range(len(w)):
        for r in range(offsets[g], offsets[g + 1]):
            row = a[r if gather is None else gather[r]]
            out[r] = row @ w[g]
            size[r] = np.abs(row) @ np.abs(w[g])
    return out, size


def gated(x):
    gate, value = x[..., 0::2], x[..., 1::2]
    return gate / (1 + np.exp(-gate)) * value


def quantize(x):
    """(codes, scales of rows x blocks, what they stand for) of a matrix in 64 bits."""
    rows, k = x.shape
    blocks = -(-k // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :k] = x
    v = v.reshape(rows, blocks, 32)
    top = np.abs(v).max(-1)
    bad = ~np.isfinite(v).all(-1)
    exponent = np.clip(np.floor(np.log2(np.where((top > 0) & ~bad, top, 1.0))) - 2, -127, 127)
    exponent = np.where(top > 0, exponent, -127)
    scaled = np.where(bad[..., None], 0.0, v / np.exp2(exponent)[..., None])
    far = np.abs(np.abs(scaled)[..., None] - E2M1)
    # the nearest; of two as near the even code
    code = np.argmin(far + np.where(np.arange(8) % 2, 1e-12, 0.0), -1)
    value = np.sign(scaled) * E2M1[code] * np.exp2(exponent)[..., None]
    value[bad] = np.nan
    code = code + 8 * np.signbit(scaled)
    code[bad] = 0
    code = code.reshape(rows, -1).astype(np.uint8)
    scales = np.where(bad, 255, exponent + 127).astype(np.uint8)
    return (code[:, 0::2] | code[:, 1::2] << 4), scales, value.reshape(rows, -1)[:, :k]


def panels(scales, lds=None, fill=0):
    """Scales of rows x blocks in panels of eight blocks."""
    rows, blocks = scales.shape
    lds = lds or rows + rows % 2
    out = np.full((-(-blocks // 8), lds, 8), fill, np.uint8)
    for b in range(blocks):
        out[b // 8, :rows, b % 8] = scales[:, b]
    return out


def packed(codes, pitch, fill=0):
    out = np.full((codes.shape[0], pitch), fill, np.uint8)
    out[:, :codes.shape[1]] = codes
    return out
