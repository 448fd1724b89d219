"""Plain 64-bit forms of the 4-bit weight operators and of the gated residual norm, and the error bounds their fp16 / fp32
results are held to. Written from the formulas alone."""
import torch

HALF = 2.0 ** -11       # an fp16 rounding is off by at most this much of the value
SUB = 2.0 ** -25        # ... or by this much among fp16's subnormals
F32 = 2.0 ** -24        # the same for fp32


def codes(q):
    """uint8 [N, K/2] -> float64 codes [N, K]."""
    return torch.stack([q & 15, q >> 4], 2).reshape(q.shape[0], -1).double()


def per_k(v, group, K):
    return v.double().repeat_interleave(group, 1)[:, :K]


def weights(q, scale, zero, group):
    c = codes(q)
    K = c.shape[1]
    return per_k(scale, group, K) * (c - (8.0 if zero is None else per_k(zero, group, K)))


def quantize(w, group):
    """(codes, scale): scale = bf16(max |w| / 7), code = 8 + rint(w / scale), ties to even."""
    N, K = w.shape
    J = -(-K // group)
    pad = torch.zeros(N, J * group, dtype=torch.float64, device=w.device)
    pad[:, :K] = w.double()
    pad = pad.view(N, J, group)
    scale = (pad.abs().amax(2) / 7).to(torch.bfloat16)
    s = scale.double()[..., None]
    c = torch.where(s > 0, pad / s, torch.zeros_like(pad)).round().clamp(-7, 7) + 8
    return c.reshape(N, -1)[:, :K], scale


def linear(x, q, scale, zero, group, bias, residual, silu, out_scale):
    """(value, bound). fp32 accumulation of K products of exact operands, in any order: each of at most K additions rounds
    (toward zero on the tensor cores: a whole step, 2^-23) a partial sum of at most sum |x w|. With zero points a weight
    rounds once to fp16. Then bias, SiLU (slope at most 1.1; exponential and division a few steps of 2^-22), residual and
    scale in fp32 and one rounding to fp16."""
    w = weights(q, scale, zero, group)
    K = w.shape[1]
    v = x.double() @ w.T
    mag = x.double().abs() @ w.abs().T
    err = mag * (K * 2 * F32 + (0.0 if zero is None else HALF))
    if bias is not None:
        v = v + bias.double()
    err = err + F32 * v.abs()
    if silu:
        err = 1.1 * err + 2.0 ** -20 * v.abs()
        v = v * torch.sigmoid(v)
    if residual is not None:
        v = v + residual.double()
    v = v * out_scale
    err = abs(out_scale) * err + 3 * F32 * v.abs()
    return v, err * (1 + HALF) + HALF * v.abs() + SUB


def norm(v, err, kind, weight, bias, eps):
    """Norm of v known to within err (both [..., C]): (value, bound). The statistics are fp32 sums of C terms in which no
    term passes through more than 48 additions and a handful of products and a square root: 64 roundings in all."""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    d = v - mean
    rstd = (d.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    # mean is off by at most 64 steps of the mean magnitude, and by the mean error of v
    derr = err + F32 * v.abs()
    if kind == "layer":
        derr = derr + err.mean(-1, keepdim=True) + 64 * F32 * v.abs().mean(-1, keepdim=True) + F32 * d.abs()
    # sqrt(mean d^2) moves by at most sqrt(mean derr^2), and by 64 steps of its size
    rel = derr.pow(2).mean(-1, keepdim=True).sqrt() * rstd + 64 * F32
    z = d * rstd
    zerr = derr * rstd * (1 + rel) + z.abs() * (rel + 4 * F32)
    if weight is not None:
        z, zerr = z * weight.double(), zerr * weight.double().abs()
        zerr = zerr + F32 * z.abs()
    if bias is not None:
        z = z + bias.double()
        zerr = zerr + F32 * z.abs()
    return z, zerr


def spread(v, dims):
    return v.double() if v.dim() != 2 or dims == 2 else v.double()[:, None]


def residual_norm(x, y, gate, post, pre, scale, shift, residual_scale):
    """((h, bound), (z, bound) or None); post and pre: (kind, weight, bias, eps) or None."""
    h = x.double() * residual_scale
    err = 2 * F32 * h.abs()
    if y is not None:
        u, uerr = y.double(), torch.zeros_like(h)
        if post is not None:
            u, uerr = norm(u, uerr, *post)
        if gate is not None:
            g = spread(gate, x.dim())
            u, uerr = u * g, uerr * g.abs() + F32 * (u * g).abs()
        h, err = h + u, err + uerr + F32 * (h + u).abs()
    step, low = (HALF, SUB) if x.dtype == torch.float16 else (F32, 0.0)
    first = (h, err * (1 + step) + step * h.abs() + low)
    if pre is None:
        return first, None
    z, zerr = norm(h, err, *pre)
    if scale is not None:
        s = spread(scale, x.dim())
        z, zerr = z * (1 + s), zerr * (1 + s).abs() + 2 * F32 * (z.abs() + (z * s).abs())
    if shift is not None:
        z = z + spread(shift, x.dim())
        zerr = zerr + F32 * z.abs()
    return first, (z, zerr * (1 + HALF) + HALF * z.abs() + SUB)


def assert_within(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values outside; first at %s: got %r, want %r, bound %r" % (
        what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), bound[bad][0].item())
