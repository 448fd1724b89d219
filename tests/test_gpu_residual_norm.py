"""The gated residual norm against its 64-bit form (tests/w4_reference.py has the bounds)."""
import pytest
import torch

from tests import w4_reference as ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _norm_args(n):
    return None if n is None else (n.kind, n.weight, n.bias, n.eps)


def _check(x, y=None, gate=None, post=None, pre=None, scale=None, shift=None, residual_scale=1.0, what="", **kw):
    from katz_b200 import ops
    first, second = ref.residual_norm(x, y, gate, _norm_args(post), _norm_args(pre), scale, shift, residual_scale)
    h, z = ops.residual_norm(x, y, gate=gate, post=post, pre=pre, scale=scale, shift=shift, residual_scale=residual_scale, **kw)
    assert h.dtype == x.dtype and h.shape == x.shape
    ref.assert_within(h, *first, "h " + what)
    if pre is None:
        assert z is None
    else:
        assert z.dtype == torch.float16 and z.shape == x.shape
        ref.assert_within(z, *second, "z " + what)
    return h, z


def _norm(g, kind, C, affine):
    from katz_b200 import ops
    if kind is None:
        return None
    w = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).half() if affine else None
    b = (0.2 * torch.randn(C, generator=g, device="cuda")).half() if affine else None
    return ops.Norm(kind, w, b)


def _vector(g, how, B, S, C):
    lead = {"channel": (), "sample": (B,), "token": (B, S)}
    return None if how is None else (0.5 * torch.randn(*lead[how], C, generator=g, device="cuda")).half()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("C", [1, 7, 8, 64, 255, 256, 320, 513, 640, 768, 1280, 1283, 2048, 2049, 4096, 5120, 8192, 10000, 16384])
def test_sizes(cuda_device, C, dtype):
    g = _gen(C)
    B, S = 2, 5
    x = (torch.randn(B, S, C, generator=g, device="cuda") + 0.5).to(dtype)
    y = torch.randn(B, S, C, generator=g, device="cuda").half()
    _check(x, y, _vector(g, "sample", B, S, C), _norm(g, "rms", C, True), _norm(g, "layer", C, False), _vector(g, "sample", B, S, C),
           _vector(g, "sample", B, S, C), 0.75, what="C=%d" % C)
    _check(x, y, None, _norm(g, "layer", C, False), _norm(g, "rms", C, True), what="C=%d" % C)


HOW = [None, "channel", "sample", "token"]


@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("pre,mod", [(None, None)] + [(k, m) for k in ("layer", "rms") for m in HOW])      # scale and shift need pre
@pytest.mark.parametrize("gate", HOW)
def test_every_combination(cuda_device, post, pre, gate, mod):
    g = _gen(1)
    for B, S, C, dtype in ((3, 7, 320, torch.float16), (2, 3, 77, torch.float32)):
        x, y = (torch.randn(B, S, C, generator=g, device="cuda") for _ in range(2))
        _check(x.to(dtype), y.half(), _vector(g, gate, B, S, C), _norm(g, post, C, True), _norm(g, pre, C, post == "rms"),
               _vector(g, mod, B, S, C), _vector(g, mod, B, S, C), 0.5)


def test_norm_alone_and_sum_alone(cuda_device):
    """Without y: a modulated norm (x comes back itself); without pre: a gated residual."""
    from katz_b200 import ops
    g = _gen(2)
    x = torch.randn(2, 9, 640, generator=g, device="cuda").half()
    h, _ = _check(x, pre=_norm(g, "layer", 640, False), scale=_vector(g, "sample", 2, 9, 640))
    assert h is x
    h, _ = _check(x, pre=_norm(g, "layer", 640, False), residual_scale=0.5)
    assert h is not x
    out = torch.empty_like(x)
    h, _ = _check(x, pre=ops.Norm("rms", eps=1e-6), shift=_vector(g, "channel", 2, 9, 640), out=out)
    assert h is out and torch.equal(out, x)
    _check(x, x.clone(), gate=_vector(g, "token", 2, 9, 640))


def test_two_dimensional_rows_broadcasts_and_views(cuda_device):
    """[rows, C]; views of wider rows; sizes of 1; offsets that rule 16-byte vectors out; what lies around is left alone."""
    g = _gen(3)
    from katz_b200 import ops
    for C, off, pad in ((64, 0, 8), (64, 3, 2), (320, 8, 16), (65, 1, 0)):
        B, S = 3, 6
        wide = torch.randn(B, S + 2, 3 * C + off + pad, generator=g, device="cuda").half()
        x, y = wide[:, 1:S + 1, off:off + C], wide[:, 1:S + 1, off + C:off + 2 * C]
        six = torch.randn(B, 6 * C, generator=g, device="cuda").half()
        gate, scale, shift = six[:, C:2 * C], six[:, 3 * C:4 * C], six[:, 5 * C:]
        ob, zb = torch.full_like(wide, 4.0), torch.full_like(wide, 4.0)
        out, normed = ob[:, 1:S + 1, off:off + C], zb[:, 1:S + 1, off + C:off + 2 * C]
        _check(x, y, gate, ops.Norm("rms"), ops.Norm("layer"), scale, shift, out=out, normed=normed)
        keep = torch.ones_like(ob, dtype=torch.bool)
        keep[:, 1:S + 1, off:off + C] = False
        assert (ob[keep] == 4).all()
        keep = torch.ones_like(ob, dtype=torch.bool)
        keep[:, 1:S + 1, off + C:off + 2 * C] = False
        assert (zb[keep] == 4).all()
        _check(x[1], y[1], gate[:1], None, ops.Norm("layer"), scale[0], wide[0, :S, :C])
        _check(x, y, gate[:, None], None, ops.Norm("rms"), wide[:1, :S, :C], wide[:, :1, :C])
        _check(x.expand(B, S, C), y, gate[:1].expand(B, C), None, ops.Norm("rms"))
        h1, z1 = ops.residual_norm(x[:1, :1], y[:1, :1], pre=ops.Norm("rms"))
        hb, z2 = ops.residual_norm(x, y, pre=ops.Norm("rms"))
        assert torch.equal(h1, hb[:1, :1]) and torch.equal(z1, z2[:1, :1])


@pytest.mark.parametrize("C", [320, 321, 5120])
def test_in_place(cuda_device, C):
    from katz_b200 import ops
    g = _gen(4)
    x = torch.randn(4, 33, C, generator=g, device="cuda").half()
    y = torch.randn(4, 33, C, generator=g, device="cuda").half()
    n = ops.Norm("layer")
    h, z = ops.residual_norm(x, y, post=n, pre=n)
    x2, y2 = x.clone(), y.clone()
    h2, z2 = ops.residual_norm(x2, y2, post=n, pre=n, out=x2, normed=y2)
    assert h2 is x2 and z2 is y2 and torch.equal(h2, h) and torch.equal(z2, z)


def test_large_means_and_constant_rows(cuda_device):
    """A mean a thousand times the spread; rows without any spread; rows of zeros; rows with NaN or infinity stay alone."""
    from katz_b200 import ops
    g = _gen(5)
    x = 1000 + torch.randn(1, 8, 1280, generator=g, device="cuda")
    x[0, 3] = 3.0
    x[0, 4] = 0.0
    _check(x, pre=ops.Norm("layer"))
    _check(x, pre=ops.Norm("rms"))
    _, z = ops.residual_norm(x, pre=ops.Norm("layer"))
    assert (z[0, 3:5] == 0).all()
    x[0, 5, 7], x[0, 6, 1279] = float("nan"), float("inf")
    y = torch.zeros(1, 8, 1280, device="cuda").half()
    h, z = ops.residual_norm(x, y, pre=ops.Norm("layer"))
    rows = torch.tensor([0, 1, 2, 3, 4, 7], device="cuda")
    assert z[0, rows].isfinite().all() and z[0, 5].isnan().all() and z[0, 6].isnan().all()
    assert h[0, 6].isinf().sum() == 1 and h[0, 5].isnan().sum() == 1


def test_streams_graphs_and_repeats(cuda_device):
    from katz_b200 import ops
    g = _gen(6)
    x = torch.randn(2, 300, 2048, generator=g, device="cuda").half()
    y = torch.randn(2, 300, 2048, generator=g, device="cuda").half()
    n = ops.Norm("layer")
    h, z = ops.residual_norm(x, y, post=n, pre=n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h2, z2 = ops.residual_norm(x, y, post=n, pre=n)
    s.synchronize()
    assert torch.equal(h, h2) and torch.equal(z, z2)
    xs = x.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        hg, zg = ops.residual_norm(xs, y, post=n, pre=n)
        hg, zg = ops.residual_norm(hg, zg, pre=n)
    xs.copy_(2 * x)
    gr.replay()
    h3, z3 = ops.residual_norm(2 * x, y, post=n, pre=n)
    h3, z3 = ops.residual_norm(h3, z3, pre=n)
    assert torch.equal(hg, h3) and torch.equal(zg, z3)


def test_more_than_four_gigabytes(cuda_device):
    from katz_b200 import ops
    B, S, C = 3, 600000, 1280      # 2.3e9 elements
    x = torch.zeros(B, S, C, device="cuda", dtype=torch.float16)
    g = _gen(5)
    x[:, -3:] = torch.randn(B, 3, C, generator=g, device="cuda").half()
    scale = _vector(g, "sample", B, S, C)
    h, z = ops.residual_norm(x, x, pre=ops.Norm("rms"), scale=scale, residual_scale=0.5)
    first, second = ref.residual_norm(x[:, -3:], x[:, -3:], None, None, ("rms", None, None, 1e-5), scale, None, 0.5)
    ref.assert_within(h[:, -3:], *first, "h")
    ref.assert_within(z[:, -3:], *second, "z")
    assert not h[:, :-3].any() and not z[:, :-3].any()


def test_empty_and_refusals(cuda_device):
    from katz_b200 import KatzError, ops
    n = ops.Norm("rms")
    h, z = ops.residual_norm(torch.empty(2, 0, 64, device="cuda").half(), torch.empty(2, 0, 64, device="cuda").half(), pre=n)
    assert h.shape == z.shape == (2, 0, 64)
    x = torch.zeros(2, 4, 64, device="cuda").half()
    v = torch.zeros(64, device="cuda").half()
    buf = torch.zeros(2 * 4 * 64 * 2, device="cuda").half()
    bad = [
        lambda: ops.residual_norm(x), lambda: ops.residual_norm(x.cpu(), x.cpu(), pre=n), lambda: ops.residual_norm(x.bfloat16(), x, pre=n),
        lambda: ops.residual_norm(x, x.float(), pre=n), lambda: ops.residual_norm(x, x[:, :3], pre=n), lambda: ops.residual_norm(x, x.cpu(), pre=n),
        lambda: ops.residual_norm(x, gate=v, pre=n), lambda: ops.residual_norm(x, post=n, pre=n), lambda: ops.residual_norm(x, x, scale=v),
        lambda: ops.residual_norm(x, x, shift=v), lambda: ops.residual_norm(x, x, normed=x), lambda: ops.residual_norm(x, x, gate=v[:32]),
        lambda: ops.residual_norm(x, x, gate=v.float()), lambda: ops.residual_norm(x, x, gate=v.expand(3, 64)), lambda: ops.residual_norm(x, x, gate=v.cpu()),
        lambda: ops.residual_norm(x, x, gate=x[:, :3]), lambda: ops.residual_norm(x[0], x[0], gate=x), lambda: ops.residual_norm(x, x, gate=x.transpose(1, 2)[:, :, :1].expand(2, 64, 64)),
        lambda: ops.residual_norm(x[0, 0], x[0, 0], pre=n), lambda: ops.residual_norm(x[None], x[None], pre=n),
        lambda: ops.residual_norm(x.transpose(1, 2), pre=n), lambda: ops.residual_norm(torch.zeros(2, 16392, device="cuda"), pre=n),
        lambda: ops.residual_norm(x, pre=ops.Norm("rms", v[:8])), lambda: ops.residual_norm(x, pre=ops.Norm("rms", v.float())),
        lambda: ops.residual_norm(x, pre=ops.Norm("layer", v, v.cpu())), lambda: ops.Norm("batch"), lambda: ops.Norm("rms", eps=-1.0),
        lambda: ops.Norm("rms", eps=float("nan")),
        lambda: ops.residual_norm(x, x.clone(), pre=n, normed=x), lambda: ops.residual_norm(x, x.clone(), pre=n, out=v.expand(2, 4, 64)),
        lambda: ops.residual_norm(x, x.clone(), out=x.float()), lambda: ops.residual_norm(x, x.clone(), pre=n, normed=torch.zeros(2, 4, 64, device="cuda")),
        lambda: ops.residual_norm(buf.as_strided((2, 4, 64), (512, 128, 1)), x, out=buf.as_strided((2, 4, 64), (256, 64, 1))),
    ]
    y = x.clone()
    bad.append(lambda: ops.residual_norm(x, y, pre=n, out=y))
    for i, c in enumerate(bad):
        with pytest.raises(KatzError):
            c()
            pytest.fail("call %d was not refused" % i)


def test_a_conditioned_block_with_four_bit_weights(cuda_device):
    """The operators together, as a conditioned block runs them: the conditioning vector's product gives shift, scale and gate
    of both halves; norm -> 4-bit linear -> gated residual and next norm -> 4-bit linears -> gated residual."""
    from katz_b200 import ops
    g = _gen(7)
    B, S, C = 2, 64, 640
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ws = [ops.quantize_w4((rnd(n, k) * k ** -0.5).half()) for n, k in ((6 * C, 320), (C, C), (4 * C, C), (C, 4 * C))]
    cond, x = rnd(B, 320).half(), rnd(B, S, C).half()
    rows = lambda t: t.reshape(B * S, -1)  # noqa: E731
    n = ops.Norm("layer")

    def block(x):
        mod = ops.linear_w4(ops.silu(cond), *ws[0]).view(B, 6, C)
        x, z = ops.residual_norm(x, pre=n, shift=mod[:, 0], scale=mod[:, 1])
        a = ops.linear_w4(rows(z), *ws[1]).view(B, S, C)
        x, z = ops.residual_norm(x, a, gate=mod[:, 2], pre=n, shift=mod[:, 3], scale=mod[:, 4])
        f = ops.linear_w4(ops.linear_w4(rows(z), *ws[2], act=ops.ACT_SILU), *ws[3]).view(B, S, C)
        return ops.residual_norm(x, f, gate=mod[:, 5])[0]

    got = block(x)
    W = [ref.weights(q, s, None, 64) for q, s in ws]
    sil = lambda t: t * torch.sigmoid(t)  # noqa: E731
    ln = lambda t: (t - t.mean(-1, keepdim=True)) * ((t - t.mean(-1, keepdim=True)).pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()  # noqa: E731
    m = (sil(cond.double()) @ W[0].T).view(B, 6, 1, C).unbind(1)
    h = x.double()
    h = h + m[2] * ((ln(h) * (1 + m[1]) + m[0]) @ W[1].T)
    want = h + m[5] * (sil((ln(h) * (1 + m[4]) + m[3]) @ W[2].T) @ W[3].T)
    # nine fp16 roundings (half a step, 2^-11, each) on the way of a value, of which each product averages its inputs'; the
    # gains between them (gates, 1 + scale, the linears) are near one in the mean square: within 9 * 2^-11 in norm
    assert float((got.double() - want).norm() / want.norm()) < 9 * 2.0 ** -11
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        again = block(x)
    gr.replay()
    assert torch.equal(again, got)
