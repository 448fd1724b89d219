"""CPU: argument checks of the 4-bit weight and residual-norm entry points that return before any launch, and the 64-bit forms
the GPU tests compare with."""
import ctypes

import pytest
import torch

from tests import w4_reference as ref

P = 1 << 20      # a 16-byte aligned address that is never read: every call below is refused on the host


def test_entry_points_refuse_bad_arguments_without_a_device():
    from katz_b200 import _lib
    lib = _lib.load()
    quant = lambda w=P, ldw=256, q=P, s=P, N=4, K=256, g=64: lib.katz_quantize_w4_f16(w, ldw, q, s, N, K, g, None)  # noqa: E731
    deq = lambda q=P, s=P, z=None, w=P, ldw=256, N=4, K=256, g=64: lib.katz_dequantize_w4_f16(q, s, z, w, ldw, N, K, g, None)  # noqa: E731
    for f in (quant, deq):
        assert f(w=None) == f(q=None) == f(s=None) == -1
        assert f(g=0) == f(g=16) == f(g=256) == -1
        assert f(N=0) == f(K=0) == f(K=48) == f(ldw=248) == -3
        assert f(w=P + 2) == f(q=P + 8) == f(s=P + 1) == f(ldw=260) == -2

    def lin(x=P, ldx=256, q=P, s=P, z=None, g=64, o=P, ldo=8, M=4, N=8, K=256, b=None, r=None, ldr=0, act=0):
        a = _lib.LinearW4Args(x=x, q=q, scale=s, zero=z, bias=b, residual=r, out=o, ldx=ldx, ldo=ldo, ldr=ldr, M=M, N=N, K=K, group=g, act=act,
                              out_scale=1.0)
        return lib.katz_linear_w4_f16(ctypes.byref(a), None)
    assert lib.katz_linear_w4_f16(None, None) == -1
    assert lin(x=None) == lin(q=None) == lin(s=None) == lin(o=None) == lin(act=2) == lin(act=-1) == lin(g=33) == -1
    assert lin(M=0) == lin(N=0) == lin(K=0) == lin(K=250) == lin(M=-1) == lin(ldx=255) == lin(ldo=7) == lin(r=P, ldr=7) == -3
    assert lin(q=P + 1) == lin(s=P + 1) == lin(x=P + 1) == lin(o=P + 1) == lin(b=P + 1) == lin(r=P + 1, ldr=8) == -2


def test_residual_norm_refuses_bad_arguments_without_a_device():
    from katz_b200 import _lib
    lib = _lib.load()

    def call(**kw):
        a = _lib.ResidualNormArgs(x=P, y=P, h=P, z=P, B=2, S=3, C=64, pre_kind=1, x_ss=64, x_sb=192)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.katz_residual_norm_f16(ctypes.byref(a), None)
    assert lib.katz_residual_norm_f16(None, None) == -1
    assert call(x=None) == call(x_dtype=2) == call(post_kind=3) == call(pre_kind=-1) == call(z=None) == call(pre_kind=0) == -1
    assert call(y=None, gate=P) == call(y=None, post_kind=1) == call(pre_kind=0, z=None, scale=P) == call(pre_kind=0, z=None, h=None) == -1
    assert call(B=0) == call(S=0) == call(C=0) == call(C=16385) == call(B=1 << 20, S=1 << 20) == -3
    assert call(x=P + 1) == call(gate=P + 1) == call(x_dtype=1, h=P + 2) == -2


def test_struct_mirrors_the_header():
    from katz_b200 import _lib, ops
    assert ctypes.sizeof(_lib.ResidualNormArgs) == 11 * 8 + 14 * 8 + 6 * 4 + 3 * 4 + 4      # padded to 8
    assert ctypes.sizeof(_lib.LinearW4Args) == 7 * 8 + 3 * 8 + 5 * 4 + 4
    a = _lib.LinearW4Args.from_buffer_copy(ops._LINEAR_W4_ARGS.pack(*range(1, 16), 0.25))
    assert [getattr(a, n) for n, _ in a._fields_] == list(range(1, 16)) + [0.25]
    # the packed form that the wrapper passes is the same record
    packed = ops._RESIDUAL_NORM_ARGS.pack(*range(1, 32), 0.25, 0.5, 0.75)
    a = _lib.ResidualNormArgs.from_buffer_copy(packed)
    values = [getattr(a, n) for n, _ in a._fields_]
    assert values == list(range(1, 32)) + [0.25, 0.5, 0.75]


def test_wrappers_refuse_cpu_tensors_and_bad_norms():
    from katz_b200 import KatzError, ops
    h = torch.zeros(4, 64, dtype=torch.float16)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16)
    for f in (lambda: ops.quantize_w4(h), lambda: ops.dequantize_w4(q, s), lambda: ops.linear_w4(h, q, s),
              lambda: ops.residual_norm(h, pre=ops.Norm("rms")), lambda: ops.Norm("group"), lambda: ops.Norm("rms", eps=float("inf"))):
        with pytest.raises(KatzError):
            f()


def test_reference_forms():
    """The 64-bit forms agree with torch's own operators where those exist."""
    g = torch.Generator().manual_seed(0)
    w = (torch.randn(5, 96, generator=g) * 0.05).half()
    c, s = ref.quantize(w, 64)
    q = (c[:, 0::2].to(torch.uint8) | (c[:, 1::2].to(torch.uint8) << 4))
    assert torch.equal(ref.codes(q), c) and s.shape == (5, 2)
    back = ref.weights(q, s, None, 64)
    assert ((back - w.double()).abs() <= ref.per_k(s, 64, 96) * (0.5 + 7 * 2.0 ** -8)).all()
    assert torch.equal(back, back.half().double())      # a 4-bit weight is an fp16 number
    x = torch.randn(3, 96, generator=g).half()
    v, bound = ref.linear(x, q, s, None, 64, None, None, True, 2.0)
    want = 2 * torch.nn.functional.silu(x.double() @ back.T)
    assert torch.allclose(v, want, rtol=1e-12) and (bound > 0).all()
    t = torch.randn(2, 3, 40, generator=g)
    wt, b = torch.randn(40, generator=g).half(), torch.randn(40, generator=g).half()
    (h, _), (z, _) = ref.residual_norm(t, t.half(), None, ("rms", wt, None, 1e-6), ("layer", wt, b, 1e-5), None, None, 0.5)
    want_h = 0.5 * t.double() + torch.nn.functional.rms_norm(t.half().double(), (40,), wt.double(), 1e-6)
    assert torch.allclose(h, want_h, rtol=1e-10, atol=1e-12)
    assert torch.allclose(z, torch.nn.functional.layer_norm(want_h, (40,), wt.double(), b.double(), 1e-5), rtol=1e-9, atol=1e-11)
