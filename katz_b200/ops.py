"""Tensor-level wrappers over the C ABI: each takes torch CUDA tensors, checks layout, and launches on the current
torch stream. No op here computes anything in torch; a missing library or a failing launch raises KatzError."""
import ctypes
import os
import struct

import torch

from . import _lib
from ._lib import ACT_NONE, ACT_SILU, KatzError, call  # noqa: F401


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _f16(t, name):
    if t.dtype != torch.float16 or not t.is_cuda:
        raise KatzError("%s must be a CUDA fp16 tensor (got %s on %s)" % (name, t.dtype, t.device))
    return t


def _use_tc05():
    return os.environ.get("KATZ_GEMM", "tc05") != "mma"


def _al16(t):
    return t is None or t.data_ptr() % 16 == 0


def _tc05_linear_ok(x, w, bias, residual, rowvec, out):
    """Shapes/alignments the tcgen05 GEMM takes; anything else goes to the mma.sync kernel."""
    M, K = x.shape
    N = w.shape[0]
    if K % 64 or N % 8 or x.stride(0) % 8 or out.stride(0) % 8:
        return False
    if not (_al16(x) and _al16(w) and _al16(out) and _al16(bias) and _al16(residual) and _al16(rowvec)):
        return False
    if residual is not None and residual.stride(0) % 8:
        return False
    if rowvec is not None and rowvec.stride(0) % 8:
        return False
    return True


def _tc05_rowvec_ok(rowvec, rows_per_batch):
    """The tcgen05 epilogue adds one row vector per 128-row tile."""
    return rowvec is None or (rows_per_batch > 0 and rows_per_batch % 128 == 0)


def gemm_kernel_name():
    """Which GEMM family `linear` dispatches large aligned shapes to."""
    return "tcgen05" if _use_tc05() else "mma.sync"


def tc05_status():
    """Status word of the tcgen05 kernels (0 = no bounded wait ever gave up). Synchronises the device."""
    return _lib.load().katz_tc05_status()


class LnFold:
    """A LayerNorm folded into the linear layer that consumes it: `wf` = W diag(gamma) (fp16), `c12` = per output column
    (sum_k W'[n,k], sum_k W[n,k] beta[k] + bias[n]) in fp32, `eps` the norm's epsilon. Built by `ln_fold`."""

    def __init__(self, wf, c12, eps):
        self.wf, self.c12, self.eps = wf, c12, float(eps)


def ln_fold(w, gamma, beta, bias=None, eps=1e-5, out=None):
    """(Re)compute the folded constants of LayerNorm(gamma, beta) followed by linear(w, bias). Pass `out` (an LnFold) to
    refresh it in place after `w` changed."""
    _f16(w, "w"), _f16(gamma, "gamma"), _f16(beta, "beta")
    if not w.is_contiguous() or w.dim() != 2 or gamma.numel() != w.shape[1] or beta.numel() != w.shape[1]:
        raise KatzError("ln_fold: w must be a contiguous [N, K] tensor and gamma/beta [K]")
    N, K = w.shape
    if out is None:
        out = LnFold(torch.empty_like(w), torch.empty((N, 2), dtype=torch.float32, device=w.device), eps)
    call("katz_ln_fold_f16", _p(w), _p(gamma), _p(beta), _p(bias), _p(out.wf), _p(out.c12), N, K, _stream())
    return out


def ln_fusable(M, K, N):
    """Whether `linear(layer_norm(x), w)` with x [M, K], w [N, K] can run as one folded GEMM on the tcgen05 path."""
    return _use_tc05() and K % 64 == 0 and N % 8 == 0


def _extras(x, ln, ln_stats, stats_out, M, K, N):
    from ._lib import LinearExtras
    ex = LinearExtras()
    keep = []
    if ln is not None:
        if ln_stats is None or ln_stats.dtype != torch.float32 or not ln_stats.is_contiguous() or ln_stats.dim() != 3 \
                or ln_stats.shape[1] != M or ln_stats.shape[2] != 2 or ln_stats.shape[0] != (K + 31) // 32:
            raise KatzError("folded LayerNorm needs the producer's statistics [ceil(K/32), M, 2] fp32")
        ex.ln_stats, ex.ln_c12, ex.ln_slots, ex.ln_eps = ln_stats.data_ptr(), ln.c12.data_ptr(), ln_stats.shape[0], ln.eps
    if stats_out is True:
        stats_out = torch.empty(((N + 31) // 32, M, 2), dtype=torch.float32, device=x.device)
    if stats_out is not None:
        if stats_out.dtype != torch.float32 or not stats_out.is_contiguous() or tuple(stats_out.shape) != ((N + 31) // 32, M, 2):
            raise KatzError("stats_out must be a contiguous fp32 [ceil(N/32), M, 2] tensor")
        ex.stats_out = stats_out.data_ptr()
    return ex, stats_out


def feed_forward_geglu(x, w, bias, out=None, ln=None, ln_stats=None):
    """GEGLU feed-forward projection: x[M,K], w[2F,K] (the unsplit `proj`), bias[2F] -> [M,F] = h * gelu(g).
    One fused tcgen05 GEMM when the shape allows, else GEMM + gating kernel. With `ln` (an LnFold whose `wf` replaces `w`;
    `bias` is already inside it) and `ln_stats` (the row statistics of x) x is the input of the LayerNorm."""
    _f16(x, "x")
    if ln is not None:
        w, bias = ln.wf, None
    _f16(w, "w")
    M, K = x.shape
    F = w.shape[0] // 2
    if out is None:
        out = torch.empty((M, F), dtype=torch.float16, device=x.device)
    fused_ok = (_use_tc05() and os.environ.get("KATZ_FUSED_GEGLU", "1") == "1" and K % 64 == 0 and F % 16 == 0
                and x.stride(1) == 1 and x.stride(0) % 8 == 0 and w.is_contiguous() and _al16(x) and _al16(w) and _al16(out)
                and _al16(bias) and out.stride(0) % 8 == 0)
    if ln is not None:
        if not fused_ok:
            raise KatzError("feed_forward_geglu: this shape cannot take a folded LayerNorm")
        ex, _ = _extras(x, ln, ln_stats, None, M, K, 2 * F)
        call("katz_linear_geglu_ex_f16", _p(x), x.stride(0), _p(w), _p(out), out.stride(0), M, F, K, None, ctypes.byref(ex), _stream())
        return out
    if fused_ok:
        call("katz_linear_geglu_f16", _p(x), x.stride(0), _p(w), _p(out), out.stride(0), M, F, K, _p(bias), _stream())
        return out
    return geglu_erf(linear(x, w, bias), out=out)


def upsample_nearest2x(x, out=None):
    _f16(x, "x")
    B, H, W, C = x.shape
    if out is None:
        out = torch.empty((B, 2 * H, 2 * W, C), dtype=torch.float16, device=x.device)
    call("katz_upsample_nearest2x_nhwc_f16", _p(x), _p(out), B, H, W, C, _stream())
    return out


def linear(x, w, bias=None, residual=None, act=ACT_NONE, rowvec=None, rows_per_batch=0, out=None, out_scale=1.0,
           ln=None, ln_stats=None, stats_out=None):
    """out[M,N] = x[M,K] @ w[N,K]^T (+bias) (+rowvec[m // rows_per_batch]) -> act -> (+residual) * out_scale.
    `x`, `residual`, `out` may be row-strided 2-D views (unit column stride).
    Folded LayerNorm: with `ln` (an LnFold; its `wf` replaces `w` and holds the bias) and `ln_stats` the call computes
    linear(layer_norm(x)); with `stats_out=True` (or a buffer) it also returns the row statistics of its own output for the
    next folded LayerNorm: `(out, stats)`."""
    _f16(x, "x")
    if ln is not None:
        w, bias = ln.wf, None
    _f16(w, "w")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise KatzError("linear: shape mismatch x%s w%s" % (tuple(x.shape), tuple(w.shape)))
    if x.stride(1) != 1 or not w.is_contiguous():
        raise KatzError("linear: x must have unit column stride and w must be contiguous")
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=x.device)
    if out.stride(1) != 1 or out.shape != (M, N):
        raise KatzError("linear: bad out")
    if residual is not None and (residual.shape != (M, N) or residual.stride(1) != 1):
        raise KatzError("linear: bad residual")
    tc05 = _use_tc05() and _tc05_linear_ok(x, w, bias, residual, rowvec, out) and _tc05_rowvec_ok(rowvec, rows_per_batch)
    if ln is not None or stats_out is not None:
        if not tc05:
            raise KatzError("linear: this shape cannot take a folded LayerNorm / emit row statistics (tcgen05 path only)")
        ex, stats = _extras(x, ln, ln_stats, stats_out, M, K, N)
        call("katz_linear_ex_f16", _p(x), x.stride(0), _p(w), _p(out), out.stride(0), M, N, K, _p(bias), _p(rowvec),
             rowvec.stride(0) if rowvec is not None else 0, rows_per_batch, _p(residual),
             residual.stride(0) if residual is not None else 0, act, float(out_scale), ctypes.byref(ex), _stream())
        return (out, stats) if stats is not None else out
    name = "katz_linear_f16" if tc05 else "katz_linear_f16_mma"
    call(name, _p(x), x.stride(0), _p(w), _p(out), out.stride(0), M, N, K, _p(bias), _p(rowvec),
         rowvec.stride(0) if rowvec is not None else 0, rows_per_batch, _p(residual),
         residual.stride(0) if residual is not None else 0, act, float(out_scale), _stream())
    return out


_F16, _F32, _BF16, _U8 = torch.float16, torch.float32, torch.bfloat16, torch.uint8
# the raw handle of a device's current stream; torch.cuda.current_stream() builds an object around it, which takes 3 us, a
# quarter of a small call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call_on(index, name, *args):
    """Launch on the current stream of CUDA device `index`, which need not be the current device."""
    if index == _current_device():
        call(name, *args, _raw_stream(index))
        return
    with torch.cuda.device(index):
        call(name, *args, _raw_stream(index))


def _expect(t, what, name, dtype, index):
    """t is a tensor of `dtype` on CUDA device `index` (None: on any)."""
    at = t.get_device()
    if t.dtype is not dtype or at < 0 or (index is not None and at != index):
        where = "" if index is None else " %d" % index
        raise KatzError("%s: %s must be a %s tensor on CUDA device%s (got %s on %s)" % (what, name, dtype, where, t.dtype, t.device))
    return at


def _row_stride(t, what, name, M, N):
    """Row stride of an [M, N] tensor with unit column stride and rows that do not overlap."""
    if t.shape != (M, N):
        raise KatzError("%s: %s must be %s (got %s)" % (what, name, (M, N), tuple(t.shape)))
    ld, one = t.stride()
    if one != 1 and N != 1:
        raise KatzError("%s: %s must have unit column stride (got strides %s)" % (what, name, t.stride()))
    if M < 2:
        return N
    if ld < N:
        raise KatzError("%s: the rows of %s overlap (strides %s)" % (what, name, t.stride()))
    return ld


def _w4_check(what, q, scale, zero, group):
    """(device index, N, K) of a 4-bit weight; see quantize_w4 for the format."""
    if group not in (32, 64, 128):
        raise KatzError("%s: group must be 32, 64 or 128 (got %r)" % (what, group))
    index = q.get_device()
    if q.dtype is not _U8 or index < 0:
        _expect(q, what, "q", _U8, None)
    if q.dim() != 2 or not q.is_contiguous():
        raise KatzError("%s: q must be a contiguous [N, K/2] tensor" % what)
    N, K = q.shape
    K *= 2
    if K == 0 or K % 32:
        raise KatzError("%s: K must be a positive multiple of 32 (got %d)" % (what, K))
    if q.data_ptr() % 16:
        raise KatzError("%s: q must start on a 16-byte boundary" % what)
    shape = (N, (K + group - 1) // group)
    if scale.dtype is not _BF16 or scale.get_device() != index:
        _expect(scale, what, "scale", _BF16, index)
    if scale.shape != shape or not scale.is_contiguous():
        raise KatzError("%s: scale must be a contiguous [N, ceil(K/group)] = %s tensor" % (what, shape))
    if zero is not None:
        _expect(zero, what, "zero", _U8, index)
        if zero.shape != shape or not zero.is_contiguous():
            raise KatzError("%s: zero must be a contiguous %s tensor" % (what, shape))
    return index, N, K


def quantize_w4(w, group=64, out=None):
    """fp16 weights [N, K] -> (q, scale), 4 bits a weight. K is a multiple of 32; w may be row-strided.
    q: uint8 [N, K/2], two codes a byte, the even k in the low four bits; scale: bf16 [N, ceil(K/group)], one for `group` (32,
    64 or 128) consecutive k of a row, the last group may be short; weight = scale * (code - 8), |code - 8| <= 7, ties to even.
    A group that holds an infinity or a NaN reads back as NaN. Rows are independent: row slices of (q, scale) are the 4-bit
    form of the same rows of w. `out` = (q, scale) rewrites an existing pair, as after an adapter switch."""
    index = _expect(w, "quantize_w4", "w", _F16, None)
    if w.dim() != 2 or w.shape[1] == 0 or w.shape[1] % 32:
        raise KatzError("quantize_w4: w must be [N, K] with K a positive multiple of 32 (got %s)" % (tuple(w.shape),))
    N, K = w.shape
    ld = _row_stride(w, "quantize_w4", "w", N, K)
    if w.data_ptr() % 16 or ld % 8:
        raise KatzError("quantize_w4: the rows of w must start on 16-byte boundaries")
    if group not in (32, 64, 128):
        raise KatzError("quantize_w4: group must be 32, 64 or 128 (got %r)" % (group,))
    if out is None:
        q, scale = w.new_empty(N, K // 2, dtype=_U8), w.new_empty(N, (K + group - 1) // group, dtype=_BF16)
    else:
        q, scale = out
        if _w4_check("quantize_w4", q, scale, None, group) != (index, N, K):
            raise KatzError("quantize_w4: out does not match w %s on %s" % (tuple(w.shape), w.device))
    if N:
        _call_on(index, "katz_quantize_w4_f16", w.data_ptr(), ld, q.data_ptr(), scale.data_ptr(), N, K, group)
    return q, scale


def dequantize_w4(q, scale, zero=None, group=64, out=None):
    """4-bit weights -> fp16 [N, K] = scale * (code - zero), rounded once. `zero`: uint8 of scale's shape, 0..15 (None: 8)."""
    index, N, K = _w4_check("dequantize_w4", q, scale, zero, group)
    ld = K
    if out is None:
        out = q.new_empty(N, K, dtype=_F16)
    else:
        _expect(out, "dequantize_w4", "out", _F16, index)
        ld = _row_stride(out, "dequantize_w4", "out", N, K)
        if out.data_ptr() % 16 or ld % 8:
            raise KatzError("dequantize_w4: the rows of out must start on 16-byte boundaries")
    if N:
        _call_on(index, "katz_dequantize_w4_f16", q.data_ptr(), scale.data_ptr(), zero.data_ptr() if zero is not None else None,
                 out.data_ptr(), ld, N, K, group)
    return out


# the C records as bytes: packed in 0.2 us, where converting as many arguments one by one takes ctypes 1 us
_LINEAR_W4_ARGS = struct.Struct("=7Q3q5if")               # katz_linear_w4_args
_RESIDUAL_NORM_ARGS = struct.Struct("=11Q14q6i3f4x")      # katz_residual_norm_args


def linear_w4(x, q, scale, zero=None, group=64, bias=None, residual=None, act=ACT_NONE, out=None, out_scale=1.0):
    """`linear` with 4-bit weights (the format of quantize_w4, optionally with zero points): out[M,N] = x[M,K] @ w[N,K]^T
    (+bias) -> act -> (+residual) * out_scale, fp32 accumulation, one rounding. Any M (0 included) and N.
    `x`, `residual`, `out` may be row-strided 2-D views (unit column stride); `out` may be `residual` and overlaps nothing else.
    Rows of x that do not start on 16-byte boundaries are read by a slower kernel. Scales of 2^-23 to 64 are covered: the
    weights of larger ones may overflow fp16 to infinity (from 1023 on), those of smaller ones lose bits."""
    index, N, K = _w4_check("linear_w4", q, scale, zero, group)
    if x.dtype is not _F16 or x.get_device() != index:
        _expect(x, "linear_w4", "x", _F16, index)
    M = x.shape[0] if x.dim() == 2 else -1
    ldx = _row_stride(x, "linear_w4", "x", M, K)
    if act != ACT_NONE and act != ACT_SILU:
        raise KatzError("linear_w4: unknown activation %r" % (act,))
    ldo = N
    if out is None:
        out = x.new_empty(M, N)
    else:
        _expect(out, "linear_w4", "out", _F16, index)
        ldo = _row_stride(out, "linear_w4", "out", M, N)
        if M and N and out.data_ptr() == x.data_ptr():
            raise KatzError("linear_w4: out must not be x")
    bias_p = residual_p = ldr = 0
    if bias is not None:
        if bias.dtype is not _F16 or bias.get_device() != index:
            _expect(bias, "linear_w4", "bias", _F16, index)
        if bias.dim() != 1 or bias.numel() != N or not bias.is_contiguous():
            raise KatzError("linear_w4: bias must be a contiguous [N] tensor")
        bias_p = bias.data_ptr()
    if residual is not None:
        _expect(residual, "linear_w4", "residual", _F16, index)
        ldr = _row_stride(residual, "linear_w4", "residual", M, N)
        residual_p = residual.data_ptr()
        if ldr != ldo and residual_p == out.data_ptr():
            raise KatzError("linear_w4: residual starts where out does, with another row stride")
    if M and N:
        _call_on(index, "katz_linear_w4_f16", _LINEAR_W4_ARGS.pack(
            x.data_ptr(), q.data_ptr(), scale.data_ptr(), 0 if zero is None else zero.data_ptr(), bias_p, residual_p, out.data_ptr(),
            ldx, ldo, ldr, M, N, K, group, act, out_scale))
    return out


def conv2d(x, w, bias=None, ksize=3, stride=1, pad=1, upsample=False, x2=None, rowvec=None, residual=None,
           act=ACT_NONE, out=None, out_scale=1.0, pad_h=None):
    """NHWC convolution. x: [B,Hs,Ws,C1] (+ optional x2 [B,Hs,Ws,C2] concatenated along channels); w: [Cout,k,k,C1+C2].
    With upsample=True the input is read through a nearest 2x upsample. rowvec: [B, >=Cout] row-strided view added per
    batch element; residual: [B,Hout,Wout,Cout]. `pad_h` overrides the vertical padding (0 for a row shard whose input
    already carries its halo rows)."""
    _f16(x, "x"), _f16(w, "w")
    if not x.is_contiguous() or not w.is_contiguous():
        raise KatzError("conv2d: x and w must be contiguous")
    B, Hs, Ws, C1 = x.shape
    C2 = 0
    if x2 is not None:
        if not x2.is_contiguous() or x2.shape[:3] != x.shape[:3]:
            raise KatzError("conv2d: bad x2")
        C2 = x2.shape[3]
    Cout = w.shape[0]
    if w.numel() != Cout * ksize * ksize * (C1 + C2):
        raise KatzError("conv2d: weight does not match [Cout,k,k,Cin]")
    ph = pad if pad_h is None else pad_h
    Hin, Win = (Hs * 2, Ws * 2) if upsample else (Hs, Ws)
    Hout = (Hin + 2 * ph - ksize) // stride + 1
    Wout = (Win + 2 * pad - ksize) // stride + 1
    if out is None:
        out = torch.empty((B, Hout, Wout, Cout), dtype=torch.float16, device=x.device)
    if residual is not None and (tuple(residual.shape) != (B, Hout, Wout, Cout) or not residual.is_contiguous()):
        raise KatzError("conv2d: bad residual")
    tw = min(Wout, 128)
    if (_use_tc05() and ksize == 3 and stride in (1, 2) and pad == 1 and ph in (0, 1) and x2 is None and C1 % 64 == 0
            and Cout % 8 == 0 and tw >= 8 and (tw & (tw - 1)) == 0 and Wout % tw == 0 and (stride == 1 or Win % 2 == 0)
            and _al16(x) and _al16(w) and _al16(out)
            and _al16(bias) and _al16(residual) and (rowvec is None or (_al16(rowvec) and rowvec.stride(0) % 8 == 0))):
        src = upsample_nearest2x(x) if upsample else x
        call("katz_conv3x3_nhwc_f16", _p(src), _p(w), _p(out), B, Hin, Win, C1, Cout, stride, ph, _p(bias), _p(rowvec),
             rowvec.stride(0) if rowvec is not None else 0, _p(residual), act, float(out_scale), _stream())
        return out
    if (ksize == 3 and stride in (1, 2) and pad == 1 and ph in (0, 1) and x2 is None and not upsample and rowvec is None
            and residual is None and out_scale == 1.0 and C1 in (8, 16, 32) and Cout % 8 == 0 and Cout <= 1024
            and _al16(x) and _al16(w) and _al16(out) and _al16(bias) and os.environ.get("KATZ_CONV_SMALL", "1") != "0"):
        # few input channels (the ControlNet conditioning embedding): direct convolution from a shared-memory patch
        call("katz_conv3x3_small_nhwc_f16", _p(x), _p(w), _p(out), B, Hin, Win, C1, Cout, stride, ph, _p(bias), act, _stream())
        return out
    call("katz_conv2d_nhwc_f16_mma", _p(x), _p(x2), _p(w), _p(out), B, Hin, Win, C1, C2, Cout, ksize, stride, ph, pad,
         1 if upsample else 0, _p(bias), _p(rowvec), rowvec.stride(0) if rowvec is not None else 0, _p(residual), act,
         float(out_scale), _stream())
    return out


_gn_scratch = {}


def _scratch(device, nbytes):
    # one buffer per (device, stream): launches that share a scratch buffer must be ordered, and two branches of a CUDA
    # graph (the two halves of a CFG batch on two streams) are not
    key = (device, torch.cuda.current_stream(device).cuda_stream)
    buf = _gn_scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        # zero-filled: the head of the scratch holds the GroupNorm ticket counters, which the kernels return to zero
        buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _gn_scratch[key] = buf
    return buf


def group_norm_nhwc(x, gamma, beta, groups, eps, act=ACT_NONE, out=None):
    """GroupNorm (+SiLU) over an NHWC tensor [B,H,W,C] (or [B,HW,C])."""
    _f16(x, "x")
    if not x.is_contiguous():
        raise KatzError("group_norm: x must be contiguous")
    B, C = x.shape[0], x.shape[-1]
    HW = x.numel() // (B * C)
    if out is None:
        out = torch.empty_like(x)
    lib = _lib.load()
    need = lib.katz_group_norm_scratch_bytes(B, HW, C, groups)
    if need < 0:
        raise KatzError("group_norm: bad shape")
    # The scratch buffer is shared by every GroupNorm call on this device: calls are ordered on one stream.
    scratch = _scratch(x.device, need)
    call("katz_group_norm_nhwc_f16", _p(x), _p(out), _p(gamma), _p(beta), B, HW, C, groups, float(eps), act,
         _p(scratch), scratch.numel(), _stream())
    return out


def group_norm_stats(x, groups):
    """fp64 (sum, sum of squares) per (batch, group) of an NHWC shard: [B, G, 2]. First half of a GroupNorm whose
    statistics span several GPUs."""
    _f16(x, "x")
    if not x.is_contiguous():
        raise KatzError("group_norm: x must be contiguous")
    B, C = x.shape[0], x.shape[-1]
    HW = x.numel() // (B * C)
    lib = _lib.load()
    need = lib.katz_group_norm_scratch_bytes(B, HW, C, groups)
    if need < 0:
        raise KatzError("group_norm: bad shape")
    scratch = _scratch(x.device, need)
    sums = torch.empty((B, groups, 2), dtype=torch.float64, device=x.device)
    call("katz_group_norm_stats_nhwc_f16", _p(x), _p(sums), B, HW, C, groups, _p(scratch), scratch.numel(), _stream())
    return sums


def group_norm_apply(x, sums, gamma, beta, groups, n_total, eps, act=ACT_NONE, out=None):
    """Second half: normalise the shard with the statistics of the whole tensor; n_total = elements per (batch, group)
    over the WHOLE tensor. sums: fp64 [B, G, 2] (already summed over the shards) or [P, B, G, 2] (one entry per shard,
    added here in shard order)."""
    _f16(x, "x")
    B, C = x.shape[0], x.shape[-1]
    HW = x.numel() // (B * C)
    if sums.dtype != torch.float64 or not sums.is_contiguous() or tuple(sums.shape[-3:]) != (B, groups, 2) or sums.dim() not in (3, 4):
        raise KatzError("group_norm_apply: sums must be a contiguous fp64 [B, G, 2] or [P, B, G, 2] tensor")
    n_parts = sums.shape[0] if sums.dim() == 4 else 1
    if out is None:
        out = torch.empty_like(x)
    call("katz_group_norm_apply_nhwc_f16", _p(x), _p(out), _p(sums), n_parts, _p(gamma), _p(beta), B, HW, C, groups,
         float(n_total), float(eps), act, _stream())
    return out


def group_norm_nchw(x, gamma, beta, groups, eps, act=ACT_NONE, out=None):
    _f16(x, "x")
    if not x.is_contiguous():
        raise KatzError("group_norm: x must be contiguous")
    B, C = x.shape[0], x.shape[1]
    HW = x.numel() // (B * C)
    if out is None:
        out = torch.empty_like(x)
    call("katz_group_norm_nchw_f16", _p(x), _p(out), _p(gamma), _p(beta), B, HW, C, groups, float(eps), act, _stream())
    return out


def layer_norm(x, gamma, beta, eps=1e-5, out=None):
    _f16(x, "x")
    if not x.is_contiguous():
        raise KatzError("layer_norm: x must be contiguous")
    C = x.shape[-1]
    rows = x.numel() // C
    if out is None:
        out = torch.empty_like(x)
    call("katz_layer_norm_f16", _p(x), _p(out), _p(gamma), _p(beta), rows, C, float(eps), _stream())
    return out


_INF = float("inf")


class Norm:
    """A norm of `residual_norm`: kind "layer" ((v - mean) / sqrt(var + eps)) or "rms" (v / sqrt(mean of v^2 + eps)), with optional
    fp16 weight [C] and bias [C]."""

    __slots__ = ("kind", "code", "weight", "bias", "eps")
    _CODES = {"layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}

    def __init__(self, kind, weight=None, bias=None, eps=1e-5):
        code = self._CODES.get(kind)
        if code is None:
            raise KatzError('Norm: kind must be "layer" or "rms" (got %r)' % (kind,))
        if not 0.0 <= eps < _INF:
            raise KatzError("Norm: eps must be finite and not negative (got %r)" % (eps,))
        self.kind = kind
        self.code = code
        self.weight = weight
        self.bias = bias
        self.eps = eps


def _row_strides(t, name, shape):
    """(batch, token) strides of an activation [rows, C] or [B, S, C] of the given shape with unit channel stride."""
    st = t.stride()
    if t.shape != shape or (st[-1] != 1 and shape[-1] != 1):
        raise KatzError("residual_norm: %s must be %s with unit channel stride (got %s, strides %s)" % (name, tuple(shape), tuple(t.shape), st))
    if len(st) == 2:
        return 0, (st[0] if shape[0] > 1 else 0)
    return (st[0] if shape[0] > 1 else 0), (st[1] if shape[1] > 1 else 0)


def _written_rows(t, name, shape, B, S, C):
    sb, ss = _row_strides(t, name, shape)
    if (S > 1 and ss < C) or (B > 1 and sb < (S - 1) * ss + C):
        raise KatzError("residual_norm: the rows of %s overlap (strides %s)" % (name, t.stride()))
    return sb, ss


def _vector(t, name, shape, index):
    """(address, batch stride, token stride) of a gate, scale or shift: [C], [B, C] ([rows, C] for a 2-D x) or [B, S, C], sizes
    of 1 broadcast."""
    if t.dtype is not _F16 or t.get_device() != index:
        _expect(t, "residual_norm", name, _F16, index)
    ts = t.shape
    if len(ts) == 1 and ts[0] == shape[-1] and t.is_contiguous():
        return t.data_ptr(), 0, 0
    st = t.stride()
    d, full = len(ts), len(shape)
    ok = 0 < d <= full and ts[-1] == shape[-1] and (st[-1] == 1 or ts[-1] == 1)
    sb = ss = 0
    if ok and d > 1:
        if ts[0] != 1:
            ok = ts[0] == shape[0]
            if full == 2:      # a 2-D x is one batch of rows
                ss = st[0]
            else:
                sb = st[0]
        if d == 3 and ts[1] != 1:
            ok = ok and ts[1] == shape[1]
            ss = st[1]
    if not ok:
        raise KatzError("residual_norm: %s %s (strides %s) does not fit x %s" % (name, tuple(ts), st, tuple(shape)))
    return t.data_ptr(), sb, ss


def _norm_vector(v, side, C, index):
    """Address of a norm's weight or bias."""
    if v is None:
        return 0
    if v.dtype is not _F16 or v.get_device() != index or v.shape != (C,) or not v.is_contiguous():
        raise KatzError("residual_norm: weight and bias of %s must be contiguous fp16 [C] = [%d] tensors on CUDA device %d (got %s %s on %s)"
                        % (side, C, index, v.dtype, tuple(v.shape), v.device))
    return v.data_ptr()


def residual_norm(x, y=None, gate=None, post=None, pre=None, scale=None, shift=None, residual_scale=1.0, out=None, normed=None):
    """The norms after and before a block with its gate and the residual scale between them, in one kernel:
    `h = residual_scale * x + gate * post(y)`, `z = pre(h) * (1 + scale) + shift`; returns (h, z).
    x: [rows, C] or [B, S, C], the residual stream, fp16 or fp32; y: the block's output, fp16, x's shape; C <= 16384.
    post, pre: Norm or None. gate, scale, shift: fp16, per channel [C], per sample [B, C], per token [B, S, C] (a 2-D x: [C]
    or [rows, C]); sizes of 1 broadcast and any may be a view into a wider row. h has x's type, z is fp16 and None without
    `pre`; both are rounded once, z from the unrounded h. Without y, h is residual_scale * x (x itself where that is 1 and no
    `out` is given). `out` (for h) may be x, `normed` (for z) may be y, and overlap nothing else; all last strides are 1."""
    dtype = x.dtype
    if dtype is not _F16 and dtype is not _F32:
        raise KatzError("residual_norm: x must be a CUDA fp16 or fp32 tensor (got %s on %s)" % (dtype, x.device))
    index = x.get_device()
    if index < 0:
        _expect(x, "residual_norm", "x", dtype, None)
    shape = x.shape
    if len(shape) == 3:
        B, S, C = shape
    elif len(shape) == 2:
        B, (S, C) = 1, shape
    else:
        B = S = C = 0
    if not 0 < C <= _lib.RESIDUAL_NORM_MAX_C:
        raise KatzError("residual_norm: x must be [rows, C] or [B, S, C] with 1 <= C <= %d (got %s)" % (_lib.RESIDUAL_NORM_MAX_C, tuple(shape)))
    if y is None and (gate is not None or post is not None):
        raise KatzError("residual_norm: gate and post need y")
    if pre is None and (scale is not None or shift is not None or normed is not None):
        raise KatzError("residual_norm: scale, shift and normed need pre")
    if y is None and pre is None:
        raise KatzError("residual_norm: neither y nor pre: nothing to compute")
    x_p = x.data_ptr()
    plain = x.is_contiguous()
    x_sb, x_ss = (S * C, C) if plain else _row_strides(x, "x", shape)
    y_p = y_sb = y_ss = gate_p = gate_sb = gate_ss = scale_p = scale_sb = scale_ss = shift_p = shift_sb = shift_ss = 0
    post_kind = post_w = post_b = pre_kind = pre_w = pre_b = 0
    post_eps = pre_eps = 0.0
    plain_y = False
    if y is not None:
        if y.dtype is not _F16 or y.get_device() != index:
            _expect(y, "residual_norm", "y", _F16, index)
        plain_y = y.shape == shape and y.is_contiguous()
        y_sb, y_ss = (S * C, C) if plain_y else _row_strides(y, "y", shape)
        y_p = y.data_ptr()
        if gate is not None:
            gate_p, gate_sb, gate_ss = _vector(gate, "gate", shape, index)
        if post is not None:
            post_kind, post_eps = post.code, post.eps
            post_w, post_b = _norm_vector(post.weight, "post", C, index), _norm_vector(post.bias, "post", C, index)
    if pre is not None:
        pre_kind, pre_eps = pre.code, pre.eps
        pre_w, pre_b = _norm_vector(pre.weight, "pre", C, index), _norm_vector(pre.bias, "pre", C, index)
        if scale is not None:
            scale_p, scale_sb, scale_ss = _vector(scale, "scale", shape, index)
        if shift is not None:
            shift_p, shift_sb, shift_ss = _vector(shift, "shift", shape, index)
    h, h_p, h_sb, h_ss = out, 0, S * C, C
    if out is not None:
        _expect(out, "residual_norm", "out", dtype, index)
        h_sb, h_ss = _written_rows(out, "out", shape, B, S, C)
        h_p = out.data_ptr()
        if h_p == y_p or (h_p == x_p and (h_sb, h_ss) != (x_sb, x_ss)):
            raise KatzError("residual_norm: out may be x (with the same strides), not y")
    elif y is None and residual_scale == 1.0:
        h = x
    else:
        h = torch.empty_like(x) if plain else x.new_empty(shape)      # empty_like is the faster of the two
        h_p = h.data_ptr()
    z, z_p, z_sb, z_ss = normed, 0, S * C, C
    if normed is not None:
        _expect(normed, "residual_norm", "normed", _F16, index)
        z_sb, z_ss = _written_rows(normed, "normed", shape, B, S, C)
        z_p = normed.data_ptr()
        if z_p == x_p or z_p == h_p or (z_p == y_p and (z_sb, z_ss) != (y_sb, y_ss)):
            raise KatzError("residual_norm: normed may be y (with the same strides), not x or out")
    elif pre is not None:
        z = torch.empty_like(y) if plain_y else torch.empty_like(x) if plain and dtype is _F16 else x.new_empty(shape, dtype=_F16)
        z_p = z.data_ptr()
    if B and S:
        _call_on(index, "katz_residual_norm_f16", _RESIDUAL_NORM_ARGS.pack(
            x_p, y_p, gate_p, scale_p, shift_p, post_w, post_b, pre_w, pre_b, h_p, z_p, x_sb, x_ss, y_sb, y_ss, h_sb, h_ss, z_sb, z_ss,
            gate_sb, gate_ss, scale_sb, scale_ss, shift_sb, shift_ss, B, S, C, 0 if dtype is _F16 else 1, post_kind, pre_kind, post_eps, pre_eps,
            residual_scale))
    return h, z


def geglu_erf(hg, out=None):
    """hg: [M, 2F] contiguous -> [M, F] = hg[:, :F] * gelu(hg[:, F:])."""
    _f16(hg, "hg")
    M, F2 = hg.shape
    F = F2 // 2
    if out is None:
        out = torch.empty((M, F), dtype=torch.float16, device=hg.device)
    call("katz_geglu_erf_f16", _p(hg), _p(out), M, F, hg.stride(0), _stream())
    return out


def fast_gelu_mul(x, m, out=None):
    _f16(x, "x"), _f16(m, "m")
    if x.shape != m.shape:
        raise KatzError("Input tensors x and m must have the same shape.")
    if not x.is_contiguous():
        raise KatzError("Input tensor x must be contiguous.")
    if not m.is_contiguous():
        raise KatzError("Input tensor m must be contiguous.")
    if out is None:
        out = torch.empty_like(x)
    call("katz_fast_gelu_mul_f16", _p(x), _p(m), _p(out), x.numel(), _stream())
    return out


def softmax_rows(x, out=None):
    """Row softmax of a 2-D fp16 matrix of logits (fp32 arithmetic); `out` may be `x`. Rows may be strided."""
    _f16(x, "x")
    if x.dim() != 2 or x.stride(1) != 1:
        raise KatzError("softmax_rows: x must be 2-D with unit column stride")
    if out is None:
        out = torch.empty_like(x)
    if out.shape != x.shape or out.stride(1) != 1 or out.dtype != torch.float16:
        raise KatzError("softmax_rows: bad out")
    call("katz_softmax_rows_f16", _p(x), _p(out), x.shape[0], x.shape[1], x.stride(0), out.stride(0), _stream())
    return out


_attn_scratch = {}


def _attention_scratch(device):
    """Scratch of the attention kernel's cut query tiles: one zero-filled buffer per device, of the size that is enough
    for every shape, allocated once (a captured graph keeps pointing at it)."""
    key = (device, torch.cuda.current_stream(device).cuda_stream)      # per stream, as the GroupNorm scratch
    buf = _attn_scratch.get(key)
    if buf is None:
        buf = torch.zeros(int(_lib.load().katz_attention_split_scratch_bytes()), dtype=torch.uint8, device=device)
        _attn_scratch[key] = buf
    return buf


def attention(q, k, v, heads, out=None, scale=None, kv_chunks=None, peer=None):
    """q: [B,Sq,>=H*64] view, k/v: [B,Sk,...] views (unit last stride, any row/batch stride); returns [B,Sq,H*64].
    kv_chunks=(n_chunks, chunk_rows, chunk_stride): k/v describe the FIRST chunk ([B, chunk_rows, ...]); chunk c of the
    keys/values starts `c * chunk_stride` elements later (the [P, B, s, C] result of an all-gather of row shards).
    peer=(address of this rank's arena control words, this rank's chunk): the chunks were pushed WITHOUT waiting
    (PeerArena.allgather(wait=False)) and the kernel waits for each peer's flag before it first touches that peer's chunk."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _f16(t, n)
        if t.dim() != 3 or t.stride(2) != 1:
            raise KatzError("attention: %s must be [B,S,C] with unit last stride" % n)
    B, Sq, _ = q.shape
    Sk = k.shape[1]
    chunk_rows, chunk_stride = 0, 0
    if kv_chunks is not None:
        n_chunks, chunk_rows, chunk_stride = kv_chunks
        Sk = n_chunks * chunk_rows
    D = 64
    if out is None:
        out = torch.empty((B, Sq, heads * D), dtype=torch.float16, device=q.device)
    if scale is None:
        scale = D ** -0.5
    args = (_p(q), _p(k), _p(v), _p(out), B, heads, Sq, Sk, D, q.stride(1), k.stride(1), v.stride(1), out.stride(1),
            q.stride(0), k.stride(0), v.stride(0), out.stride(0), float(scale), chunk_rows, chunk_stride, _stream())
    strides_ok = all(t.stride(1) % 8 == 0 and t.stride(0) % 8 == 0 and _al16(t) for t in (q, k, v, out))
    # KATZ_ATTN: "tc05" / "mma" force a kernel; by default a single key tile (cross-attention over 77 text tokens) goes to
    # the mma.sync kernel, whose CTAs share an SM (measured 9.5 us against 13.5 us for 2x20 heads x 1024 queries)
    mode = os.environ.get("KATZ_ATTN", "auto")
    if (_use_tc05() and (mode == "tc05" or (mode == "auto" and Sk > 128)) and strides_ok
            and (chunk_rows == 0 or (chunk_rows % 128 == 0 and chunk_stride % 8 == 0))):
        if peer is not None:
            scratch = _attention_scratch(q.device)
            call("katz_attention_peer_f16", *args[:-1], _p(scratch), scratch.numel(), ctypes.c_void_p(int(peer[0])), int(peer[1]),
                 args[-1])
        elif os.environ.get("KATZ_ATTN_SPLIT", "1") != "0":
            scratch = _attention_scratch(q.device)
            call("katz_attention_split_f16", *args[:-1], _p(scratch), scratch.numel(), args[-1])
        else:
            call("katz_attention_f16", *args)
    else:
        if peer is not None:
            raise KatzError("attention: chunks that are still in flight need the tcgen05 kernel (128-row chunks, aligned strides)")
        call("katz_attention_f16_mma", *args)
    return out


def residual_intake(src, residuals, scales, out=None):
    """out = src + half(sum_i scales[i] * residuals[i])."""
    _f16(src, "src")
    n = len(residuals)
    if out is None:
        out = torch.empty_like(src)
    ptrs = (ctypes.c_void_p * n)(*[r.data_ptr() for r in residuals])
    for r in residuals:
        _f16(r, "residual")
        if r.numel() != src.numel() or not r.is_contiguous():
            raise KatzError("residual_intake: residual shape/layout mismatch")
    sc = (ctypes.c_float * n)(*[float(s) for s in scales])
    call("katz_residual_intake_f16", _p(src), _p(out), ptrs, sc, n, src.numel(), _stream())
    return out


def timestep_embedding(t, dim, out=None):
    """t: fp32 CUDA tensor [rows] -> fp16 [rows, dim]."""
    if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
        raise KatzError("timestep_embedding: t must be a contiguous CUDA fp32 tensor")
    rows = t.numel()
    if out is None:
        out = torch.empty((rows, dim), dtype=torch.float16, device=t.device)
    call("katz_timestep_embedding_f16", _p(t), _p(out), rows, dim, out.stride(0), _stream())
    return out


def silu(x, out=None):
    _f16(x, "x")
    if out is None:
        out = torch.empty_like(x)
    call("katz_silu_f16", _p(x), _p(out), x.numel(), _stream())
    return out


def add(a, b, out=None):
    _f16(a, "a"), _f16(b, "b")
    if out is None:
        out = torch.empty_like(a)
    call("katz_add_f16", _p(a), _p(b), _p(out), a.numel(), _stream())
    return out


def concat_channels(a, b, out=None):
    """[..., C1] ++ [..., C2] -> [..., C1+C2] (skip-connection concat of the up blocks)."""
    _f16(a, "a"), _f16(b, "b")
    C1, C2 = a.shape[-1], b.shape[-1]
    rows = a.numel() // C1
    if out is None:
        out = torch.empty(tuple(a.shape[:-1]) + (C1 + C2,), dtype=torch.float16, device=a.device)
    call("katz_concat_channels_f16", _p(a), _p(b), _p(out), rows, C1, C2, _stream())
    return out


def halo_assemble(x, edges, rank, world, top=True, bottom=True, upsample=False, out=None):
    """x [B,h,W,C] + gathered edge rows [P,2,B,W,C] (None when world == 1) -> the padded (optionally 2x upsampled) input
    of a row shard's 3x3 convolution."""
    _f16(x, "x")
    if not x.is_contiguous() or (edges is not None and not edges.is_contiguous()):
        raise KatzError("halo_assemble: x and edges must be contiguous")
    B, h, W, C = x.shape
    shape = (B, 2 * h + 2, 2 * W, C) if upsample else (B, h + int(top) + int(bottom), W, C)
    if out is None:
        out = torch.empty(shape, dtype=torch.float16, device=x.device)
    call("katz_halo_assemble_f16", _p(x), _p(edges), _p(out), B, h, W, C, int(top), int(bottom), 1 if upsample else 0, rank,
         world, _stream())
    return out


def nchw_to_nhwc(x, cpad=None, out=None):
    _f16(x, "x")
    B, C, H, W = x.shape
    cpad = cpad or C
    if out is None:
        out = torch.empty((B, H, W, cpad), dtype=torch.float16, device=x.device)
    call("katz_nchw_to_nhwc_f16", _p(x.contiguous()), _p(out), B, C, H * W, cpad, _stream())
    return out


def nhwc_to_nchw(x, c=None, out=None):
    _f16(x, "x")
    B, H, W, cpad = x.shape
    c = c or cpad
    if out is None:
        out = torch.empty((B, c, H, W), dtype=torch.float16, device=x.device)
    call("katz_nhwc_to_nchw_f16", _p(x), _p(out), B, c, H * W, cpad, _stream())
    return out


def euler_scale_input(x, sigma, copies=1, out=None, cpu_torch_rounding=False):
    """half(x / sqrt(sigma^2 + 1)), written `copies` times. See euler_cfg_step for `cpu_torch_rounding`."""
    _f16(x, "x")
    if out is None:
        out = torch.empty((copies * x.shape[0],) + tuple(x.shape[1:]), dtype=torch.float16, device=x.device)
    call("katz_euler_scale_input", _p(x), _p(out), x.numel(), float(sigma), copies, 1 if cpu_torch_rounding else 0, _stream())
    return out


def euler_cfg_step(x, eps_uncond, eps_cond, guidance, sigma, sigma_next, cpu_torch_rounding=False):
    """In-place Euler step on the fp16 latent x with classifier-free guidance. The default reproduces torch's CUDA
    kernels (division by a host scalar = multiplication by its reciprocal; fp32 sigma); `cpu_torch_rounding`
    reproduces torch's CPU kernels (true division; sigma rounded to fp16 before `sigma * eps`)."""
    _f16(x, "x"), _f16(eps_uncond, "eps_uncond")
    call("katz_euler_cfg_step", _p(x), _p(eps_uncond), _p(eps_cond), x.numel(), float(guidance), float(sigma),
         float(sigma_next), 1 if cpu_torch_rounding else 0, _stream())
    return x
