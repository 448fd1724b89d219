"""4-bit weights: quantize, dequantize and the product, against 64-bit forms (tests/w4_reference.py has the bounds)."""
import pytest
import torch

from tests import w4_reference as ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight(g, N, K, group, zeros, spread=0.3):
    """Codes and scales as a quantiser leaves them: all sixteen codes, scales that differ by row and group."""
    J = -(-K // group)
    q = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (0.004 * torch.exp(spread * torch.randn(N, J, generator=g, device="cuda"))).bfloat16()
    zero = torch.randint(0, 16, (N, J), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return q, scale, zero


def _linear_case(M, N, K, group=64, zeros=False, bias=False, residual=False, silu=False, out_scale=1.0, seed=0):
    from katz_b200 import ops
    g = _gen(seed)
    q, scale, zero = _weight(g, N, K, group, zeros)
    x = torch.randn(M, K, generator=g, device="cuda").half()
    b = torch.randn(N, generator=g, device="cuda").half() if bias else None
    r = torch.randn(M, N, generator=g, device="cuda").half() if residual else None
    out = ops.linear_w4(x, q, scale, zero=zero, group=group, bias=b, residual=r, act=ops.ACT_SILU if silu else ops.ACT_NONE,
                        out_scale=out_scale)
    assert out.shape == (M, N) and out.dtype == torch.float16
    ref.assert_within(out, *ref.linear(x, q, scale, zero, group, b, r, silu, out_scale), "linear_w4 %s" % ((M, N, K, group),))
    assert ops.tc05_status() == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(64, 256), (1, 32), (17, 96), (200, 1280), (127, 352), (640, 64)])
def test_quantize_and_back(cuda_device, N, K, group):
    from katz_b200 import ops
    g = _gen(N + K)
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.03).half()
    q, scale = ops.quantize_w4(w, group=group)
    want_c, want_s = ref.quantize(w, group)
    assert torch.equal(scale, want_s)
    assert torch.equal(ref.codes(q), want_c)
    back = ops.dequantize_w4(q, scale, group=group)
    assert torch.equal(back.double(), ref.weights(q, scale, None, group))      # exact: 8 + 3 bits
    # half a step of the scale, and the scale's own rounding on seven steps
    assert ((back.double() - w.double()).abs() <= ref.per_k(scale, group, K) * (0.5 + 7 * 2.0 ** -8)).all()


def test_quantize_ties_and_extremes(cuda_device):
    """Quotients exactly half way between two codes go to the even one; tiny, zero and huge groups."""
    from katz_b200 import ops
    w = torch.zeros(6, 64, device="cuda")
    w[0, :15] = torch.arange(-7, 8, device="cuda") * 0.5                       # scale 0.5: -7..7 halves
    w[0, 0] = 3.5
    w[1, :8] = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5, 6.5, -6.5], device="cuda")
    w[2, 3] = 2.0 ** -24                                                       # the smallest fp16
    w[3, 40] = -65504.0
    w[4, :] = 2.0 ** -20
    w = w.half()
    q, scale = ops.quantize_w4(w, group=64)
    want_c, want_s = ref.quantize(w, 64)
    assert torch.equal(scale, want_s) and torch.equal(ref.codes(q), want_c)
    assert (ref.codes(q)[5] == 8).all() and float(scale[5, 0]) == 0.0
    # the value is rounded to fp16 once (the smallest weight's scale is not a multiple of fp16's smallest step)
    assert torch.equal(ops.dequantize_w4(q, scale), ref.weights(q, scale, None, 64).half())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_quantize_of_non_finite_groups_reads_back_as_nan(cuda_device, bad):
    from katz_b200 import ops
    g = _gen(3)
    w = torch.randn(4, 192, generator=g, device="cuda").half()
    w[1, 70] = bad
    q, scale = ops.quantize_w4(w, group=64)
    back = ops.dequantize_w4(q, scale)
    want = torch.zeros(4, 192, dtype=torch.bool, device="cuda")
    want[1, 64:128] = True
    assert torch.equal(back.isnan(), want)
    for M in (1, 40, 200):
        out = ops.linear_w4(torch.ones(M, 192, device="cuda").half(), q, scale)
        assert out[:, 1].isnan().all() and out[:, [0, 2, 3]].isfinite().all()


def test_quantize_strided_rows_and_out(cuda_device):
    """Row-strided sources; `out` rewritten in place; row slices stand for the same rows; nothing else is touched."""
    from katz_b200 import ops
    g = _gen(4)
    big = torch.randn(40, 512, generator=g, device="cuda").half()
    w = big[:, 128:448]
    q, scale = ops.quantize_w4(w, group=64)
    assert torch.equal(ref.codes(q), ref.quantize(w, 64)[0])
    qb, sb = torch.full((60, 160), 99, dtype=torch.uint8, device="cuda"), torch.full((60, 5), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.quantize_w4(w, group=64, out=(qb[10:50], sb[10:50]))
    assert torch.equal(qb[10:50], q) and torch.equal(sb[10:50], scale)
    assert (qb[:10] == 99).all() and (qb[50:] == 99).all() and (sb[:10] == 3).all() and (sb[50:] == 3).all()
    dst = torch.full((40, 512), 7.0, dtype=torch.float16, device="cuda")
    ops.dequantize_w4(q, scale, out=dst[:, 64:384])
    assert torch.equal(dst[:, 64:384], ops.dequantize_w4(q, scale)) and (dst[:, :64] == 7).all() and (dst[:, 384:] == 7).all()
    x = torch.randn(3, 320, generator=g, device="cuda").half()
    whole = ops.linear_w4(x, q, scale)
    assert torch.equal(ops.linear_w4(x, q[8:24], scale[8:24]), whole[:, 8:24])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K", [32, 160, 640])
def test_dequantize_with_zero_points(cuda_device, K, group):
    from katz_b200 import ops
    q, scale, zero = _weight(_gen(K), 33, K, group, True)
    want = ref.weights(q, scale, zero, group)
    got = ops.dequantize_w4(q, scale, zero, group=group)
    assert torch.equal(got, want.half())


@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 16, 17, 31, 33, 64, 77, 129, 154, 257, 600])
@pytest.mark.parametrize("N,K,group,zeros", [(320, 640, 64, False), (1283, 352, 32, True), (131, 1312, 128, False)])
def test_linear_rows(cuda_device, M, N, K, group, zeros):
    _linear_case(M, N, K, group, zeros, bias=True, residual=M % 2 == 1, silu=M % 3 == 0, seed=M)


@pytest.mark.parametrize("M", [1, 5, 40, 130])
@pytest.mark.parametrize("N", [1, 8, 15, 16, 127, 128, 129])
@pytest.mark.parametrize("K", [32, 64, 96, 128, 4128])
def test_linear_edges(cuda_device, M, N, K):
    _linear_case(M, N, K, group=(32, 64, 128)[(M + N + K // 32) % 3], zeros=(M + N) % 2 == 0, bias=N % 2 == 0, seed=N + K)


# the same kinds of sizes where the tcgen05 kernel takes them: more work, odd numbers of rows on either side, short last steps
@pytest.mark.parametrize("M", [17, 31, 64, 77, 129, 257, 600])
@pytest.mark.parametrize("N,K,group,zeros", [(5123, 1312, 32, True), (2051, 2400, 64, False), (10003, 416, 128, False), (1283, 7200, 32, False)])
def test_linear_more_rows(cuda_device, M, N, K, group, zeros):
    _linear_case(M, N, K, group=group, zeros=zeros, bias=M % 2 == 0, residual=M > 60, silu=M == 77, out_scale=0.5 if M == 129 else 1.0, seed=M)


@pytest.mark.parametrize("N", [15, 16, 127, 128, 129, 257])
@pytest.mark.parametrize("K", [1440, 4128])
def test_linear_many_rows_of_few_weights(cuda_device, N, K):
    _linear_case(8000, N, K, group=64, bias=True, residual=True, seed=N)


@pytest.mark.parametrize("M,N,K", [(2, 13760, 1280), (1, 16384, 8192), (8, 10240, 1280), (77, 5120, 1280), (154, 20480, 2048),
                                   (2048, 1280, 5120), (300, 5120, 10240)])
def test_linear_sizes_of_the_step(cuda_device, M, N, K):
    _linear_case(M, N, K, group=64, bias=True, residual=M > 100, seed=1)
    _linear_case(M, N, K, group=32, zeros=True, silu=True, out_scale=0.5, seed=2)


@pytest.mark.parametrize("M,N,K", [(1, 16, 102432), (3, 40, 102432), (8, 17, 13600), (16, 20, 9600), (5, 33, 40992)])
def test_linear_few_rows_of_many_k(cuda_device, M, N, K):
    """x that does not fit shared memory in one piece, or not at all."""
    _linear_case(M, N, K, group=64, zeros=True, bias=True)
    _linear_case(M, N, K, group=32)


# weights that are streamed: odd numbers of groups and rows, short last blocks, and x that leaves shared memory for eight warps
# but not for sixteen (8 x 10240)
@pytest.mark.parametrize("M", [1, 3, 8])
@pytest.mark.parametrize("N,K,group,zeros", [(640, 10240, 64, False), (640, 10240, 64, True), (2403, 1312, 32, True), (1700, 2080, 64, False),
                                             (2500, 1440, 128, True), (311, 16416, 128, False), (9000, 1376, 32, False)])
def test_linear_streamed_rows(cuda_device, M, N, K, group, zeros):
    _linear_case(M, N, K, group=group, zeros=zeros, bias=True, residual=True, silu=M == 3, out_scale=0.5, seed=M + N)


@pytest.mark.parametrize("group", [32, 128])
def test_linear_streamed_rows_of_any_alignment_and_scale(cuda_device, group):
    from katz_b200 import ops
    g = _gen(31)
    N, K = 1700, 2080      # the last block of 128 k is a quarter full
    q, scale, _ = _weight(g, N, K, group, False)
    q[:, :] = 0x88      # weights of zero but for one a row ...
    q[torch.arange(N), torch.arange(N) % (K // 2)] = 0x89
    scale[:] = 900.0      # ... of 900: code 0 would stand for -7200, outside fp16
    x = torch.randn(3, K + 9, generator=g, device=cuda_device).half()[:, 1:K + 1]
    out = ops.linear_w4(x, q, scale, group=group)
    want = 900.0 * x.double()[:, 2 * (torch.arange(N, device=cuda_device) % (K // 2))]
    assert torch.allclose(out.double(), want, rtol=2.0 ** -11 + 2.0 ** -23, atol=0)      # one product, one rounding


@pytest.mark.parametrize("M", [3, 50, 200])
def test_linear_strided_unaligned_and_untouched_rows(cuda_device, M):
    """Views with row strides, sources and outputs that start off a 16-byte boundary, `out` = `residual`, and what lies around
    the output left as it was."""
    from katz_b200 import ops
    g = _gen(M)
    N, K = 264, 320
    q, scale, _ = _weight(g, N, K, 64, False)
    for off, pad in ((0, 8), (8, 8), (1, 0), (3, 5)):
        xb = torch.randn(M + 2, K + pad + off + 3, generator=g, device="cuda").half()
        ob = torch.full((M + 2, N + pad + off + 2), 5.0, dtype=torch.float16, device="cuda")
        x, out = xb[1:M + 1, off:off + K], ob[1:M + 1, off:off + N]
        ops.linear_w4(x, q, scale, out=out)
        ref.assert_within(out, *ref.linear(x, q, scale, None, 64, None, None, False, 1.0), "strided %d %d" % (off, pad))
        keep = torch.ones_like(ob, dtype=torch.bool)
        keep[1:M + 1, off:off + N] = False
        assert (ob[keep] == 5).all()
        before = torch.randn(M, N, generator=g, device="cuda").half()
        out.copy_(before)
        ops.linear_w4(x, q, scale, residual=out, out=out, out_scale=0.25)
        ref.assert_within(out, *ref.linear(x, q, scale, None, 64, None, before, False, 0.25), "residual in place")
        assert (ob[keep] == 5).all()


@pytest.mark.parametrize("M", [1, 20, 100])
def test_linear_scale_range(cuda_device, M):
    """Scales from 2^-23 to 64 keep every bit; above, a result is right or not finite (few rows multiply the scale in fp32 and
    are right; more rows take 64 * weight in fp16), never a plausible wrong number."""
    from katz_b200 import ops
    g = _gen(5)
    N, K = 48, 128
    q, _, _ = _weight(g, N, K, 64, False)
    x = torch.randn(M, K, generator=g, device="cuda").half()
    for s, out_scale in ((2.0 ** -23, 2.0 ** 16), (1.7 * 2.0 ** -21, 2.0 ** 14), (64.0, 2.0 ** -7)):
        scale = torch.full((N, 2), s, device="cuda").bfloat16()
        out = ops.linear_w4(x, q, scale, out_scale=out_scale)
        ref.assert_within(out, *ref.linear(x, q, scale, None, 64, None, None, False, out_scale), "scale %g" % s)
    scale = torch.full((N, 2), 2.0 ** 14, device="cuda").bfloat16()
    out = ops.linear_w4(x, q, scale, out_scale=2.0 ** -20)
    want, bound = ref.linear(x, q, scale, None, 64, None, None, False, 2.0 ** -20)
    assert ((out.double() - want).abs() <= bound)[out.isfinite()].all()
    assert out.isfinite().all() or not out.isfinite().any()


@pytest.mark.parametrize("M", [1, 40])
def test_linear_non_finite_inputs_stay_in_their_rows(cuda_device, M):
    from katz_b200 import ops
    g = _gen(6)
    q, scale, _ = _weight(g, 64, 256, 64, False)
    x = torch.randn(M + 2, 256, generator=g, device="cuda").half()
    x[M, 3], x[M + 1, 200] = float("nan"), float("inf")
    out = ops.linear_w4(x, q, scale)
    assert out[:M].isfinite().all() and out[M].isnan().all() and not out[M + 1].isfinite().any()


def test_linear_empty(cuda_device):
    from katz_b200 import ops
    q, scale, _ = _weight(_gen(7), 64, 256, 64, False)
    assert ops.linear_w4(torch.empty(0, 256, device="cuda").half(), q, scale).shape == (0, 64)
    assert ops.linear_w4(torch.ones(3, 256, device="cuda").half(), q[:0], scale[:0]).shape == (3, 0)
    assert ops.quantize_w4(torch.empty(0, 256, device="cuda").half())[0].shape == (0, 128)
    assert ops.dequantize_w4(q[:0], scale[:0]).shape == (0, 256)


@pytest.mark.parametrize("M,N,K", [(2, 1280, 1280), (3, 5120, 2560), (100, 1280, 2048), (500, 640, 2560)])
def test_linear_repeats_bit_for_bit_on_streams_and_in_graphs(cuda_device, M, N, K):
    from katz_b200 import ops
    g = _gen(8)
    q, scale, _ = _weight(g, N, K, 64, False)
    x, x2 = (torch.randn(M, K, generator=g, device="cuda").half() for _ in range(2))
    want, want2 = ops.linear_w4(x, q, scale), ops.linear_w4(x2, q, scale)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):                                   # two calls at once
        for s, v in zip(streams, (x, x2)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(ops.linear_w4(v, q, scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, [want, want2] * 20))
    graphs, results, inputs = [], [], []
    for v in (x, x2):                                     # two graphs, replayed on two streams at once
        static = v.clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r = ops.linear_w4(static, q, scale)
            r = ops.linear_w4(static, q, scale, residual=r)
        graphs.append(gr), results.append(r), inputs.append(static)
    for i in range(5):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0], ops.linear_w4(x, q, scale, residual=want))
    inputs[1].copy_(x)
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[1], results[0])
    assert ops.tc05_status() == 0


# K split, small groups: the scales arrive later than the codes
@pytest.mark.parametrize("M,N,K,zeros", [(147, 3663, 7168, False), (300, 5120, 10240, True), (96, 1280, 5120, True)])
def test_linear_is_the_same_whatever_runs_around_it(cuda_device, M, N, K, zeros):
    from katz_b200 import ops
    g = _gen(9)
    q, scale, zero = _weight(g, N, K, 32, zeros)
    x = torch.randn(M, K, generator=g, device="cuda").half()
    r = torch.randn(M, N, generator=g, device="cuda").half()
    other = torch.randn(1500, 1500, device="cuda")
    first = ops.linear_w4(x, q, scale, zero=zero, group=32, residual=r)
    ref.assert_within(first, *ref.linear(x, q, scale, zero, 32, None, r, False, 1.0), "linear_w4")
    for i in range(20):
        outs = []
        for j in range(25):
            if (i + j) % 3 == 0:
                other @ other
            if (i + j) % 5 == 0:
                torch.cuda._sleep(1000 * (j + 1))
            if (i + j) % 4 == 0:
                x + 0
            outs.append(ops.linear_w4(x, q, scale, zero=zero, group=32, residual=r))
        assert not any(torch.stack([(o != first).any() for o in outs]).tolist())
    assert ops.tc05_status() == 0


def test_linear_from_threads(cuda_device):
    import threading

    from katz_b200 import ops
    g = _gen(13)
    q, scale, _ = _weight(g, 1280, 1280, 64, False)
    xs = [torch.randn(m, 1280, generator=g, device="cuda").half() for m in (1, 8, 77, 600)]
    want = [ops.linear_w4(x, q, scale) for x in xs]
    torch.cuda.synchronize()
    equal = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [ops.linear_w4(x, q, scale) for _ in range(30) for x in xs]
        stream.synchronize()
        equal.append(all(torch.equal(o, w) for o, w in zip(outs, want * 30)))
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert equal == [True] * 4 and ops.tc05_status() == 0


def test_weights_past_four_gigabytes(cuda_device):
    from katz_b200 import ops
    g = _gen(12)
    N, K, group = 270000, 32768, 128      # 4.4 GB of codes, 17.7 GB as fp16: byte and element offsets beyond 32 bits
    q = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (0.004 * torch.exp(0.3 * torch.randn(N, K // group, generator=g, device="cuda"))).bfloat16()
    wide = torch.randn(40, K + 8, generator=g, device="cuda").half()
    ends = [slice(0, 200), slice(N - 333, N)]
    for x in (wide[:2, :K], wide[:2, 1:K + 1], wide[:12, :K], wide[:40, :K]):      # streamed, direct, few rows, tcgen05
        out = ops.linear_w4(x, q, scale, group=group)
        for e in ends:
            ref.assert_within(out[:, e], *ref.linear(x, q[e], scale[e], None, group, None, None, False, 1.0), "M=%d" % x.shape[0])
    w = ops.dequantize_w4(q, scale, group=group)
    for e in ends:
        assert torch.equal(w[e], ref.weights(q[e], scale[e], None, group).half())
    q2, scale2 = ops.quantize_w4(w, group=group)
    for e in ends:
        c, s = ref.quantize(w[e], group)
        assert torch.equal(ref.codes(q2[e]), c) and torch.equal(scale2[e], s)
    assert ops.tc05_status() == 0


def test_adapter_switch_on_four_bit_weights(cuda_device):
    """The operators as an adapter switch uses them: merge in fp16, remake the 4-bit form in place, multiply; then back."""
    from collections import OrderedDict
    from katz_b200 import ops
    from katz_b200.lora import LoraMerger
    g = _gen(9)
    N, K, r = 640, 1280, 16
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.03).half()
    up, down = (torch.randn(N, r, generator=g, device="cuda") * 0.05).half(), (torch.randn(r, K, generator=g, device="cuda") * 0.1).half()
    x = torch.randn(2, K, generator=g, device="cuda").half()
    q, scale = ops.quantize_w4(w)
    plain = ops.linear_w4(x, q, scale)
    live = w.clone()
    m = LoraMerger(OrderedDict(a=live))
    m.merge(OrderedDict(a=(up, down)), 1.0)
    ops.quantize_w4(live, out=(q, scale))
    want_c, want_s = ref.quantize(live, 64)
    assert torch.equal(ref.codes(q), want_c) and torch.equal(scale, want_s)
    merged = ops.linear_w4(x, q, scale)
    ref.assert_within(merged, *ref.linear(x, q, scale, None, 64, None, None, False, 1.0), "merged")
    assert not torch.equal(merged, plain)
    m.restore()
    ops.quantize_w4(live, out=(q, scale))
    assert torch.equal(ops.linear_w4(x, q, scale), plain)


def test_refusals(cuda_device):
    from katz_b200 import KatzError, ops
    q, scale, zero = _weight(_gen(10), 64, 256, 64, True)
    x, w = torch.zeros(4, 256, device="cuda").half(), torch.zeros(64, 256, device="cuda").half()
    buf = torch.zeros(4 * 300, device="cuda").half()
    calls = [
        lambda: ops.linear_w4(x.float(), q, scale), lambda: ops.linear_w4(x.bfloat16(), q, scale), lambda: ops.linear_w4(x.cpu(), q, scale),
        lambda: ops.linear_w4(x, q.cpu(), scale), lambda: ops.linear_w4(x, q, scale.cpu()), lambda: ops.linear_w4(x, q, scale.half()),
        lambda: ops.linear_w4(x, q.to(torch.int8), scale), lambda: ops.linear_w4(x, q, scale, group=48), lambda: ops.linear_w4(x, q, scale, group=32),
        lambda: ops.linear_w4(x, q, scale, zero=zero.float()), lambda: ops.linear_w4(x, q, scale, zero=zero[:, :2]),
        lambda: ops.linear_w4(x[:, :224], q, scale), lambda: ops.linear_w4(x[0], q, scale), lambda: ops.linear_w4(x[:, ::2], q[:, :64], scale[:, :2]),
        lambda: ops.linear_w4(x[:1].expand(4, 256), q, scale), lambda: ops.linear_w4(x, q, scale, act=2),
        lambda: ops.linear_w4(x, q, scale, bias=x[0]), lambda: ops.linear_w4(x, q, scale, bias=torch.zeros(64, device="cuda")),
        lambda: ops.linear_w4(x, q, scale, residual=x), lambda: ops.linear_w4(x, q, scale, out=torch.zeros(4, 64, device="cuda")),
        lambda: ops.linear_w4(x, q, scale, out=x[:, :64]), lambda: ops.linear_w4(x, q, scale, out=buf[:64].expand(4, 64)),
        lambda: ops.linear_w4(x, q, scale, out=buf.as_strided((4, 64), (300, 1)), residual=buf.as_strided((4, 64), (64, 1))),
        lambda: ops.linear_w4(x[:, :240], q[:, :120].contiguous(), scale), lambda: ops.linear_w4(x, q.t().contiguous().t(), scale),
        lambda: ops.linear_w4(x, torch.zeros(64 * 128 + 1, dtype=torch.uint8, device="cuda")[1:].view(64, 128), scale),
        lambda: ops.quantize_w4(w[:, :250]), lambda: ops.quantize_w4(w.float()), lambda: ops.quantize_w4(w[:, 4:132]), lambda: ops.quantize_w4(w.t()),
        lambda: ops.quantize_w4(w, group=16), lambda: ops.quantize_w4(w, out=(q[:32], scale[:32])), lambda: ops.quantize_w4(w, out=(q, scale.float())),
        lambda: ops.quantize_w4(w[0]), lambda: ops.quantize_w4(w.cpu()),
        lambda: ops.dequantize_w4(q, scale, out=w.float()), lambda: ops.dequantize_w4(q, scale, out=w[:, :192]), lambda: ops.dequantize_w4(q, scale, group=128),
    ]
    for i, c in enumerate(calls):
        with pytest.raises(KatzError):
            c()
            pytest.fail("call %d was not refused" % i)
