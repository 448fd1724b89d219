"""Measured cases of the 4-bit weight operators and of the gated residual norm.

Four operators: `linear_w4` (products of few or many rows with 4-bit weights), `quantize_w4` and `dequantize_w4` (the weight
format made and unmade on the device; one pass of a case makes it and reads it back), `residual_norm` (the norms before and
after a block with its gate and residual scale).

Weight format: `q` uint8 [N, K/2], the code of an even k in the low four bits; `scale` bf16 [N, ceil(K/group)]; `zero` uint8 of
the same shape or None (8 everywhere). A weight is scale * (code - zero)."""
import torch

own = False

LINEAR = [
    # the step's first small layer: time embedding of a two-image batch
    dict(name="linear time embedding", m=2, n=1280, k=320, group=64, zero=False, bias=True, act="silu", residual=False),
    # the time projections of all 17 resnets in one call
    dict(name="linear time projections", m=2, n=13760, k=1280, group=64, zero=False, bias=True, act="none", residual=False),
    # one token through a wide layer whose weights no cache holds
    dict(name="linear one token wide", m=1, n=16384, k=8192, group=128, zero=False, bias=False, act="none", residual=False),
    # a few rows, small groups with zero points, the gated projection's width
    dict(name="linear 8 rows zero points", m=8, n=10240, k=1280, group=32, zero=True, bias=True, act="none", residual=False),
    # one prompt of 77 tokens through a text-encoder-sized layer
    dict(name="linear one prompt", m=77, n=5120, k=1280, group=128, zero=False, bias=True, act="none", residual=False),
    # the text keys and values of every block of the UNet for two prompts
    dict(name="linear text keys values", m=154, n=166400, k=2048, group=64, zero=False, bias=False, act="none", residual=False),
    # feed-forward output of a transformer block over a 32 x 32 latent, two images, with its skip connection
    dict(name="linear feed-forward out", m=2048, n=1280, k=5120, group=64, zero=False, bias=True, act="none", residual=True),
]
QUANT = [
    # one attention projection after an adapter switch
    dict(name="quantize projection", n=1280, k=1280, group=32),
    # the text projections of the whole UNet after an adapter switch
    dict(name="quantize text projections", n=166400, k=2048, group=64),
]
NORM = [
    # two prompts: norms on both sides of the block, gate per channel
    dict(name="norm two prompts", b=2, s=77, c=1280, stream="fp16", post="rms", pre="rms", gate="channel", mod="none", affine=True, rscale=1.0),
    # a conditioned block over a 32 x 32 latent: gate, scale and shift per image
    dict(name="norm conditioned block", b=2, s=1024, c=1280, stream="fp16", post="none", pre="layer", gate="sample", mod="sample",
         affine=False, rscale=1.0),
    # the largest token count of a 2048 x 2048 image with the residual stream in 32 bits
    dict(name="norm large image", b=2, s=16384, c=640, stream="fp32", post="rms", pre="layer", gate="sample", mod="sample", affine=True,
         rscale=0.7071),
]


def listed():
    return [dict(c, op="linear") for c in LINEAR] + [dict(c, op="quant") for c in QUANT] + [dict(c, op="norm") for c in NORM]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "quant", "norm", "norm"])
    if op == "linear":
        n, k = _log(rng, 64, 32768), 32 * _log(rng, 2, 320)
        if rng.random() < 0.6:
            n = max(8, n // 8 * 8)
        m = _log(rng, 1, 16) if rng.random() < 0.5 else _log(rng, 1, 2048)
        m = max(1, min(m, int(4e10 / (n * k))))
        return dict(op=op, m=m, n=n, k=k, group=rng.choice([32, 64, 128]), zero=rng.random() < 0.4, bias=rng.random() < 0.5,
                    act=rng.choice(["none", "silu"]), residual=rng.random() < 0.4)
    if op == "quant":
        return dict(op=op, n=_log(rng, 1, 65536), k=32 * _log(rng, 1, 256), group=rng.choice([32, 64, 128]))
    c = _log(rng, 32, 8192)
    if rng.random() < 0.7:
        c = max(8, c // 8 * 8)
    b = rng.randint(1, 4)
    s = max(1, min(_log(rng, 1, 16384), int(2e7 / (b * c))))
    return dict(op=op, b=b, s=s, c=c, stream=rng.choice(["fp16", "fp32"]), post=rng.choice(["none", "layer", "rms"]),
                pre=rng.choice(["layer", "rms"]), gate=rng.choice(["none", "channel", "sample", "token"]),
                mod=rng.choice(["none", "channel", "sample", "token"]), affine=rng.random() < 0.5, rscale=rng.choice([1.0, 0.5, 0.7071]))


def _groups(c):
    return -(-c["k"] // c["group"])


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": dict(c)}
    if c["op"] == "norm":
        B, S, C = c["b"], c["s"], c["c"]
        # a residual stream with a drifting mean and a few loud channels, a branch output of its own scale
        loud = 1 + 4 * (torch.rand(C, generator=g, device=dev) < 0.01)
        s["x"] = ((randn(B, S, C) + 0.3 * randn(B, S, 1)) * loud).to(torch.float16 if c["stream"] == "fp16" else torch.float32)
        s["y"] = (0.5 * randn(B, S, C)).half()
        # the vectors of one conditioning product lie side by side in one row: gate, scale and shift are views of it
        lead = {"channel": (), "sample": (B,), "token": (B, S)}
        s["gate"] = s["scale"] = s["shift"] = None
        if c["gate"] != "none":
            s["gate"] = (0.5 * randn(*lead[c["gate"]], 3 * C)).half()[..., :C]
        if c["mod"] != "none":
            t = (0.3 * randn(*lead[c["mod"]], 3 * C)).half()
            s["scale"], s["shift"] = t[..., C:2 * C], t[..., 2 * C:]
        for side in ("post", "pre"):
            s[side + "_w"] = (1 + 0.1 * randn(C)).half() if c["affine"] else None
            s[side + "_b"] = (0.1 * randn(C)).half() if c["affine"] and c[side] == "layer" else None
        return s
    N, K, G = c["n"], c["k"], c["group"]
    w = randn(N, K).mul_(0.03).mul_(torch.exp(0.3 * randn(N, 1)))
    if c["op"] == "quant":
        s["w"] = w.half()
        return s
    pad = (-K) % G
    wg = torch.nn.functional.pad(w, (0, pad)).view(N, -1, G)
    if c["zero"]:
        lo, hi = wg.amin(2).clamp_(max=0), wg.amax(2).clamp_(min=0)
        s["scale"] = ((hi - lo) / 15).bfloat16()
        zero = (-lo / s["scale"].float()).round_().clamp_(0, 15)
        s["zero"] = zero.to(torch.uint8)
    else:
        s["scale"] = (wg.abs().amax(2) / 7).bfloat16()
        zero = torch.full_like(s["scale"], 8, dtype=torch.float32)
        s["zero"] = None
    code = wg.div_(s["scale"].float()[..., None]).round_().add_(zero[..., None]).clamp_(0, 15).to(torch.uint8).view(N, -1)[:, :K]
    s["q"] = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    s["x"] = randn(c["m"], K).half()
    s["bias"] = (0.1 * randn(N)).half() if c["bias"] else None
    s["residual"] = randn(c["m"], N).half() if c["residual"] else None
    return s


def _weights(q, scale, zero, group, k):
    code = torch.stack([q & 15, q >> 4], 2).view(q.shape[0], k).float()
    code -= 8.0 if zero is None else zero.float().repeat_interleave(group, 1)[:, :k]
    return code.mul_(scale.float().repeat_interleave(group, 1)[:, :k])


def _norm(t, kind, weight, bias, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    t = t if weight is None else t * weight.float()
    return t if bias is None else t + bias.float()


def _over_tokens(v):
    return v.float()[:, None] if v.dim() == 2 else v.float()


def run(state):
    s, c = state, state["case"]
    if own:
        from katz_b200 import ops
        if c["op"] == "linear":
            return ops.linear_w4(s["x"], s["q"], s["scale"], zero=s["zero"], group=c["group"], bias=s["bias"], residual=s["residual"],
                                 act=ops.ACT_SILU if c["act"] == "silu" else ops.ACT_NONE)
        if c["op"] == "quant":
            q, scale = ops.quantize_w4(s["w"], group=c["group"])
            return scale, ops.dequantize_w4(q, scale, group=c["group"])
        post = None if c["post"] == "none" else ops.Norm(c["post"], s["post_w"], s["post_b"])
        pre = ops.Norm(c["pre"], s["pre_w"], s["pre_b"])
        return ops.residual_norm(s["x"], s["y"], gate=s["gate"], post=post, pre=pre, scale=s["scale"], shift=s["shift"],
                                 residual_scale=c["rscale"])
    if c["op"] == "linear":
        t = s["x"].float() @ _weights(s["q"], s["scale"], s["zero"], c["group"], c["k"]).t()
        t = t if s["bias"] is None else t + s["bias"].float()
        t = t * torch.sigmoid(t) if c["act"] == "silu" else t
        t = t if s["residual"] is None else t + s["residual"].float()
        return t.half()
    if c["op"] == "quant":
        K, G = c["k"], c["group"]
        w = torch.nn.functional.pad(s["w"].float(), (0, (-K) % G)).view(c["n"], -1, G)
        scale = (w.abs().amax(2) / 7).bfloat16()
        code = (w / scale.float()[..., None]).round().clamp(-7, 7)
        code = torch.where(scale[..., None] == 0, torch.zeros_like(code), code)
        return scale, (code * scale.float()[..., None]).view(c["n"], -1)[:, :K].half()
    u = s["y"].float()
    if c["post"] != "none":
        u = _norm(u, c["post"], s["post_w"], s["post_b"], 1e-5)
    u = u if s["gate"] is None else u * _over_tokens(s["gate"])
    h = c["rscale"] * s["x"].float() + u
    z = _norm(h, c["pre"], s["pre_w"], s["pre_b"], 1e-5)
    if s["scale"] is not None:
        z = z * (1 + _over_tokens(s["scale"])) + _over_tokens(s["shift"])
    return h.to(s["x"].dtype), z.half()


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "linear":
        N, K, G, J = c["n"], c["k"], c["group"], _groups(c)
        x, q = s["x"].double(), s["q"]
        col = torch.arange(K // 2, device=q.device) * 2 // G          # the group of each pair of codes
        off = torch.full((N, J), 8, device=q.device, dtype=torch.uint8) if s["zero"] is None else s["zero"]
        y = torch.zeros(c["m"], N, device=q.device, dtype=torch.float64)
        for odd in (0, 1):
            w = (q // 16 if odd else q % 16).double()
            w = (w - off.double()[:, col]) * s["scale"].double()[:, col]
            y += torch.matmul(x[:, odd::2], w.T)
            del w
        if c["bias"]:
            y += s["bias"].double()
        if c["act"] == "silu":
            y = y / (1 + torch.exp(-y))
        return y + s["residual"].double() if c["residual"] else y
    if c["op"] == "quant":
        K, G, J = c["k"], c["group"], _groups(c)
        idx = (torch.arange(K, device=s["w"].device) // G).expand(c["n"], K)
        w = s["w"].double()
        top = torch.zeros(c["n"], J, device=w.device, dtype=torch.float64).scatter_reduce(1, idx, w.abs(), "amax")
        scale = (top / 7).to(torch.bfloat16).double()
        each = scale.gather(1, idx)
        steps = torch.where(each > 0, w / each, torch.zeros_like(w)).round().clamp(-7, 7)
        return scale, steps * each
    x, u = s["x"].double(), s["y"].double()

    def normed(t, kind, w, b):
        m = t.mean(-1, keepdim=True) if kind == "layer" else 0
        t = (t - m) * ((t - m).pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
        return t * (1 if w is None else w.double()) + (0 if b is None else b.double())

    def spread(v):
        return v.double().reshape((v.shape[0], 1, v.shape[1]) if v.dim() == 2 else v.shape)

    if c["post"] != "none":
        u = normed(u, c["post"], s["post_w"], s["post_b"])
    h = x * c["rscale"] + (u if s["gate"] is None else u * spread(s["gate"]))
    z = normed(h, c["pre"], s["pre_w"], s["pre_b"])
    return h, z if s["scale"] is None else z + z * spread(s["scale"]) + spread(s["shift"])


def work(case):
    c = case
    if c["op"] == "norm":
        r = c["b"] * c["s"] * c["c"]
        per = {"none": 0, "channel": c["c"], "sample": c["b"] * c["c"], "token": r}
        wide = 2 if c["stream"] == "fp16" else 4
        sides = [c["post"], c["pre"]]
        vectors = c["c"] * (sum(k != "none" for k in sides) + sides.count("layer")) if c["affine"] else 0
        return {"bytes": 2 * r * wide + 4 * r + 2 * (per[c["gate"]] + 2 * per[c["mod"]] + vectors),
                "flops": r * (3 + 5 * sum(k != "none" for k in sides) + (2 if c["mod"] != "none" else 0))}
    n, k, j = c["n"], c["k"], _groups(c)
    if c["op"] == "quant":
        # weights in, codes and scales out; codes and scales in, weights out
        return {"bytes": 2 * (2 * n * k + n * k / 2 + 2 * n * j), "flops": 5 * n * k}
    m = c["m"]
    return {"bytes": n * k / 2 + n * j * (3 if c["zero"] else 2) + 2 * m * k + 2 * m * n * (2 if c["residual"] else 1) + (2 * n if c["bias"] else 0),
            "flops": 2 * m * n * k}
