"""Cases for the operators that stand beside the DiT's Linear, RoPE and norms: 8-bit block quantisation, the 8-bit
block-scaled Linear, rotary positions, and GroupNorm (+ SiLU) over channel-last rows.

Formulas
  quant   blocks of 128 columns x (1 row | 128 rows): s = 2^k, the smallest k >= -126 with max|x| <= 448 * 2^k
          (largest finite |x| of the block; a block of zeros takes 2^-126), code = e4m3(x / s), ties to even.
          Row scales are laid out [column block][row], block scales [row block][column block].
  linear  y[m, n] = sum_b xs[b, m] * ws[n // 128, b] * sum_{k in b} xq[m, k] * wq[n, k] + bias[n]
  rope    pair i of a head turns by pos[axis(i)] * f_i; interleaved pairs are (2i, 2i + 1), half pairs (i, i + P);
          dims past the 2 P rotated ones are copied; `inverse` turns back (the gradient's direction).
  norm    y = act((x - mean_g) / sqrt(var_g + eps) * gamma_c + beta_c), mean and variance over the rows and the channels
          of group g of one sample.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the SwiGLU product of a 1080p frame's rows on its way into the 8-bit output projection
        dict(name="quant rows 1080p mlp", op="quant", rows=5498, cols=6912, block_rows=1, type="bf16"),
        # one qkv weight, quantised when a model is loaded
        dict(name="quant blocks qkv weight", op="quant", rows=7680, cols=2560, block_rows=128, type="fp32"),
        # one conditioning row through a qkv-wide projection: the single-token form
        dict(name="linear one token", op="linear", M=1, K=2560, N=7680, bias=True, out="bf16"),
        # the text rows of one prompt into the model's width
        dict(name="linear txt rows", op="linear", M=58, K=5120, N=2560, bias=True, out="bf16"),
        # a 720p frame's rows through the down projection; ragged in M, fp32 out as the residual stream takes it
        dict(name="linear 720p down", op="linear", M=2443, K=6912, N=2560, bias=False, out="fp32"),
        # a 1080p frame's rows through the gated up projection: the largest product of a layer
        dict(name="linear 1080p up", op="linear", M=5498, K=2560, N=13824, bias=True, out="bf16"),
        # a decode step: one new token's q and k heads behind 8191 earlier ones
        dict(name="rope one token", op="rope", batch=1, tokens=1, heads=40, dim=128, axes=1, axis_dim=128,
             layout="half", scaling="none", start=8191, row=40 * 128, type="bf16", inverse=False),
        # q and k of a 1080p frame out of the fused qkv rows, rotated by (t, h, w) on 3 x 42 of 128 dims
        dict(name="rope 1080p grid", op="rope", batch=1, tokens=5440, heads=40, dim=128, axes=3, axis_dim=42,
             layout="interleaved", scaling="none", start=0, row=7680, type="bf16", inverse=False),
        # gradient of a long stream's keys under YaRN scaling, a quarter of each head rotated
        dict(name="rope long yarn back", op="rope", batch=2, tokens=65521, heads=8, dim=128, axes=1, axis_dim=32,
             layout="half", scaling="yarn", start=0, row=8 * 128, type="fp32", inverse=True),
        # a decoder's innermost norm on a small tile: latency
        dict(name="norm latent tile", op="norm", batch=1, rows=34 * 40, channels=512, groups=32, act="silu", type="bf16"),
        # the latent grid of 1080p frames (136 x 160), three frames, no activation
        dict(name="norm latent frames", op="norm", batch=3, rows=136 * 160, channels=512, groups=32, act="none", type="bf16"),
        # a decoder's last block at full resolution (1088 x 1280)
        dict(name="norm full frame", op="norm", batch=1, rows=1088 * 1280, channels=128, groups=32, act="silu", type="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quant", "linear", "linear", "rope", "norm"))
    if op == "quant":
        return dict(op=op, rows=_spread(rng, 1, 7680), cols=_spread(rng, 16, 6912), block_rows=rng.choice((1, 1, 128)),
                    type=rng.choice(("fp32", "fp16", "bf16")))
    if op == "linear":
        return dict(op=op, M=_spread(rng, 1, 5498), K=_spread(rng, 32, 6912), N=_spread(rng, 16, 6912),
                    bias=rng.random() < 0.5, out=rng.choice(("fp32", "fp16", "bf16", "bf16")))
    if op == "rope":
        axes = rng.choice((1, 1, 3))
        dim = rng.choice((64, 80, 96, 128, 256))
        most = dim // axes // 2
        pairs = rng.randint(most // 2, most)
        heads = rng.choice((1, 3, 8, 20, 40))
        tokens = _spread(rng, 1, max(2, 200_000 // heads))
        return dict(op=op, batch=rng.choice((1, 1, 2, 3)), tokens=tokens, heads=heads, dim=dim, axes=axes,
                    axis_dim=2 * pairs, layout=rng.choice(("half", "interleaved")),
                    scaling=rng.choice(("none", "linear", "ntk", "yarn")), start=rng.choice((0, 0, 1000, 1_000_000)),
                    row=heads * dim * rng.choice((1, 1, 3)), type=rng.choice(("fp32", "fp16", "bf16", "bf16")),
                    inverse=rng.random() < 0.3)
    groups = rng.choice((1, 8, 16, 32))
    channels = groups * rng.choice((1, 2, 3, 4, 8, 10, 16))
    rows = _spread(rng, 1, max(2, 100_000_000 // channels // 3))
    return dict(op=op, batch=rng.choice((1, 1, 2, 3)), rows=rows, channels=channels, groups=groups,
                act=rng.choice(("none", "silu")), type=rng.choice(("fp32", "fp16", "bf16", "bf16")))


def work(case):
    op = case["op"]
    if op == "quant":
        e = DTYPES[case["type"]].itemsize
        n, kb = case["rows"] * case["cols"], -(-case["cols"] // 128)
        scales = kb * (case["rows"] if case["block_rows"] == 1 else -(-case["rows"] // 128))
        return {"bytes": n * (e + 1) + 4 * scales, "flops": 2 * n}
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        kb = -(-K // 128)
        e = DTYPES[case["out"]].itemsize
        return {"bytes": M * K + N * K + M * N * e + 4 * kb * (M + -(-N // 128)) + 4 * N * case["bias"],
                "flops": 2 * M * K * N}
    e = DTYPES[case["type"]].itemsize
    if op == "rope":
        n = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * e + 4 * case["tokens"] * case["axes"], "flops": 3 * n}
    n = case["batch"] * case["rows"] * case["channels"]
    return {"bytes": 2 * n * e + 8 * case["channels"], "flops": 10 * n}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _pitch(cols):
    """Bytes of one row of codes: a multiple of 16."""
    return (cols + 15) // 16 * 16


def _activations(g, rows, cols):
    """Rows of differing size with a few far larger columns, as activations have."""
    x = _normal(g, rows, cols)
    x *= torch.exp(0.5 * _normal(g, rows, 1))
    big = torch.rand(cols, generator=g, device="cuda") < 0.01
    x[:, big] *= 20
    return x


def _codes(x, block_rows):
    """Codes with their row pitch, and scales, of x: what a program has in hand before a Linear."""
    q, s = _quant_plain(x, block_rows)
    buf = torch.zeros(x.shape[0], _pitch(x.shape[1]), dtype=torch.uint8, device="cuda")
    buf[:, : x.shape[1]] = q.view(torch.uint8)
    return buf, s


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = {"case": case}
    if op == "quant":
        R, C = case["rows"], case["cols"]
        x = _activations(g, R, C) if case["block_rows"] == 1 else 0.02 * _normal(g, R, C)
        kb = -(-C // 128)
        st["x"] = x.to(DTYPES[case["type"]])
        st["q"] = torch.empty(R, _pitch(C), dtype=torch.uint8, device="cuda")
        st["scale"] = torch.empty((kb, R) if case["block_rows"] == 1 else (-(-R // 128), kb), device="cuda")
    elif op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        st["xq"], st["xs"] = _codes(_activations(g, M, K), 1)
        st["wq"], st["ws"] = _codes(0.02 * _normal(g, N, K), 128)
        st["bias"] = 0.1 * _normal(g, N) if case["bias"] else None
        st["y"] = torch.empty(M, N, dtype=DTYPES[case["out"]], device="cuda")
    elif op == "rope":
        B, T, H, D, A = (case[k] for k in ("batch", "tokens", "heads", "dim", "axes"))
        st["x"] = _normal(g, B * T, case["row"]).to(DTYPES[case["type"]])
        t = torch.arange(T, device="cuda", dtype=torch.int32)
        if A == 1:
            pos = (t + case["start"])[:, None]
        else:  # a grid 80 wide and 68 high, frame after frame, behind 58 text positions
            pos = torch.stack((58 + t // 5440, t // 80 % 68, t % 80), 1) + case["start"]
        st["pos"] = pos.to(torch.int32).contiguous()
        st["y"] = torch.empty(B, T, H, D, dtype=st["x"].dtype, device="cuda")
    else:
        B, S, C = case["batch"], case["rows"], case["channels"]
        x = torch.empty(B, S, C, dtype=DTYPES[case["type"]], device="cuda")
        spread, mean = torch.exp(0.3 * _normal(g, C)), 2 * _normal(g, C)
        for b in range(B):  # one sample at a time: the fp32 draft of a full frame is large
            x[b] = _normal(g, S, C) * spread + mean
        st["x"] = x
        st["gamma"], st["beta"] = 1 + 0.1 * _normal(g, C), 0.1 * _normal(g, C)
        st["y"] = torch.empty_like(x)
    return st


# ---------------------------------------------------------------- plain forms (32 bits; angles in 64)
def _blocks_of(x, block_rows):
    """x padded with zeros and cut as [row blocks, block rows, column blocks, 128]."""
    R, C = x.shape
    pr, pc = -R % block_rows, -C % 128
    if pr or pc:
        x = torch.nn.functional.pad(x, (0, pc, 0, pr))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)


def _quant_plain(x, block_rows):
    R, C = x.shape
    b = _blocks_of(x.float(), block_rows)
    amax = b.abs().amax(dim=(1, 3))
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 9, e - 8)
    k = torch.where(amax > 0, k, torch.full_like(k, -126)).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(amax), k)
    q = (b / s[:, None, :, None]).to(E4M3).reshape(b.shape[0] * block_rows, -1)[:R, :C]
    return q, s.t().contiguous() if block_rows == 1 else s


def _linear_plain(st):
    c = st["case"]
    M, K, N = c["M"], c["K"], c["N"]
    x = st["xq"].view(E4M3)[:, :K].float() * st["xs"].t().repeat_interleave(128, 1)[:, :K]
    w = st["wq"].view(E4M3)[:, :K].float() * st["ws"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = x @ w.t()
    if st["bias"] is not None:
        y = y + st["bias"]
    return y.to(DTYPES[c["out"]])


THETA, FACTOR, ORIGINAL, FAST, SLOW = 10000.0, 4.0, 32768, 32.0, 1.0


def _frequencies(case):
    """64-bit angles a position for one axis, and the factor on the rotated values."""
    d = case["axis_dim"]
    j = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    theta = THETA
    if case["scaling"] == "ntk" and d > 2:
        theta = THETA * FACTOR ** (d / (d - 2))
    f = theta ** (-2 * j / d)
    if case["scaling"] == "linear":
        f = f / FACTOR
    if case["scaling"] != "yarn":
        return f, 1.0
    # dims that turn more than FAST times over the original length keep their angle, those under SLOW take f / FACTOR
    edge = lambda turns: d * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
    lo, hi = max(math.floor(edge(FAST)), 0), min(math.ceil(edge(SLOW)), d - 1)
    keep = 1 - ((j - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f * keep + f / FACTOR * (1 - keep), 0.1 * math.log(FACTOR) + 1


def _rope_plain(st):
    c = st["case"]
    B, T, H, D = c["batch"], c["tokens"], c["heads"], c["dim"]
    f, amp = _frequencies(c)
    angle = (st["pos"].double()[:, :, None] * f).reshape(T, -1)  # axis after axis
    cos, sin = (angle.cos() * amp).float()[None, :, None], (angle.sin() * amp).float()[None, :, None]
    if c["inverse"]:
        sin = -sin
    P = angle.shape[1]
    x = st["x"].view(B, T, -1)[:, :, : H * D].reshape(B, T, H, D).float()
    y = x.clone()
    a, b = (slice(0, P), slice(P, 2 * P)) if c["layout"] == "half" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y.to(st["x"].dtype)


EPS = 1e-6


def _norm_plain(st):
    c = st["case"]
    B, S, C, G = c["batch"], c["rows"], c["channels"], c["groups"]
    x = st["x"].float().view(B, S, G, C // G)
    mean = x.mean(dim=(1, 3), keepdim=True)
    x = x - mean
    var = (x * x).mean(dim=(1, 3), keepdim=True)
    y = (x * torch.rsqrt(var + EPS)).view(B, S, C) * st["gamma"] + st["beta"]
    if c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(st["x"].dtype)


# ---------------------------------------------------------------- the framework's calls
_s2b = _ctx = None


def _framework():
    global _s2b, _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "seedvr2-2b-ncnn_b200"))
        import s2b as _s2b
        _ctx = _s2b.DitB200(0, _s2b.PREC_BF16)
    return _s2b, _ctx


def _own(st):
    s2b, ctx = _framework()
    c, op = st["case"], st["case"]["op"]
    types = {torch.float32: s2b.PREC_FP32, torch.float16: s2b.PREC_FP16, torch.bfloat16: s2b.PREC_BF16}
    stream = torch.cuda.current_stream().cuda_stream
    if op == "quant":
        x, q, s = st["x"], st["q"], st["scale"]
        R, C = x.shape
        ctx.fp8_quant_dev(x.data_ptr(), types[x.dtype], R, C, C, c["block_rows"], q.data_ptr(), q.shape[1], s.data_ptr(), stream)
        return {"q": q.view(E4M3)[:, :C], "scale": s}
    if op == "linear":
        xq, wq, y, b = st["xq"], st["wq"], st["y"], st["bias"]
        ctx.linear_fp8_dev(xq.data_ptr(), xq.shape[1], st["xs"].data_ptr(), c["M"], c["K"], wq.data_ptr(), wq.shape[1],
                           st["ws"].data_ptr(), c["N"], None if b is None else b.data_ptr(), y.data_ptr(), types[y.dtype],
                           c["N"], stream)
        return y
    if op == "rope":
        x, y = st["x"], st["y"]
        B, T, H, D = y.shape
        if "plan" not in st:  # a program makes it once for its model
            st["plan"] = s2b.rope_plan([c["axis_dim"]] * c["axes"], layout=c["layout"], theta=THETA, scaling=c["scaling"],
                                       factor=FACTOR, original_length=ORIGINAL, beta_fast=FAST, beta_slow=SLOW)
        ctx.rope_dev(st["plan"], x.data_ptr(), types[x.dtype], B, T, H, D, (T * c["row"], c["row"], D), st["pos"].data_ptr(),
                     0, 0, y.data_ptr(), (T * H * D, H * D, D), c["inverse"], stream)
        return y
    x, y = st["x"], st["y"]
    B, S, C = x.shape
    if "work" not in st:  # a program keeps its workspace
        st["work"] = torch.empty(max(1, s2b.groupnorm_workspace(B, S, C, c["groups"])), dtype=torch.uint8, device="cuda")
    ctx.groupnorm_dev(x.data_ptr(), types[x.dtype], B, S, C, C, c["groups"], st["gamma"].data_ptr(), st["beta"].data_ptr(), EPS,
                      c["act"] == "silu", y.data_ptr(), types[y.dtype], C, st["work"].data_ptr(), st["work"].numel(), stream)
    return y


def run(st):
    if own:
        return _own(st)
    op = st["case"]["op"]
    if op == "quant":
        q, s = _quant_plain(st["x"], st["case"]["block_rows"])
        return {"q": q, "scale": s}
    return {"linear": _linear_plain, "rope": _rope_plain, "norm": _norm_plain}[op](st)


# ---------------------------------------------------------------- 64 bits, from the definitions
def _decode64(codes):
    """e4m3 bytes to the numbers they stand for: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    v = codes.to(torch.int64)
    e, f = (v >> 3 & 15).double(), (v & 7).double()
    mag = torch.where(e > 0, torch.exp2(e - 7) * (1 + f / 8), torch.exp2(torch.full_like(e, -6)) * f / 8)
    return torch.where(v >= 128, -mag, mag)


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "quant":
        R, C = st["x"].shape
        b = _blocks_of(st["x"].double(), case["block_rows"])
        amax = b.abs().amax(dim=(1, 3))
        k = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / 448)).clamp(min=-126)
        k = torch.where(amax > 448 * torch.exp2(k), k + 1, k)  # where the logarithm landed on the wrong side
        k = torch.where((amax <= 448 * torch.exp2(k - 1)) & (k > -126), k - 1, k)
        s = torch.exp2(k)
        v = (b / s[:, None, :, None]).reshape(b.shape[0] * case["block_rows"], -1)[:R, :C]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
        return {"q": torch.round(v / step) * step, "scale": s.t().contiguous() if case["block_rows"] == 1 else s}
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        y = torch.zeros(M, N, dtype=torch.float64, device="cuda")
        if st["bias"] is not None:
            y += st["bias"].double()
        row_block = torch.arange(N, device="cuda") // 128
        for b in range(-(-K // 128)):
            cut = slice(128 * b, min(K, 128 * b + 128))
            x, w = _decode64(st["xq"][:, cut]), _decode64(st["wq"][:, cut])
            x *= st["xs"][b].double()[:, None]
            w *= st["ws"][:, b].double()[row_block][:, None]
            y.addmm_(x, w.t())
        return y
    if op == "rope":
        B, T, H, D = st["y"].shape
        f, amp = _frequencies(case)
        out = st["x"].view(B, T, -1)[..., : H * D].reshape(B, T, H, D).double()
        P = case["axes"] * f.numel()
        for i in range(P):  # pair after pair, as one complex number
            turn = torch.polar(torch.full((T,), amp, dtype=torch.float64, device="cuda"),
                               st["pos"][:, i // f.numel()].double() * f[i % f.numel()] * (-1 if case["inverse"] else 1))
            p, q = (i, i + P) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(out[..., p], out[..., q]) * turn[None, :, None]
            out[..., p], out[..., q] = z.real, z.imag
        return out
    B, S, C = st["x"].shape
    G, out = case["groups"], []
    for b in range(B):
        y = torch.empty(S, C, dtype=torch.float64, device="cuda")
        for g in range(G):
            cut = slice(g * (C // G), (g + 1) * (C // G))
            x = st["x"][b, :, cut].double()
            var, mean = torch.var_mean(x, correction=0)
            v = (x - mean) / torch.sqrt(var + EPS) * st["gamma"][cut].double() + st["beta"][cut].double()
            y[:, cut] = v * torch.sigmoid(v) if case["act"] == "silu" else v
        out.append(y)
    return torch.stack(out)
