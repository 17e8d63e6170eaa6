"""The operators beside the DiT against plain 64-bit forms: 8-bit block
quantisation, the 8-bit Linear, rotary positions, GroupNorm, and the chain of
them in front of an attention block.

Tolerances count roundings: an output type rounds by at most half a step
(HALF), fp32 arithmetic by 2^-24 a step; each test says how many it allows."""
import ctypes
import math

import pytest

import s2b

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FP32, FP16, BF16 = s2b.PREC_FP32, s2b.PREC_FP16, s2b.PREC_BF16
DT = {FP32: torch.float32, FP16: torch.float16, BF16: torch.bfloat16}
HALF = {FP32: 2.0 ** -24, FP16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {FP32: 2.0 ** -149, FP16: 2.0 ** -24, BF16: 2.0 ** -133}     # the smallest step of the type
IDS = {FP32: "fp32", FP16: "fp16", BF16: "bf16"}.get
E4M3 = torch.float8_e4m3fn
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    c = s2b.DitB200(0, s2b.PREC_BF16)
    yield c
    torch.cuda.synchronize()
    c.check_errors()                   # no bounded wait expired in any call of this file
    c.close()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def stream():
    return torch.cuda.current_stream().cuda_stream


def decode(codes):
    """e4m3 bytes to the numbers they stand for, in 64 bits."""
    v = codes.to(torch.int64)
    e, f = (v >> 3 & 15).double(), (v & 7).double()
    mag = torch.where(e > 0, torch.exp2(e - 7) * (1 + f / 8), f / 512)
    mag = torch.where((v & 127) == 127, torch.full_like(mag, math.nan), mag)
    return torch.where(v >= 128, -mag, mag)


# ---------------------------------------------------------------- quantisation
def quantise(ctx, x, block_rows, cols=None, ldq=None):
    R = x.shape[0]
    cols = x.shape[1] if cols is None else cols
    ldq = (cols + 15) // 16 * 16 if ldq is None else ldq
    kb = -(-cols // 128)
    q = torch.full((R + 2, ldq), 0x5A, dtype=torch.uint8, device=DEV)
    s = torch.full((kb * (R if block_rows == 1 else -(-R // 128)) + 3,), -7.0, device=DEV)
    t = {v: k for k, v in DT.items()}[x.dtype]
    ctx.fp8_quant_dev(x.data_ptr(), t, R, cols, x.stride(0), block_rows, q.data_ptr(), ldq, s.data_ptr(), stream())
    assert (q[R:] == 0x5A).all() and (q[:, cols:] == 0x5A).all() and (s[-3:] == -7).all()      # nothing else is written
    s = s[:-3].view(kb, R) if block_rows == 1 else s[:-3].view(-(-R // 128), kb)
    return q[:R, :cols], s


def quantise64(x, block_rows):
    """Codes as numbers (NaN where x is not finite) and scales, from the definition."""
    R, C = x.shape
    p = torch.nn.functional.pad(x.double(), (0, -C % 128, 0, -R % block_rows))
    b = p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // 128, 128)
    amax = torch.where(b.isfinite(), b.abs(), 0).amax(dim=(1, 3))
    k = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -150) / 448)).clamp(min=-126)
    k = torch.where(amax > 448 * torch.exp2(k), k + 1, k)
    k = torch.where((amax <= 448 * torch.exp2(k - 1)) & (k > -126), k - 1, k)
    s = torch.exp2(k)
    v = (b / s[:, None, :, None]).reshape(p.shape)[:R, :C]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6, max=448))).clamp(min=-6) - 3)
    return torch.where(v.isfinite(), torch.round(v / step) * step, math.nan), s.t() if block_rows == 1 else s


def check_quant(ctx, x, block_rows):
    q, s = quantise(ctx, x, block_rows)
    qr, sr = quantise64(x, block_rows)
    assert torch.equal(s.double(), sr)
    torch.testing.assert_close(decode(q), qr, rtol=0, atol=0, equal_nan=True)       # every code, bit for bit
    return q, s


@pytest.mark.parametrize("t", [FP32, FP16, BF16], ids=IDS)
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 2560), (3, 127), (31, 129), (58, 5120), (128, 128), (129, 2500), (300, 7), (257, 640)])
def test_quant_codes_equal_the_definition(ctx, R, C, br, t):
    g = gen(R * 1000 + C)
    x = normal(g, R, C) * torch.exp(2 * normal(g, R, 1))
    x[:, ::17] *= 30
    check_quant(ctx, x.to(DT[t]), br)


@pytest.mark.parametrize("t", [FP32, FP16, BF16], ids=IDS)
@pytest.mark.parametrize("br", [1, 128])
def test_quant_borders(ctx, br, t):
    """Zeros, values on both sides of 448 * 2^k, ties of the code, the smallest and
    largest values of the type, subnormals, NaN and infinities."""
    x = torch.zeros(256, 512, device=DEV, dtype=DT[t])
    fin = torch.finfo(DT[t])
    if br == 1:
        x[1, 0] = 448.0
        x[2, 0], x[3, 0] = 448 * (1 + 2 * fin.eps), 448 * (1 - 2 * fin.eps)
        x[4, :128] = torch.arange(128, device=DEV) / 8.0 - 8           # ties at every odd sixteenth
        x[4, 127] = 448.0
        x[5, 0], x[5, 1] = fin.max, fin.tiny
        x[6, 0] = fin.tiny
        x[7, :4] = torch.tensor([fin.tiny / 4, -fin.tiny / 4, 0, fin.tiny / 2], device=DEV, dtype=DT[t])
        x[8, 0], x[8, 1] = math.nan, 3.0
        x[9, 0], x[9, 1], x[9, 2] = math.inf, -math.inf, 100.0
        x[10, :128] = math.nan
        x[11, 130], x[11, 3] = math.inf, 5.0
        x[12, 0], x[12, 1] = -448.0, 2.0 ** -9
    else:
        x[:128, :128] = normal(gen(3), 128, 128).to(DT[t])
        x[5, 7] = math.nan
        x[0, 128], x[127, 255] = 448.0, -1.0
        x[1, 256], x[2, 257] = math.inf, 7.0
        x[128:, 128] = fin.tiny / 2
        x[200, 300] = fin.max
    check_quant(ctx, x, br)


@pytest.mark.parametrize("br", [1, 128])
def test_quant_pitches_and_unaligned_rows(ctx, br):
    g = gen(5)
    for t in (FP32, BF16):
        big = normal(g, 200, 333).to(DT[t])
        check_quant(ctx, big[:, 1:301], br)             # rows that start off a 16-byte boundary
        x = normal(g, 64, 512).to(DT[t])
        q, s = quantise(ctx, x, br, cols=300, ldq=304 + 48)
        qr, sr = quantise64(x[:, :300], br)
        assert torch.equal(s.double(), sr) and torch.equal(decode(q), qr)


# ---------------------------------------------------------------- 8-bit Linear
def codes(x, block_rows):
    """Pitched codes, scales and decoded values (64 bits) of x, made without the library."""
    v, s = quantise64(x, block_rows)
    q = torch.zeros(x.shape[0], (x.shape[1] + 15) // 16 * 16, dtype=torch.uint8, device=DEV)
    q[:, : x.shape[1]] = v.to(E4M3).view(torch.uint8)
    return q, s.float().contiguous()


def linear64(xq, xs, wq, ws, K, bias):
    """y and sum |x||w| in 64 bits."""
    N = wq.shape[0]
    x = decode(xq[:, :K]) * xs.double().t().repeat_interleave(128, 1)[:, :K]
    w = decode(wq[:, :K]) * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.abs().double()
    return y, mag


def run_linear(ctx, xq, xs, wq, ws, K, bias, t, ldy=None, st=None):
    M, N = xq.shape[0], wq.shape[0]
    ldy = N if ldy is None else ldy
    y = torch.full((M + 1, ldy), 123.0, dtype=DT[t], device=DEV)
    ctx.linear_fp8_dev(xq.data_ptr(), xq.stride(0), xs.data_ptr(), M, K, wq.data_ptr(), wq.stride(0), ws.data_ptr(), N,
                       None if bias is None else bias.data_ptr(), y.data_ptr(), t, ldy, stream() if st is None else st)
    return y


def check_linear(y, M, N, ref, mag, K, t):
    """Products of two codes are exact in fp32 and so are their scales' where those are powers of two; K additions,
    one scale product a block and the bias each err by at most 2^-23 of the running sum (rounded or cut), which stays
    below sum |x||w|."""
    assert (y[M:] == 123).all() and (y[:, N:] == 123).all()
    got = y[:M, :N].double()
    tol = (K + 2 * (-(-K // 128)) + 2) * 2.0 ** -23 * mag + HALF[t] * ref.abs() + TINY[t]
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (bad.sum().item(), ((got - ref).abs() / mag.clamp(min=1e-30)).max().item())


SHAPES = [(1, 128, 128), (1, 2560, 7680), (2, 16, 1), (5, 132, 77), (16, 640, 64), (17, 2500, 300), (33, 5120, 129), (58, 5120, 2560),
          (64, 256, 512), (65, 2560, 2560), (129, 384, 257), (256, 1024, 256), (257, 128, 513), (300, 2500, 1000), (511, 4000, 384),
          (513, 6912, 640), (1000, 2560, 2560), (2443, 1280, 1285), (5498, 2560, 512)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("t", [FP32, FP16, BF16], ids=IDS)
def test_linear_vs_64bit(ctx, M, K, N, t):
    g = gen(M + K + N)
    xq, xs = codes(normal(g, M, K) * torch.exp(normal(g, M, 1)), 1)
    wq, ws = codes(0.02 * normal(g, N, K), 128)
    bias = 0.1 * normal(g, N) if (M + N) % 2 else None
    ref, mag = linear64(xq, xs, wq, ws, K, bias)
    check_linear(run_linear(ctx, xq, xs, wq, ws, K, bias, t), M, N, ref, mag, K, t)


@pytest.mark.parametrize("M,K,N,ldy", [(3, 300, 200, 208), (70, 256, 130, 133), (700, 512, 640, 648), (700, 512, 600, 603), (1400, 300, 1300, 1304),
                                       (1400, 1100, 1303, 1304)])
def test_linear_any_scales_and_pitches(ctx, M, K, N, ldy):
    """Scales that are no powers of two, among them 0, negative and far apart ones; codes inside wider rows whose rest is
    NaN; y inside wider rows."""
    g = gen(M)
    kb = -(-K // 128)
    xq = torch.full((M, (K + 15) // 16 * 16 + 32), 0x7F, dtype=torch.uint8, device=DEV)
    wq = torch.full((N, (K + 15) // 16 * 16 + 16), 0x7F, dtype=torch.uint8, device=DEV)
    xq[:, :K] = codes(normal(g, M, K), 1)[0][:, :K]
    wq[:, :K] = codes(normal(g, N, K), 128)[0][:, :K]
    xs = torch.exp(3 * normal(g, kb, M))
    ws = 0.3 * normal(g, -(-N // 128), kb)
    xs[0, 0], ws[0, kb - 1] = 0.0, 0.0
    bias = normal(g, N)
    ref, mag = linear64(xq, xs, wq, ws, K, bias)
    for t in (FP32, BF16):
        check_linear(run_linear(ctx, xq, xs, wq, ws, K, bias, t, ldy), M, N, ref, mag, K, t)


# sizes that the CTA-pair kernel takes: odd numbers of blocks, one block, rows of y off 16 bytes, both tile widths
PAIR_SHAPES = [(1500, 128, 1000), (700, 300, 2000), (2049, 640, 1281), (300, 1664, 4000), (1400, 16, 1300), (4200, 900, 776), (900, 2200, 2563),
               (2600, 640, 13824), (5000, 384, 9000)]            # nine and eleven tiles a pair of CTAs


@pytest.mark.parametrize("M,K,N", PAIR_SHAPES)
@pytest.mark.parametrize("t", [FP32, BF16], ids=IDS)
def test_linear_many_rows_scaled_general_and_mixed(ctx, M, K, N, t):
    """Scales that are powers of two, scales that are none, and a few of these among those (so that some tiles of a call
    run one way and some the other), each with bias and with the rows of y inside wider ones."""
    g = gen(M + N)
    kb = -(-K // 128)
    xq, xs = codes(normal(g, M, K) * torch.exp(normal(g, M, 1)), 1)
    wq, ws = codes(0.02 * normal(g, N, K), 128)
    bias = normal(g, N)
    some = xs.clone()
    some[0, M // 2], some[kb - 1, 3] = 0.3, 0.0
    wsome = ws.clone()
    wsome[ws.shape[0] - 1, 0] = 3.0e-3
    wsome[:: 7, kb // 2] *= 1.3
    for a, b in ((xs, ws), (some, ws), (xs, wsome), (xs * 1.1, ws * 0.7)):
        ref, mag = linear64(xq, a, wq, b, K, bias)
        for ldy in (N, N + 5):
            check_linear(run_linear(ctx, xq, a, wq, b, K, bias, t, ldy), M, N, ref, mag, K, t)


def test_linear_extreme_scales(ctx):
    """Scales at both ends of what one byte of exponent holds, and past it (subnormal, zero): products stay fp32's."""
    M, K, N = 1500, 256, 1024
    g = gen(77)
    xq, xs = codes(normal(g, M, K), 1)
    wq, ws = codes(normal(g, N, K), 128)
    for ex, ew in ((2.0 ** -126, 2.0 ** 100), (2.0 ** 120, 2.0 ** -126), (2.0 ** -130, 2.0 ** 120), (0.0, 1.0), (2.0 ** 60, 2.0 ** -60)):
        a, b = torch.full_like(xs, ex), torch.full_like(ws, ew)
        ref, mag = linear64(xq, a, wq, b, K, None)
        check_linear(run_linear(ctx, xq, a, wq, b, K, None, FP32), M, N, ref, mag, K, FP32)


@pytest.mark.parametrize("M,N", [(1, 256), (40, 300), (600, 512), (1700, 1280)])
def test_linear_nan_stays_in_its_row_and_column(ctx, M, N):
    g, K = gen(9), 700
    xq, xs = codes(normal(g, M, K), 1)
    wq, ws = codes(normal(g, N, K), 128)
    ref, mag = linear64(xq, xs, wq, ws, K, None)
    xq[M - 1, 650] = 0x7F
    wq[N - 3, 5] = 0xFF
    y = run_linear(ctx, xq, xs, wq, ws, K, None, FP32)[:M]
    assert y[M - 1].isnan().all() and y[:, N - 3].isnan().all()
    keep = torch.ones(M, N, dtype=torch.bool, device=DEV)
    keep[M - 1], keep[:, N - 3] = False, False
    assert y[keep].isfinite().all()
    assert ((y.double() - ref).abs() <= 2 * K * 2.0 ** -23 * mag)[keep].all()


def test_linear_same_bits_every_time_and_on_two_streams(ctx):
    """Calls in flight together on two streams, with sizes of every kernel, give the bits of calls alone."""
    g = gen(11)
    sets = []
    for M, K, N in ((1, 2560, 2560), (58, 5120, 2560), (600, 2560, 2560), (1300, 1280, 1024)):
        xq, xs = codes(normal(g, M, K), 1)
        wq, ws = codes(0.02 * normal(g, N, K), 128)
        sets.append((xq, xs, wq, ws, K))
    alone = [run_linear(ctx, *s, None, BF16) for s in sets]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for rep in range(3):
        for i, s in enumerate(sets):
            with torch.cuda.stream((a, b)[(i + rep) % 2]):
                got.append((i, run_linear(ctx, *s, None, BF16)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y.view(torch.int16), alone[i].view(torch.int16))


@pytest.mark.parametrize("K", [2560, 5120, 6912])
@pytest.mark.parametrize("M,N", [(1, 512), (40, 768), (1536, 1280)])
def test_linear_error_against_the_norm_of_y(ctx, M, N, K):
    """What the header promises of fp32 outputs, against y's norm.  Scales that are no powers of two, and few rows: a
    block's sum is cut at most four times (2^-23 of it: 4.8e-7 at the very most, half that on average) and added with a
    rounding (2^-24 * sqrt(blocks / 2) against independent blocks, 3.1e-7 at the most, 1.8e-7 in rms): 5e-7.  Powers of
    two in the CTA-pair kernel: the tensor core's accumulator takes all of K, cut at each 32 codes: 2e-6, a quarter of what
    24 bits would lose.  Sums held in 16 bits anywhere would be off by 1e-3."""
    g = gen(K + M)
    xq, xs = codes(normal(g, M, K) * torch.exp(0.5 * normal(g, M, 1)), 1)
    wq, ws = codes(0.02 * normal(g, N, K), 128)
    for a, b, bound in ((xs, ws, 2e-6 if M > 1000 else 5e-7), (xs * 1.1, ws * 0.7, 5e-7)):
        ref, _ = linear64(xq, a, wq, b, K, None)
        y = run_linear(ctx, xq, a, wq, b, K, None, FP32)[:M].double()
        assert ((y - ref).norm() / ref.norm()).item() <= bound


def test_linear_error_flag_reaches_check_errors():
    c = s2b.DitB200(0, s2b.PREC_BF16)
    try:
        xq, xs = codes(normal(gen(1), 4, 128), 1)
        c.debug_raise_kernel_error(1)
        run_linear(c, xq, xs, xq, torch.ones(1, 1, device=DEV), 128, None, FP32)
        torch.cuda.synchronize()
        with pytest.raises(s2b.S2BError) as e:
            c.check_errors()
        assert e.value.code == 7
        c.check_errors()
    finally:
        c.close()


# ---------------------------------------------------------------- rotary positions
def frequencies(plan):
    return torch.tensor([plan.turns[i] for i in range(plan.pairs)], dtype=torch.float64, device=DEV) / 2.0 ** 64 * 2 * math.pi


def rope64(plan, x, pos, inverse):
    """x (B, T, H, D), pos (B, T, axes) -> the turned heads in 64 bits, and |a| + |b| of each pair in its places."""
    f = frequencies(plan)
    axis = torch.tensor([plan.axis[i] for i in range(plan.pairs)], device=DEV, dtype=torch.long)
    angle = pos.double()[:, :, axis] * f * (-1 if inverse else 1)
    P, y = plan.pairs, x.double().clone()
    mag = torch.zeros_like(y)
    a, b = (slice(0, P), slice(P, 2 * P)) if plan.half else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    cos, sin = angle.cos()[:, :, None] * plan.amplitude, angle.sin()[:, :, None] * plan.amplitude
    xa, xb = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = xa * cos - xb * sin, xa * sin + xb * cos
    mag[..., a] = mag[..., b] = (xa.abs() + xb.abs()) * plan.amplitude
    return y, mag


def run_rope(ctx, plan, x, t, pos, pbs, pos0, y, inverse=False):
    """x, y: (B, T, H, D) views with unit stride inside a head."""
    B, T, H, D = x.shape
    ctx.rope_dev(plan, x.data_ptr(), t, B, T, H, D, x.stride()[:3], None if pos is None else pos.data_ptr(), pbs, pos0,
                 y.data_ptr(), y.stride()[:3], inverse, stream())
    return y


def check_rope(got, ref, mag, t, reach, plan):
    """The fraction of a turn goes to fp32 (2^-24 of at most half a turn: pi 2^-24 rad), sine and cosine err by 2 units of
    2^-23, the amplitude's product and the pair's two products and sum by 2^-24 each: under 12 * 2^-24 of |a| + |b|.  The
    64-bit angle of the reference is cut at `reach` * 2^-52 of it."""
    tol = (12 * 2.0 ** -24 + reach * 2.0 ** -51) * mag + HALF[t] * ref.abs() + TINY[t]
    tol = torch.where(mag == 0, torch.zeros_like(tol), tol) if 2 * plan.pairs < got.shape[-1] else tol
    assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() - tol).max().item()


PLANS = [dict(axis_dims=[128], layout="half"), dict(axis_dims=[42, 42, 42]), dict(axis_dims=[32], layout="half"), dict(axis_dims=[10, 6], layout="half"),
         dict(axis_dims=[2]), dict(axis_dims=[64], scaling="yarn", factor=8.0, original_length=4096),
         dict(axis_dims=[16, 0, 48], scaling="ntk", factor=2.0), dict(axis_dims=[0])]


@pytest.mark.parametrize("t", [FP32, FP16, BF16], ids=IDS)
@pytest.mark.parametrize("B,T,H,D", [(1, 1, 40, 128), (2, 37, 3, 128), (3, 5, 1, 256), (1, 300, 8, 160)])
@pytest.mark.parametrize("kw", PLANS, ids=[f"{p['axis_dims']}{p.get('layout', '')}{p.get('scaling', '')}" for p in PLANS])
def test_rope_vs_64bit(ctx, kw, B, T, H, D, t):
    plan = s2b.rope_plan(**kw)
    g = gen(T + H)
    x = normal(g, B, T, H, D).to(DT[t])
    pos = torch.randint(-5000, 5000, (B, T, plan.axes), generator=g, device=DEV, dtype=torch.int32)
    for inverse in (False, True):
        buf = torch.full((B * T * H * D + 64,), 55.0, dtype=DT[t], device=DEV)
        y = run_rope(ctx, plan, x, t, pos, T * plan.axes, 0, buf[:-64].view(B, T, H, D), inverse)
        ref, mag = rope64(plan, x, pos, inverse)
        check_rope(y, ref, mag, t, 5000, plan)
        assert (buf[-64:] == 55).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t,D,dims,off", [(BF16, 80, 80, 0), (BF16, 50, 46, 0), (FP32, 7, 6, 0), (FP16, 128, 128, 1), (BF16, 33, 0, 0), (FP32, 64, 36, 2)])
def test_rope_odd_heads_and_unaligned_buffers(ctx, t, D, dims, off, layout):
    plan = s2b.rope_plan([dims], layout=layout)
    B, T, H = 2, 19, 3
    g = gen(D)
    src = normal(g, B * T * H * D + off).to(DT[t])
    x = src[off:].view(B, T, H, D)
    dst = torch.full((B * T * H * D + off + 8,), 9.0, dtype=DT[t], device=DEV)
    y = run_rope(ctx, plan, x, t, None, 0, 3, dst[off:-8].view(B, T, H, D))
    pos = (torch.arange(T, device=DEV) + 3)[None, :, None].expand(B, T, 1)
    ref, mag = rope64(plan, x, pos, False)
    check_rope(y, ref, mag, t, T + 3, plan)
    assert (dst[-8:] == 9).all() and (dst[:off] == 9).all()


@pytest.mark.parametrize("kw", [dict(axis_dims=[128], layout="half"), dict(axis_dims=[42, 42, 42])], ids=["half", "grid"])
@pytest.mark.parametrize("t", [FP32, BF16], ids=IDS)
def test_rope_inside_qkv_rows_in_place_and_heads_outermost(ctx, kw, t):
    """q and k of q|k|v rows: out into dense heads, in place with v and the other rows left as they were, and out into
    (heads, tokens) order; positions shared by the samples."""
    plan = s2b.rope_plan(**kw)
    B, T, H, D = 2, 45, 6, 128
    g = gen(1)
    qkv = normal(g, B, T + 2, 3 * H // 2 * D).to(DT[t])
    keep = qkv.clone()
    pos = torch.randint(0, 200, (T, plan.axes), generator=g, device=DEV, dtype=torch.int32)
    x = qkv[:, :T, : H * D].unflatten(2, (H, D))
    ref, mag = rope64(plan, x, pos[None].expand(B, -1, -1), False)
    y = run_rope(ctx, plan, x, t, pos, 0, 0, torch.empty(B, T, H, D, dtype=DT[t], device=DEV))
    check_rope(y, ref, mag, t, 200, plan)
    z = torch.empty(B, H, T, D, dtype=DT[t], device=DEV).transpose(1, 2)
    assert torch.equal(run_rope(ctx, plan, x, t, pos, 0, 0, z), y)
    run_rope(ctx, plan, x, t, pos, 0, 0, x)
    assert torch.equal(x, y)
    keep[:, :T, : H * D] = x.flatten(2)
    assert torch.equal(qkv, keep)


def test_rope_far_positions(ctx):
    """Positions to both ends of 32 bits: the reference's angles are reduced with Python's whole numbers."""
    plan = s2b.rope_plan([64], layout="half", theta=1e6)
    ps = [0, 1, 131071, 1 << 20, (1 << 24) + 1, 10 ** 9 + 7, 2 ** 31 - 1, -1, -(2 ** 31)]
    x = normal(gen(2), 1, len(ps), 2, 64)
    pos = torch.tensor(ps, dtype=torch.int32, device=DEV).view(1, -1, 1)
    y = run_rope(ctx, plan, x, FP32, pos, 0, 0, torch.empty_like(x))
    ang = torch.tensor([[(p * plan.turns[i] % 2 ** 64) / 2.0 ** 64 * 2 * math.pi for i in range(32)] for p in ps], dtype=torch.float64, device=DEV)
    a, b = x[..., :32].double(), x[..., 32:].double()
    c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]
    ref = torch.cat((a * c - b * s, a * s + b * c), -1)
    mag = torch.cat((a.abs() + b.abs(),) * 2, -1)
    check_rope(y, ref, mag, FP32, 1, plan)
    # pos0 counts on from any position, past 2^31 too
    z = run_rope(ctx, plan, x[:, :2], FP32, None, 0, 2 ** 31 - 1, torch.empty_like(x[:, :2]))
    assert torch.equal(z[:, 0], run_rope(ctx, plan, x[:, :1], FP32, pos[:, 6:7].contiguous(), 0, 0, torch.empty_like(x[:, :1]))[:, 0])
    ang = torch.tensor([2 ** 31 * plan.turns[i] % 2 ** 64 / 2.0 ** 64 * 2 * math.pi for i in range(32)], dtype=torch.float64, device=DEV)
    ref = torch.cat((a[:, 1] * ang.cos() - b[:, 1] * ang.sin(), a[:, 1] * ang.sin() + b[:, 1] * ang.cos()), -1)
    assert ((z[:, 1].double() - ref).abs() <= 13 * 2.0 ** -24 * mag[:, 1]).all()


def test_rope_angles_are_as_exact_as_documented(ctx):
    """Pairs (1, 0) become (cos, sin) of the angle: off by the documented 2^-26 + 2^-31 of a turn and by 2 ulp (2^-24 each
    below 1) of the sine or cosine, anywhere in 32 bits; the multiplications by 1 and 0 are exact."""
    plan = s2b.rope_plan([256], layout="interleaved", theta=500.0)
    g = gen(6)
    ps = [0, 1, -1, 2 ** 31 - 1, -(2 ** 31)] + torch.randint(-(2 ** 31), 2 ** 31, (300,), generator=g, device=DEV).tolist()
    x = torch.zeros(1, len(ps), 1, 256, device=DEV)
    x[..., ::2] = 1
    pos = torch.tensor(ps, dtype=torch.int32, device=DEV).view(1, -1, 1)
    y = run_rope(ctx, plan, x, FP32, pos, 0, 0, torch.empty_like(x))[0, :, 0].double()
    ang = torch.tensor([[(p * plan.turns[i] % 2 ** 64) / 2.0 ** 64 * 2 * math.pi for i in range(128)] for p in ps], dtype=torch.float64, device=DEV)
    tol = 2 * math.pi * (2.0 ** -26 + 2.0 ** -31) + 2 * 2.0 ** -24
    assert (y[:, ::2] - ang.cos()).abs().max().item() <= tol and (y[:, 1::2] - ang.sin()).abs().max().item() <= tol


def test_rope_inverse_is_the_gradient(ctx):
    """<rope(x), w> differs by <inverse(w), d> along d: the map is linear, so the difference is exact but for rounding."""
    plan = s2b.rope_plan([64], layout="half", scaling="yarn", factor=4.0, original_length=1000)
    g = gen(4)
    x, w, d = (normal(g, 2, 50, 4, 96) for _ in range(3))
    go = lambda v, inv=False: run_rope(ctx, plan, v, FP32, None, 0, 700, torch.empty_like(v), inv).double()  # noqa: E731
    lhs = ((go(x + d) - go(x)) * w.double()).sum()
    rhs = (go(w, True) * d.double()).sum()
    size = plan.amplitude * 2 * (w.abs() * (d.abs() + 2 * x.abs())).sum().item()
    assert abs(lhs.item() - rhs.item()) <= 30 * 2.0 ** -24 * size
    back = run_rope(ctx, plan, go(x).float(), FP32, None, 0, 700, torch.empty_like(x), True)
    assert torch.equal(back[..., 64:], x[..., 64:])
    assert ((back / plan.amplitude ** 2 - x)[..., :64].abs() <= 30 * 2.0 ** -24 * 2 * x.abs().max()).all()


# ---------------------------------------------------------------- GroupNorm
def norm64(x, G, gamma, beta, eps, act):
    B, S, C = x.shape
    v = x.double().view(B, S, G, C // G)
    mean = v.mean(dim=(1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    hat = ((v - mean) * rstd).view(B, S, C)
    gm = torch.ones(C, dtype=torch.float64, device=DEV) if gamma is None else gamma.double()
    y = hat * gm + (0 if beta is None else beta.double())
    pre = (mean.abs() * rstd).expand(B, S, G, C // G).reshape(B, S, C)
    return (y * torch.sigmoid(y) if act else y), y, hat, pre, gm.abs()


def run_norm(ctx, x, G, gamma, beta, eps, act, yt, y=None, work=None):
    """x (B, S, C), rows evenly strided."""
    B, S, C = x.shape
    t = {v: k for k, v in DT.items()}[x.dtype]
    y = torch.empty(B, S, C, dtype=DT[yt], device=DEV) if y is None else y
    n = s2b.groupnorm_workspace(B, S, C, G)
    work = torch.full((n + 16,), 0xFF, dtype=torch.uint8, device=DEV) if work is None else work
    ctx.groupnorm_dev(x.data_ptr(), t, B, S, C, x.stride(1), G, None if gamma is None else gamma.data_ptr(),
                      None if beta is None else beta.data_ptr(), eps, int(act), y.data_ptr(), yt, y.stride(1), work.data_ptr(), n,
                      stream())
    assert (work[n:] == 0xFF).all()
    return y


def check_norm(got, x, G, gamma, beta, eps, act, yt, steps=24):
    """Mean and variance: `steps` fp32 roundings relative to the spread about a near value, plus the mean's own rounding
    to fp32 (pre = |mean| / std) twice, in the mean and in x - mean; then 3 roundings of the affine map.  SiLU has slope
    below 1.1 and its exponential and reciprocal err by under 2^-20 relative (fast forms)."""
    ref, y, hat, pre, gm = norm64(x, G, gamma, beta, eps, act)
    tol = gm * 2.0 ** -24 * (steps * (1 + hat.abs()) + 2 * pre) + 3 * 2.0 ** -24 * y.abs()
    if act:
        tol = 1.1 * tol + 2.0 ** -20 * ref.abs() * (1 + y.abs() * 2.0 ** -3)
    tol = tol + HALF[yt] * ref.abs() + TINY[yt]
    assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() / tol).max().item()


NORMS = [(1, 1, 1, 1), (1, 1, 32, 8), (2, 7, 33, 3), (1, 1360, 512, 32), (3, 100, 48, 16), (1, 5000, 10, 1), (2, 333, 320, 32), (1, 257, 2560, 32),
         (1, 64, 5120, 5120), (5, 1025, 96, 32), (1, 40000, 128, 32), (2, 2, 64, 64), (1, 3000, 2056, 8)]


@pytest.mark.parametrize("xt,yt", [(BF16, BF16), (FP32, FP32), (FP16, FP16), (FP32, BF16), (BF16, FP32), (FP16, BF16)],
                         ids=lambda t: IDS(t))
@pytest.mark.parametrize("B,S,C,G", NORMS)
def test_groupnorm_vs_64bit(ctx, B, S, C, G, xt, yt):
    g = gen(S + C)
    x = (normal(g, B, S, C) * torch.exp(0.5 * normal(g, C)) + 2 * normal(g, C)).to(DT[xt])
    gamma, beta = normal(g, C), normal(g, C)
    for act, ga, be in ((True, gamma, beta), (False, None, None), (False, gamma, None), (True, None, beta)):
        check_norm(run_norm(ctx, x, G, ga, be, 1e-5, act, yt), x, G, ga, be, 1e-5, act, yt)


def test_groupnorm_far_means_and_flat_groups(ctx):
    """A mean 4096 times the spread cancels nothing but the mean's own fp32 rounding; a constant group gives beta."""
    g = gen(8)
    x = normal(g, 2, 3000, 64) + 4096.0
    x[1] += torch.arange(64, device=DEV) * 100.0
    check_norm(run_norm(ctx, x, 64, None, None, 1e-6, False, FP32), x, 64, None, None, 1e-6, False, FP32)
    check_norm(run_norm(ctx, x, 8, None, None, 1e-6, True, FP32), x, 8, None, None, 1e-6, True, FP32)
    c = torch.full((1, 500, 32), 3.25, device=DEV, dtype=torch.bfloat16)
    beta = normal(g, 32)
    y = run_norm(ctx, c, 4, normal(g, 32), beta, 1e-6, False, FP32)
    assert torch.equal(y, beta.expand(1, 500, 32))


@pytest.mark.parametrize("S", [40, 40000])
@pytest.mark.parametrize("t", [FP32, FP16, BF16], ids=IDS)
def test_groupnorm_silu_over_its_whole_range(ctx, t, S):
    """Constant groups, so that y = beta * sigmoid(beta) of known betas: from where the exponential leaves fp32's range to
    where it is 1.  fp32: the exponential errs by 2 ulp, the sum in the denominator by a rounding, its quotient by 2 ulp,
    the product by a rounding: 10 * 2^-24; for 16-bit outputs the fast exponential errs by |beta| + 5 ulp, the rest by 2
    more, next to their own half step.  Exponentials below 2^-126 are held to a few steps of 2^-149."""
    C = 512
    beta = torch.linspace(-120.0, 30.0, C, device=DEV)
    x = torch.full((1, S, C), 2.5, device=DEV, dtype=DT[t])
    y = run_norm(ctx, x, 4, None, beta, 1e-6, True, t)
    ref = (beta.double() * torch.sigmoid(beta.double()))[None, None]
    units = 10 if t == FP32 else 2 * (7 + beta.abs().double())
    tol = (1.01 * units * 2.0 ** -24 + (0 if t == FP32 else HALF[t])) * ref.abs() + 3 * 2.0 ** -149 * beta.abs().double() + TINY[t]
    err = (y.double() - ref).abs()
    assert (err <= tol).all(), ((err / tol).max().item(), beta[(err / tol).amax(dim=(0, 1)).argmax()].item())


@pytest.mark.parametrize("S,C,G", [(40, 64, 8), (20000, 64, 8), (300, 10, 2), (30000, 60, 20)])
@pytest.mark.parametrize("t", [FP32, BF16], ids=IDS)
def test_groupnorm_squares_past_fp32(ctx, t, S, C, G):
    """Finite values whose squared deviations leave fp32: the variance is infinite, as in plain fp32 statistics, and y is
    act(beta) in that group; the other groups are what they are without it."""
    g = gen(S)
    x, beta = normal(g, 1, S, C).to(DT[t]), normal(g, C)
    ref = run_norm(ctx, x, G, None, beta, 1e-6, False, FP32)
    for rows in ([0], [S - 1], list(range(0, S, 3)), [S // 2, S // 2 + 1]):
        z = x.clone()
        z[0, rows, 0] = 1e25
        if len(rows) == 2:
            z[0, rows[1], 0] = -1e25
        y = run_norm(ctx, z, G, None, beta, 1e-6, False, FP32)
        assert torch.equal(y[..., : C // G], beta[: C // G].expand(1, S, -1)) and torch.equal(y[..., C // G:], ref[..., C // G:])


def test_groupnorm_nan_and_inf_stay_in_their_group(ctx):
    g = gen(12)
    x = normal(g, 2, 900, 64)
    ref = run_norm(ctx, x, 8, None, None, 1e-6, True, FP32)
    x[0, 450, 9], x[1, 0, 63] = math.nan, math.inf
    y = run_norm(ctx, x, 8, None, None, 1e-6, True, FP32)
    assert y[0, :, 8:16].isnan().all() and y[1, :, 56:].isnan().all()
    y[0, :, 8:16], y[1, :, 56:] = ref[0, :, 8:16], ref[1, :, 56:]
    assert torch.equal(y, ref)


def unlike_first_values(kind, size, B, S, C, G, t):
    """Inputs whose groups begin with values unlike the rest."""
    g = gen(S + C + G)
    x = normal(g, B, S, C)
    if kind == "first":                    # one value: the group's first
        x[:, 0, :: C // G] = size
    elif kind == "head":                   # the first rows, which many threads begin with
        x[:, : max(1, min(64, S // 4))] *= size
    elif kind == "padding":                # rows of zeros ahead of far values
        x += size
        x[:, : max(1, S // 16)] = 0
    else:                                  # a lone value in zeros
        x.zero_()
        x[:, 0, :: C // G] = size
    return x.to(DT[t])


@pytest.mark.parametrize("kind", ["first", "head", "padding", "lone"])
@pytest.mark.parametrize("B,S,C,G", [(2, 300, 64, 8), (1, 300, 64, 64), (1, 7000, 64, 16), (2, 40000, 64, 8), (1, 40000, 64, 64), (1, 21760, 128, 32),
                                     (1, 30000, 60, 4), (1, 300, 10, 1), (1, 200000, 10, 2), (1, 40003, 64, 1)])
def test_groupnorm_first_values_unlike_the_rest(ctx, B, S, C, G, kind):
    """No value of a group is special: one that lies 30 to 300000 deviations off the rest, where the group begins or in
    every thread's first rows, costs no accuracy anywhere.  Deviations are differences to a batch's own mean (rounded
    relative to themselves), their squares sum to what the group's M2 holds, and means move by a share of a difference
    that M2 holds too: the roundings of check_norm, counted against the group's spread, are all there are."""
    for xt in (FP32, BF16):
        for size in (30.0, 1000.0, 4097.0, 300000.0):
            x = unlike_first_values(kind, size, B, S, C, G, xt)
            check_norm(run_norm(ctx, x, G, None, None, 1e-6, False, FP32), x, G, None, None, 1e-6, False, FP32)


@pytest.mark.parametrize("C,pad,off", [(64, 8, 0), (64, 3, 0), (60, 0, 2), (512, 16, 8)])
@pytest.mark.parametrize("t", [FP32, BF16], ids=IDS)
def test_groupnorm_pitches_in_place_and_unaligned(ctx, t, C, pad, off):
    B, S, G = 2, 210, 4
    g = gen(C)
    buf = normal(g, B * S * (C + pad) + off).to(DT[t])
    keep = buf.clone()
    x = buf[off:].view(B, S, C + pad)[:, :, :C]
    out = torch.full((B, S, C + pad), 7.0, dtype=DT[t], device=DEV)
    run_norm(ctx, x, G, None, None, 1e-6, True, t, y=out[:, :, :C])
    check_norm(out[:, :, :C], x, G, None, None, 1e-6, True, t)
    assert (out[:, :, C:] == 7).all()
    run_norm(ctx, x, G, None, None, 1e-6, True, t, y=x)
    assert torch.equal(x, out[:, :, :C])
    assert torch.equal(buf[:off], keep[:off]) and torch.equal(buf[off:].view(B, S, C + pad)[:, :, C:], keep[off:].view(B, S, C + pad)[:, :, C:])


def test_groupnorm_two_streams_with_a_workspace_each(ctx):
    g = gen(20)
    xs = [normal(g, 1, n, 512).bfloat16() for n in (1360, 21760, 9000)]
    alone = [run_norm(ctx, x, 32, None, None, 1e-6, True, BF16) for x in xs]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in xs]
    got = []
    for rep in range(3):
        for i, x in enumerate(xs):
            with torch.cuda.stream(st[i]):
                got.append((i, run_norm(ctx, x, 32, None, None, 1e-6, True, BF16)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, alone[i])


# ---------------------------------------------------------------- together
class Front:
    """GroupNorm + SiLU -> row codes -> 8-bit q|k|v Linear -> rotary q and k in place, over a latent grid's rows."""

    def __init__(self, ctx, T, C=512, H=4, D=128, seed=3):
        g = gen(seed)
        self.ctx, self.T, self.C, self.H, self.D, self.N = ctx, T, C, H, D, 3 * H * D
        self.x = torch.empty(1, T, C, dtype=torch.bfloat16, device=DEV)
        self.fill(seed)
        self.gamma, self.beta, self.bias = 1 + 0.1 * normal(g, C), 0.1 * normal(g, C), 0.1 * normal(g, self.N)
        w = 0.05 * normal(g, self.N, C)
        self.wq, self.ws = (v.clone() for v in quantise(ctx, w, 128))
        self.plan = s2b.rope_plan([42, 42, 42])
        t = torch.arange(T, device=DEV, dtype=torch.int32)
        self.pos = torch.stack((58 + t // 160, t // 16 % 10, t % 16), 1).contiguous().int()
        self.n = torch.empty(T, C, dtype=torch.bfloat16, device=DEV)
        self.xq, self.xs = torch.empty(T, C, dtype=torch.uint8, device=DEV), torch.empty(C // 128, T, device=DEV)
        self.qkv = torch.empty(T, self.N, dtype=torch.bfloat16, device=DEV)
        self.y = torch.empty_like(self.qkv)
        self.work = torch.empty(s2b.groupnorm_workspace(1, T, C, 32) + 16, dtype=torch.uint8, device=DEV)

    def fill(self, seed):
        self.x.copy_(normal(gen(seed), 1, self.T, self.C) * 3 + 1)

    def run(self):
        c, st, T, C, N, qk = self.ctx, stream(), self.T, self.C, self.N, 2 * self.H
        c.groupnorm_dev(self.x.data_ptr(), BF16, 1, T, C, C, 32, self.gamma.data_ptr(), self.beta.data_ptr(), 1e-6, s2b.ACT_SILU,
                        self.n.data_ptr(), BF16, C, self.work.data_ptr(), self.work.numel(), st)
        c.fp8_quant_dev(self.n.data_ptr(), BF16, T, C, C, 1, self.xq.data_ptr(), C, self.xs.data_ptr(), st)
        c.linear_fp8_dev(self.xq.data_ptr(), C, self.xs.data_ptr(), T, C, self.wq.data_ptr(), C, self.ws.data_ptr(), N, self.bias.data_ptr(),
                         self.qkv.data_ptr(), BF16, N, st)
        self.y.copy_(self.qkv)
        c.rope_dev(self.plan, self.y.data_ptr(), BF16, 1, T, qk, self.D, (0, N, self.D), self.pos.data_ptr(), 0, 0, self.y.data_ptr(),
                   (0, N, self.D), False, st)

    def check(self):
        T, C, N = self.T, self.C, self.N
        check_norm(self.n[None], self.x, 32, self.gamma, self.beta, 1e-6, True, BF16)
        qr, sr = quantise64(self.n, 1)
        assert torch.equal(decode(self.xq), qr) and torch.equal(self.xs.double(), sr)
        ref, mag = linear64(self.xq, self.xs, self.wq, self.ws, C, self.bias)
        tol = (C + 10) * 2.0 ** -23 * mag + HALF[BF16] * ref.abs()
        assert ((self.qkv.double() - ref).abs() <= tol).all()
        qk = self.qkv[:, : 2 * N // 3].view(1, T, -1, self.D)
        ref, mag = rope64(self.plan, qk, self.pos[None], False)
        check_rope(self.y[:, : 2 * N // 3].view(1, T, -1, self.D), ref, mag, BF16, 5000, self.plan)
        assert torch.equal(self.y[:, 2 * N // 3:], self.qkv[:, 2 * N // 3:])


@pytest.mark.parametrize("T", [1, 58, 333, 1440])
def test_front_of_an_attention_block(ctx, T):
    f = Front(ctx, T)
    f.run()
    f.check()


def test_front_captured_and_replayed_on_new_inputs(ctx):
    """The chain in two graphs that are replayed in turn and at the same time, against eager runs."""
    fs = [Front(ctx, 160, seed=5), Front(ctx, 700, seed=6)]
    for f in fs:
        f.run()
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for f in fs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f.run()
        graphs.append(gr)
    for seed in (7, 8):
        for f in fs:
            f.fill(seed)
            f.y.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for f in fs:
            f.check()
            y = f.y.clone()
            f.run()
            assert torch.equal(f.y, y)


# ---------------------------------------------------------------- far offsets, broadcasts
def test_offsets_past_32_bits(ctx):
    """Rows, samples and heads that start more than 2^32 elements (or bytes) into their buffers."""
    g = gen(31)
    far = (1 << 32) + 1024
    # rotary: the second sample far away, in and out
    plan = s2b.rope_plan([128], layout="half")
    big, out = (torch.empty(far + 4096, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    x, y = (torch.as_strided(b, (2, 3, 2, 128), (far, 256, 128, 1)) for b in (big, out))
    x.copy_(normal(g, 2, 3, 2, 128))
    run_rope(ctx, plan, x, BF16, None, 0, 5, y)
    pos = (torch.arange(3, device=DEV) + 5)[None, :, None].expand(2, 3, 1)
    ref, mag = rope64(plan, x.contiguous(), pos, False)
    check_rope(y, ref, mag, BF16, 10, plan)
    # GroupNorm: rows 2^17 apart, streamed and in place
    S, C, ld = 40000, 64, 1 << 17
    assert S * ld > 1 << 32
    del big, out, x, y
    buf = torch.empty(S * ld // 2 + C, dtype=torch.bfloat16, device=DEV)
    x = torch.as_strided(buf, (1, S, C), (S * ld // 2, ld // 2, 1))
    x.copy_(normal(g, 1, S, C))
    keep = x.contiguous()
    run_norm(ctx, x, 8, None, None, 1e-6, False, BF16, y=x)
    check_norm(x.contiguous(), keep, 8, None, None, 1e-6, False, BF16)
    # quantisation: codes and rows far apart
    x = torch.as_strided(buf, (S, 32), (ld // 2, 1))
    x.copy_(normal(g, S, 32))
    q = torch.empty(S * ld, dtype=torch.uint8, device=DEV)
    s = torch.empty(1, S, device=DEV)
    ctx.fp8_quant_dev(x.data_ptr(), BF16, S, 32, ld // 2, 1, q.data_ptr(), ld, s.data_ptr(), stream())
    qr, sr = quantise64(x.contiguous(), 1)
    codes_ = torch.as_strided(q, (S, 32), (ld, 1)).contiguous()
    assert torch.equal(decode(codes_), qr) and torch.equal(s.double(), sr)
    # Linear: those codes as x, y's rows far apart, by both kernels
    wq, ws = codes(normal(g, 1000, 32), 128)
    for M in (40, 36000):
        ref, mag = linear64(codes_[:M], s[:, :M].contiguous(), wq, ws, 32, None)
        xs = s[:, :M].contiguous()
        ctx.linear_fp8_dev(q.data_ptr(), ld, xs.data_ptr(), M, 32, wq.data_ptr(), wq.stride(0), ws.data_ptr(), 1000, None,
                           buf.data_ptr(), BF16, ld // 2, stream())
        y = torch.as_strided(buf, (M, 1000), (ld // 2, 1)).double()
        assert ((y - ref).abs() <= 40 * 2.0 ** -23 * mag + HALF[BF16] * ref.abs() + TINY[BF16]).all()


def test_rope_broadcast_heads(ctx):
    """One head read for many (stride 0), as shared keys are: the gradient's inverse takes the heads apart again."""
    plan = s2b.rope_plan([64], layout="half")
    x = normal(gen(3), 1, 40, 1, 64)
    y = run_rope(ctx, plan, x.expand(1, 40, 6, 64), FP32, None, 0, 0, torch.empty(1, 40, 6, 64, device=DEV))
    one = run_rope(ctx, plan, x, FP32, None, 0, 0, torch.empty_like(x))
    assert torch.equal(y, one.expand(1, 40, 6, 64))


# ---------------------------------------------------------------- refusals that need the context
def test_host_memory_is_refused_and_writes_nothing(ctx):
    h = torch.zeros(16, 128)
    d = torch.zeros(16, 128, device=DEV)
    q, s = torch.zeros(16, 128, dtype=torch.uint8, device=DEV), torch.zeros(16, device=DEV)
    plan = s2b.rope_plan([128])
    pinned = torch.zeros(16, 128).pin_memory()
    calls = [lambda: ctx.fp8_quant_dev(h.data_ptr(), FP32, 16, 128, 128, 1, q.data_ptr(), 128, s.data_ptr(), stream()),
             lambda: ctx.fp8_quant_dev(d.data_ptr(), FP32, 16, 128, 128, 1, q.data_ptr(), 128, h.data_ptr(), stream()),
             lambda: ctx.linear_fp8_dev(q.data_ptr(), 128, s.data_ptr(), 16, 128, q.data_ptr(), 128, s.data_ptr(), 16, h.data_ptr(),
                                        d.data_ptr(), FP32, 128, stream()),
             lambda: ctx.rope_dev(plan, d.data_ptr(), FP32, 1, 16, 1, 128, (0, 128, 0), None, 0, 0, pinned.data_ptr(), (0, 128, 0), False, stream()),
             lambda: ctx.groupnorm_dev(d.data_ptr(), FP32, 1, 16, 128, 128, 8, h.data_ptr(), None, 1e-6, 0, d.data_ptr(), FP32, 128,
                                       q.data_ptr(), q.numel() * 64, stream())]
    for c in calls:
        with pytest.raises(s2b.S2BError) as e:
            c()
        assert e.value.code == 1 and "context's device" in str(e.value) or "device memory" in str(e.value)
    torch.cuda.synchronize()
    assert not h.any() and not d.any() and not q.any() and not pinned.any()


def test_host_memory_is_refused_with_its_code(ctx):
    """Each operator with one buffer on the host, pageable or page-locked: the argument code, whatever the words."""
    d = torch.zeros(64, 128, device=DEV)
    q, s = torch.zeros(64, 128, dtype=torch.uint8, device=DEV), torch.zeros(64, device=DEV)
    plan, n = s2b.rope_plan([128]), 1 << 14
    for h in (torch.zeros(64, 128), torch.zeros(64, 128).pin_memory()):
        p = h.data_ptr()
        calls = [lambda: ctx.fp8_quant_dev(p, FP32, 16, 128, 128, 1, q.data_ptr(), 128, s.data_ptr(), stream()),
                 lambda: ctx.fp8_quant_dev(d.data_ptr(), FP32, 16, 128, 128, 1, p, 128, s.data_ptr(), stream()),
                 lambda: ctx.linear_fp8_dev(q.data_ptr(), 128, p, 16, 128, q.data_ptr(), 128, s.data_ptr(), 16, None, d.data_ptr(), FP32, 128, stream()),
                 lambda: ctx.linear_fp8_dev(q.data_ptr(), 128, s.data_ptr(), 16, 128, q.data_ptr(), 128, s.data_ptr(), 16, None, p, FP32, 128, stream()),
                 lambda: ctx.rope_dev(plan, p, FP32, 1, 16, 1, 128, (0, 128, 0), None, 0, 0, d.data_ptr(), (0, 128, 0), False, stream()),
                 lambda: ctx.rope_dev(plan, d.data_ptr(), FP32, 1, 16, 1, 128, (0, 128, 0), p, 0, 0, d.data_ptr(), (0, 128, 0), False, stream()),
                 lambda: ctx.groupnorm_dev(d.data_ptr(), FP32, 1, 16, 128, 128, 8, None, p, 1e-6, 0, d.data_ptr(), FP32, 128, q.data_ptr(), n, stream()),
                 lambda: ctx.groupnorm_dev(d.data_ptr(), FP32, 1, 16, 128, 128, 8, None, None, 1e-6, 0, d.data_ptr(), FP32, 128, p, n, stream())]
        for c in calls:
            with pytest.raises(s2b.S2BError) as e:
                c()
            assert e.value.code == 1
        torch.cuda.synchronize()
        assert not h.any() and not d.any() and not q.any() and not s.any()


def test_empty_calls_write_nothing(ctx):
    y = torch.full((4, 128), 5.0, device=DEV)
    plan = s2b.rope_plan([128])
    ctx.fp8_quant_dev(None, FP32, 0, 128, 128, 1, None, 128, None, stream())
    ctx.linear_fp8_dev(None, 128, None, 0, 128, None, 128, None, 128, None, y.data_ptr(), FP32, 128, stream())
    ctx.linear_fp8_dev(None, 128, None, 4, 128, None, 128, None, 0, None, y.data_ptr(), FP32, 128, stream())
    ctx.rope_dev(plan, None, FP32, 1, 0, 1, 128, (0, 0, 0), None, 0, 0, None, (0, 0, 0), False, stream())
    ctx.groupnorm_dev(None, FP32, 1, 0, 128, 128, 8, None, None, 1e-6, 0, None, FP32, 128, None, 0, stream())
    torch.cuda.synchronize()
    assert (y == 5).all()


def test_calls_leave_the_current_device(ctx):
    before = torch.cuda.current_device()
    q, s = quantise(ctx, normal(gen(1), 4, 128), 1)
    assert torch.cuda.current_device() == before and ctypes.CDLL(None) is not None


# ---------------------------------------------------------------- back to back
@pytest.mark.parametrize("T,C,N", [(1, 256, 256), (40, 512, 384), (150, 1280, 640), (700, 640, 1280)])
def test_back_to_back_calls_see_what_the_calls_before_wrote(ctx, T, C, N):
    """Calls of one stream overlap at their ends.  A run of them over buffers that every step writes anew -- codes and
    scales, and the weights' scales, bias, gamma and positions, copied by a rotary call without pairs -- gives what the
    same calls give with the device idle before each; eager and from a graph."""
    g = gen(T + C)
    n = 24
    copy, turned = s2b.rope_plan([0]), s2b.rope_plan([64])
    nwb, kb = -(-N // 128), -(-C // 128)
    src = [dict(x=normal(g, T, C).bfloat16(), gamma=normal(g, C), bias=normal(g, N), ws=torch.exp2(torch.randint(-3, 3, (nwb * kb,), generator=g, device=DEV).float()),
                pos=torch.randint(0, 5000, (T,), generator=g, device=DEV, dtype=torch.int32)) for _ in range(n)]
    for i in range(0, n, 3):
        src[i]["ws"] *= 1.25                                   # not powers of two
    wq, _ = quantise(ctx, normal(g, N, C), 128, ldq=C)
    now = {k: torch.empty_like(v) for k, v in src[0].items() if k != "x"}
    work = torch.empty(max(1, s2b.groupnorm_workspace(1, T, C, 32)), dtype=torch.uint8, device=DEV)
    h = torch.empty(T, C, dtype=torch.bfloat16, device=DEV)
    xq = torch.empty(T, C, dtype=torch.uint8, device=DEV)
    xs = torch.empty(kb, T, device=DEV)

    def run(out, idle):
        st = stream()
        for i, s in enumerate(src):
            y = out[i].data_ptr()
            calls = [lambda k=k: ctx.rope_dev(copy, s[k].data_ptr(), FP32, 1, 1, 1, s[k].numel(), (0, 0, 0), None, 0, 0, now[k].data_ptr(),
                                              (0, 0, 0), False, st) for k in now]
            calls += [
                lambda: ctx.groupnorm_dev(s["x"].data_ptr(), BF16, 1, T, C, C, 32, now["gamma"].data_ptr(), None, 1e-6, s2b.ACT_SILU,
                                          h.data_ptr(), BF16, C, work.data_ptr(), work.numel(), st),
                lambda: ctx.fp8_quant_dev(h.data_ptr(), BF16, T, C, C, 1, xq.data_ptr(), C, xs.data_ptr(), st),
                lambda: ctx.linear_fp8_dev(xq.data_ptr(), C, xs.data_ptr(), T, C, wq.data_ptr(), C, now["ws"].data_ptr(), N,
                                           now["bias"].data_ptr(), y, BF16, N, st),
                lambda: ctx.rope_dev(turned, y, BF16, 1, T, N // 64, 64, (0, N, 64), now["pos"].data_ptr(), 0, 0, y, (0, N, 64), False, st)]
            for c in calls:
                c()
                if idle:
                    torch.cuda.synchronize()

    ref = torch.zeros(n, T, N, dtype=torch.bfloat16, device=DEV)
    run(ref, True)
    assert ref.isfinite().all() and not torch.equal(ref[0], ref[1])
    got = torch.zeros_like(ref)
    for _ in range(8):
        got.zero_()
        run(got, False)
        assert torch.equal(got, ref)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        run(got, False)
    for _ in range(8):
        got.zero_()
        gr.replay()
        assert torch.equal(got, ref)


@pytest.mark.parametrize("t,T,H,D,kw", [
    (BF16, 60000, 8, 64, dict(axis_dims=[32], layout="half")), (FP32, 60000, 9, 32, dict(axis_dims=[32], layout="half")),
    (FP16, 80000, 12, 24, dict(axis_dims=[6, 8, 4])), (BF16, 60000, 6, 62, dict(axis_dims=[62])), (BF16, 21000, 6, 33, dict(axis_dims=[32])),
    (FP32, 3, 2, 4200, dict(axis_dims=[256], layout="half")), (BF16, 3, 2, 4201, dict(axis_dims=[254])),
])
def test_rope_many_tokens_and_wide_heads(ctx, t, T, H, D, kw):
    """CTAs that take several batches of heads, and heads that take several CTAs; into another buffer and in place."""
    plan = s2b.rope_plan(**kw)
    x = normal(gen(T + D), 1, T, H, D).to(DT[t])
    y = torch.full((T * H * D + 64,), 55.0, dtype=DT[t], device=DEV)
    run_rope(ctx, plan, x, t, None, 0, 7, y[:-64].view(1, T, H, D))
    pos = (torch.arange(T, device=DEV) + 7)[None, :, None].expand(1, T, plan.axes)
    ref, mag = rope64(plan, x, pos, False)
    check_rope(y[:-64].view(1, T, H, D), ref, mag, t, T + 7, plan)
    assert (y[-64:] == 55).all()
    run_rope(ctx, plan, x, t, None, 0, 7, x)
    assert torch.equal(x, y[:-64].view(1, T, H, D))


# ---------------------------------------------------------------- errors that are not a call's
def test_pending_cuda_error_stays_the_callers(tmp_path):
    """A CUDA error left pending before an operator call is still there after it, and the call succeeds."""
    import glob
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    objs = glob.glob(os.path.join(root, "seedvr2-2b-ncnn_b200", "build", "*.o"))
    if not objs:
        pytest.skip("the library's objects are not here")
    exe = str(tmp_path / "pending_error")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), "-I/usr/local/cuda/include",
                        os.path.join(root, "tests", "cpp", "pending_error.cpp"), *objs, "-L/usr/local/cuda/lib64", "-lcudart_static", "-lpthread",
                        "-ldl", "-lrt", "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr
