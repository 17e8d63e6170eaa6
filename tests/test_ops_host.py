"""The operators beside the DiT, host side: refusals come before any device is
touched (a null context reports them through s2b_last_error(NULL)), the rotary
plan against its formula, and the workspace size."""
import ctypes
import math

import numpy as np
import pytest

import s2b

A = 1 << 20            # addresses that are never read: far apart, 16-byte aligned
X, Q, S, W, V, Y, B = (A * k for k in range(1, 8))
FP32, FP16, BF16 = s2b.PREC_FP32, s2b.PREC_FP16, s2b.PREC_BF16


def refused(rc, needle):
    msg = s2b.lib().s2b_last_error(None).decode()
    assert rc == 1 and needle in msg, (rc, msg)


def quant(x=X, t=BF16, rows=4, cols=256, ldx=256, br=1, q=Q, ldq=256, s=S):
    return s2b.lib().s2b_fp8_quant_dev(None, x, t, rows, cols, ldx, br, q, ldq, s, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(t=3), "x_type"), (dict(t=-1), "x_type"), (dict(rows=-1), "negative"), (dict(br=2), "block_rows"),
    (dict(x=None), "null buffer"), (dict(q=None), "null buffer"), (dict(s=None), "null buffer"),
    (dict(ldx=255), "pitch below"), (dict(ldq=240), "pitch below"), (dict(ldq=264), "multiple of 16"),
    (dict(q=Q + 8), "16-byte"), (dict(x=X + 1), "aligned to its type"), (dict(s=S + 2), "aligned to its type"),
    (dict(q=X), "overlap"), (dict(s=Q + 16), "overlap"), (dict(), "null context"), (dict(rows=0, x=None), "null context"),
])
def test_quant_refusals(kw, needle):
    refused(quant(**kw), needle)


def linear(xq=X, ldx=256, xs=S, M=4, K=256, wq=W, ldw=256, ws=V, N=64, b=None, y=Y, t=BF16, ldy=64):
    return s2b.lib().s2b_linear_fp8_dev(None, xq, ldx, xs, M, K, wq, ldw, ws, N, b, y, t, ldy, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(t=5), "y_type"), (dict(M=-1), "negative"), (dict(K=0), "K must be positive"), (dict(N=-2), "negative"),
    (dict(xq=None), "null"), (dict(xs=None), "null"), (dict(wq=None), "null"), (dict(ws=None), "null"),
    (dict(y=None), "null"), (dict(ldx=240), "pitch below"), (dict(ldw=255), "pitch below"), (dict(ldy=63), "pitch below"),
    (dict(ldx=264), "multiples of 16"), (dict(ldw=257), "multiples of 16"), (dict(xq=X + 1), "16-byte"),
    (dict(wq=W + 8), "16-byte"), (dict(y=Y + 1), "aligned"), (dict(b=B + 2), "aligned"), (dict(xs=S + 1), "aligned"),
    (dict(y=X), "overlaps"), (dict(y=W + 256), "overlaps"), (dict(y=S), "overlaps"), (dict(y=V), "overlaps"),
    (dict(b=Y + 4), "overlaps"), (dict(), "null context"),
])
def test_linear_refusals(kw, needle):
    refused(linear(**kw), needle)


L3 = ctypes.c_long * 3


def rope(plan=None, x=X, t=BF16, batch=2, tokens=3, heads=4, dim=128, xs=(1536, 512, 128), pos=None, pbs=0, pos0=0,
         y=Y, ys=(1536, 512, 128), inverse=0):
    plan = s2b.rope_plan([64]) if plan is None else plan
    return s2b.lib().s2b_rope_dev(None, plan, x, t, batch, tokens, heads, dim, L3(*xs), pos, pbs, pos0, y, L3(*ys),
                                  inverse, None)


def broken(**kw):
    p = s2b.rope_plan([64])
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,needle", [
    (dict(t=9), "type"), (dict(batch=-1), "negative"), (dict(dim=0), "head_dim"), (dict(dim=62), "more than head_dim"),
    (dict(plan=broken(pairs=129)), "not a plan"), (dict(plan=broken(axes=0)), "not a plan"),
    (dict(plan=broken(amplitude=math.inf)), "not a plan"), (dict(x=None), "null"), (dict(y=None), "null"),
    (dict(x=X + 1), "aligned"), (dict(pos=Q + 2), "aligned"), (dict(xs=(-1, 512, 128)), "negative"),
    (dict(ys=(1536, 512, -128)), "negative"), (dict(ys=(1 << 41, 512, 128)), "2^40"), (dict(pos=Q, pbs=-1), "negative"),
    (dict(ys=(1536, 512, 127)), "overlap"), (dict(ys=(1536, 256, 128)), "overlap"), (dict(ys=(0, 512, 128)), "overlap"),
    (dict(y=X, ys=(1536, 512, 128), xs=(1536, 0, 128)), "overlap without"), (dict(y=X + 2), "overlap without"),
    (dict(pos=Y + 8), "overlaps the positions"), (dict(), "null context"), (dict(y=X), "null context"),
    # heads outermost, and a broadcast input, are fine
    (dict(ys=(1536, 128, 384)), "null context"), (dict(xs=(0, 512, 0)), "null context"),
    (dict(batch=0, x=None), "null context"),
])
def test_rope_refusals(kw, needle):
    refused(rope(**kw), needle)


def test_rope_null_strides_and_plan():
    L = s2b.lib()
    refused(L.s2b_rope_dev(None, s2b.rope_plan([64]), X, BF16, 1, 1, 1, 64, None, None, 0, 0, Y, L3(0, 0, 0), 0, None), "null strides")
    refused(L.s2b_rope_dev(None, None, X, BF16, 1, 1, 1, 64, L3(0, 0, 0), None, 0, 0, Y, L3(0, 0, 0), 0, None), "null plan")
    refused(L.s2b_rope_plan(None, None), "null")


def norm(x=X, xt=BF16, batch=2, rows=10, C=64, ldx=64, G=8, gamma=S, beta=V, eps=1e-6, act=1, y=Y, yt=BF16, ldy=64,
         work=B, nbytes=1 << 19):
    return s2b.lib().s2b_groupnorm_dev(None, x, xt, batch, rows, C, ldx, G, gamma, beta, eps, act, y, yt, ldy, work,
                                       nbytes, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(xt=3), "types"), (dict(yt=-1), "types"), (dict(batch=-1), "negative"), (dict(C=0), "positive"),
    (dict(G=0), "positive"), (dict(G=7), "multiple of groups"), (dict(act=2), "act"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(x=None), "null"), (dict(y=None), "null"),
    (dict(ldx=63), "pitch"), (dict(ldy=63), "pitch"), (dict(x=X + 1), "aligned"), (dict(gamma=S + 2), "aligned"),
    (dict(nbytes=0), "workspace smaller"), (dict(work=None), "workspace smaller"), (dict(work=B + 8), "not 16-byte"),
    (dict(y=X + 64), "overlap without"), (dict(y=X, yt=FP32), "overlap without"), (dict(gamma=Y), "overlaps gamma"),
    (dict(work=Y), "workspace overlaps"), (dict(batch=70000), "65535"), (dict(), "null context"), (dict(y=X), "null context"),
    (dict(rows=0, work=None, nbytes=0), "null context"),
])
def test_groupnorm_refusals(kw, needle):
    refused(norm(**kw), needle)


def test_groupnorm_workspace_is_small_next_to_the_data():
    assert s2b.groupnorm_workspace(0, 10, 64, 8) == 0 and s2b.groupnorm_workspace(1, 0, 64, 8) == 0
    for b, r, c, g in ((1, 1, 64, 8), (1, 1360, 512, 32), (3, 21760, 512, 32), (1, 1088 * 1280, 128, 32), (65535, 1, 8, 1)):
        assert s2b.groupnorm_workspace(b, r, c, g) <= b * r * c // 2 + 16 * b * c + 16 * b * g
    with pytest.raises(s2b.S2BError):
        s2b.groupnorm_workspace(1, 1, 0, 1)


def turns(plan):
    return np.array([plan.turns[i] for i in range(plan.pairs)], dtype=np.float64) / 2.0 ** 64


@pytest.mark.parametrize("d,theta", [(2, 10000.0), (42, 10000.0), (128, 10000.0), (256, 5e5)])
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_rope_plan_follows_the_formula(d, theta, scaling):
    """Fractions of a turn to 1e-15 relative: both sides hold the frequency in
    at least 53 bits, and the fraction is cut at 2^-64 of a turn."""
    factor, orig, fast, slow = 4.0, 4096, 32.0, 1.0
    p = s2b.rope_plan([d], theta=theta, scaling=scaling, factor=factor, original_length=orig, beta_fast=fast, beta_slow=slow)
    j = np.arange(d // 2)
    th = theta * factor ** (d / (d - 2)) if scaling == "ntk" and d > 2 else theta
    f = th ** (-2 * j / d)
    amp = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        edge = lambda n: d * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(edge(fast)), 0), min(math.ceil(edge(slow)), d - 1)
        ramp = np.clip((j - lo) / max(hi - lo, 0.001), 0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        amp = 0.1 * math.log(factor) + 1
    np.testing.assert_allclose(turns(p), f / (2 * math.pi), rtol=1e-14, atol=2.0 ** -64)
    assert p.pairs == d // 2 and p.axes == 1 and abs(p.amplitude - amp) < 1e-6


def test_rope_plan_axes_and_the_dits_own_frequencies():
    p = s2b.rope_plan([42, 42, 42])
    assert p.pairs == 63 and p.half == 0 and [p.axis[i] for i in range(63)] == [i // 21 for i in range(63)]
    w = s2b.make_win(1, 2, 2, (1, 1, 1), 3, False)      # the library's own angle tables: position 58-style txt rows
    txt = w.txt_freq.reshape(w.nwin, 3, 126)[0, 2]      # position 2 on every axis, angles of pairs side by side
    np.testing.assert_allclose(2 * 2 * math.pi * turns(p), txt[::2], rtol=2.0 ** -23)
    q = s2b.rope_plan([0, 16, 4], layout="half")
    assert q.pairs == 10 and q.half == 1 and [q.axis[i] for i in range(10)] == [1] * 8 + [2] * 2


@pytest.mark.parametrize("kw", [
    dict(axis_dims=[3]), dict(axis_dims=[-2]), dict(axis_dims=[258]), dict(axis_dims=[128, 128, 2]),
    dict(axis_dims=[64], theta=0.0), dict(axis_dims=[64], theta=math.nan), dict(axis_dims=[64], scaling="linear", factor=0.5),
    dict(axis_dims=[64], scaling="yarn", factor=2.0), dict(axis_dims=[64], scaling="yarn", factor=2.0, original_length=10, beta_fast=0.5),
    dict(axis_dims=[64], scaling="ntk", factor=math.inf),
])
def test_rope_plan_refusals(kw):
    with pytest.raises(s2b.S2BError) as e:
        s2b.rope_plan(**kw)
    assert e.value.code == 1 and "rope plan" in str(e.value)


def test_rope_plan_python_refusals():
    for kw in (dict(axis_dims=[]), dict(axis_dims=[2] * 4), dict(axis_dims=[64], layout="x"), dict(axis_dims=[64], scaling="x")):
        with pytest.raises(ValueError):
            s2b.rope_plan(**kw)


def packed(op, *words):
    import struct
    return s2b.lib().s2b_op_packed(struct.pack("@24q", *([op, 0, 0] + [w or 0 for w in words] + [0] * (21 - len(words)))))


def test_packed_calls_are_checked_like_the_others():
    plan = s2b.rope_plan([64])
    at = ctypes.addressof(plan)
    refused(packed(0, X, 3, 4, 256, 256, 1, Q, 256, S), "x_type")
    refused(packed(0, X, BF16, 4, 256, 256, 1, Q, 256, S), "null context")
    refused(packed(1, X, 256, S, 4, 0, W, 256, V, 64, 0, Y, BF16, 64), "K must be positive")
    refused(packed(1, X, 256, S, 4, 256, W, 256, V, 64, 0, Y, BF16, 64), "null context")
    refused(packed(2, at, X, BF16, 2, 3, 4, 62, 1536, 512, 128, 0, 0, 0, Y, 1536, 512, 128, 0), "more than head_dim")
    refused(packed(2, at, X, BF16, 2, 3, 4, 128, 1536, 512, 128, 0, 0, 0, Y, 1536, 512, 128, 0), "null context")
    eps = np.array([1e-6]).view(np.int64)[0]
    refused(packed(3, X, BF16, 2, 10, 64, 64, 7, S, V, eps, 1, Y, BF16, 64, B, 1 << 19), "multiple of groups")
    refused(packed(3, X, BF16, 2, 10, 64, 64, 8, S, V, eps, 1, Y, BF16, 64, B, 1 << 19), "null context")
    refused(packed(4), "unknown operator")
    refused(s2b.lib().s2b_op_packed(None), "null argument")
    for bad in (1 << 31, -(1 << 31) - 1, 1 << 40):
        refused(packed(0, X, BF16, bad, 256, 256, 1, Q, 256, S), "out of range")
        refused(packed(1, X, 256, S, 4, 256, W, 256, V, bad, 0, Y, BF16, 64), "out of range")
        refused(packed(2, at, X, BF16, 2, bad, 4, 128, 1536, 512, 128, 0, 0, 0, Y, 1536, 512, 128, 0), "out of range")
        refused(packed(3, X, BF16, 2, bad, 64, 64, 8, S, V, eps, 1, Y, BF16, 64, B, 1 << 19), "out of range")


def test_sizes_past_the_limits_are_refused():
    """Sizes whose tile counts or offsets would leave their integers."""
    big, far = 2 ** 31 - 1, 1 << 40
    refused(linear(M=big), "2^30")
    refused(linear(N=big, ldy=big), "2^30")
    refused(linear(K=big, ldx=big - 15, ldw=big - 15), "2^30")
    refused(linear(M=big, N=0), "2^30")
    refused(rope(dim=big), "2^30")
    # 2^40 values a step is a stride, 2^30 such steps wrap a 64-bit offset
    refused(rope(tokens=2 ** 30, ys=(1536, far, 128)), "reaches over")
    refused(rope(tokens=2 ** 30, xs=(1536, far, 128)), "reaches over")
    refused(rope(batch=big, xs=(1 << 33, 512, 128), ys=(1 << 33, 512, 128)), "reaches over")
    refused(rope(batch=3, pos=Q, pbs=far), "positions reach")
    refused(rope(batch=1, pos=Q, pbs=far, xs=(far, 512, 128), ys=(far, 512, 128)), "null context")    # no step is taken
    refused(norm(C=1 << 24, ldx=1 << 24, ldy=1 << 24), "2^23 channels")
    refused(norm(rows=big), "2^30 rows")
    for sizes in ((1, big, 64, 8), (65536, 1, 64, 8), (1, 1, big, 1)):
        with pytest.raises(s2b.S2BError) as e:
            s2b.groupnorm_workspace(*sizes)
        assert "more than" in str(e.value)


def test_pair_linear_orders_what_crosses_between_its_ctas():
    """What one CTA of a pair hands to the other, besides TMA and MMA completions: TMEM that it has read or written, as a
    cluster-scope signal between the fences that order TMEM accesses; a verdict's words, as asynchronous stores that carry
    their own signal; and, ahead of the next such store, that the verdict's readers are done, as a cluster-scope release.
    Read from the source: no run shows a missing order."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(s2b.__file__))), "csrc")
    text = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, "k_fp8_linear.cu")).read())
    text = text[text.index("k_fp8_linear_pair("):]
    assert "st_cluster" not in text
    remote = re.findall(r"(mbar_arrive_cluster\w*)\(([^;]*)\);", text)
    relaxed = [a for f, a in remote if f == "mbar_arrive_cluster_relaxed"]
    release = [a for f, a in remote if f == "mbar_arrive_cluster"]
    assert len(remote) == len(relaxed) + len(release) == 4
    assert all("sfull" in a or "tempty" in a for a in relaxed) and all("mgone" in a for a in release), remote
    for m in re.finditer(r"mbar_arrive_cluster_relaxed", text):
        assert "tc_fence_before()" in text[m.start() - 200: m.start()]
    cluster_waits = {"wait_cluster", "wait_flag_idle<true>", "mbar_try_wait_cluster"}
    for bar in ("sfull", "tempty", "mfull", "mgone"):
        used = set(re.findall(r"([\w<>]+)\(&ctl->%s\[" % bar, text)) - {"mbar_init", "map_to_rank", "mbar_arrive", "mbar_arrive_expect_tx"}
        assert used and used <= cluster_waits, (bar, used)
    # the stores: after the wait for both CTAs' readers
    post = text[text.index("wait_flag_idle<true>(&ctl->mgone"):]
    assert post.index("st_async_u32") < 700 and text.count("st_async_u32") == 1
    assert "map_to_rank(&ctl->mempty" not in text
    arrive = re.search(r"mbar_arrive_cluster_relaxed\(.*?\n}", open(os.path.join(csrc, "sm100.cuh")).read(), re.S).group(0)
    assert "mbarrier.arrive.relaxed.cluster.shared::cluster" in arrive


def test_python_calls_check_what_they_pack():
    """The short calls pack their arguments themselves: None is the default stream as in the other methods, strides are
    three, and a plan is one that rope_plan made."""
    c = s2b.DitB200.__new__(s2b.DitB200)
    c._ctx, c._h, c._op = ctypes.c_void_p(), 0, s2b.lib().s2b_op_packed
    plan, st = s2b.rope_plan([64]), (1536, 512, 128)
    calls = [lambda s: c.fp8_quant_dev(X, BF16, 4, 256, 256, 1, Q, 256, S, s),
             lambda s: c.linear_fp8_dev(X, 256, S, 4, 256, W, 256, V, 64, None, Y, BF16, 64, s),
             lambda s: c.rope_dev(plan, X, BF16, 2, 3, 4, 128, st, None, 0, 0, Y, st, False, s),
             lambda s: c.groupnorm_dev(X, BF16, 2, 10, 64, 64, 8, S, V, 1e-6, 1, Y, BF16, 64, B, 1 << 19, s)]
    for call in calls:
        for s in (0, None):
            with pytest.raises(s2b.S2BError, match="null context"):
                call(s)
    for xs, ys in ((st[:2], st), (st, st + (1,)), (st + (1,), st[:2]), ((), st * 2)):
        with pytest.raises(ValueError, match="strides"):
            c.rope_dev(plan, X, BF16, 2, 3, 4, 128, xs, None, 0, 0, Y, ys, False, 0)
    for p in (None, s2b.s2b_rope_config(), ctypes.c_int(0)):
        with pytest.raises(TypeError, match="rope_plan"):
            c.rope_dev(p, X, BF16, 2, 3, 4, 128, st, None, 0, 0, Y, st, False, 0)
