"""residual_norm_out: h = x + scale * act(gate) * Post(y), out = Pre(h).

The refusals need no GPU.  The results are compared with the formulas in 64
bits, to bounds that follow from the arithmetic (bounds(), below): everything
is fp32 until one rounding to the element type.
"""
import ctypes

import pytest
import torch

import gpipes

F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24  # half a step of fp32
C = 64 * U      # a sum of up to 32 values a thread, then over lanes and waves: fewer than 64 roundings a value


# ---------------------------------------------------------------------------
# Refusals, through the C ABI with pointers that are never dereferenced
# ---------------------------------------------------------------------------

def _call(M=16, D=128, x=16, y=16, post=2, pg=16, pb=0, peps=1e-5, gate=0, rows=0, gact=0, scale=1.0, pre=2, g=16, b=0,
          eps=1e-5, h=32, out=48, dtype=0):
    vp = ctypes.c_void_p
    P = lambda v: vp(v) if v else None  # noqa: E731
    return gpipes.lib.gp_residual_norm_out(M, D, P(x), P(y), post, P(pg), P(pb), peps, P(gate), rows, gact, scale, pre,
                                           P(g), P(b), eps, P(h), P(out), dtype, None)


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(M=1 << 41), -2), (dict(D=0), -2), (dict(D=-4), -2), (dict(D=32769), -2), (dict(dtype=2), -1),
    (dict(post=3), -1), (dict(pre=-1), -1), (dict(post=0), -1), (dict(post=0, pg=0, pb=16), -1), (dict(pre=0, out=0), -1),
    (dict(peps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1), (dict(scale=float("inf")), -1),
    (dict(scale=float("nan")), -1), (dict(gate=16, rows=0), -2), (dict(gate=16, rows=3), -2), (dict(gate=16, rows=32), -2),
    (dict(gate=16, rows=-16), -2), (dict(gate=16, rows=16, gact=5), -1), (dict(x=0), -1), (dict(y=0), -1),
    (dict(y=0, post=0, pg=0, gate=16, rows=1), -1), (dict(out=0), -1), (dict(pre=0, g=0), -1),
    (dict(pre=0, g=0, out=0, h=0), -1), (dict(h=48), -1), (dict(x=17), -3), (dict(out=49), -3), (dict(b=3), -3),
])
def test_argument_errors(kw, code):
    assert _call(**kw) == code
    assert gpipes.lib.gp_last_error().decode() != ""


@pytest.mark.parametrize("kw", [
    dict(h=(1 << 20) + 2), dict(out=(1 << 20) - 4094), dict(h=(1 << 21) + 4094), dict(out=(1 << 21) + 256),
    dict(h=1 << 24, out=(1 << 24) + 4094), dict(gate=1 << 24, rows=1, h=1 << 24), dict(gate=1 << 24, rows=8, out=1 << 24),
    dict(gate=(1 << 24) + 4094, rows=1, out=1 << 24), dict(gate=1 << 24, rows=16, h=(1 << 24) + 256),
    dict(pg=(1 << 22) + 4094), dict(g=(1 << 23) - 254), dict(pb=1 << 23), dict(b=(1 << 22) + 256),
])
def test_overlaps_are_refused(kw):
    a = dict(x=1 << 20, y=1 << 21, h=1 << 22, out=1 << 23, pg=0, g=0)  # 16 rows of 128: 4,096 bytes
    assert _call(**{**a, **kw}) == -1
    assert "overlap" in gpipes.lib.gp_last_error().decode()


def test_empty_batch_is_a_noop():
    assert _call(M=0, x=0, y=0, h=0, out=0) == 0
    assert _call(M=0, gate=16, rows=0) == 0
    assert gpipes.lib.gp_last_error().decode() == ""


def test_other_calls_still_refuse_silu():
    vp = ctypes.c_void_p
    assert gpipes.lib.gp_linear_out(16, 128, vp(16), vp(16), None, None, 4, vp(16), None) == -1
    assert gpipes.lib.gp_gemm_out(16, 128, 64, vp(16), vp(16), None, None, 4, vp(16), None) == -1


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 128, dtype=F16)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.residual_norm_out(x)
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        gpipes.residual_norm(None)


# ---------------------------------------------------------------------------
# The formulas in 64 bits, and how far fp32 arithmetic may be from them
# ---------------------------------------------------------------------------

def act64(v, act):
    sig = torch.sigmoid(v)
    return {"none": v, "relu": torch.where(v > 0, v, 0 * v), "sigmoid": sig, "silu": v * sig,
            "gelu_tanh": v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))}[act]


def norm64(v, dv, kind, gamma, beta, eps):
    """The norm of v [M, D] and a bound on the kernel's distance from it, dv [M, 1] bounding that of its input.

    With u = (v - m) r: m is off by at most max dv + C max|v|; d = v - m by dd = 2 dv + C max|v|; the variance, a
    mean of d^2, by 2 dd mean|d| + C var, so r by r (dd r + C / 2) as mean|d| <= 1 / r; u by r dd (1 + |u|) + C |u|."""
    if kind == "none":
        return v, dv + 0 * v
    m = v.mean(1, keepdim=True) if kind == "layer" else 0 * v[:, :1]
    r = 1 / torch.sqrt(((v - m) ** 2).mean(1, keepdim=True) + eps)
    u = (v - m) * r
    dd = 2 * dv + C * v.abs().amax(1, keepdim=True)
    du = r * dd * (1 + u.abs()) + C * u.abs()
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    w = u * g + b
    return w, du * (g.abs() if gamma is not None else 1.0) + 4 * U * ((u * g).abs() + w.abs())


def ref(a):
    """(h, its bound), (out, its bound), without the last roundings."""
    d = lambda t: None if t is None else t.double().cpu()  # noqa: E731
    x = d(a["x"])
    h, dh = x, 0 * x
    if a["y"] is not None:
        y = d(a["y"])
        v, dv = norm64(y, 0 * y[:, :1], a["post"], d(a["post_gamma"]), d(a["post_beta"]), a["post_eps"])
        if a["gate"] is not None:
            gate = d(a["gate"])
            gate = gate[None] if gate.dim() == 1 else gate
            g = act64(gate, a["gate_act"]).repeat_interleave(x.shape[0] // gate.shape[0], 0)
            # e^z from a power of two whose exponent is off by |z| 2^-23, the reciprocal and products by a few steps
            z = gate.abs().amax() * 4 + 4
            dv = dv * g.abs() + (z * 2.0 ** -22 if a["gate_act"] != "none" else 0) * (v * g).abs() + 4 * U * (v * g).abs()
            v = v * g
        s = float(torch.tensor(a["scale"], dtype=torch.float32))
        h = x + s * v
        dh = abs(s) * dv + 4 * U * ((s * v).abs() + x.abs())
    o, do = norm64(h, dh.amax(1, keepdim=True), a["norm"], d(a["gamma"]), d(a["beta"]), a["eps"])
    return (h, dh), (o, do)


def check(got, want, bound, dt):
    """Off by the bound and half a step of dt (at fp16's smallest values half of 2^-24)."""
    got, eps = got.double().cpu(), torch.finfo(dt).eps
    tol = bound + (want.abs() + bound) * eps / 2 + (2.0 ** -25 if dt == F16 else 0)
    over = ((got - want).abs() / tol.clamp(min=1e-300))
    assert torch.isfinite(got).all()
    assert over.max() <= 1, (over.max().item(), int(over.argmax()))


def make(M, D, dt, dev, post="rms", norm="rms", gate=None, gate_act="none", scale=1.0, gamma=True, beta=True, y=True,
         seed=0, post_eps=1e-6, eps=1e-5):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, m=0.0, k=1.0: (torch.randn(*s, generator=g) * k + m).to(dt).to(dev)  # noqa: E731
    a = dict(x=n(M, D, k=2), y=n(M, D, m=0.3) if y else None, post=post, norm=norm, gate_act=gate_act, scale=scale,
             post_eps=post_eps, eps=eps)
    a["gate"] = None if gate is None else n(D) if gate == 0 else n(gate, D)
    for side, kind in (("post_", post), ("", norm)):
        a[side + "gamma"] = n(D, m=1, k=0.3) if gamma and kind != "none" else None
        a[side + "beta"] = n(D, k=0.3) if beta and kind != "none" else None
    return a


def run_and_check(a, **kw):
    x = a["x"]
    dt = x.dtype
    (h64, dh), (o64, do) = ref(a)
    h, out = gpipes.residual_norm_out(**a, h=torch.empty_like(x), **kw)
    check(h, h64, dh, dt)
    if a["norm"] == "none":
        assert out is None
    else:
        check(out, o64, do, dt)
    return h, out


SIZES = [(1, 1), (1, 7), (3, 8), (5, 64), (2, 1021), (130, 128), (7, 4096), (1, 8192), (3, 8200), (2, 32768), (301, 513),
         (5000, 96), (9, 2047), (2600, 1024), (700, 5000)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,D", SIZES)
@pytest.mark.parametrize("dt", [F16, BF16])
def test_sizes(cuda, M, D, dt):
    print(M, D, dt, flush=True)
    run_and_check(make(M, D, dt, cuda, seed=M + D))
    run_and_check(make(M, D, dt, cuda, post="layer", norm="layer", gate=1, gate_act="sigmoid", scale=0.5, seed=M * D))


@pytest.mark.gpu
@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("norm", ["none", "layer", "rms"])
@pytest.mark.parametrize("gate", [None, 0, 1, 6, 24])
def test_kinds(cuda, post, norm, gate):
    for D, act in ((200, "silu"), (257, "gelu_tanh"), (1544, "relu"), (4104, "none")):
        run_and_check(make(24, D, BF16, cuda, post=post, norm=norm, gate=gate, gate_act=act, scale=-1.25, seed=D,
                           gamma=D != 257, beta=D != 1544))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["none", "layer", "rms"])
def test_without_y(cuda, norm):
    for M, D in ((1, 4096), (33, 130)):
        a = make(M, D, F16, cuda, post="none", norm=norm, y=False, seed=D)
        h, _ = run_and_check(a)
        assert torch.equal(h, a["x"])


@pytest.mark.gpu
def test_out_alone_equals_both(cuda):
    a = make(37, 1032, F16, cuda, seed=3)
    h, out = run_and_check(a)
    none, alone = gpipes.residual_norm_out(**a)
    assert none is None and torch.equal(alone, out)
    h2, out2 = gpipes.residual_norm(**a)
    assert torch.equal(h2, h) and torch.equal(out2, out)


@pytest.mark.gpu
@pytest.mark.parametrize("M,D", [(3, 77), (40, 1024), (2, 9000)])
def test_unaligned_rows_and_what_lies_around_them(cuda, M, D):
    """Tensors that start one element into their memory; nothing outside h and out is written."""
    for dt in (F16, BF16):
        a = make(M, D, dt, cuda, post="layer", norm="rms", gate=M, gate_act="silu", seed=D)
        want = run_and_check(a)

        def shifted(t):
            buf = torch.full((t.numel() + 64,), 7.0, dtype=dt, device=cuda)
            buf[1:1 + t.numel()] = t.reshape(-1)
            return buf, buf[1:1 + t.numel()].view(t.shape)

        b = {k: shifted(v)[1] if isinstance(v, torch.Tensor) else v for k, v in a.items()}
        (hb, h), (ob, o) = shifted(torch.zeros_like(a["x"])), shifted(torch.zeros_like(a["x"]))
        gpipes.residual_norm_out(**b, h=h, out=o)
        assert torch.equal(h, want[0]) and torch.equal(o, want[1])
        for buf in (hb, ob):
            assert (buf[:1] == 7).all() and (buf[1 + M * D:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,D", [(1, 4096), (50, 1021), (3, 20000)])
def test_in_place(cuda, M, D):
    a = make(M, D, BF16, cuda, post="rms", norm="layer", gate=M, gate_act="sigmoid", seed=9)
    want = run_and_check(a)
    for hn, on in (("x", "y"), ("y", "x"), ("gate", "x"), ("x", "gate")):
        b = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
        gpipes.residual_norm_out(**b, h=b[hn], out=b[on])
        assert torch.equal(b[hn], want[0]) and torch.equal(b[on], want[1])


@pytest.mark.gpu
def test_constant_and_large_rows(cuda):
    """A row of equal values has no variance, and eps decides; a mean far from zero costs no more than the bound says;
    eps 0 with a row of zeros divides by zero, in that row alone."""
    for norm in ("layer", "rms"):
        a = make(6, 1000, F16, cuda, post=norm, norm=norm, seed=4)
        a["y"][0], a["y"][1], a["y"][2] = 3.0, 0.0, a["y"][2] + 300
        a["x"][3], a["y"][3] = 0.0, 0.0
        run_and_check(a)
        b = make(3, 512, F16, cuda, post="none", norm=norm, y=False, beta=False, eps=0.0, seed=5)
        b["x"][1] = 0.0
        _, out = gpipes.residual_norm_out(**b)
        (_, _), (want, bound) = ref(b)
        assert torch.isnan(out[1]).all()
        for r in (0, 2):
            check(out[r:r + 1], want[r:r + 1], bound[r:r + 1], F16)


@pytest.mark.gpu
def test_infinities_and_nans_stay_in_their_rows(cuda):
    for M, D in ((64, 384), (5, 4097)):
        a = make(M, D, BF16, cuda, post="rms", norm="layer", gate=1, seed=6)
        (h64, dh), (o64, do) = ref(a)
        a["y"][1, 5], a["x"][2, 300], a["y"][4, D - 1] = float("inf"), float("nan"), float("-inf")
        h, out = gpipes.residual_norm_out(**a, h=torch.empty_like(a["x"]))
        for r in range(M):
            if r in (1, 2, 4):
                assert torch.isnan(out[r]).all()
            else:
                check(h[r:r + 1], h64[r:r + 1], dh[r:r + 1], BF16)
                check(out[r:r + 1], o64[r:r + 1], do[r:r + 1], BF16)


@pytest.mark.gpu
def test_many_rows_twice_the_same(cuda):
    """More rows than one round of workgroups, a row a gate; two calls give the same bits."""
    M, D = 40001, 72
    a = make(M, D, F16, cuda, post="layer", norm="rms", gate=M, gate_act="sigmoid", seed=8)
    h, out = run_and_check(a)
    h2, out2 = gpipes.residual_norm(**a)
    assert torch.equal(h, h2) and torch.equal(out, out2)


@pytest.mark.gpu
def test_graph_and_side_stream(cuda):
    a = make(19, 2048, BF16, cuda, seed=10)
    h, out = torch.empty_like(a["x"]), torch.empty_like(a["x"])
    gpipes.residual_norm_out(**a, h=h, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gpipes.residual_norm_out(**a, h=h, out=out)
        gpipes.residual_norm_out(h, out, norm="none", post="none", scale=0.5, h=h)
    side = torch.cuda.Stream(cuda)
    for r in range(3):
        a["x"].copy_(make(19, 2048, BF16, cuda, seed=20 + r)["x"])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            w, o = gpipes.residual_norm(**a)
            w2, _ = gpipes.residual_norm_out(w, o, norm="none", scale=0.5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, w2) and torch.equal(out, o)


@pytest.mark.gpu
def test_python_refusals(cuda):
    a = make(8, 64, F16, cuda)
    x = a["x"]
    with pytest.raises(RuntimeError, match="contiguous"):
        gpipes.residual_norm_out(torch.zeros(64, 8, dtype=F16, device=cuda).t())
    with pytest.raises(RuntimeError, match="shape"):
        gpipes.residual_norm_out(x, a["y"][:4])
    with pytest.raises(RuntimeError, match="gate"):
        gpipes.residual_norm_out(x, a["y"], gate=torch.zeros(8, 32, dtype=F16, device=cuda))
    with pytest.raises(RuntimeError, match="divisor"):
        gpipes.residual_norm_out(x, a["y"], gate=torch.zeros(3, 64, dtype=F16, device=cuda))
    with pytest.raises(RuntimeError, match="bfloat16|float16"):
        gpipes.residual_norm_out(x, a["y"].to(BF16))
    with pytest.raises(RuntimeError, match="2-D"):
        gpipes.residual_norm_out(x[0])
    e = x[:0]
    h, out = gpipes.residual_norm(e, e, gate=e)
    assert h.shape == out.shape == (0, 64)


@pytest.mark.gpu
def test_more_values_than_32_bits_count(cuda):
    """2^31 values and more: rows on both sides of that offset, and the last."""
    M, D = (1 << 31) // 4093 + 700, 4093
    a = make(256, D, BF16, cuda, post="rms", norm="layer", scale=0.5, seed=4)
    x, y = (a[k].repeat(M // 256 + 1, 1)[:M] for k in ("x", "y"))
    h, out = gpipes.residual_norm_out(**{**a, "x": x, "y": y}, h=torch.empty_like(x))
    for i in (0, (1 << 31) // D - 8, (1 << 31) // D, M - 8):
        rows = slice(i, i + 8)
        (h64, dh), (o64, do) = ref({**a, "x": x[rows], "y": y[rows]})
        check(h[rows], h64, dh, BF16)
        check(out[rows], o64, do, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(norm="foo"), dict(post="foo"), dict(gate_act="foo"), dict(scale="1"), dict(eps=None),
                                dict(post_eps="x"), dict(norm=7), dict(gate_act=-1)])
def test_unknown_names_and_no_numbers_raise_runtime_errors(cuda, kw):
    x = torch.zeros(2, 64, dtype=F16, device=cuda)
    with pytest.raises(RuntimeError):
        gpipes.residual_norm_out(x, x, gate=x, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("M,gated", [((1 << 28) + 5, False), ((1 << 28) + 6, True), ((1 << 31) + 9, False)])
def test_more_rows_than_a_launch_has_threads(cuda, M, gated):
    """2^28 rows of one value and more, sixteen a workgroup of 256, are 2^32 threads: every row all the same."""
    x = torch.randn(1 << 20, dtype=F16, device=cuda).repeat((M >> 20) + 1)[:M].view(M, 1)
    gate = torch.tensor([[0.5], [2.0]], dtype=F16, device=cuda) if gated else None
    h = torch.full((M + 64,), 7.0, dtype=F16, device=cuda)
    gpipes.residual_norm_out(x, x, gate=gate, scale=0.5, norm="none", h=h[:M].view(M, 1))
    # h = 1.5 x, or with the gate 1.25 x in the first half and 2 x in the second: fp32 holds all, so one rounding
    for at in range(0, M, 1 << 28):
        v, n = x[at:at + (1 << 28), 0], min(1 << 28, M - at)
        k = 1.5 if not gated else torch.where(torch.arange(at, at + n, device=cuda) < M // 2, 1.25, 2.0)
        assert torch.equal(h[at:at + n], (v.float() * k).half())
    assert (h[M:] == 7).all()
