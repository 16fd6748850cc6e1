"""Products with 4-bit weights: q4_gemm_out and q4_gated_out, and gpipes.q4, which makes such weights.

The refusals and gpipes.q4 need no GPU.  Results are compared with the formulas in 64 bits, to a
bound from the arithmetic (product(), below), and as a whole: the error's norm may hardly be
larger than that of the exact result rounded to the element type.
"""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import gpipes
from gpipes import q4

F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24


# ---------------------------------------------------------------------------
# Without a GPU
# ---------------------------------------------------------------------------

def _call(M=4, N=256, K=512, group=128, x=16, wq=16, s=16, z=0, b=0, r=0, act=0, out=32, dtype=0, two=False, u=16,
          ws=0, wsb=0):
    vp = ctypes.c_void_p
    P = lambda v: vp(v) if v else None  # noqa: E731
    if two:
        return gpipes.lib.gp_q4_gated_out(M, N, K, group, P(x), P(wq), P(s), P(z), P(b), P(u), P(s), P(z), P(b), act,
                                          P(out), P(ws), wsb, dtype, None)
    return gpipes.lib.gp_q4_gemm_out(M, N, K, group, P(x), P(wq), P(s), P(z), P(b), P(r), act, P(out), P(ws), wsb, dtype,
                                     None)


@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(M=(1 << 21) + 1), -2), (dict(N=0), -2), (dict(N=(1 << 20) + 1), -2), (dict(K=0), -2),
    (dict(K=12), -2), (dict(K=65544), -2), (dict(K=65536, N=65536), -2), (dict(group=16), -2), (dict(group=256), -2),
    (dict(group=0), -2), (dict(dtype=2), -1), (dict(act=5), -1), (dict(act=-1), -1), (dict(x=0), -1), (dict(wq=0), -1),
    (dict(s=0), -1), (dict(out=0), -1), (dict(x=24), -3), (dict(wq=20), -3), (dict(s=18), -3), (dict(z=8), -3),
    (dict(b=2), -3), (dict(out=40), -3), (dict(wsb=-1), -1), (dict(wsb=64), -1), (dict(ws=24, wsb=64), -3),
])
def test_argument_errors(kw, code, two):
    assert _call(**kw, two=two) == code
    assert gpipes.lib.gp_last_error().decode() != ""


def test_argument_errors_of_one_form():
    assert _call(r=16, act=1) == -1
    assert _call(r=8) == -3
    assert _call(u=0, two=True) == -1
    assert _call(u=24, two=True) == -3


@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("kw", [
    dict(out=1 << 20), dict(out=(1 << 20) + 4080), dict(out=(1 << 20) - 2032), dict(ws=(1 << 20) - 64, wsb=80),
    dict(ws=(1 << 21) + 2032, wsb=64),
])
def test_overlaps_are_refused(kw, two):
    a = dict(x=1 << 20, out=1 << 21)  # x 4 x 512, out 4 x 256: 4,096 and 2,048 bytes
    assert _call(**{**a, **kw}, two=two) == -1
    assert "overlap" in gpipes.lib.gp_last_error().decode()


def test_a_residual_that_overlaps_is_refused():
    assert _call(x=1 << 20, out=1 << 21, r=(1 << 21) + 16) == -1
    assert _call(x=1 << 20, out=1 << 21, r=1 << 22, ws=(1 << 22) + 2032, wsb=16) == -1


@pytest.mark.parametrize("what,size,two", [
    (what, size, two) for what, size in (("wq", 512 * 256 // 2), ("s", 4 * 256 * 2), ("z", 4 * 256 * 2), ("b", 256 * 2),
                                         ("u", 512 * 256 // 2)) for two in (False, True) if two or what != "u"])
def test_overlaps_with_the_weight_are_refused(what, size, two):
    """out and the workspace over the first or the last 16 bytes of a weight's tensors."""
    at = 1 << 24
    far = dict(x=1 << 20, out=1 << 21, wq=1 << 22, s=1 << 23, z=5 << 21, b=11 << 20, u=13 << 20)
    for lo, n in ((at - 2048 + 16, 2048), (at + size - 16, 2048)):  # out's 4 x 256 values
        assert _call(**{**far, what: at, "out": lo}, two=two) == -1
        assert "out must not overlap" in gpipes.lib.gp_last_error().decode()
        assert _call(**{**far, what: at}, ws=lo, wsb=n, two=two) == -1
        assert "workspace must not overlap" in gpipes.lib.gp_last_error().decode()


def test_empty_batch_is_a_noop():
    assert _call(M=0, x=0, out=0) == 0
    assert _call(M=0, x=0, out=0, two=True) == 0
    assert gpipes.lib.gp_last_error().decode() == ""


@pytest.mark.parametrize("args,code", [((-1, 64, 64, 32, 1), -1), ((64, 0, 64, 32, 1), -2), ((64, 64, 60, 32, 1), -2),
                                       ((64, 64, 64, 33, 1), -2), ((64, 64, 64, 32, 3), -1), ((64, 64, 64, 32, 0), -1),
                                       ((0, 64, 64, 32, 1), 0)])
def test_workspace_arguments(args, code):
    assert gpipes.lib.gp_q4_workspace_bytes(*args) == code


def test_python_refuses():
    x, wq, s = torch.zeros(1, 64, dtype=F16), torch.zeros(8, 32, dtype=torch.int32), torch.zeros(1, 32, dtype=F16)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.q4_gemm_out(x, wq, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.q4_gated_out(x, wq, s, None, wq, s, None)


@pytest.mark.parametrize("group", [0, 16, 256, -32, 1.5, None, "128"])
def test_python_refuses_groups(group):
    x, wq, s = torch.zeros(1, 64, dtype=F16), torch.zeros(8, 32, dtype=torch.int32), torch.zeros(1, 32, dtype=F16)
    with pytest.raises(RuntimeError):
        gpipes.q4_gemm_out(x, wq, s, group=group)
    with pytest.raises(RuntimeError):
        gpipes.q4_gated_out(x, wq, s, None, wq, s, None, group=group)


def test_the_package_has_the_weights_module():
    """As it is named in the documents: gpipes.q4 after `import gpipes` alone."""
    code = "import gpipes; assert gpipes.q4.pack and 'q4' in gpipes.__all__"
    path = os.path.dirname(os.path.dirname(gpipes.__file__))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=path, timeout=120)


def test_pack_and_unpack():
    g = torch.Generator().manual_seed(0)
    q = torch.randint(0, 16, (40, 13), generator=g)
    wq = q4.pack(q)
    assert wq.dtype == torch.int32 and wq.shape == (5, 13)
    assert torch.equal(q4.unpack(wq).long(), q)
    assert (int(wq[2, 3]) & 15, (int(wq[2, 3]) >> 28) & 15) == (int(q[16, 3]), int(q[23, 3]))
    for bad in (q[:7], q - 1, q + 1):
        with pytest.raises(RuntimeError):
            q4.pack(bad)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_quantize(group, zeros, dt):
    """Off by half a step, and by what rounding the step to dt moves the ends by: seven or fifteen steps of a step that
    is off by half of dt's eps; and a whole zero moves an end by up to half a step."""
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(200, 17, generator=g) * 0.05 + 0.02).to(dt)
    w[:, 3], w[:, 4], w[:, 5] = 0, 0.75, -0.5
    wq, s, z = q4.quantize(w, group, zeros)
    assert s.shape == (-(-200 // group), 17) and (z is None) == (not zeros)
    step = s.double().repeat_interleave(group, 0)[:200]
    got = q4.dequantize(wq, s, z, group).double()
    assert ((got - w.double()).abs() <= step * (1.0 if zeros else 0.5) + step * 16 * torch.finfo(dt).eps).all()
    assert (got[:, 3] == 0).all()


@pytest.mark.parametrize("dt", [torch.uint8, torch.int64, torch.float32])
def test_pack_takes_any_strides(dt):
    q = torch.randint(0, 16, (13, 40), generator=torch.Generator().manual_seed(0)).to(dt).t()
    wq = q4.pack(q)
    assert wq.is_contiguous() and torch.equal(wq, q4.pack(q.contiguous())) and torch.equal(q4.unpack(wq).to(dt), q)


@pytest.mark.parametrize("v", [3.7, -0.5, 15.5, 1e-3, float("nan"), float("inf")])
def test_pack_refuses_what_is_no_whole_number(v):
    q = torch.full((8, 3), 7.0)
    assert torch.equal(q4.unpack(q4.pack(q)).float(), q)  # whole numbers of any type
    q[5, 1] = v
    with pytest.raises(RuntimeError, match="whole numbers"):
        q4.pack(q)


def test_quantize_refuses():
    w = torch.ones(16, 4, dtype=F16)
    for bad, kw in ((w[:9], {}), (w.float(), {}), (w, dict(group=16)), (w * float("inf"), {})):
        with pytest.raises(RuntimeError):
            q4.quantize(bad, **kw)


# ---------------------------------------------------------------------------
# The formulas in 64 bits
# ---------------------------------------------------------------------------

def act64(v, act):
    return {"none": v, "relu": v.clamp(min=0), "sigmoid": torch.sigmoid(v), "silu": v * torch.sigmoid(v),
            "gelu_tanh": v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))}[act]


def weight(K, N, group, zeros, dt, gen):
    q = torch.randint(0, 16, (K, N), generator=gen)
    groups = -(-K // group)
    s = ((0.3 + torch.rand(groups, N, generator=gen)) / (4.6 * K ** 0.5)).to(dt)
    z = (torch.randint(0, 31, (groups, N), generator=gen) / 2).to(dt) if zeros else None
    return q, s, z


def product(x, q, s, z, group):
    """x W, and a bound on the kernel's distance from it.  Products of x with B + q (B 64 in fp16, 128 in bf16) are
    exact; a group's sum of at most 128 of them, and that of x, which B + z multiplies, take sixteen roundings each
    at most (eight products a step), the running sum one a group and one a wave, under 100 for what the tests use.  Up to four rows may be taken in whole numbers
    instead, each value to 2^-19 of the largest of its 128: 2^-19 of that largest times |W| a product."""
    B = 64 if x.dtype == F16 else 128
    x, q, s = x.double(), q.double(), s.double()
    K = q.shape[0]
    zz = z.double() if z is not None else torch.full_like(s, 8)
    sr, zr = (t.repeat_interleave(group, 0)[:K] for t in (s, zz))
    out = x @ (sr * (q - zr))
    near = 16 * U * (x.abs() @ (sr * (2 * B + q + zr)))
    if x.shape[0] <= 4:
        for k in range(0, K, 128):
            top = x[:, k:k + 128].abs().amax(1, keepdim=True)
            near += 2.0 ** -19 * top * (sr * (q - zr)).abs()[k:k + 128].sum(0)
    run = torch.zeros_like(out)
    for k in range(0, K, group):
        run += (x[:, k:k + group] @ (sr * (q - zr))[k:k + group]).abs()
    return out, near + 100 * U * run


def moved(v, dv, act):
    """act(v), and the bound on from where v is off by dv: no activation here is steeper than 1.13."""
    a = act64(v, act)
    return a, 1.13 * dv + 2.0 ** -20 * a.abs() + 2.0 ** -22 * v.abs() * (act not in ("none", "relu"))


def check(got, want, bound, dt):
    got = got.double().cpu()
    half = torch.finfo(dt).eps / 2
    tol = bound + (want.abs() + bound) * half + (2.0 ** -25 if dt == F16 else 0)
    assert torch.isfinite(got).all()
    over = (got - want).abs() / tol.clamp(min=1e-300)
    assert over.max() <= 1, (over.max().item(), divmod(int(over.argmax()), got.shape[1]))
    if got.numel() >= 256:  # errors that are half a step at most, spread evenly: those of fp32 add little to them
        best = (want.to(dt).double() - want).norm()
        assert (got - want).norm() <= 1.1 * best, ((got - want).norm() / want.norm(), best / want.norm())


def dev(t, d):
    return None if t is None else t.to(d)


def run_gemm(M, K, N, group, zeros, dt, d, bias=False, residual=False, act="none", seed=0, x=None):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *sh: torch.randn(*sh, generator=gen).to(dt)  # noqa: E731
    x = n(M, K) if x is None else x
    q, s, z = weight(K, N, group, zeros, dt, gen)
    b, r = n(N) if bias else None, n(M, N) if residual else None
    v, dv = product(x, q, s, z, group)
    if bias:
        v, dv = v + b.double(), dv + 2 * U * (v.abs() + b.double().abs())
    v, dv = moved(v, dv, act)
    if residual:
        v, dv = v + r.double(), dv + 2 * U * (v.abs() + r.double().abs())
    # what lies behind the last row stays as it was
    buf = torch.full((M * N + 512,), 7.0, dtype=dt, device=d)
    out = buf[:M * N].view(M, N)
    got = gpipes.q4_gemm_out(dev(x, d), dev(q4.pack(q), d), dev(s, d), dev(z, d), dev(b, d), dev(r, d), act, group, out)
    check(got, v, dv, dt)
    assert (buf[M * N:] == 7).all()
    return got


def run_gated(M, K, N, group, zeros, dt, d, bias=False, act="silu", seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *sh: torch.randn(*sh, generator=gen).to(dt)  # noqa: E731
    x = n(M, K)
    sides, args, bs = [], [], []
    for _ in range(2):
        q, s, z = weight(K, N, group, zeros, dt, gen)
        b = n(N) if bias else None
        v, dv = product(x, q, s, z, group)
        if bias:
            v, dv = v + b.double(), dv + 2 * U * (v.abs() + b.double().abs())
        sides.append((v, dv))
        args += [dev(q4.pack(q), d), dev(s, d), dev(z, d)]
        bs.append(dev(b, d))
    g, dg = moved(*sides[0], act)
    u, du = sides[1]
    want, bound = g * u, dg * (u.abs() + du) + g.abs() * du + 2 * U * (g * u).abs()
    buf = torch.full((M * N + 512,), 7.0, dtype=dt, device=d)
    got = gpipes.q4_gated_out(dev(x, d), *args, bg=bs[0], bu=bs[1], act=act, group=group, out=buf[:M * N].view(M, N))
    check(got, want, bound, dt)
    assert (buf[M * N:] == 7).all()
    return got


ROWS = [1, 2, 3, 4, 5, 15, 16, 17, 31, 33, 48, 64, 65, 130, 255, 300]
SHAPES = [(8, 1), (24, 3), (32, 16), (64, 61), (96, 64), (128, 128), (136, 65), (1000, 257), (2048, 512), (520, 1021)]


@pytest.mark.gpu
@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_sizes(cuda, M, group):
    for i, (K, N) in enumerate(SHAPES):
        dt = (F16, BF16)[(i + M) % 2]
        print(M, K, N, group, dt, flush=True)
        run_gemm(M, K, N, group, i % 3 == 0, dt, cuda, bias=i % 2 == 0, residual=i % 4 == 1,
                 act="none" if i % 4 == 1 else ("none", "relu", "gelu_tanh", "sigmoid", "silu")[i % 5], seed=i + M)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 5, 20, 64, 200, 520])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_gated_sizes(cuda, M, dt):
    for i, (K, N) in enumerate(SHAPES):
        group = (32, 64, 128)[i % 3]
        print(M, K, N, group, dt, flush=True)
        run_gated(M, K, N, group, i % 2 == 0, dt, cuda, bias=i % 3 == 1,
                  act=("silu", "gelu_tanh", "none", "relu", "sigmoid")[i % 5], seed=i + M)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,group,zeros", [
    (1, 512, 8192, 64, True), (3, 256, 8209, 32, True), (2, 264, 16384, 128, False), (16, 128, 16411, 128, True),
    (40, 384, 9001, 64, False), (1, 16384, 96, 128, True), (7, 16376, 40, 32, False), (70, 4096, 130, 64, True),
    (1, 65536, 16, 128, False), (4, 16384, 50, 64, True), (4, 15000, 33, 32, False), (3, 65536, 20, 128, True), (129, 8200, 260, 32, True), (1024, 256, 2048, 128, False), (2100, 136, 300, 64, True)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_wide_and_deep(cuda, M, K, N, group, zeros, dt):
    run_gemm(M, K, N, group, zeros, dt, cuda, bias=True, seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 1024, 16390), (4, 2048, 4100), (30, 512, 8192), (513, 1024, 1088)])
def test_gated_wide(cuda, M, K, N):
    run_gated(M, K, N, 128, True, BF16, cuda, bias=True, seed=N)
    run_gated(M, K, N, 64, False, F16, cuda, act="gelu_tanh", seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 9, 40, 130])
def test_gated_with_zeros_on_one_side(cuda, M):
    gen = torch.Generator().manual_seed(M)
    x = torch.randn(M, 512, generator=gen).to(F16)
    (qg, sg, zg), (qu, su, _) = (weight(512, 192, 64, True, F16, gen) for _ in range(2))
    for a, b in ((zg, None), (None, zg)):
        g, dg = moved(*product(x, qg, sg, a, 64), "silu")
        u, du = product(x, qu, su, b, 64)
        got = gpipes.q4_gated_out(x.to(cuda), q4.pack(qg).to(cuda), sg.to(cuda), dev(a, cuda), q4.pack(qu).to(cuda),
                                  su.to(cuda), dev(b, cuda), group=64)
        check(got, g * u, dg * (u.abs() + du) + g.abs() * du + 2 * U * (g * u).abs(), F16)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 17, 64, 150, 300])
def test_large_and_small_values_of_x(cuda, M):
    """Rows far apart in size, zeros among them, and fp16's largest and smallest values."""
    gen = torch.Generator().manual_seed(M)
    for dt in (F16, BF16):
        x = torch.randn(M, 640, generator=gen)
        x *= 10.0 ** torch.randint(-3, 4, (M, 1), generator=gen)
        x[M // 2, ::2] = 0
        x = x.to(dt)
        if M > 1:
            x[0] = 0
        run_gemm(M, 640, 144, 64, True, dt, cuda, seed=M, x=x / 64)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 16, 64, 200])
def test_outlying_channels(cuda, M):
    """A few channels a thousand times as large as the others, as activations have them."""
    gen = torch.Generator().manual_seed(M)
    x = torch.randn(M, 1024, generator=gen)
    x[:, [3, 500, 1000]] *= 1000
    for dt in (F16, BF16):
        run_gemm(M, 1024, 256, 128, True, dt, cuda, seed=M, x=x.to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 5, 40, 100, 300])
def test_infinities_and_nans_stay_in_their_rows(cuda, M):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(M, 512, generator=gen).to(BF16)
    q, s, z = weight(512, 200, 64, True, BF16, gen)
    args = [dev(t, cuda) for t in (q4.pack(q), s, z)]
    clean = gpipes.q4_gemm_out(x.to(cuda), *args, group=64)
    bad = x.clone()
    bad[M // 2, 100], bad[M - 1, 511] = float("inf"), float("nan")
    got = gpipes.q4_gemm_out(bad.to(cuda), *args, group=64)
    rows = {M // 2, M - 1}
    for m in range(M):
        assert torch.isnan(got[m]).all() if m in rows else torch.equal(got[m], clean[m])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 16, 50, 200, 600])
def test_rows_do_not_depend_on_their_neighbours(cuda, M):
    """Two calls give the same bits, residual in place too."""
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(M, 1024, generator=gen).to(F16).to(cuda)
    q, s, z = weight(1024, 328, 128, True, F16, gen)
    r = torch.randn(M, 328, generator=gen).to(F16).to(cuda)
    args = [dev(t, cuda) for t in (q4.pack(q), s, z)]
    a = gpipes.q4_gemm_out(x, *args, r=r)
    b = r.clone()
    gpipes.q4_gemm_out(x, *args, r=b, out=b)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,two", [(65, 4096, 520, False), (100, 4096, 4098, False), (64, 8200, 4104, True),
                                       (128, 8192, 256, True), (200, 5000, 250, False)])
def test_parts_of_k(cuda, M, K, N, two):
    """With the workspace that is asked for, without one, and with one that is too small: within the bounds each time,
    nothing behind the workspace's end written, the last two the same bits."""
    L, vp = gpipes.lib, ctypes.c_void_p
    weights = 2 if two else 1
    need = L.gp_q4_workspace_bytes(M, N, K, 64, weights)
    assert need > 0
    gen = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=gen).to(BF16)
    sides = [weight(K, N, 64, True, BF16, gen) for _ in range(weights)]
    v, dv = product(x, *sides[0], 64)
    if two:
        u, du = product(x, *sides[1], 64)
        g, dg = moved(v, dv, "silu")
        v, dv = g * u, dg * (u.abs() + du) + g.abs() * du + 2 * U * (g * u).abs()
    xd, ts = x.to(cuda), [[dev(t, cuda) for t in (q4.pack(q), s, z)] for q, s, z in sides]
    ws = torch.full((need // 4 + 1024,), 7.0, device=cuda)
    outs = []
    for n in (need, need - 16, 0):
        out = torch.empty(M, N, dtype=BF16, device=cuda)
        args = [vp(t.data_ptr()) for side in ts for t in side]
        stream = vp(torch.cuda.current_stream().cuda_stream)
        if two:
            rc = L.gp_q4_gated_out(M, N, K, 64, vp(xd.data_ptr()), *args[:3], None, *args[3:], None, 4,
                                   vp(out.data_ptr()), vp(ws.data_ptr()), n, 1, stream)
        else:
            rc = L.gp_q4_gemm_out(M, N, K, 64, vp(xd.data_ptr()), *args, None, None, 0, vp(out.data_ptr()),
                                  vp(ws.data_ptr()), n, 1, stream)
        assert rc == 0, L.gp_last_error().decode()
        check(out, v, dv, BF16)
        outs.append(out)
    assert (ws[need // 4:] == 7).all()
    assert torch.equal(outs[1], outs[2])


@pytest.mark.gpu
def test_python_refusals(cuda):
    gen = torch.Generator().manual_seed(6)
    q, s, z = weight(256, 64, 64, True, F16, gen)
    wq, s, z = q4.pack(q).to(cuda), s.to(cuda), z.to(cuda)
    x = torch.zeros(3, 256, dtype=F16, device=cuda)
    ok = dict(group=64)
    for args, kw, what in (
            ((x, wq, s, z), dict(group=128), "scales"), ((x, wq, s, z), dict(group=48), "group"),
            ((x[:, :128].contiguous(), wq, s, z), ok, "wq"), ((x, wq.long(), s, z), ok, "int32"),
            ((x, wq.t(), s, z), ok, "contiguous|shape"), ((x, wq, s.to(BF16), z), ok, "float16"),
            ((x, wq, s, z[:2]), ok, "zeros"), ((x.t(), wq, s, z), ok, "contiguous"), ((x, wq, s, z, x), ok, "b must"),
            ((x, wq, s, z, None, x), ok, "r must"), ((x[0], wq, s, z), ok, "2-D"), ((x.float(), wq, s, z), ok, "float16"),
            ((x, wq, s, z), dict(group=64, out=x), "out"), ((x[:, :252].contiguous(), wq, s, z), ok, "multiple of 8"),
            ((x, wq, s, z), dict(group=64, act=9), "activation")):
        with pytest.raises(RuntimeError, match=what):
            gpipes.q4_gemm_out(*args, **kw)
    with pytest.raises(RuntimeError, match="_u"):
        gpipes.q4_gated_out(x, wq, s, z, wq[:, :32].contiguous(), s, z, group=64)
    assert gpipes.q4_gemm_out(x[:0], wq, s, z, group=64).shape == (0, 64)


# ---------------------------------------------------------------------------
# The operators together: the feed-forward half of a block, as a program runs it
# ---------------------------------------------------------------------------

def block64(x, y, p):
    """x, y -> (h1, z1) after norm + residual, gated product, product, norm + residual, rounded where the kernels store."""
    def rms(v, g):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * g
    rnd = lambda t: t.to(p["dt"]).double()  # noqa: E731
    d = lambda t: t.double()  # noqa: E731
    h = d(x) + rms(d(y), d(p["g0"]))
    z = rnd(rms(h, d(p["g1"])))
    h = rnd(h)
    w = [q4.dequantize(*p[k], group=64).double() for k in ("wg", "wu", "wd")]
    a = z @ w[0]
    a = rnd(a * torch.sigmoid(a) * (z @ w[1]))
    f = rnd(a @ w[2])
    h2 = h + 0.5 * rms(f, d(p["g2"]))
    return rnd(h2), rnd(rms(h2, d(p["g3"])))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 12, 77, 260])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_block(cuda, M, dt):
    """Eager, and captured into a graph that is replayed with other work between: the same bits each time, and close
    to the block in 64 bits.  Three roundings to dt between input and output, each relative to its row (2^-8 and less
    in bf16) and passed on by products whose outputs are sums of many such terms: as a whole off by a few half steps."""
    H, FF = 512, 1088
    gen = torch.Generator().manual_seed(M)
    n = lambda *sh, m=0.0, k=1.0: (torch.randn(*sh, generator=gen) * k + m).to(dt)  # noqa: E731
    p = {"dt": dt, **{k: n(H, m=1, k=0.1) for k in ("g0", "g1", "g2", "g3")}}
    for k, a, b in (("wg", H, FF), ("wu", H, FF), ("wd", FF, H)):
        p[k] = q4.quantize(n(a, b, k=a ** -0.5), 64, zeros=k == "wu")
    c = {k: tuple(dev(t, cuda) for t in v) if isinstance(v, tuple) else v.to(cuda) for k, v in p.items() if k != "dt"}
    x, y = n(M, H), n(M, H)
    xc, yc = x.to(cuda), y.to(cuda)
    bufs = {k: torch.empty(M, w, dtype=dt, device=cuda) for k, w in (("h", H), ("z", H), ("a", FF), ("f", H), ("h2", H), ("o", H))}

    def step():
        gpipes.residual_norm_out(xc, yc, post="rms", post_gamma=c["g0"], gamma=c["g1"], h=bufs["h"], out=bufs["z"])
        gpipes.q4_gated_out(bufs["z"], *c["wg"], *c["wu"], group=64, out=bufs["a"])
        gpipes.q4_gemm_out(bufs["a"], *c["wd"], group=64, out=bufs["f"])
        gpipes.residual_norm_out(bufs["h"], bufs["f"], post="rms", post_gamma=c["g2"], scale=0.5, gamma=c["g3"],
                                 h=bufs["h2"], out=bufs["o"])

    def close():
        want = block64(xc.cpu(), yc.cpu(), p)
        for got, w in zip((bufs["h2"], bufs["o"]), want):
            assert (got.double().cpu() - w).norm() / w.norm() <= 3 * torch.finfo(dt).eps / 2

    step()
    torch.cuda.synchronize()
    close()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        xc.copy_(n(M, H)), yc.copy_(n(M, H))
        step()
        eager = [bufs[k].clone() for k in ("h2", "o")]
        for t in bufs.values():
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bufs["h2"], eager[0]) and torch.equal(bufs["o"], eager[1])
        close()


@pytest.mark.gpu
def test_two_streams_and_two_graphs(cuda):
    """Calls on two streams at once, and two graphs replayed together: nothing is shared between them."""
    gen = torch.Generator().manual_seed(8)
    sets = []
    for M in (1, 33):
        q, s, z = weight(2048, 1024, 128, True, F16, gen)
        x = torch.randn(M, 2048, generator=gen).to(F16).to(cuda)
        args = [dev(t, cuda) for t in (q4.pack(q), s, z)]
        out = torch.empty(M, 1024, dtype=F16, device=cuda)
        want = gpipes.q4_gemm_out(x, *args)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            for _ in range(20):
                gpipes.q4_gemm_out(x, *args, out=out)
        sets.append((x, args, out, want, g, torch.cuda.Stream(cuda)))
    for _ in range(3):
        for x, args, out, want, g, st in sets:
            out.zero_()
        torch.cuda.synchronize()
        for x, args, out, want, g, st in sets:
            with torch.cuda.stream(st):
                g.replay()
                gpipes.q4_gemm_out(x, *args, out=out)
        torch.cuda.synchronize()
        for x, args, out, want, g, st in sets:
            assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 16384, 1040), (4, 8192, 520), (100, 4096, 1032), (64, 8192, 8200)])
def test_graph_of_a_deep_product(cuda, M, K, N):
    """Calls whose LDS is above the default limit, and calls with parts of k in a workspace: a graph replayed with other
    calls before and behind it gives the eager call's bits each time."""
    gen = torch.Generator().manual_seed(K + M)
    q, s, z = weight(K, N, 128, True, BF16, gen)
    args = [dev(t, cuda) for t in (q4.pack(q), s, z)]
    x, x2 = (torch.randn(M, K, generator=gen).to(BF16).to(cuda) for _ in range(2))
    out = torch.empty(M, N, dtype=BF16, device=cuda)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gpipes.q4_gemm_out(x, *args, out=out)
    for i in range(3):
        x.copy_(torch.randn(M, K, generator=gen).to(BF16))
        want = gpipes.q4_gemm_out(x, *args)
        out.zero_()
        gpipes.q4_gemm_out(x2, *args)
        torch.cuda.synchronize()
        graph.replay()
        gpipes.q4_gemm_out(x2, *args)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("K,N,two", [(64, 1088, False), (1088, 64, False), (32, 1032, True)])
def test_more_values_than_32_bits_count(cuda, K, N, two):
    """2^31 values of x or out and more, at the largest M: rows on both sides of that offset, and the last."""
    M, group = 1 << 21, 32
    gen = torch.Generator().manual_seed(K)
    w = [weight(K, N, group, True, F16, gen) for _ in range(2)]
    args = [[dev(t, cuda) for t in (q4.pack(q), s, z)] for q, s, z in w]
    x = torch.randn(1 << 20, generator=gen).to(F16).to(cuda).repeat(M * K >> 20).view(M, K)
    if two:
        out = gpipes.q4_gated_out(x, *args[0], *args[1], group=group)
    else:
        r = torch.randn(1 << 20, generator=gen).to(F16).to(cuda).repeat(M * N >> 20).view(M, N)
        out = gpipes.q4_gemm_out(x, *args[0], r=r, group=group)
    mid = (1 << 31) // max(K, N)
    for i in (0, mid - 80, mid, M - 80):
        rows = slice(i, i + 80)
        sides = [product(x[rows].cpu(), *t, group) for t in w]
        if two:
            (g, dg), (u, du) = moved(*sides[0], "silu"), sides[1]
            want, bound = g * u, dg * (u.abs() + du) + g.abs() * du + 2 * U * (g * u).abs()
        else:
            v, d = sides[0][0], r[rows].double().cpu()
            want, bound = v + d, sides[0][1] + 2 * U * (v.abs() + d.abs())
        check(out[rows], want, bound, F16)


# ---------------------------------------------------------------------------
# What an fp32 sum keeps
# ---------------------------------------------------------------------------

def outlying(M, K, N, group, zeros, dt, seed):
    """x with a few channels thousands of times as large as the others, and a weight that is exactly zero there."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen)
    at = [3, K // 2 + 7, K - 30]
    x[:, at] = 5000 * (1 + torch.rand(M, len(at), generator=gen)) * torch.tensor([1.0, -1.0, 1.0])
    q, s, _ = weight(K, N, group, False, dt, gen)
    z = torch.randint(0, 16, s.shape, generator=gen).to(dt) if zeros else None
    for c in at:
        q[c] = 8 if z is None else z[c // group].long()
    return x.to(dt), q, s, z


def near(x, q, s, z, group):
    """x W, and a bound for sums in fp32: a group's sum of x q and z times that of x, up to 128 terms of both, take
    sixteen roundings each at most (eight products a step), of what they have come to."""
    x, q, s = x.double(), q.double(), s.double()
    K = q.shape[0]
    zz = z.double() if z is not None else torch.full_like(s, 8)
    sr, zr = (t.repeat_interleave(group, 0)[:K] for t in (s, zz))
    run = torch.zeros(x.shape[0], q.shape[1], dtype=torch.float64, device=x.device)
    for k in range(0, K, group):
        run += (x[:, k:k + group] @ (sr * (q - zr))[k:k + group]).abs()
    return x @ (sr * (q - zr)), 16 * U * (x.abs() @ (sr * (q + zr.abs()))) + 100 * U * run


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(3, 1024, 257), (5, 1024, 256), (16, 1024, 512), (16, 2048, 8192), (40, 1024, 320),
                                   (64, 1024, 256), (100, 4096, 520), (200, 1024, 256), (600, 1024, 1024)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_large_values_under_zero_weights(cuda, M, K, N, zeros, dt):
    """They leave behind what an fp32 sum does: 2^-24 of 15 x 10,000 in a rounding, 0.009, three groups with some ten of
    them at random, 0.05 at most of results that are about 4.6 sqrt(1024) = 147 (all in units of a scale), 3.4e-4 of
    them against a half step of 4.9e-4 in fp16, uniform, 2.8e-4.  Typically a quarter of that: a few hundredths more
    than rounding's own, whose limit is 1.1 in check()."""
    x, q, s, z = outlying(M, K, N, 64, zeros, dt, M + N)
    want, bound = near(x, q, s, z, 64)
    got = gpipes.q4_gemm_out(x.to(cuda), dev(q4.pack(q), cuda), s.to(cuda), dev(z, cuda), group=64)
    check(got, want, bound, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("K,N,group", [(1024, 256, 64), (4096, 512, 128), (1000, 8208, 32), (2048, 16448, 64)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_large_values_of_few_tokens_under_zero_weights(cuda, M, K, N, group, zeros, dt):
    """A single row's x may be taken to 2^-29 of the largest of its 128: 2^-29 of that largest times |W| a product, 2e-5
    at most, which add up at random to 2e-5 x 6.5 sqrt(3 x 128) / sqrt(3) = 0.0015 in units of a scale, where a result
    is about 6.5 sqrt(1000) = 200 and its rounding in fp16 0.04 (uniform)."""
    x, q, s, z = outlying(M, K, N, group, zeros, dt, M + N)
    want, bound = near(x, q, s, z, group)
    zr = (z if z is not None else torch.full_like(s, 8)).double().repeat_interleave(group, 0)[:K]
    w = (s.double().repeat_interleave(group, 0)[:K] * (q - zr)).abs()
    for k in range(0, K if M == 1 else 0, 128):
        bound += 2.0 ** -29 * x[:, k:k + 128].abs().amax(1, keepdim=True).double() * w[k:k + 128].sum(0)
    got = gpipes.q4_gemm_out(x.to(cuda), dev(q4.pack(q), cuda), s.to(cuda), dev(z, cuda), group=group)
    check(got, want, bound, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4])
def test_values_of_one_token_do_not_reach_another(cuda, M):
    """Tokens share a matrix instruction: what the others hold, large, infinite or NaN, leaves a token's bits alone."""
    gen = torch.Generator().manual_seed(M)
    for dt, N in ((F16, 128), (BF16, 8208)):
        x = torch.randn(M, 640, generator=gen).to(dt).to(cuda)
        q, s, z = weight(640, N, 32, True, dt, gen)
        args = [dev(t, cuda) for t in (q4.pack(q), s, z)]
        want = gpipes.q4_gemm_out(x, *args, group=32)
        for m in range(M):
            for v in (0.0, 30000.0, float("inf"), float("nan")):
                other = torch.full_like(x, v)
                other[m] = x[m]
                assert torch.equal(gpipes.q4_gemm_out(other, *args, group=32)[m], want[m])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["foo", 9, 1.5, None])
def test_unknown_activations_raise_runtime_errors(cuda, act):
    q, s, _ = weight(64, 32, 32, False, F16, torch.Generator().manual_seed(0))
    x, wq, s = torch.zeros(2, 64, dtype=F16, device=cuda), q4.pack(q).to(cuda), s.to(cuda)
    with pytest.raises(RuntimeError):
        gpipes.q4_gemm_out(x, wq, s, act=act, group=32)
    with pytest.raises(RuntimeError):
        gpipes.q4_gated_out(x, wq, s, None, wq, s, None, act=act, group=32)


# ---------------------------------------------------------------------------
# Every kernel that a call can select, at sizes that no tile divides
# ---------------------------------------------------------------------------

def run_case(M, K, N, group, zeros, dt, d, two, seed):
    """A product with bias (and a residual), or a gated pair with biases, against the formulas; in 64 bits on the GPU."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *sh: torch.randn(*sh, generator=gen).to(dt).to(d)  # noqa: E731
    x, sides, args = n(M, K), [], []
    for _ in range(2 if two else 1):
        q, s, z = weight(K, N, group, zeros, dt, gen)
        q, s, z, b = q.to(d), s.to(d), dev(z, d), n(N)
        v, dv = near(x, q, s, z, group)
        sides.append((v + b.double(), dv + 2 * U * (v.abs() + b.double().abs())))
        args.append((q4.pack(q), s, z, b))
    buf = torch.full((M * N + 512,), 7.0, dtype=dt, device=d)
    out = buf[:M * N].view(M, N)
    if two:
        (g, dg), (u, du) = moved(*sides[0], "silu"), sides[1]
        want, bound = g * u, dg * (u.abs() + du) + g.abs() * du + 2 * U * (g * u).abs()
        gpipes.q4_gated_out(x, *args[0][:3], *args[1][:3], bg=args[0][3], bu=args[1][3], group=group, out=out)
    else:
        r = n(M, N)
        v, dv = sides[0]
        want, bound = v + r.double(), dv + 2 * U * (v.abs() + r.double().abs())
        gpipes.q4_gemm_out(x, *args[0], r=r, group=group, out=out)
    check(out, want.cpu(), bound.cpu(), dt)
    assert (buf[M * N:] == 7).all()


# (rows, k, columns), of the pair each weight's: tiles of 64, 128 and 256 columns, k whole and in parts (256 CUs)
TILES = [(130, 136, 61, False), (130, 520, 61, False), (1030, 136, 5001, False), (700, 4104, 1030, False),
         (257, 136, 11003, False), (65, 2056, 6001, False), (130, 136, 61, True), (130, 520, 61, True),
         (257, 136, 8195, True), (700, 4104, 515, True), (130, 136, 8195, True), (65, 2056, 3001, True)]
# one to four tiles of 16 rows, and up to four rows, by one, two and four columns a lane
FEW = [(M, K, N, two) for M in (1, 3, 4, 9, 25, 45) for K, N, two in ((1160, 67, False), (392, 8195, False),
                                                                     (136, 16387, False), (1160, 35, True),
                                                                     (392, 4099, True), (136, 8195, True))]
FEW += [(60, 1160, 67, False), (64, 136, 8192, False), (100, 1160, 67, False), (60, 1160, 35, True), (52, 392, 4096, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,two", TILES + FEW)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_every_kernel(cuda, M, K, N, two, group, zeros):
    for dt in (F16, BF16):
        print(M, K, N, two, group, zeros, dt, flush=True)
        run_case(M, K, N, group, zeros, dt, cuda, two, M + N)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,two", [(1, 1160, 66, False), (1, 392, 8194, False), (1, 136, 16386, False),
                                       (1, 520, 130, True), (1, 392, 8198, True), (1, 136, 16390, True)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_every_width_of_the_one_token_kernel(cuda, M, K, N, two, group, zeros):
    for dt in (F16, BF16):
        run_case(M, K, N, group, zeros, dt, cuda, two, N)


# ---------------------------------------------------------------------------
# Rows and calls that must not see each other
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(2, 640, 200), (4, 640, 200), (16, 1024, 328), (40, 1024, 328), (64, 1024, 328),
                                   (100, 4096, 1032), (200, 1024, 328), (700, 512, 2056)])
@pytest.mark.parametrize("two", [False, True])
def test_a_row_keeps_its_bits_among_other_rows(cuda, M, K, N, two):
    """Other values in every other row, large and not finite ones among them, leave a row's bits as they were."""
    gen = torch.Generator().manual_seed(M + N)
    sides = []
    for _ in range(2):
        q, s, z = weight(K, N, 64, True, BF16, gen)
        sides += [dev(t, cuda) for t in (q4.pack(q), s, z)]

    def call(x):
        return gpipes.q4_gated_out(x, *sides, group=64) if two else gpipes.q4_gemm_out(x, *sides[:3], group=64)

    x = torch.randn(M, K, generator=gen).to(BF16).to(cuda)
    want = call(x)
    for m in sorted({0, 1, M // 2, M - 1}):
        for k in (1.0, 1e4, float("nan")):
            other = (torch.randn(M, K, generator=gen) * k).to(BF16).to(cuda)
            other[m] = x[m]
            assert torch.equal(call(other)[m], want[m])


@pytest.mark.gpu
def test_two_streams_and_two_graphs_with_workspaces(cuda):
    """Calls with parts of k in a workspace, on two streams at once, eager and replayed together."""
    gen = torch.Generator().manual_seed(9)
    sets = []
    for M, K, N in ((100, 4096, 1032), (65, 4096, 520)):
        assert gpipes.lib.gp_q4_workspace_bytes(M, N, K, 128, 1) > 0
        q, s, z = weight(K, N, 128, True, F16, gen)
        x = torch.randn(M, K, generator=gen).to(F16).to(cuda)
        args = [dev(t, cuda) for t in (q4.pack(q), s, z)]
        outs = [torch.empty(M, N, dtype=F16, device=cuda) for _ in range(2)]
        want = gpipes.q4_gemm_out(x, *args)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            for _ in range(20):
                gpipes.q4_gemm_out(x, *args, out=outs[0])
        sets.append((x, args, outs, want, g, torch.cuda.Stream(cuda), torch.cuda.Stream(cuda)))
    for _ in range(3):
        for _, _, outs, *_ in sets:
            outs[0].zero_(), outs[1].zero_()
        torch.cuda.synchronize()
        for x, args, outs, want, g, a, b in sets:
            with torch.cuda.stream(a):
                g.replay()
            with torch.cuda.stream(b):
                for _ in range(20):
                    gpipes.q4_gemm_out(x, *args, out=outs[1])
        torch.cuda.synchronize()
        for x, args, outs, want, *_ in sets:
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 20, 64, 150, 300])
def test_the_largest_values_of_fp16(cuda, M):
    """Rows of +-65,504, of fp16's smallest values, and both together, with scales that keep the results in range."""
    gen = torch.Generator().manual_seed(M)
    K, N, G = 640, 144, 64
    x = torch.where(torch.rand(M, K, generator=gen) < 0.5, -65504.0, 65504.0)
    x[1::3] = torch.randint(-9, 10, x[1::3].shape, generator=gen) * 2.0 ** -24
    x[2::3, ::2] = torch.randint(-9, 10, x[2::3, ::2].shape, generator=gen) * 2.0 ** -24
    x = x.to(F16)
    q, s, z = weight(K, N, G, True, F16, gen)
    s = (s.double() / 64).to(F16)
    want, bound = near(x, q, s, z, G)
    got = gpipes.q4_gemm_out(x.to(cuda), *(dev(t, cuda) for t in (q4.pack(q), s, z)), group=G)
    if M == 1:
        bound += 2.0 ** -29 * 65504 * (s.double().repeat_interleave(G, 0) * (q - z.double().repeat_interleave(G, 0))).abs().sum(0)
    check(got, want, bound, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 4, 6, 14, 18])
def test_one_token_of_few_columns(cuda, N):
    for K, group, two in ((8, 32, False), (64, 32, True), (264, 64, False), (1400, 128, True)):
        for dt in (F16, BF16):
            run_case(1, K, N, group, K != 264, dt, cuda, two, N)


@pytest.mark.gpu
@pytest.mark.parametrize("K,group,zeros,two", [(19968, 128, False, False), (19976, 128, False, False),
                                               (15872, 32, True, False), (15872, 64, True, True), (15880, 64, True, True),
                                               (15872, 32, False, True), (65536, 128, True, True)])
def test_one_token_of_the_deepest_k_that_lds_holds(cuda, K, group, zeros, two):
    """All of a CU's 160 KiB, and the next k, which another kernel takes."""
    for dt in (F16, BF16):
        run_case(1, K, 66, group, zeros, dt, cuda, two, K)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 144), (1, 145), (3, 144), (20, 144), (64, 145), (150, 144), (300, 145)])
@pytest.mark.parametrize("zeros", [False, True])
def test_large_values_of_bf16(cuda, M, N, zeros):
    """x up to some 1e35: 15 times a group's sum of |x| stays below fp32's largest number, 3.4e38, and so do results."""
    gen = torch.Generator().manual_seed(M)
    K, G = 640, 128
    x = (torch.randn(M, K, generator=gen) * 2e34).to(BF16)
    q, s, z = weight(K, N, G, zeros, BF16, gen)
    assert 16 * 128 * x.double().abs().max() < 3.4e38
    want, bound = near(x, q, s, z, G)
    got = gpipes.q4_gemm_out(x.to(cuda), *(dev(t, cuda) for t in (q4.pack(q), s, z)), group=G)
    check(got / 2.0 ** 110, want / 2.0 ** 110, bound / 2.0 ** 110, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 520), (1, 521), (2, 520), (16, 521), (48, 520), (64, 521), (130, 520), (700, 1031)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_zeros_of_any_value(cuda, M, N, dt):
    """Negative, fractional and larger than any q."""
    gen = torch.Generator().manual_seed(M + N)
    K, G = 1000, 64
    x = torch.randn(M, K, generator=gen).to(dt)
    q, s, z = weight(K, N, G, True, dt, gen)
    z = (torch.randn(z.shape, generator=gen) * 30).to(dt)
    want, bound = near(x, q, s, z, G)
    got = gpipes.q4_gemm_out(x.to(cuda), *(dev(t, cuda) for t in (q4.pack(q), s, z)), group=G)
    check(got, want, bound, dt)
