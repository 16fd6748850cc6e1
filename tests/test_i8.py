"""Products in 8-bit integers: i8_gemm_out and i8_gated_out, and gpipes.i8, which makes their weights.

The refusals and gpipes.i8 need no GPU.  The sums over k are whole numbers and exact, so results
are compared with the formulas in 64 bits to a bound that holds only the roundings behind them:
the sum, its two scales, bias and activation in fp32, and the result's own.
"""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import gpipes
from gpipes import i8

F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24
MAX_K = 131056


# ---------------------------------------------------------------------------
# Without a GPU
# ---------------------------------------------------------------------------

def _call(M=4, N=256, K=512, x=1 << 20, xs=0, wq=1 << 24, s=1 << 25, b=0, r=0, act=0, out=1 << 21, dtype=0, two=False,
          u=1 << 26, su=1 << 27, ws=0, wsb=0):
    vp = ctypes.c_void_p
    P = lambda v: vp(v) if v else None  # noqa: E731
    if two:
        return gpipes.lib.gp_i8_gated_out(M, N, K, P(x), P(xs), P(wq), P(s), P(b), P(u), P(su), P(b), act, P(out), P(ws),
                                          wsb, dtype, None)
    return gpipes.lib.gp_i8_gemm_out(M, N, K, P(x), P(xs), P(wq), P(s), P(b), P(r), act, P(out), P(ws), wsb, dtype, None)


@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(M=(1 << 21) + 1), -2), (dict(N=0), -2), (dict(N=(1 << 20) + 1), -2), (dict(K=0), -2),
    (dict(K=-16), -2), (dict(K=8), -2), (dict(K=520), -2), (dict(K=MAX_K + 16), -2), (dict(K=65536, N=32768), -2),
    (dict(dtype=2), -1), (dict(act=5), -1), (dict(act=-1), -1), (dict(x=0), -1), (dict(wq=0), -1), (dict(s=0), -1),
    (dict(out=0), -1), (dict(x=24), -3), (dict(wq=20), -3), (dict(s=10), -3), (dict(xs=6), -3), (dict(b=2), -3),
    (dict(out=40), -3), (dict(wsb=-1), -1), (dict(wsb=64), -1), (dict(ws=24, wsb=64), -3),
])
def test_argument_errors(kw, code, two):
    assert _call(**kw, two=two) == code
    assert gpipes.lib.gp_last_error().decode() != ""


def test_argument_errors_of_one_form():
    assert _call(r=1 << 28, act=1) == -1
    assert _call(r=8) == -3
    assert _call(u=0, two=True) == -1
    assert _call(su=0, two=True) == -1
    assert _call(u=24, two=True) == -3
    assert _call(su=26, two=True) == -3


SIZES = {"x": 4 * 512 * 2, "xs": 16, "wq": 256 * 512, "s": 1024, "b": 512, "u": 256 * 512, "su": 1024}


@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("what", SIZES)
def test_overlaps_are_refused(what, two):
    """out and the workspace over the first and the last 16 bytes of every other operand."""
    if what in ("u", "su") and not two:
        return
    at, size = 1 << 29, SIZES[what] // 2 if what == "x" else SIZES[what]
    kw = {"b": 1 << 28, "xs": 3 << 28, what: at}  # x in 8 bits
    for lo, n in ((at - 2048 + 16, 2048), (at + size - 16, 2048)):  # out's 4 x 256 values
        assert _call(**{**kw, "out": lo}, two=two) == -1
        assert "out must not overlap" in gpipes.lib.gp_last_error().decode()
        assert _call(**kw, ws=lo, wsb=n, two=two) == -1
        assert "workspace must not overlap" in gpipes.lib.gp_last_error().decode()


def test_overlaps_of_residual_and_workspace():
    assert _call(r=(1 << 21) + 16) == -1
    assert _call(r=1 << 22, ws=(1 << 22) + 2032, wsb=16) == -1
    assert _call(ws=(1 << 21) + 2032, wsb=16) == -1
    assert "workspace" in gpipes.lib.gp_last_error().decode()


@pytest.mark.parametrize("two", [False, True])
def test_empty_batch_is_a_noop(two):
    assert _call(M=0, x=0, out=0, two=two) == 0
    assert gpipes.lib.gp_last_error().decode() == ""


@pytest.mark.parametrize("args,code", [
    ((-1, 64, 64, 0, 1), -1), ((64, 0, 64, 0, 1), -2), ((64, 64, 72, 0, 1), -2), ((64, 64, 64, 2, 1), -1),
    ((64, 64, 64, 0, 3), -1), ((64, 64, 64, 0, 0), -1), ((0, 64, 64, 0, 1), 0)])
def test_workspace_arguments(args, code):
    assert gpipes.lib.gp_i8_workspace_bytes(*args) == code


def test_python_refuses():
    x, wq, s = torch.zeros(1, 64, dtype=F16), torch.zeros(2, 1, 1024, dtype=torch.int8), torch.zeros(32)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.i8_gemm_out(x, wq, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.i8_gated_out(x, wq, s, wq, s)
    for bad in (None, 3, "x"):
        with pytest.raises(RuntimeError):
            gpipes.i8_gemm_out(bad, wq, s)


def test_the_package_has_the_weights_module():
    code = "import gpipes; assert gpipes.i8.pack and 'i8' in gpipes.__all__"
    path = os.path.dirname(os.path.dirname(gpipes.__file__))
    env = {**os.environ, "PYTHONPATH": os.pathsep.join([path, os.environ.get("PYTHONPATH", "")])}
    assert subprocess.run([sys.executable, "-c", code], env=env).returncode == 0


@pytest.mark.parametrize("K,N", [(16, 1), (64, 16), (80, 17), (144, 33), (1, 5)])
@pytest.mark.parametrize("experts", [0, 3])
def test_pack_and_unpack(K, N, experts):
    gen = torch.Generator().manual_seed(K)
    q = torch.randint(-128, 128, (experts, K, N) if experts else (K, N), generator=gen).to(torch.int8)
    w = i8.pack(q)
    assert w.shape == ((experts,) if experts else ()) + i8.packed_shape(K, N) and w.is_contiguous()
    assert torch.equal(i8.unpack(w, K, N), q)
    flat = (w if experts else w[None]).flatten(1).long()
    for e, k, n in ((0, 0, 0), (max(experts, 1) - 1, K - 1, N - 1), (0, K // 2, N // 2)):
        at = (n // 16 * -(-K // 64) + k // 64) * 1024 + k % 64 // 16 * 256 + n % 16 * 16 + k % 16
        assert flat[e, at] == (q if experts else q[None])[e, k, n]
    assert flat.abs().sum() == q.long().abs().sum()  # zeros behind K and N
    s = torch.rand((experts, N) if experts else (N,), generator=gen)
    assert torch.equal(i8.dequantize(w, s, K), q.float() * s[..., None, :])


@pytest.mark.parametrize("dt", [torch.int64, torch.int32, torch.float32, torch.uint8])
def test_pack_takes_other_types_and_strides(dt):
    q = torch.arange(128).view(4, 32).to(dt)
    assert torch.equal(i8.unpack(i8.pack(q.t()), 32, 4).to(dt), q.t())


@pytest.mark.parametrize("v", [3.5, 128, -129, float("nan"), float("inf")])
def test_pack_refuses_what_is_no_byte(v):
    q = torch.zeros(16, 4)
    q[3, 2] = v
    with pytest.raises(RuntimeError, match="-128 .. 127"):
        i8.pack(q)


@pytest.mark.parametrize("dt", [F16, BF16, torch.float32])
def test_quantize(dt):
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(2, 96, 40, generator=gen).to(dt)
    w[0, :, 5] = 0
    w[1, 3, 7] = 100  # one value far from the others
    wq, s = i8.quantize(w)
    assert s.dtype == torch.float32 and s.shape == (2, 40) and s[0, 5] == 0
    q = i8.unpack(wq, 96, 40)
    assert q.abs().max() == 127 and not bool((q[0, :, 5]).any())
    d = w.double()
    # half a step, max / 254; the scale's and the product's roundings in fp32 are 2^-24 of at most the maximum each,
    # together 2 * 254 * 2^-24 < 2^-15 of the half step
    assert bool(((i8.dequantize(wq, s, 96).double() - d).abs() <= d.abs().amax(1, keepdim=True) / 254 * (1 + 2 ** -15)).all())
    one, t = i8.quantize(w[1])
    assert torch.equal(one, wq[1]) and torch.equal(t, s[1])


def test_quantize_refuses():
    for bad in (torch.zeros(4, dtype=F16), torch.zeros(0, 4), torch.zeros(4, 4, dtype=torch.float64),
                torch.full((4, 4), float("nan"))):
        with pytest.raises(RuntimeError):
            i8.quantize(bad)
    for bad in (torch.zeros(16), torch.zeros(0, 4), torch.zeros(2, 2, 2, 2)):
        with pytest.raises(RuntimeError):
            i8.pack(bad)
    with pytest.raises(RuntimeError):
        i8.unpack(torch.zeros(1, 1, 1024, dtype=torch.int8), 65, 16)
    with pytest.raises(RuntimeError):
        i8.quantize_rows(torch.zeros(4, 16))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_quantize_rows(dt):
    x = torch.tensor([[127, 0.5, 1.5, -2.5, 126.5, 0], [0] * 6, [1, float("nan"), 2, 3, 4, 5], [2, -2, 1, 0, 0, 0]]).to(dt)
    if dt == BF16:
        x[0, 4] = 126
    q, s = i8.quantize_rows(x)
    assert q[0].tolist() == [127, 0, 2, -2, 126, 0] and s[0] == 1  # halves to even
    assert not bool(q[1].any()) and s[1] == 0
    assert not bool(q[2].any()) and bool(s[2].isnan())
    assert q[3].tolist() == [127, -127, 64, 0, 0, 0]  # 63.5


# ---------------------------------------------------------------------------
# On a GPU
# ---------------------------------------------------------------------------

def act64(v, act):
    return {"none": lambda: v, "relu": lambda: v.clamp(min=0), "sigmoid": lambda: torch.sigmoid(v),
            "silu": lambda: v * torch.sigmoid(v),
            "gelu_tanh": lambda: v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))}[act]()


def moved(v, d, act):
    """An activation of v, which is off by d: no slope is above 1.13, and the activation's own arithmetic takes some
    ulp, the exponent's argument |1.6 v (1 + 0.045 v^2)| of them (past 30 the result is v or nothing)."""
    a = act64(v, act)
    if act == "none":
        return a, d
    return a, 1.13 * d + U * (8 + 2 * v.abs().clamp(max=30) * (1 + 0.045 * v.abs().clamp(max=30) ** 2)) * a.abs()


def side(q, xs, w, b):
    """x W + b in 64 bits, and a bound of fp32's roundings: the sum's, two products', the bias'."""
    wq, s = w
    v = (q.double() @ wq.double()) * s.double() * xs.double()[:, None]
    d = 3 * U * v.abs()
    if b is not None:
        v = v + b.double()
        d = d + U * v.abs()
    return v, d


def check(out, want, bound, dt):
    """Each value to within half a step of its own type and the bound (and half of a denormal's step)."""
    eps, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == F16 else 2.0 ** -134
    out = out.double()
    err = (out - want).abs()
    tol = eps * (want.abs() + bound) + bound + tiny
    big = want.abs() + bound >= torch.finfo(dt).max * (1 - eps)  # may round to an infinity
    bad = ~(err <= tol) & ~(big & torch.isinf(out))
    assert not bool(bad.any()), (int(bad.sum()), (err / tol)[bad].max().item(), bad.nonzero()[:3].tolist())


def weight(K, N, gen, dev):
    q = torch.randint(-128, 128, (K, N), generator=gen, dtype=torch.int16).to(torch.int8).to(dev)
    s = (torch.rand(N, generator=gen) + 0.5) / (74 * K ** 0.5)
    return q, s.to(dev)


def rows(M, K, dt, gen, dev, int8=False):
    if int8:
        return (torch.randint(-128, 128, (M, K), generator=gen, dtype=torch.int16).to(torch.int8).to(dev),
                ((torch.rand(M, generator=gen) + 0.5) / 74).to(dev))
    x = torch.randn(M, K, generator=gen)
    x[:, :: max(1, K // 3)] *= 6
    return x.to(dt).to(dev), None


def whole(x, xs):
    return i8.quantize_rows(x) if xs is None else (x, xs)


def linear(cuda, M, K, N, dt, int8=False, bias=False, residual=False, act="none", seed=0):
    gen = torch.Generator().manual_seed(seed + M * 7 + K * 3 + N)
    x, xs = rows(M, K, dt, gen, cuda, int8)
    wq, s = weight(K, N, gen, cuda)
    b = torch.randn(N, generator=gen).to(dt).to(cuda) if bias else None
    r = torch.randn(M, N, generator=gen).to(dt).to(cuda) if residual else None
    out = gpipes.i8_gemm_out(x, i8.pack(wq), s, xs=xs, b=b, r=r, act=act,
                             out=torch.full((M, N), float("nan"), dtype=dt, device=cuda))
    want, d = moved(*side(*whole(x, xs), (wq, s), b), act)
    if r is not None:
        want = want + r.double()
        d = d + U * want.abs()
    check(out, want, d, dt)


def gated(cuda, M, K, N, dt, int8=False, bias=False, act="silu", seed=0):
    gen = torch.Generator().manual_seed(seed + M * 7 + K * 3 + N)
    x, xs = rows(M, K, dt, gen, cuda, int8)
    w = [weight(K, N, gen, cuda) for _ in range(2)]
    b = [torch.randn(N, generator=gen).to(dt).to(cuda) if bias else None for _ in range(2)]
    out = gpipes.i8_gated_out(x, i8.pack(w[0][0]), w[0][1], i8.pack(w[1][0]), w[1][1], xs=xs, bg=b[0], bu=b[1], act=act,
                              out=torch.full((M, N), float("nan"), dtype=dt, device=cuda))
    q, xs = whole(x, xs)
    (g, dg), (u, du) = moved(*side(q, xs, w[0], b[0]), act), side(q, xs, w[1], b[1])
    want = g * u
    check(out, want, dg * (u.abs() + du) + g.abs() * du + U * want.abs(), dt)


FORMS = [dict(), dict(int8=True), dict(bias=True, act="gelu_tanh"), dict(residual=True), dict(int8=True, bias=True, residual=True),
         dict(act="relu"), dict(bias=True, act="silu"), dict(act="sigmoid")]


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 15, 16, 17, 32, 33, 48, 64, 65, 127, 128, 129, 200, 256, 257, 520])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_sizes(cuda, M, dt):
    i = 0
    for K in (16, 48, 64, 80, 128, 144, 192, 528, 1040):
        for N in (1, 15, 16, 17, 63, 100, 257):
            linear(cuda, M, K, N, dt, **FORMS[i % len(FORMS)])
            i += 1


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 4, 5, 16, 20, 40, 64, 65, 130, 300])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_gated_sizes(cuda, M, dt):
    i = 0
    for K in (16, 80, 256, 592):
        for N in (1, 16, 33, 130, 264):
            gated(cuda, M, K, N, dt, int8=i % 3 == 1, bias=i % 2 == 0, act=("silu", "gelu_tanh", "relu", "sigmoid", "none")[i % 5])
            i += 1


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [
    (1, 16384, 1040), (1, 16400, 520), (1, 131056, 40), (3, 4096, 8200), (4, 4096, 16400), (4, 4112, 4100), (2, 8192, 2050),
    (16, 8192, 8200), (16, 16384, 16400), (30, 4096, 16390), (60, 2064, 16400), (64, 8192, 4100), (70, 16384, 300),
    (203, 4080, 4093), (600, 1040, 4100), (1000, 2048, 8190), (2500, 528, 2100), (70, 131056, 20)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_wide_and_deep(cuda, M, K, N, dt):
    linear(cuda, M, K, N, dt)
    linear(cuda, M, K, N, dt, int8=True, bias=True, residual=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 4096, 16400), (1, 1040, 4100), (4, 4096, 4104), (16, 2048, 8200), (48, 2048, 8192),
                                   (60, 528, 16390), (130, 4112, 1100), (700, 1040, 4100), (1030, 2048, 8190)])
def test_gated_wide(cuda, M, K, N):
    gated(cuda, M, K, N, BF16)
    gated(cuda, M, K, N, F16, int8=True, bias=True, act="gelu_tanh")


@pytest.mark.gpu
@pytest.mark.parametrize("K,N,two", [(528, 300, False), (4096, 2064, False), (4096, 5000, True), (16384, 272, False)])
def test_a_row_keeps_its_bits_among_other_rows(cuda, K, N, two):
    """Whole sums: whichever kernel a number of rows selects, a row's result is the same to the bit."""
    gen = torch.Generator().manual_seed(K)
    x, _ = rows(600, K, BF16, gen, cuda)
    w = [(i8.pack(q), s) for q, s in (weight(K, N, gen, cuda) for _ in range(2))]
    b = torch.randn(N, generator=gen).to(BF16).to(cuda)

    def call(x, xs=None):
        out = torch.empty(x.shape[0], N, dtype=BF16, device=cuda)
        if two:
            return gpipes.i8_gated_out(x, *w[0], *w[1], xs=xs, bg=b, out=out)
        return gpipes.i8_gemm_out(x, *w[0], xs=xs, b=b, act="gelu_tanh", out=out)
    full = call(x)
    q, xs = i8.quantize_rows(x)
    assert torch.equal(call(q, xs), full)
    for n in (1, 2, 3, 4, 5, 16, 17, 33, 64, 65, 128, 200, 300):
        assert torch.equal(call(x[-n:].contiguous()), full[-n:])
        assert torch.equal(call(q[-n:].contiguous(), xs[-n:].contiguous()), full[-n:])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 16, 70])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_rows_are_rounded_to_even_and_to_the_last_bit(cuda, M, dt):
    """x against a weight that picks single k out: the whole numbers that the call makes of a row, and ties among them."""
    K = 528
    gen = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=gen)
    ties = torch.arange(K) + 0.5
    x[0] = torch.where(ties < 127, ties, x[0].clamp(-3, 3))  # exact halves under a largest value of 127
    x[0, K - 1] = 127
    if M > 2:
        x[1] = torch.randint(-255, 256, (K,), generator=gen) / 2
        x[1, 5] = 127
        x[2] = torch.randint(0, 2, (K,), generator=gen) * 2.0 - 1  # every value the largest
        x[3] = 0
    x = x.to(dt)
    one = torch.eye(K, dtype=torch.int8)
    out = gpipes.i8_gemm_out(x.to(cuda), i8.pack(one).to(cuda), torch.ones(K, device=cuda)).cpu()
    q, s = i8.quantize_rows(x)
    assert torch.equal(out, (q.float() * s[:, None]).to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 16, 100])
def test_largest_and_smallest_values(cuda, M):
    K, N = 272, 80
    gen = torch.Generator().manual_seed(M)
    wq, s = weight(K, N, gen, cuda)
    for dt, scales in ((BF16, (3e38, 1e30, 1e-30, 1e-38)), (F16, (65504.0, 1e-4, 6e-8))):
        for top in scales:
            x = torch.randn(M, K, generator=gen).clamp(-3, 3) * (top / 3)
            x[:, 7] = top
            x = x.to(dt).to(cuda)
            x = torch.where(torch.isfinite(x), x, torch.finfo(dt).max)
            out = gpipes.i8_gemm_out(x, i8.pack(wq), s)
            q, xs = i8.quantize_rows(x)
            want, d = side(q, xs, (wq, s), None)
            check(out, want, d + 2.0 ** -149, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 20, 64, 100, 300])
@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_rows_that_are_not_finite(cuda, M, two, act):
    """NaN in their own rows of out, under every activation, and nowhere else; a row of zeros gives the bias."""
    K, N = 528, 130
    gen = torch.Generator().manual_seed(M)
    x, _ = rows(M, K, F16, gen, cuda)
    w = [(i8.pack(q), s) for q, s in (weight(K, N, gen, cuda) for _ in range(2))]
    b = torch.randn(N, generator=gen).to(F16).to(cuda)
    call = lambda x: (gpipes.i8_gated_out(x, *w[0], *w[1], bu=b, act=act) if two  # noqa: E731
                      else gpipes.i8_gemm_out(x, *w[0], b=b, act=act))
    good = call(x)
    bad = x.clone()
    for i, v in ((0, float("nan")), (M // 2, float("inf")), (M - 1, float("-inf"))):
        bad[i, (i * 5) % K] = v
    out = call(bad)
    hit = torch.zeros(M, dtype=torch.bool, device=cuda)
    hit[[0, M // 2, M - 1]] = True
    assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], good[~hit])
    x[-1] = 0
    zero = call(x)[-1].float()
    bias = torch.zeros_like(zero) if two and act != "sigmoid" else b.float()
    if act == "none" or two:
        assert torch.equal(zero, act64(bias, act) if not two else bias)


@pytest.mark.gpu
def test_the_largest_sums(cuda):
    """Every product 128 * 128, K at its largest: the sum just fits 32 bits, in one part of k and in several."""
    for M in (1, 16, 70, 300):
        x = torch.full((M, MAX_K), -128, dtype=torch.int8, device=cuda)
        wq = torch.full((MAX_K, 18), -128, dtype=torch.int8, device=cuda)
        wq[:, 1] = 127
        out = torch.empty(M, 18, dtype=BF16, device=cuda)
        gpipes.i8_gemm_out(x, i8.pack(wq), torch.ones(18, device=cuda), xs=torch.ones(M, device=cuda), out=out)
        want = torch.full((M, 18), 128.0 * 128 * MAX_K, dtype=torch.float64)
        want[:, 1] = -127.0 * 128 * MAX_K
        assert torch.equal(out.cpu(), want.to(BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("K,N,two,int8", [(64, 1088, False, False), (1088, 64, False, True), (1040, 48, True, False)])
def test_more_values_than_32_bits_count(cuda, K, N, two, int8):
    """2^31 values of x or out and more, at the largest M: rows on both sides of that offset, and the last."""
    M = 1 << 21
    gen = torch.Generator().manual_seed(K)
    w = [weight(K, N, gen, cuda) for _ in range(2)]
    xs = None
    if int8:
        x = torch.randint(-128, 128, (1 << 20,), generator=gen, dtype=torch.int16).to(torch.int8).to(cuda)
        xs = (torch.rand(M, generator=gen) / 74).to(cuda)
    else:
        x = torch.randn(1 << 20, generator=gen).to(F16).to(cuda)
    x = x.repeat(M * K >> 20).view(M, K)
    out = torch.empty(M, N, dtype=F16, device=cuda)
    if two:
        gpipes.i8_gated_out(x, i8.pack(w[0][0]), w[0][1], i8.pack(w[1][0]), w[1][1], xs=xs, out=out)
    else:
        r = torch.randn(1 << 20, generator=gen).to(F16).to(cuda).repeat(M * N >> 20).view(M, N)
        gpipes.i8_gemm_out(x, i8.pack(w[0][0]), w[0][1], xs=xs, r=r, out=out)
    mid = (1 << 31) // max(K, N)
    for i in (0, mid - 80, mid, M - 80):
        at = slice(i, i + 80)
        q, t = whole(x[at], None if xs is None else xs[at])
        if two:
            (g, dg), (u, du) = moved(*side(q, t, w[0], None), "silu"), side(q, t, w[1], None)
            check(out[at], g * u, dg * (u.abs() + du) + g.abs() * du + U * (g * u).abs(), F16)
        else:
            v, d = side(q, t, w[0], None)
            want = v + r[at].double()
            check(out[at], want, d + U * want.abs(), F16)


@pytest.mark.gpu
def test_python_refusals(cuda):
    gen = torch.Generator().manual_seed(6)
    q, s = weight(256, 64, gen, cuda)
    wq = i8.pack(q)
    x = torch.zeros(3, 256, dtype=F16, device=cuda)
    x8, xs, out = x.to(torch.int8), torch.ones(3, device=cuda), torch.empty(3, 64, dtype=F16, device=cuda)
    for args, kw, what in (
            ((x, wq, s[:48]), {}, "wq must have shape"), ((x[:, :128].contiguous(), wq, s), {}, "wq"),
            ((x, wq.int(), s), {}, "int8"), ((x, wq.transpose(0, 1), s), {}, "contiguous|shape"), ((x, wq, s.half()), {}, "float32"),
            ((x, wq, s[None]), {}, r"\[N\]"), ((x.t(), wq, s), {}, "contiguous"), ((x[0], wq, s), {}, "2-D"),
            ((x.float(), wq, s), {}, "float16"), ((x[:, :248].contiguous(), wq, s), {}, "multiple of 16"),
            ((x, wq, s), dict(b=x), "b must"), ((x, wq, s), dict(r=x), "r must"), ((x, wq, s), dict(out=x), "out"),
            ((x, wq, s), dict(act=9), "activation"), ((x, wq, s), dict(act="foo"), "invalid"), ((x8, wq, s), {}, "float16"),
            ((x8, wq, s), dict(xs=xs), "out must be given"), ((x, wq, s), dict(xs=xs, out=out), "int8"),
            ((x8, wq, s), dict(xs=xs[:2], out=out), "xs"), ((x8, wq, s), dict(xs=xs.half(), out=out), "float32"),
            ((x8, wq, s), dict(xs=xs, out=out.float()), "float16"), ((x8, wq, s), dict(xs=xs.cpu(), out=out), "CUDA"),
            ((x, wq, s.cpu()), {}, "CUDA"), ((x, wq, s), dict(out=out.to(BF16)), "float16")):
        with pytest.raises(RuntimeError, match=what):
            gpipes.i8_gemm_out(*args, **kw)
    with pytest.raises(RuntimeError, match="wq_u"):
        gpipes.i8_gated_out(x, wq, s, wq[:3].contiguous(), s)
    with pytest.raises(RuntimeError, match="scales_u"):
        gpipes.i8_gated_out(x, wq, s, wq, s[:60])
    assert gpipes.i8_gemm_out(x[:0], wq, s).shape == (0, 64)
    r = out.clone()
    assert gpipes.i8_gemm_out(x, wq, s, r=r, out=r) is r  # in place


@pytest.mark.gpu
def test_a_short_workspace_is_refused(cuda):
    M, K, N = 100, 4096, 80
    need = gpipes.lib.gp_i8_workspace_bytes(M, N, K, 0, 1)
    assert need > 0
    t = [torch.zeros(n, dtype=torch.uint8, device=cuda) for n in (M * K * 2, 80 * 4096, 320, M * N * 2, need)]
    p = [ctypes.c_void_p(v.data_ptr()) for v in t]
    call = lambda n: gpipes.lib.gp_i8_gemm_out(M, N, K, p[0], None, p[1], p[2], None, None, 0, p[3], p[4], n, 0, None)  # noqa: E731
    assert call(need - 1) == -1 and str(need) in gpipes.lib.gp_last_error().decode()
    assert call(0) == -1
    assert call(need) == 0
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,int8", [(1, 16384, 1040, False), (4, 4096, 520, False), (16, 8192, 520, False), (100, 4096, 1032, False),
                                        (64, 8192, 8200, True), (1, 131056, 40, False), (300, 16384, 100, False)])
def test_streams_and_graphs(cuda, M, K, N, int8):
    """Two calls at once on two streams and in two graphs, each with its workspace, other calls between the replays."""
    gen = torch.Generator().manual_seed(K + M)
    wq, s = weight(K, N, gen, cuda)
    wq = i8.pack(wq)
    sets = []
    for _ in range(2):
        x, xs = rows(M, K, BF16, gen, cuda, int8)
        out = torch.empty(M, N, dtype=BF16, device=cuda)
        gpipes.i8_gemm_out(x, wq, s, xs=xs, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                gpipes.i8_gemm_out(x, wq, s, xs=xs, out=out)
        sets.append((x, xs, out, out.clone(), g, torch.cuda.Stream(cuda)))
    for _ in range(3):
        want = []
        for x, xs, out, eager, g, st in sets:
            x.copy_(rows(M, K, BF16, gen, cuda, int8)[0])
            want.append(gpipes.i8_gemm_out(x, wq, s, xs=xs, out=torch.empty_like(out)))
            out.zero_(), eager.zero_()
        torch.cuda.synchronize()
        for x, xs, out, eager, g, st in sets:
            with torch.cuda.stream(st):
                g.replay()
                gpipes.i8_gemm_out(x, wq, s, xs=xs, out=eager)
        torch.cuda.synchronize()
        for (x, xs, out, eager, g, st), w in zip(sets, want):
            assert torch.equal(out, w) and torch.equal(eager, w)


@pytest.mark.gpu
def test_rows_behind_out_stay(cuda):
    """out is a part of a larger tensor: nothing around it is written."""
    gen = torch.Generator().manual_seed(9)
    for M, K, N in ((1, 272, 40), (3, 528, 24), (17, 144, 72), (65, 80, 8), (130, 528, 264), (300, 272, 136)):
        wq, s = weight(K, N, gen, cuda)
        x, _ = rows(M, K, F16, gen, cuda)
        full = torch.full((M + 64, N), 7.0, dtype=F16, device=cuda)
        out = full[32:32 + M]
        gpipes.i8_gemm_out(x, i8.pack(wq), s, out=out)
        assert bool((full[:32] == 7).all()) and bool((full[32 + M:] == 7).all())
        want, d = side(*i8.quantize_rows(x), (wq, s), None)
        check(out, want, d, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,two", [
    (4090, 4096, 8190, False),  # 512 tiles of 256 x 256: two a workgroup, the last ones short
    (2040, 4096, 8190, True), (4090, 2064, 8200, False), (1040, 4096, 4100, False), (300, 2064, 4100, True),
    (70, 16384, 40, False), (90, 8208, 72, True)])  # few tiles: parts of k
def test_every_size_of_tile(cuda, M, K, N, two):
    if two:
        gated(cuda, M, K, N, F16, bias=True)
        gated(cuda, M, K, N, BF16, int8=True, act="gelu_tanh")
    else:
        linear(cuda, M, K, N, F16, bias=True, residual=True)
        linear(cuda, M, K, N, BF16, int8=True, act="silu")


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 17, 40, 100, 300])
def test_scales_of_any_alignment(cuda, M):
    """Scales that begin 4, 8 and 12 bytes behind a 16-byte border, as a slice's do."""
    K, N = 528, 101
    gen = torch.Generator().manual_seed(M)
    for off in (1, 2, 3):
        wq, s = weight(K, N, gen, cuda)
        x, xs = rows(M, K, F16, gen, cuda, True)
        ss, xx = (torch.full((v.numel() + 8,), float("nan"), device=cuda) for v in (s, xs))
        ss[off:off + N], xx[off:off + M] = s, xs
        out = torch.empty(M, N, dtype=F16, device=cuda)
        gpipes.i8_gemm_out(x, i8.pack(wq), ss[off:off + N], xs=xx[off:off + M], out=out)
        want, d = side(x, xs, (wq, s), None)
        check(out, want, d, F16)


@pytest.mark.gpu
def test_one_weight_for_both_sides(cuda):
    """The same tensors as gate and as the other weight, and calls one after the other with one output."""
    K, N = 272, 80
    gen = torch.Generator().manual_seed(1)
    wq, s = weight(K, N, gen, cuda)
    for M in (1, 20, 130):
        x, _ = rows(M, K, F16, gen, cuda)
        out = torch.empty(M, N, dtype=F16, device=cuda)
        for _ in range(3):
            gpipes.i8_gated_out(x, i8.pack(wq), s, i8.pack(wq), s, act="none", out=out)
        v, d = side(*i8.quantize_rows(x), (wq, s), None)
        check(out, v * v, 2 * d * v.abs() + d * d + U * v * v, F16)
