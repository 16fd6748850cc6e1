"""The feed-forward block of experts in 8-bit integers: i8_experts_out.

The refusals need no GPU.  An expert's first half is i8_gated_out's to the bit (whole sums, and one
arithmetic behind them), which has its own tests; what follows it is compared with the formulas in 64
bits, to a bound that holds the roundings of fp32 and the result's own.
"""
import ctypes

import pytest
import torch

import gpipes
from gpipes import i8

F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24
NAN = float("nan")


# ---------------------------------------------------------------------------
# Without a GPU
# ---------------------------------------------------------------------------

AT = dict(x=1 << 20, ids=2 << 20, w=3 << 20, wg=1 << 30, sg=4 << 20, wu=2 << 30, su=5 << 20, wd=3 << 30, sd=6 << 20,
          r=7 << 20, out=8 << 20)


def _call(T=4, H=256, F=512, E=8, k=2, act=4, ws=0, wsb=0, dtype=0, **at):
    P = lambda n: ctypes.c_void_p({**AT, **at}[n]) if {**AT, **at}[n] else None  # noqa: E731
    return gpipes.lib.gp_i8_experts_out(T, H, F, E, k, P("x"), P("ids"), P("w"), P("wg"), P("sg"), P("wu"), P("su"),
                                        P("wd"), P("sd"), act, P("r"), P("out"), ctypes.c_void_p(ws) if ws else None, wsb,
                                        dtype, None)


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), -1), (dict(T=(1 << 21) + 1), -2), (dict(T=1 << 21, H=1024), -2), (dict(H=0), -2), (dict(H=24), -2),
    (dict(H=131072), -2), (dict(F=0), -2), (dict(F=8), -2), (dict(F=131072), -2), (dict(H=65536, F=32768), -2),
    (dict(E=0), -2), (dict(E=1025), -2), (dict(k=0), -2), (dict(k=33), -2), (dict(act=5), -1), (dict(act=-1), -1),
    (dict(dtype=2), -1), (dict(wsb=-1), -1), (dict(wsb=64), -1), (dict(ws=24, wsb=64), -3)]
    + [({n: 0}, -1) for n in AT if n != "r"]
    + [({n: AT[n] + 8}, -3) for n in ("x", "wg", "wu", "wd", "r", "out")]
    + [({n: AT[n] + 2}, -3) for n in ("ids", "w", "sg", "su", "sd")])
def test_argument_errors(kw, code):
    assert _call(**kw) == code
    assert gpipes.lib.gp_last_error().decode() != ""


SIZES = dict(x=2048, ids=32, w=32, wg=8 * 256 * 512, sg=8 * 2048, wu=8 * 256 * 512, su=8 * 2048, wd=8 * 256 * 512, sd=8 * 1024)


@pytest.mark.parametrize("what", SIZES)
def test_overlaps_are_refused(what):
    """out and the workspace over the first and the last 16 bytes of every other operand."""
    at = 5 << 30
    for lo in (at - 2048 + 16, at + SIZES[what] - 16):
        assert _call(**{what: at, "out": lo}) == -1
        assert "out must not overlap" in gpipes.lib.gp_last_error().decode()
        assert _call(**{what: at}, ws=lo, wsb=2048) == -1
        assert "workspace must not overlap" in gpipes.lib.gp_last_error().decode()


def test_overlaps_of_residual_and_workspace():
    assert _call(r=AT["out"] + 16) == -1
    assert _call(ws=AT["r"] + 2032, wsb=16) == -1
    assert _call(ws=AT["out"] + 2032, wsb=16) == -1


def test_no_tokens_is_a_noop():
    assert _call(T=0, x=0, ids=0, w=0, out=0) == 0
    assert gpipes.lib.gp_last_error().decode() == ""
    assert gpipes.lib.gp_i8_experts_workspace_bytes(0, 64, 64, 4, 2) == 0


@pytest.mark.parametrize("args,code", [((-1, 64, 64, 4, 2), -1), ((4, 72, 64, 4, 2), -2), ((4, 64, 72, 4, 2), -2),
                                       ((4, 64, 64, 0, 2), -2), ((4, 64, 64, 4, 0), -2)])
def test_workspace_arguments(args, code):
    assert gpipes.lib.gp_i8_experts_workspace_bytes(*args) == code


def test_python_refuses():
    x = torch.zeros(1, 64, dtype=F16)
    w = torch.zeros(2, 4, 1, 1024, dtype=torch.int8)
    s = torch.zeros(2, 64)
    args = (torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1), w, s, w, s, w, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.i8_experts_out(x, *args)
    with pytest.raises(RuntimeError):
        gpipes.i8_experts_out(None, *args)


# ---------------------------------------------------------------------------
# On a GPU
# ---------------------------------------------------------------------------

def experts(E, H, F, gen, dev):
    """Packed weights and scales (up, gate, down), q over all of -128 .. 127."""
    p = {}
    for n, K, N in (("g", H, F), ("u", H, F), ("d", F, H)):
        q = torch.randint(-128, 128, (E, K, N), generator=gen, dtype=torch.int16).to(torch.int8)
        p["w" + n] = i8.pack(q).to(dev)
        p["s" + n] = ((torch.rand(E, N, generator=gen) + 0.5) / (74 * K ** 0.5)).to(dev)
    return p


def run(x, ids, w, p, act="silu", r=None, out=None):
    return gpipes.i8_experts_out(x, ids, w, p["wg"], p["sg"], p["wu"], p["su"], p["wd"], p["sd"], act=act, r=r, out=out)


def want64(x, ids, w, p, act, r):
    """out in 64 bits behind i8_gated_out, and the bound of fp32's roundings: three for a product, one for its weight
    and one for each sum that it then is in."""
    T, H = x.shape
    E, F = p["sg"].shape
    k = ids.shape[1]
    v = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    d = torch.zeros_like(v)
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        h = gpipes.i8_gated_out(x[t].contiguous(), p["wg"][e], p["sg"][e], p["wu"][e], p["su"][e], act=act)
        q, hs = i8.quantize_rows(h)
        y = (q.double() @ i8.unpack(p["wd"][e], F, H).double()) * p["sd"][e].double() * hs.double()[:, None]
        y = y * w[t, j].double()[:, None]
        v.index_put_((t,), y, accumulate=True)
        d.index_put_((t,), (4 + k) * U * y.abs(), accumulate=True)
    if r is not None:
        v = v + r.double()
        d = d + U * v.abs()
    return v, d


def check(out, want, bound, dt):
    eps, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == F16 else 2.0 ** -134
    err = (out.double() - want).abs()
    tol = eps * (want.abs() + bound) + bound + tiny
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), (err / tol)[bad].max().item(), bad.nonzero()[:3].tolist())


def tokens(T, H, E, k, dt, gen, dev, how="spread"):
    x = torch.randn(T, H, generator=gen)
    x[:, :: max(1, H // 3)] *= 6
    ids = torch.rand(T, E, generator=gen).topk(min(k, E), 1).indices
    if k > E:
        ids = torch.randint(0, E, (T, k), generator=gen)
    if how == "one":
        ids[:] = E - 1
    elif how == "twice":
        ids = torch.randint(0, E, (T, 1), generator=gen).expand(T, k).clone()
    elif how == "some":  # none, too large, negative
        ids = torch.where(torch.rand(T, k, generator=gen) < 0.4, torch.randint(-3, 0, (T, k), generator=gen), ids)
        ids = torch.where(torch.rand(T, k, generator=gen) < 0.1, E + 5, ids)
        ids[0] = -1  # a token without an expert
    w = torch.rand(T, k, generator=gen) - 0.2
    return x.to(dt).to(dev), ids.to(torch.int32).to(dev), w.to(dev)


def case(cuda, T, H, F, E, k, dt, how="spread", act="silu", residual=False, p=None):
    gen = torch.Generator().manual_seed(T * 3 + H + F * 5 + E * 7 + k)
    p = p or experts(E, H, F, gen, cuda)
    x, ids, w = tokens(T, H, E, k, dt, gen, cuda, how)
    r = torch.randn(T, H, generator=gen).to(dt).to(cuda) if residual else None
    out = run(x, ids, w, p, act, r, torch.full((T, H), NAN, dtype=dt, device=cuda))
    check(out, *want64(x, ids, w, p, act, r), dt)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 3, 5, 8, 16, 33, 64, 100, 200, 500])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_sizes(cuda, T, dt):
    hows = ("spread", "some", "one", "twice")
    i = 0
    for H, F in ((16, 16), (64, 48), (144, 272), (272, 528)):
        for E, k in ((1, 1), (4, 2), (7, 3), (16, 6), (64, 8)):
            case(cuda, T, H, F, E, k, dt, hows[i % 4], ("silu", "gelu_tanh", "relu", "sigmoid", "none")[i % 5], i % 2 == 0)
            i += 1


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,F,E,k", [
    (1, 2048, 4096, 16, 4), (1, 4096, 1040, 8, 8), (1, 1024, 8192, 4, 1), (1, 528, 16384, 3, 2), (1, 16384, 528, 3, 2),
    (1, 2064, 1040, 9, 9), (1, 1024, 1024, 40, 17), (1, 1024, 2048, 40, 32), (2, 2048, 1024, 16, 6), (4, 1024, 4096, 8, 2),
    (24, 2048, 1024, 64, 6), (300, 1024, 2064, 8, 2), (700, 1040, 1024, 4, 2), (2000, 528, 1040, 8, 2), (3000, 1024, 528, 3, 3),
    (5000, 144, 80, 300, 2), (1000, 64, 64, 1024, 5), (40, 256, 256, 1, 32)])
@pytest.mark.parametrize("how", ["spread", "some"])
def test_wide_deep_and_many(cuda, T, H, F, E, k, how):
    case(cuda, T, H, F, E, k, BF16 if T % 2 else F16, how, residual=T % 3 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,F,E,k", [(4096, 1024, 2048, 4, 2), (4096, 2048, 4096, 8, 2), (700, 1024, 1040, 16, 2), (1000, 272, 2064, 30, 1)])
@pytest.mark.parametrize("how", ["spread", "some", "one"])
def test_every_size_of_tile(cuda, T, H, F, E, k, how):
    """Both halves on tiles of 256, of 256 and 128, of 128 and 64 rows; all tokens with one expert too."""
    case(cuda, T, H, F, E, k, BF16, how, residual=True)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 50, 400, 1500])
def test_uneven_experts(cuda, T):
    """All tokens with one expert, all but one, and none with any."""
    H, F, E = 272, 144, 5
    gen = torch.Generator().manual_seed(T)
    p = experts(E, H, F, gen, cuda)
    case(cuda, T, H, F, E, 2, F16, "one", p=p)
    x, ids, w = tokens(T, H, E, 2, F16, gen, cuda)
    ids[:] = 2
    ids[T // 2, 1] = 0
    check(run(x, ids, w, p), *want64(x, ids, w, p, "silu", None), F16)
    ids[:] = -1
    assert not bool(run(x, ids, w, p).any())
    r = torch.randn(T, H, generator=gen).to(F16).to(cuda)
    assert torch.equal(run(x, ids, w, p, r=r), r)
    keep = r.clone()
    assert run(x, ids, w, p, r=r, out=r) is r and torch.equal(r, keep)  # in place


@pytest.mark.gpu
def test_a_token_keeps_its_bits_among_other_tokens(cuda):
    H, F, E, k = 528, 272, 6, 3
    gen = torch.Generator().manual_seed(2)
    p = experts(E, H, F, gen, cuda)
    x, ids, w = tokens(2000, H, E, k, BF16, gen, cuda)
    full = run(x, ids, w, p)
    for n in (1, 2, 3, 4, 5, 8, 16, 33, 100, 300, 700):
        part = run(x[-n:].contiguous(), ids[-n:].contiguous(), w[-n:].contiguous(), p)
        assert torch.equal(part, full[-n:])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 6, 40, 300])
def test_tokens_that_are_not_finite(cuda, T):
    """NaN in their rows alone: of x, of a weight, and of a first half that passes fp16's range; what an id of no
    expert weighs does not count."""
    H, F, E, k = 272, 144, 4, 2
    gen = torch.Generator().manual_seed(T)
    p = experts(E, H, F, gen, cuda)
    x, ids, w = tokens(T, H, E, k, F16, gen, cuda)
    good = run(x, ids, w, p)
    for kind in ("nan", "inf", "weight", "half"):
        x2, w2, p2, ids2 = x.clone(), w.clone(), dict(p), ids.clone()
        at = T // 2
        if kind == "nan":
            x2[at, 5] = NAN
        elif kind == "inf":
            x2[at, H - 1] = -float("inf")
        elif kind == "weight":
            w2[at, 0] = NAN
        else:
            x2[at] = x2[at].sign() * 60000
            p2["su"] = p["su"] * 1e3
        out = run(x2, ids2, w2, p2)
        assert bool(out[at].isnan().all())
        if kind != "half":
            rest = torch.arange(T, device=cuda) != at
            assert torch.equal(out[rest], good[rest])
    ids[0, 0], w[0, 0] = -1, NAN
    assert bool(torch.isfinite(run(x, ids, w, p)).all())
    x[0] = 0
    assert not bool(run(x, ids, w, p)[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_close_to_64_bits_as_a_whole(cuda, dt):
    """Both halves in 64 bits.  A first half's value near a rounding's border may be one step of its type off, and a
    whole number of it then one off; both are rare, so that as a whole the error is that of the result's rounding
    (at most half a step, its rms 0.58 of that relative to values between powers of two)."""
    for T, H, F, E, k in ((1, 1024, 2048, 8, 4), (20, 512, 1024, 16, 4), (400, 512, 1024, 4, 2)):
        gen = torch.Generator().manual_seed(T)
        p = experts(E, H, F, gen, cuda)
        x, ids, w = tokens(T, H, E, k, dt, gen, cuda)
        out = run(x, ids, w, p).double()
        q, xs = i8.quantize_rows(x)
        want = torch.zeros(T, H, dtype=torch.float64, device=cuda)
        for e in range(E):
            t, j = torch.nonzero(ids == e, as_tuple=True)
            if t.numel() == 0:
                continue
            up = [(q[t].double() @ i8.unpack(p["w" + n][e], H, F).double()) * p["s" + n][e].double() * xs[t].double()[:, None]
                  for n in "gu"]
            hq, hs = i8.quantize_rows((up[0] * torch.sigmoid(up[0]) * up[1]).to(dt))
            y = (hq.double() @ i8.unpack(p["wd"][e], F, H).double()) * p["sd"][e].double() * hs.double()[:, None]
            want.index_put_((t,), y * w[t, j].double()[:, None], accumulate=True)
        assert (out - want).norm() / want.norm() <= torch.finfo(dt).eps / 2


@pytest.mark.gpu
def test_python_refusals(cuda):
    gen = torch.Generator().manual_seed(6)
    p = experts(3, 64, 48, gen, cuda)
    x, ids, w = tokens(5, 64, 3, 2, F16, gen, cuda)
    ok = dict(x=x, ids=ids, weights=w, wq_g=p["wg"], scales_g=p["sg"], wq_u=p["wu"], scales_u=p["su"], wq_d=p["wd"],
              scales_d=p["sd"])
    for kw, what in (
            (dict(x=x.float()), "float16"), (dict(x=x[0]), "2-D"), (dict(x=x.t()), "contiguous"), (dict(ids=ids.long()), "int32"),
            (dict(ids=ids[0]), r"\[T, k\]"), (dict(ids=ids[:3]), "ids must have shape"), (dict(weights=w.half()), "float32"),
            (dict(weights=w[:, :1].contiguous()), "weights must have shape"), (dict(wq_g=p["wg"][:2]), "wq_g"),
            (dict(wq_u=p["wd"]), "wq_u"), (dict(wq_d=p["wu"]), "wq_d"), (dict(scales_g=p["sg"][0]), r"\[E, F\]"),
            (dict(scales_u=p["sd"]), "scales_u"), (dict(scales_d=p["su"]), "scales_d"), (dict(r=x[:2]), "r must"),
            (dict(out=x.to(BF16)), "float16"), (dict(out=x), "overlap"), (dict(act="foo"), "invalid"), (dict(act=7), "activation"),
            (dict(ids=ids[:, :0], weights=w[:, :0]), "topk"), (dict(scales_g=p["sg"].cpu()), "CUDA"),
            (dict(scales_g=p["sg"][:, :40].contiguous()), "multiples of 16"), (dict(ids=None), "ids")):
        with pytest.raises(RuntimeError, match=what):
            gpipes.i8_experts_out(**{**ok, **kw})
    assert gpipes.i8_experts_out(**{**ok, "x": x[:0], "ids": ids[:0], "weights": w[:0]}).shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40, 600])
def test_graphs_and_streams(cuda, T):
    """Two captured calls replayed at once on two streams, with other tokens, experts and weights each time."""
    H, F, E, k = 272, 528, 8, 3
    gen = torch.Generator().manual_seed(T)
    p = experts(E, H, F, gen, cuda)
    sets = []
    for _ in range(2):
        x, ids, w = tokens(T, H, E, k, BF16, gen, cuda)
        out = run(x, ids, w, p)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(2):
                run(x, ids, w, p, out=out)
        sets.append((x, ids, w, out, g, torch.cuda.Stream(cuda)))
    for how in ("spread", "one", "some"):
        want = []
        for x, ids, w, out, g, st in sets:
            for to, v in zip((x, ids, w), tokens(T, H, E, k, BF16, gen, cuda, how)):
                to.copy_(v)
            want.append(run(x, ids, w, p))
            out.zero_()
        torch.cuda.synchronize()
        for x, ids, w, out, g, st in sets:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (x, ids, w, out, g, st), v in zip(sets, want):
            assert torch.equal(out, v)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 12, 260])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_block(cuda, T, dt):
    """The feed-forward half of a block as a program runs it: norm with residual, router, experts with a shared one
    beside them, norm; eager, and captured and replayed with other tokens."""
    H, F, E, k = 512, 144, 128, 4  # gemm_out's columns are a multiple of 128
    gen = torch.Generator().manual_seed(T)
    p = experts(E, H, F, gen, cuda)
    n = lambda *sh: torch.randn(*sh, generator=gen).to(dt).to(cuda)  # noqa: E731
    router = (n(H, E) * H ** -0.5).contiguous()
    bias = torch.randn(E, generator=gen).to(cuda) * 0.1
    gamma = [1 + 0.1 * n(H) for _ in range(2)]
    x, y = n(T, H), n(T, H)
    bufs = {c: torch.empty(T, H, dtype=dt, device=cuda) for c in ("h", "z", "s", "o", "h2", "z2")}
    bufs["a"] = torch.empty(T, F, dtype=dt, device=cuda)
    bufs["l"] = torch.empty(T, E, dtype=dt, device=cuda)
    bufs["w"] = torch.empty(T, k, device=cuda)
    bufs["ids"] = torch.empty(T, k, dtype=torch.int32, device=cuda)

    def step():
        gpipes.residual_norm_out(x, y, gamma=gamma[0], h=bufs["h"], out=bufs["z"])
        gpipes.gemm_out(bufs["z"], router, out=bufs["l"])
        gpipes.route_out(bufs["l"], k, bias=bias, score="sigmoid", groups=4, top_groups=2, group_score="top2", scale=1.5,
                         weights=bufs["w"], ids=bufs["ids"])
        gpipes.i8_gated_out(bufs["z"], p["wg"][0], p["sg"][0], p["wu"][0], p["su"][0], out=bufs["a"])
        gpipes.i8_gemm_out(bufs["a"], p["wd"][0], p["sd"][0], out=bufs["s"])
        run(bufs["z"], bufs["ids"], bufs["w"], p, r=bufs["s"], out=bufs["o"])
        gpipes.residual_norm_out(bufs["h"], bufs["o"], gamma=gamma[1], h=bufs["h2"], out=bufs["z2"])

    def close():
        d = lambda t: t.double()  # noqa: E731
        rms = lambda v, g: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * d(g)  # noqa: E731
        h = d(x) + d(y)
        assert (d(bufs["z"]) - rms(h, gamma[0])).norm() <= 2 * torch.finfo(dt).eps * d(bufs["z"]).norm()
        l = d(bufs["l"])
        assert (l - d(bufs["z"]) @ d(router)).norm() <= torch.finfo(dt).eps * l.norm()
        c = torch.sigmoid(l) + d(bias)
        groups = c.view(T, 4, E // 4).topk(2, 2).values.sum(2).topk(2, 1).indices
        keep = torch.zeros(T, 4, dtype=torch.bool, device=cuda)
        keep[torch.arange(T, device=cuda)[:, None], groups] = True
        c = torch.where(keep.repeat_interleave(E // 4, 1), c, -1.0)
        ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(ids, bufs["ids"].long())
        w = torch.gather(torch.sigmoid(l), 1, ids)
        w = w / w.sum(1, keepdim=True) * 1.5
        assert bool(((d(bufs["w"]) - w).abs() <= 2 * U * w).all())
        want, bound = want64(bufs["z"], bufs["ids"], bufs["w"], p, "silu", bufs["s"])
        check(bufs["o"], want, bound, dt)
        h2 = d(bufs["h"]) + d(bufs["o"])
        # h goes to memory in 16 bits; the norm takes its sum before that
        assert (d(bufs["z2"]) - rms(h2, gamma[1])).norm() <= 2 * torch.finfo(dt).eps * d(bufs["z2"]).norm()

    step()
    torch.cuda.synchronize()
    close()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        x.copy_(n(T, H)), y.copy_(n(T, H))
        step()
        eager = {c: v.clone() for c, v in bufs.items()}
        for v in bufs.values():
            v.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(v, eager[c]) for c, v in bufs.items())
        close()


@pytest.mark.gpu
def test_a_short_workspace_is_refused(cuda):
    need = gpipes.lib.gp_i8_experts_workspace_bytes(40, 64, 64, 4, 2)
    t = {c: torch.zeros(n, dtype=torch.uint8, device=cuda) for c, n in dict(
        x=5120, ids=320, w=320, wg=4 * 4096, sg=1024, wu=4 * 4096, su=1024, wd=4 * 4096, sd=1024, out=5120, ws=need).items()}
    at = {c: v.data_ptr() for c, v in t.items() if c != "ws"}
    assert need > 0 and _call(T=40, H=64, F=64, E=4, ws=t["ws"].data_ptr(), wsb=need - 1, **{**at, "r": 0}) == -1
    assert str(need) in gpipes.lib.gp_last_error().decode()
    assert _call(T=40, H=64, F=64, E=4, ws=t["ws"].data_ptr(), wsb=need, **{**at, "r": 0}) == 0
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_more_pairs_than_a_launch_of_one_axis_holds(cuda):
    """2^26 pairs: their first and last tokens have the bits that they have in calls by themselves."""
    T, H, F, E, k = 1 << 21, 16, 16, 32, 32
    p = experts(E, H, F, torch.Generator().manual_seed(5), cuda)
    gen = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(T, H, generator=gen, device=cuda).to(F16)
    ids = torch.randint(-1, E, (T, k), generator=gen, device=cuda, dtype=torch.int32)
    w = torch.rand(T, k, generator=gen, device=cuda)
    got = run(x, ids, w, p)
    for lo in (0, T // 2, T - 1000):
        part = slice(lo, lo + 1000)
        assert torch.equal(got[part], run(x[part].contiguous(), ids[part].contiguous(), w[part].contiguous(), p))
