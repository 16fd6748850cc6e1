"""Routing of tokens to experts: route_out.

The refusals need no GPU.  Results are compared with the definition, token by token in 64 bits: the
experts have to be the same, and a weight is off by half a step of fp32 and what 64 bits leave.
"""
import ctypes
import math

import pytest
import torch

import gpipes

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = math.inf, math.nan


# ---------------------------------------------------------------------------
# Without a GPU
# ---------------------------------------------------------------------------

def _call(T=4, E=64, k=6, logits=1 << 20, bias=0, score=0, groups=1, top=1, gscore=0, renorm=1, scale=1.0, w=1 << 21,
          ids=1 << 22, dtype=2):
    vp = ctypes.c_void_p
    P = lambda v: vp(v) if v else None  # noqa: E731
    return gpipes.lib.gp_route_out(T, E, k, P(logits), P(bias), score, groups, top, gscore, renorm, scale, P(w), P(ids),
                                   dtype, None)


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), -1), (dict(T=(1 << 30) + 1), -2), (dict(E=0), -2), (dict(E=1025), -2), (dict(k=0), -2), (dict(k=-1), -2),
    (dict(k=33), -2), (dict(E=5, k=6), -2), (dict(score=2), -1), (dict(score=-1), -1), (dict(gscore=2), -1),
    (dict(groups=0), -2), (dict(groups=5), -2), (dict(groups=128, E=256), -2), (dict(groups=8, top=0), -2),
    (dict(groups=8, top=9), -2), (dict(groups=16, top=1), -2), (dict(renorm=2), -1), (dict(scale=INF), -1),
    (dict(scale=NAN), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(logits=0), -1), (dict(w=0), -1),
    (dict(ids=0), -1), (dict(logits=2), -3), (dict(logits=1, dtype=0), -3), (dict(bias=2), -3), (dict(w=6), -3),
    (dict(ids=6), -3), (dict(ids=(1 << 21) + 92), -1), (dict(w=(1 << 20) + 1020), -1), (dict(ids=(1 << 20) - 92), -1),
    (dict(bias=(1 << 21) + 92), -1), (dict(bias=(1 << 22) - 252), -1)])
def test_argument_errors(kw, code):
    assert _call(**kw) == code
    assert gpipes.lib.gp_last_error().decode() != ""


def test_no_tokens_is_a_noop():
    assert _call(T=0, logits=0, w=0, ids=0) == 0
    assert gpipes.lib.gp_last_error().decode() == ""


def test_python_refuses():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        gpipes.route_out(x, 2)
    for bad in (None, 3, x.double(), x.int()):
        with pytest.raises(RuntimeError, match="logits"):
            gpipes.route_out(bad, 2)
    for k in (-1, 2.0, None, "2"):
        with pytest.raises(RuntimeError):
            gpipes.route_out(x, k)


# ---------------------------------------------------------------------------
# The definition
# ---------------------------------------------------------------------------

def route64(logits, k, bias=None, score="softmax", groups=1, top_groups=1, group_score="max", renorm=True, scale=1.0):
    T, E = logits.shape
    size = E // groups
    weights, ids = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1)
    for t in range(T):
        l = logits[t].double()
        out = l == -INF
        s = torch.softmax(l, 0) if score == "softmax" and not bool(out.all()) else torch.sigmoid(l)
        c = l if bias is None else s + bias.double()
        if bool((l.isnan() | (c.isnan() & ~out)).any()) or (score == "softmax" and bool((l == INF).any())):
            weights[t], ids[t] = NAN, torch.arange(k)
            continue
        c = torch.where(out, -INF, c).tolist()
        rank = c if bias is not None or group_score == "max" else torch.where(out, -INF, s).tolist()
        of = []
        for g in range(groups):
            best = sorted((v for v in rank[g * size:(g + 1) * size] if v > -INF), reverse=True)
            of.append(-INF if not best else best[0] if group_score == "max" else sum(best[:2]))
        chosen = sorted(range(groups), key=lambda g: (-of[g], g))[:top_groups]
        left = [e for e in range(E) if e // size in chosen and c[e] > -INF]
        left = sorted(left, key=lambda e: (-c[e], e))[:k]
        ids[t, :len(left)] = torch.tensor(left, dtype=torch.long)
        w = s[left]
        if renorm and left:
            if score == "softmax":  # relative to the best chosen one: the same quotients, no underflow
                w = torch.exp(l[left] - l[left].max())
            w = w / w.sum() if w.sum() > 0 else 0 * w
        weights[t, :len(left)] = w * scale
    return weights, ids


def check(cuda, logits, k, **kw):
    dev = {n: v.to(cuda) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    T = logits.shape[0]
    w = torch.full((T, k), 7.0, device=cuda)
    ids = torch.full((T, k), -7, dtype=torch.int32, device=cuda)
    got = gpipes.route_out(logits.to(cuda), k, weights=w, ids=ids, **dev)
    assert got[0] is w and got[1] is ids
    want, at = route64(logits, k, **kw)
    assert torch.equal(ids.cpu().long(), at)
    w = w.cpu().double()
    assert torch.equal(w.isnan(), want.isnan())
    ok = ~want.isnan()
    # half a step of fp32 (of its denormals), and 64-bit arithmetic: an exponent's argument up to 2^10 takes 2^-43
    assert bool(((w - want).abs()[ok] <= (2.0 ** -24 + 2.0 ** -40) * want.abs()[ok] + 2.0 ** -149).all())


FORMS = [dict(), dict(score="sigmoid"), dict(renorm=False), dict(score="sigmoid", renorm=False, scale=2.5)]


@pytest.mark.gpu
@pytest.mark.parametrize("E", [1, 2, 7, 8, 16, 17, 32, 60, 64, 65, 100, 128, 160, 256, 257, 512, 513, 1000, 1024])
@pytest.mark.parametrize("bias", [False, True])
def test_sizes(cuda, E, bias):
    gen = torch.Generator().manual_seed(E)
    i = 0
    for T in (1, 3, 16, 17, 37):
        for k in sorted({1, min(2, E), min(6, E), min(16, E), min(17, E), min(32, E)}):
            dt = (F32, BF16, F16)[i % 3]
            logits = (torch.randn(T, E, generator=gen) * 2).to(dt)
            b = torch.randn(E, generator=gen) * 0.2 if bias else None
            check(cuda, logits, k, bias=b, **FORMS[i % 4])
            i += 1


@pytest.mark.gpu
@pytest.mark.parametrize("E,groups", [(8, 2), (16, 16), (60, 4), (64, 8), (96, 3), (128, 8), (160, 32), (256, 8), (256, 64), (512, 16),
                                      (1024, 64), (1000, 5)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_groups(cuda, E, groups, bias, group_score):
    gen = torch.Generator().manual_seed(E + groups)
    for i, top in enumerate(sorted({1, groups // 2, groups - 1, groups})):
        logits = (torch.randn(21, E, generator=gen) * 2).to((BF16, F32, F16)[i % 3])
        b = torch.randn(E, generator=gen) * 0.2 if bias else None
        k = min(6, E // groups * top, 32)
        check(cuda, logits, k, bias=b, groups=groups, top_groups=top, group_score=group_score, **FORMS[i % 4])
        check(cuda, logits, k, bias=b, groups=groups, top_groups=top, group_score=group_score, **FORMS[(i + 1) % 4])


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_ties_go_to_the_lowest(cuda, score, bias):
    gen = torch.Generator().manual_seed(3)
    for E, groups in ((8, 1), (64, 8), (128, 4), (512, 8)):
        logits = torch.randint(-2, 3, (40, E), generator=gen).float()
        logits[0] = 0
        b = torch.randint(0, 2, (E,), generator=gen).float() if bias else None
        for gs in ("max", "top2"):
            check(cuda, logits, min(8, E), bias=b, score=score)
            check(cuda, logits, 2, bias=b, score=score, groups=groups, top_groups=max(1, groups // 2), group_score=gs)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_zeros_of_both_signs_and_steps_of_the_type(cuda, dt):
    """-0 ties with 0; logits one step of their type apart do not; 16-bit ones that nearly all tie."""
    gen = torch.Generator().manual_seed(4)
    for E in (8, 64, 128, 200, 512, 1000):
        logits = torch.zeros(12, E)
        logits[0, ::2] = -0.0
        logits[1] = -1.0
        logits[1, E // 2], logits[1, E // 3] = -0.0, 0.0
        eps = torch.finfo(dt).eps
        logits[2:6] = 1 + eps * torch.randint(0, 4, (4, E), generator=gen)
        logits[6:9] = -1 - eps * torch.randint(0, 4, (3, E), generator=gen)
        logits[9:] = torch.randn(3, E, generator=gen) * 1e-3 + 100
        logits = logits.to(dt)
        check(cuda, logits, 5)
        check(cuda, logits, 4, groups=2, top_groups=1)
        check(cuda, logits, 5, score="sigmoid", bias=torch.zeros(E))
        check(cuda, logits, 4, score="sigmoid", groups=2, top_groups=1, group_score="top2")


@pytest.mark.gpu
def test_scores_that_32_bits_cannot_tell_apart(cuda):
    """Saturated sigmoids, whose logits still differ, and biases that differ by less than a score's 32 bits keep."""
    logits = torch.tensor([[40.0, 41.0, 39.0, 60.0, 30.0, 42.0, 20.0, 50.0]])
    check(cuda, logits, 4, score="sigmoid")
    check(cuda, logits, 4, score="sigmoid", bias=torch.zeros(8))
    near = torch.tensor([[0.5, 0.5 + 2 ** -24, 0.5 - 2 ** -25, 0.5, -3.0, 0.5 + 2 ** -23, 0.0, 0.25]])
    check(cuda, near, 5, score="sigmoid", bias=torch.full((8,), 1.0))
    check(cuda, near, 5, score="softmax", bias=torch.full((8,), 64.0))
    check(cuda, near, 3, score="sigmoid", groups=2, top_groups=1, group_score="top2")


@pytest.mark.gpu
@pytest.mark.parametrize("E,groups", [(16, 4), (64, 8), (128, 8), (512, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_experts(cuda, E, groups, score, bias):
    """Rows with few experts left, with none, and groups of which nothing is left."""
    gen = torch.Generator().manual_seed(E)
    logits = torch.randn(24, E, generator=gen)
    b = torch.randn(E, generator=gen) if bias else None
    for t in range(24):
        logits[t, torch.randperm(E, generator=gen)[:E * t // 23]] = -INF  # the last row: none left
    logits[3, :E // groups] = -INF
    for gs in ("max", "top2"):
        for renorm in (True, False):
            check(cuda, logits, 4, bias=b, score=score, renorm=renorm)
            check(cuda, logits, 4, bias=b, score=score, renorm=renorm, groups=groups, top_groups=2, group_score=gs)
    if bias:
        b[::3] = -INF  # experts that the bias takes out
        check(cuda, logits, 4, bias=b, score=score, groups=groups, top_groups=2, group_score="top2")
        b[1] = INF
        check(cuda, logits, 4, bias=b, score=score, groups=groups, top_groups=2, group_score="top2")


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_rows_that_are_not_finite(cuda, score, bias):
    gen = torch.Generator().manual_seed(11)
    for E in (8, 64, 200, 600):
        logits = torch.randn(9, E, generator=gen)
        b = torch.randn(E, generator=gen) if bias else None
        logits[1, E - 1] = NAN
        logits[4, 0] = INF
        logits[6] = NAN
        logits[7] = INF
        check(cuda, logits, 4, bias=b, score=score)
        check(cuda, logits, 4, bias=b, score=score, renorm=False, groups=2, top_groups=1, group_score="top2")
        check(cuda, logits, 4, bias=b, score=score, groups=4, top_groups=2)
    if bias:
        b = torch.randn(64, generator=gen)
        b[5] = NAN
        logits = torch.randn(4, 64, generator=gen)
        logits[1, 5] = -INF
        check(cuda, logits, 4, bias=b, score=score)


@pytest.mark.gpu
def test_large_and_small_logits(cuda):
    gen = torch.Generator().manual_seed(5)
    for score in ("softmax", "sigmoid"):
        for top in (60.0, 600.0, 3e4):
            logits = torch.randn(16, 64, generator=gen) * top
            check(cuda, logits.clamp(-700, 700) if score == "sigmoid" else logits, 6, score=score)
            check(cuda, logits.clamp(-700, 700), 6, score=score, renorm=False)
    check(cuda, torch.full((2, 16), -3e38), 4)
    check(cuda, torch.full((2, 16), -800.0), 4, score="sigmoid")  # scores of 0, and their sum


@pytest.mark.gpu
def test_many_tokens(cuda):
    """Every token of a large call gives what it gives in a small one."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    for T, E, dt in ((100001, 64, BF16), (20001, 128, F32), (5003, 512, F16)):
        logits = torch.randn(T, E, generator=gen, device=cuda).to(dt)
        bias = torch.randn(E, generator=gen, device=cuda) * 0.1
        kw = dict(bias=bias, score="sigmoid", groups=8, top_groups=3, group_score="top2")
        w, ids = gpipes.route_out(logits, 6, **kw)
        for at in (0, T // 2, T - 40):
            part = gpipes.route_out(logits[at:at + 40].clone(), 6, **kw)
            assert torch.equal(part[0], w[at:at + 40]) and torch.equal(part[1], ids[at:at + 40])
            check(cuda, logits[at:at + 40].cpu(), 6, **{**kw, "bias": bias.cpu()})


@pytest.mark.gpu
def test_tokens_behind_the_last_stay(cuda):
    for T, E in ((1, 64), (5, 128), (17, 512)):
        w = torch.full((T + 8, 4), 3.0, device=cuda)
        ids = torch.full((T + 8, 4), 9, dtype=torch.int32, device=cuda)
        gpipes.route_out(torch.randn(T, E, device=cuda), 4, weights=w[4:T + 4], ids=ids[4:T + 4])
        assert bool((w[:4] == 3).all()) and bool((w[T + 4:] == 3).all())
        assert bool((ids[:4] == 9).all()) and bool((ids[T + 4:] == 9).all())


@pytest.mark.gpu
def test_python_refusals(cuda):
    x = torch.zeros(3, 16, device=cuda)
    w, ids = torch.zeros(3, 2, device=cuda), torch.zeros(3, 2, dtype=torch.int32, device=cuda)
    for args, kw, what in (
            ((x.t(), 2), {}, "contiguous"), ((x[0], 2), {}, "2-D"), ((x, 0), {}, "k must"), ((x, 17), {}, "k must"),
            ((x, -1), {}, "k must"), ((x, 2.0), {}, "k must"), ((x, 2), dict(bias=x[0].half()), "float32"),
            ((x, 2), dict(bias=x), "bias must have shape"), ((x, 2), dict(bias=x[0].cpu()), "CUDA"),
            ((x, 2), dict(weights=ids), "float32"), ((x, 2), dict(ids=w), "int32"), ((x, 3), dict(weights=w), "weights"),
            ((x, 2), dict(ids=ids.long()), "int32"), ((x, 2), dict(score="foo"), "invalid"), ((x, 2), dict(score=7), "score"),
            ((x, 2), dict(groups=3), "groups"), ((x, 2), dict(groups=16, top_groups=1), "k must"),
            ((x, 2), dict(group_score="foo"), "invalid"), ((x, 2), dict(scale=INF), "scale"), ((x, 2), dict(renorm=2), "renorm"),
            ((x, 2), dict(scale=None), "invalid"), ((x, 2), dict(groups=2.0), "invalid")):
        with pytest.raises(RuntimeError, match=what):
            gpipes.route_out(*args, **kw)
    w, ids = gpipes.route_out(x[:0], 2)
    assert w.shape == ids.shape == (0, 2)


@pytest.mark.gpu
def test_graph_and_streams(cuda):
    sets = []
    for T, E in ((1, 64), (4097, 128)):
        x = torch.randn(T, E, device=cuda)
        b = torch.randn(E, device=cuda) * 0.1
        kw = dict(bias=b, score="sigmoid", groups=8, top_groups=2, group_score="top2")
        w, ids = gpipes.route_out(x, 4, **kw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gpipes.route_out(x, 4, weights=w, ids=ids, **kw)
        sets.append((x, kw, w, ids, g, torch.cuda.Stream(cuda)))
    for _ in range(3):
        want = []
        for x, kw, w, ids, g, st in sets:
            x.normal_()
            want.append(gpipes.route_out(x, 4, **kw))
            w.zero_(), ids.zero_()
        torch.cuda.synchronize()
        for x, kw, w, ids, g, st in sets:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (x, kw, w, ids, g, st), (ww, wi) in zip(sets, want):
            assert torch.equal(w, ww) and torch.equal(ids, wi)


@pytest.mark.gpu
def test_more_tokens_than_a_launch_of_one_axis_holds(cuda):
    T = (1 << 28) + 5
    logits = torch.empty(T, 2, dtype=F16, device=cuda)
    logits[:, 0] = 0
    logits[:, 1] = torch.arange(T, device=cuda) % 3 - 1  # -1; 0, where the lower expert is first; 1
    weights, ids = gpipes.route_out(logits, 1, score="sigmoid", renorm=False)
    assert torch.equal(ids[:, 0] == 1, logits[:, 1] == 1) and bool((ids >= 0).all())
    low, high = 0.5, 1 / (1 + 2.718281828459045 ** -1)
    for n, w in ((0, low), (1, high)):  # a weight is the score in 64 bits, rounded once: 2^-24 of it
        assert bool(((weights[ids == n].double() - w).abs() <= 2.0 ** -24 * w * (1 + 1e-6)).all())
