"""Choices of route_out that 32 bits cannot settle: rows that are not finite beside rows in doubt, and groups whose
sums 32 bits do not hold.

Compared with the definition, token by token in 64 bits, as the other tests of routing are.
"""
import math

import pytest
import torch

import gpipes
from test_route import check

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = math.inf, math.nan


def in_doubt(T, E, gen):
    """Rows whose choice hangs on bits that 32 do not hold: ties, saturated scores, steps of the last bit."""
    x = torch.randint(-1, 2, (T, E), generator=gen).float()
    x[1::4] = 40 + torch.randint(0, 30, x[1::4].shape, generator=gen)
    x[2::4] = 1 + torch.finfo(F32).eps * torch.randint(0, 8, x[2::4].shape, generator=gen)
    x[3::4] = 0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("E", [8, 16, 64, 200, 512, 1000])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_a_row_that_is_not_finite_among_rows_in_doubt(cuda, E, score, bias):
    """A NaN at each of the first 64 experts (every lane's first one), in rows that are in doubt themselves and beside
    such rows: NaN weights and the ids 0 .. k - 1 there, and the other rows' choices as they are without it."""
    gen = torch.Generator().manual_seed(E)
    n = min(E, 64)
    logits = in_doubt(2 * n, E, gen)
    b = torch.randint(0, 2, (E,), generator=gen) * 0.5 if bias else None
    for v in (NAN, INF) if score == "softmax" else (NAN,):
        x = logits.clone()
        x[torch.arange(n) * 2, torch.arange(n)] = v
        for k in sorted({min(6, E // 2), min(17, E // 2)}):
            check(cuda, x, k, bias=b, score=score)
            check(cuda, x, k, bias=b, score=score, renorm=False, groups=2, top_groups=1, group_score="top2")
            check(cuda, x, min(k, E // 4), bias=b, score=score, groups=4, top_groups=1)
    x = logits[:24].clone()
    x[::2] = NAN  # whole rows
    check(cuda, x, 3, bias=b, score=score, groups=4, top_groups=2, group_score="top2")


@pytest.mark.gpu
@pytest.mark.parametrize("E", [8, 64, 200, 600])
def test_a_bias_that_is_nan(cuda, E):
    """Every row is, but those in which the logit is -inf; at each lane's first expert."""
    gen = torch.Generator().manual_seed(E)
    logits = in_doubt(24, E, gen)
    for at in sorted({0, 1, 7, min(15, E - 1), min(40, E - 1), E - 1}):
        b = torch.zeros(E)
        b[at] = NAN
        x = logits.clone()
        x[::3, at] = -INF
        check(cuda, x, 4, bias=b, score="sigmoid")
        check(cuda, x, 2, bias=b, score="softmax", groups=2, top_groups=1, group_score="top2")


LOWEST, LARGEST = torch.finfo(F32).min, torch.finfo(F32).max


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(16, 4), (64, 8), (128, 8), (256, 64), (512, 8)])
def test_biases_of_the_lowest_value(cuda, E, groups, score):
    """A mask of float32's lowest value: two of them have no sum in 32 bits, but their groups can be chosen, and only
    an expert with a logit or bias of -inf cannot."""
    gen = torch.Generator().manual_seed(E)
    size = E // groups
    logits = torch.randn(20, E, generator=gen)
    for fill in (LOWEST, LOWEST / 2, LARGEST):
        b = torch.full((E,), fill)
        b[size:2 * size] = 0.1
        k = min(size + 2, 2 * size, 32)  # more than the group that is not masked has, up to what a call takes
        for top in (1, 2, groups - 1):
            for gs in ("top2", "max"):
                check(cuda, logits, min(k, top * size), bias=b, score=score, groups=groups, top_groups=top, group_score=gs)
        b[::3] = fill
        b[1] = LARGEST
        check(cuda, logits, k, bias=b, score=score, groups=groups, top_groups=2, group_score="top2")
        b[2::5] = -INF
        check(cuda, logits, k, bias=b, score=score, groups=groups, top_groups=2, group_score="top2")


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("B", [100.0, 1e4, 1e6, 1e9])
def test_groups_whose_biases_cancel(cuda, B, score):
    """Groups whose two best have biases of B and -B: a sum near 1 of terms that keep B 2^-24 in 32 bits.  Logits of
    neighbouring groups are close, so that the order of the sums hangs on what the terms' roundings take away."""
    gen = torch.Generator().manual_seed(int(B))
    for T, E, groups, top in ((3000, 4, 2, 1), (1000, 16, 4, 2), (300, 64, 16, 5), (100, 512, 32, 3)):
        size = E // groups
        logits = torch.randn(T, 1, E, generator=gen) * torch.tensor([1.0, 0.05]).repeat((T + 1) // 2)[:T, None, None]
        b = torch.full((groups, size), -2 * B)
        b[:, 0], b[:, 1] = B, -B
        b = b.flatten()
        check(cuda, logits[:, 0], min(3, size * top), bias=b, score=score, groups=groups, top_groups=top, group_score="top2")


@pytest.mark.gpu
@pytest.mark.parametrize("E,groups", [(16, 4), (128, 8), (512, 8)])
def test_a_token_keeps_its_choice_among_other_tokens(cuda, E, groups):
    """Rows in doubt, rows whose sums cancel and rows that are not finite: as in a call of their own."""
    gen = torch.Generator().manual_seed(E)
    size = E // groups
    x = torch.cat([in_doubt(24, E, gen), torch.randn(40, E, generator=gen)])[torch.randperm(64, generator=gen)]
    x[7, 3], x[30, 0] = NAN, -INF
    x = x.to(cuda)
    for B in (0.1, 1e4, 1e6, LARGEST):
        b = torch.full((groups, size), -B)
        b[:, 0] = B
        b = b.flatten().to(cuda)
        kw = dict(bias=b, score="sigmoid", groups=groups, top_groups=2, group_score="top2")
        w, ids = gpipes.route_out(x, 4, **kw)
        for t in range(64):
            one = gpipes.route_out(x[t:t + 1].clone(), 4, **kw)
            assert torch.equal(one[0].nan_to_num(7), w[t:t + 1].nan_to_num(7)) and torch.equal(one[1], ids[t:t + 1])
