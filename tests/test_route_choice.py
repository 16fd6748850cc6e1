"""Choices of route_out that 32 bits cannot settle: rows that are not finite beside rows in doubt.

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
