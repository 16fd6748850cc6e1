"""More operators of a language model's feed-forward half whose speed is measured: products in 8
bits, and experts.

Four operators, in the order in which a block uses them:

  linear   i8_gemm_out: act(x @ W + b), or x @ W + b + r, x and W in 8-bit integers
  gated    i8_gated_out: act(x @ Wg + bg) * (x @ Wu + bu)
  route    route_out: scores of the experts for each token, the k best of them and their weights
  experts  i8_experts_out: out[t] = r[t] + sum over j of w[t, j] * Down(act(x Wg) * (x Wu)) of expert ids[t, j]

A row is a token.  A row of x is taken as whole numbers q = round(127 x / max|x|) times max|x| /
127, ties to even; W[k, n] = s[n] * q[k, n].  Packed weights are [ceil(N / 16), ceil(K / 64),
1024] bytes, zeros behind K and N: byte 256 g + 16 j + i of block [a, b] is q[64 b + 16 g + i, 16 a + j].
Between an expert's two halves the activations have x's type, as between any two products.
"""
import math
import os
import sys

import torch

own = False  # whether run() calls the framework's operators, or computes them from elementary operations

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # The second layer of a block for one token: deep and narrow, the residual added.
        {"name": "linear_token_down", "op": "linear", "M": 1, "K": 16384, "N": 4096, "x8": False, "bias": False,
         "residual": True, "act": "none", "dtype": "bf16"},
        # Sixteen sequences being answered at once.
        {"name": "linear_batch", "op": "linear", "M": 16, "K": 8192, "N": 8192, "x8": False, "bias": False,
         "residual": False, "act": "none", "dtype": "fp16"},
        # A short prompt, sizes that no tile divides, the activation fused.
        {"name": "linear_ragged", "op": "linear", "M": 203, "K": 4080, "N": 4093, "x8": False, "bias": True,
         "residual": False, "act": "gelu_tanh", "dtype": "fp16"},
        # Prompts, their tokens in 8 bits already (the operator before has rounded them).
        {"name": "linear_prompts", "op": "linear", "M": 4096, "K": 4096, "N": 4096, "x8": True, "bias": False,
         "residual": False, "act": "none", "dtype": "bf16"},

        # The first half of a gated block for one token: the largest weights of a layer.
        {"name": "gated_token", "op": "gated", "M": 1, "K": 4096, "N": 16384, "x8": False, "bias": False, "act": "silu",
         "dtype": "bf16"},
        # A few sequences with a few guessed tokens each.
        {"name": "gated_batch", "op": "gated", "M": 48, "K": 2048, "N": 8192, "x8": False, "bias": True,
         "act": "gelu_tanh", "dtype": "fp16"},
        # Prompts through the first half of a block.
        {"name": "gated_prompts", "op": "gated", "M": 2040, "K": 4096, "N": 16384, "x8": False, "bias": False,
         "act": "silu", "dtype": "bf16"},

        # One token's choice: the call is short, latency counts.
        {"name": "route_token", "op": "route", "T": 1, "E": 64, "k": 6, "score": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "group_score": "max", "renorm": True, "scale": 1.0, "masked": 0, "dtype": "fp32"},
        # Prompts: sigmoid scores, a bias that balances the experts' loads, the best groups of experts first.
        {"name": "route_prompts", "op": "route", "T": 16384, "E": 128, "k": 6, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 3, "group_score": "top2", "renorm": True, "scale": 1.5, "masked": 0, "dtype": "fp32"},

        # One token: the chosen experts' weights, once.
        {"name": "experts_token", "op": "experts", "T": 1, "H": 2048, "F": 4096, "E": 16, "k": 4, "absent": 0,
         "residual": True, "act": "silu", "dtype": "bf16"},
        # A batch being answered, many small experts, a part of them on other devices.
        {"name": "experts_batch", "op": "experts", "T": 24, "H": 2048, "F": 1024, "E": 64, "k": 6, "absent": 16,
         "residual": False, "act": "silu", "dtype": "fp16"},
        # Prompts, few large experts.
        {"name": "experts_prompts", "op": "experts", "T": 4096, "H": 2048, "F": 8192, "E": 8, "k": 2, "absent": 0,
         "residual": True, "act": "silu", "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "route", "experts"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _spread(rng, 4, 512 // groups)
        top = rng.randint(1, groups)
        bias = rng.random() < 0.5
        return {"op": op, "T": _spread(rng, 1, min(16384, 2 ** 21 // E)), "E": E,
                "k": rng.randint(1, min(12, E // groups * top)), "score": rng.choice(["softmax", "sigmoid"]), "bias": bias,
                "groups": groups, "top_groups": top, "group_score": rng.choice(["max", "top2"]),
                "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 1.5, 2.5]),
                "masked": rng.choice([0, 0, E // 4]), "dtype": rng.choice(["fp32", "fp16", "bf16"])}
    act = rng.choice(["silu", "gelu_tanh", "relu", "sigmoid"])
    if op == "experts":
        H, F = _spread(rng, 256, 4096) // 16 * 16, _spread(rng, 256, 8192) // 16 * 16
        E = _spread(rng, 4, 64)
        while E * H * F > 2 ** 27:
            E, F = max(4, E // 2), max(256, F // 32 * 16)
        k = rng.randint(1, min(8, E))
        T = _spread(rng, 1, max(1, min(4096, 2 ** 37 // (k * H * F))))
        return {"op": op, "T": T, "H": H, "F": F, "E": E, "k": k, "absent": rng.choice([0, 0, E // 4]),
                "residual": rng.random() < 0.5, "act": act, "dtype": dtype}
    K = max(64, _spread(rng, 64, 16384) // 16 * 16)
    if rng.random() < 0.6:
        K = max(128, K // 128 * 128)
    N = _spread(rng, 64, 16384)
    if rng.random() < 0.7:
        N = max(64, N // 64 * 64)
    both = 2 if op == "gated" else 1
    while both * K * N > 2 ** 27:
        N = N // 2
    M = _spread(rng, 1, max(1, min(4096, 2 ** 37 // (both * K * N))))
    case = {"op": op, "M": M, "K": K, "N": N, "x8": rng.random() < 0.25, "bias": rng.random() < 0.5, "dtype": dtype}
    if op == "gated":
        return {**case, "act": act}
    residual = rng.random() < 0.5
    return {**case, "residual": residual, "act": "none" if residual else rng.choice(["none", act])}


def _weight(gen, K, N, experts=None):
    """A weight in 8 bits, packed, and its scales: q is spread as the quantised values of a normal weight are, the
    scales such that the weight's standard deviation is about 1 / sqrt(K)."""
    K64, N16 = -(-K // 64), -(-N // 16)
    packed = torch.empty((experts or 1, N16, K64, 1024), dtype=torch.int8, device=DEV)
    for one in packed:
        q = torch.zeros((K64 * 64, N16 * 16), dtype=torch.int8, device=DEV)
        q[:K, :N] = torch.randn(K, N, generator=gen, device=DEV).mul_(32).round_().clamp_(-127, 127)
        one.view(N16, K64, 4, 16, 16).copy_(q.view(K64, 4, 16, N16, 16).permute(3, 0, 1, 4, 2))
    s = (0.5 + torch.rand(experts or 1, N, generator=gen, device=DEV)) / (32 * math.sqrt(K))
    return (packed, s) if experts else (packed[0], s[0])


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=DEV).mul_(std).to(dt)

    st = {"case": case}
    op = case["op"]
    if op == "route":
        T, E = case["T"], case["E"]
        st["logits"] = normal(T, E, std=1.5)
        if case["masked"]:  # experts that are out of use
            st["logits"][:, torch.randperm(E, generator=gen, device=DEV)[:case["masked"]]] = -math.inf
        st["bias"] = torch.randn(E, generator=gen, device=DEV).mul_(0.1) if case["bias"] else None
        return st
    if op == "experts":
        T, H, F, E, k = (case[n] for n in "THFEk")
        st["x"] = normal(T, H)
        # some experts are chosen up to four times as often as others
        liked = torch.rand(T, E, generator=gen, device=DEV).log_().div_(1 + 3 * torch.rand(E, generator=gen, device=DEV))
        ids = liked.topk(k, 1).indices.to(torch.int32)
        away = torch.zeros(E, dtype=torch.bool, device=DEV)
        away[torch.randperm(E, generator=gen, device=DEV)[:case["absent"]]] = True
        st["ids"] = torch.where(away[ids.long()], -1, ids)
        w = torch.rand(T, k, generator=gen, device=DEV) + 0.1
        st["w"] = w / w.sum(1, keepdim=True)
        st["wg"], st["sg"] = _weight(gen, H, F, E)
        st["wu"], st["su"] = _weight(gen, H, F, E)
        st["wd"], st["sd"] = _weight(gen, F, H, E)
        st["r"] = normal(T, H) if case["residual"] else None
        return st
    M, K, N = case["M"], case["K"], case["N"]
    if case["x8"]:
        st["x"] = torch.randn(M, K, generator=gen, device=DEV).mul_(30).round_().clamp_(-127, 127).to(torch.int8)
        st["xs"] = torch.rand(M, generator=gen, device=DEV).add_(0.5).div_(30)
    else:
        st["x"], st["xs"] = normal(M, K), None
        st["x"][:, :: max(1, K // 5)] *= 8  # a few channels of activations are much larger than the others
    for side in ("g", "u") if op == "gated" else ("",):
        st["w" + side], st["s" + side] = _weight(gen, K, N)
        st["b" + side] = normal(N, std=0.5) if case["bias"] else None
    st["r"] = normal(M, N) if case.get("residual") else None
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    dt = TYPES[case["dtype"]]
    if case["op"] == "route":
        st["weights"] = torch.empty((case["T"], case["k"]), device=DEV)
        st["ids"] = torch.empty((case["T"], case["k"]), dtype=torch.int32, device=DEV)
    elif case["op"] == "experts":
        st["out"] = torch.empty_like(st["x"])
    else:
        st["out"] = torch.empty((case["M"], case["N"]), dtype=dt, device=DEV)
    if own:
        sys.path[:0] = [p for p in [os.path.join(os.getcwd(), "gpu-pipes_amd")] if p not in sys.path]
        import gpipes
        st["gpipes"] = gpipes
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    case, gp = st["case"], st["gpipes"]
    if case["op"] == "route":
        return gp.route_out(st["logits"], case["k"], bias=st["bias"], score=case["score"], groups=case["groups"],
                            top_groups=case["top_groups"], group_score=case["group_score"], renorm=case["renorm"],
                            scale=case["scale"], weights=st["weights"], ids=st["ids"])
    if case["op"] == "experts":
        return gp.i8_experts_out(st["x"], st["ids"], st["w"], st["wg"], st["sg"], st["wu"], st["su"], st["wd"], st["sd"],
                                 act=case["act"], r=st["r"], out=st["out"])
    if case["op"] == "linear":
        return gp.i8_gemm_out(st["x"], st["w"], st["s"], xs=st["xs"], b=st["b"], r=st["r"], act=case["act"],
                              out=st["out"])
    return gp.i8_gated_out(st["x"], st["wg"], st["sg"], st["wu"], st["su"], xs=st["xs"], bg=st["bg"], bu=st["bu"],
                           act=case["act"], out=st["out"])


def _act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    return v


def _rows8(x):
    """Rows as whole numbers and their scales, in 32 bits: 127 x is exact there, and no quotient that is not itself
    halfway lies so near to a half that its rounding could pass it."""
    v = x.float()
    top = v.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * v / top), 0 * v), top / 127


def _unpacked(packed, K, N):
    """The whole numbers [K, N] of a packed weight, in 32 bits."""
    N16, K64 = packed.shape[:2]
    return packed.view(N16, K64, 4, 16, 16).permute(1, 2, 4, 0, 3).reshape(K64 * 64, N16 * 16)[:K, :N].float()


def _product(q, xs, packed, s):
    return torch.matmul(q, _unpacked(packed, q.shape[1], s.shape[0])) * xs * s


def _run_plain(st):
    case = st["case"]
    dt = TYPES[case["dtype"]]
    if case["op"] == "route":
        return _route_plain(st)
    if case["op"] == "experts":
        x, ids, w = st["x"], st["ids"], st["w"]
        q, xs = _rows8(x)
        y = torch.zeros((*ids.shape, x.shape[1]), device=x.device)
        for e in range(case["E"]):
            t, j = torch.nonzero(ids == e, as_tuple=True)
            if t.numel() == 0:
                continue
            g = _act(_product(q[t], xs[t], st["wg"][e], st["sg"][e]), case["act"])
            h = (g * _product(q[t], xs[t], st["wu"][e], st["su"][e])).to(dt)
            y[t, j] = _product(*_rows8(h), st["wd"][e], st["sd"][e])
        y = (y * torch.where((ids >= 0) & (ids < case["E"]), w, 0 * w)[:, :, None]).sum(1)
        return (y if st["r"] is None else y + st["r"].float()).to(dt)
    q, xs = (st["x"].float(), st["xs"][:, None]) if case["x8"] else _rows8(st["x"])
    got = []
    for side in ("g", "u") if case["op"] == "gated" else ("",):
        v = _product(q, xs, st["w" + side], st["s" + side])
        if st["b" + side] is not None:
            v = v + st["b" + side].float()
        got.append(v)
    v = _act(got[0], case["act"])
    if case["op"] == "gated":
        return (v * got[1]).to(dt)
    return (v if st["r"] is None else v + st["r"].float()).to(dt)


def _route_plain(st):
    """In 64 bits: which of two experts is better hangs on the last bits of their scores."""
    case = st["case"]
    T, E, G = case["T"], case["E"], case["groups"]
    v = st["logits"].double()
    if case["score"] == "softmax":
        s = torch.exp(v - v.amax(1, keepdim=True))
        s = s / s.sum(1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-v))
    masked = torch.isinf(v)
    key = torch.where(masked, v, v if st["bias"] is None else s + st["bias"].double())
    if case["top_groups"] < G:
        rank = key
        if case["group_score"] == "top2":
            rank = torch.where(masked, v, s if st["bias"] is None else key)
        rank = torch.sort(rank.view(T, G, E // G), dim=2, descending=True).values
        best = rank[:, :, 0]
        if case["group_score"] == "top2" and E // G > 1:
            best = best + torch.where(torch.isinf(rank[:, :, 1]), 0, rank[:, :, 1])
        order = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=v.device)
        kept[torch.arange(T, device=v.device)[:, None], order] = True
        key = torch.where(kept.repeat_interleave(E // G, 1), key, -math.inf)
    got = torch.sort(key, dim=1, descending=True, stable=True)
    ids, none = got.indices[:, :case["k"]], torch.isinf(got.values[:, :case["k"]])
    w = torch.where(none, 0.0, torch.gather(s, 1, ids))
    if case["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return (w * case["scale"]).float(), torch.where(none, -1, ids).to(torch.int32)


def work(case):
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": T * E * (4 if case["dtype"] == "fp32" else 2) + (4 * E if case["bias"] else 0) + 8 * T * k,
                "flops": 4 * T * E}
    if case["op"] == "experts":
        T, H, F, E, k = (case[n] for n in "THFEk")
        here = (E - case["absent"]) / E
        used = E * here * (1 - (1 - k / E) ** T)  # experts that some token has chosen, about
        data = 2 * T * H * (3 if case["residual"] else 2) + 8 * T * k
        return {"bytes": int(used * (3 * H * F + 8 * F + 4 * H) + data), "flops": int(6 * T * k * here * H * F)}
    M, K, N = case["M"], case["K"], case["N"]
    both = 2 if case["op"] == "gated" else 1
    weight = K * N + 4 * N + (2 * N if case["bias"] else 0)
    data = (M * K + 4 * M if case["x8"] else 2 * M * K) + 2 * M * N * (2 if case.get("residual") else 1)
    return {"bytes": both * weight + data, "flops": 2 * both * M * N * K}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "sigmoid":
        return torch.sigmoid(v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def _exact_rows(x):
    """Each row as whole numbers times its scale."""
    v = x.double()
    scale = torch.linalg.vector_norm(v, ord=math.inf, dim=1, keepdim=True) / 127
    top = scale * 127
    safe = torch.where(top == 0, torch.ones_like(top), top)
    return (v * 127 / safe).round() * scale


def _exact_product(x, packed, s):
    """x @ W, about a thousand k at a time, the bytes taken out of their blocks by their places."""
    K, N = x.shape[1], s.shape[0]
    flat = packed.reshape(-1)
    n = torch.arange(N, device=x.device)
    out = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    for k0 in range(0, K, 1024):
        k = torch.arange(k0, min(K, k0 + 1024), device=x.device)
        block = (n // 16)[None, :] * packed.shape[1] + (k // 64)[:, None]
        place = (k % 64 // 16 * 256 + k % 16)[:, None] + (n % 16 * 16)[None, :]
        out += x[:, k] @ flat[block * 1024 + place].double()
    return out * s.double()


def _exact_route(case, st):
    """The k best one after the other, the first of equal ones each time."""
    T, E, G = case["T"], case["E"], case["groups"]
    v = st["logits"].double()
    masked = v == -math.inf
    s = torch.softmax(v, 1) if case["score"] == "softmax" else torch.sigmoid(v)
    s = torch.where(masked, torch.zeros_like(s), s)
    low = torch.full_like(v, -math.inf)
    key = torch.where(masked, low, v if st["bias"] is None else s + st["bias"].double())

    def first_best(a):
        top = a.max(1, keepdim=True).values
        at = torch.where(a == top, torch.arange(a.shape[1], device=a.device), a.shape[1]).min(1).values
        return top[:, 0], at

    rows = torch.arange(T, device=v.device)
    if case["top_groups"] < G:
        of = torch.where(masked, low, key if st["bias"] is not None or case["group_score"] == "max" else s)
        best = torch.empty((T, G), dtype=torch.float64, device=v.device)
        for g in range(G):
            part = of[:, g * (E // G):(g + 1) * (E // G)].clone()
            best[:, g], at = first_best(part)
            if case["group_score"] == "top2":
                part[rows, at] = -math.inf
                second = first_best(part)[0]
                best[:, g] += torch.where(second == -math.inf, torch.zeros_like(second), second)
        allowed = torch.zeros_like(masked)
        for _ in range(case["top_groups"]):
            at = first_best(best)[1]
            best[rows, at] = -math.inf
            allowed |= (torch.arange(E, device=v.device) // (E // G))[None, :] == at[:, None]
        key = torch.where(allowed, key, low)
    ids, w = [], []
    for _ in range(case["k"]):
        top, at = first_best(key)
        found = top > -math.inf
        w.append(torch.where(found, s[rows, at], torch.zeros_like(top)))
        ids.append(torch.where(found, at, torch.full_like(at, -1)))
        key = key.clone()
        key[rows, at] = -math.inf
    ids, w = torch.stack(ids, 1), torch.stack(w, 1)
    if case["renorm"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return w * case["scale"], ids.to(torch.int32)


def exact(case, seed):
    st = _inputs(case, seed)
    dt = TYPES[case["dtype"]]
    if case["op"] == "route":
        return _exact_route(case, st)
    if case["op"] == "experts":
        x = _exact_rows(st["x"])
        out = torch.zeros_like(x) if st["r"] is None else st["r"].double()
        for e in range(case["E"]):
            share = torch.where(st["ids"] == e, st["w"].double(), 0.0).sum(1)
            t = torch.nonzero((st["ids"] == e).any(1))[:, 0]
            if t.numel():
                h = _exact_act(_exact_product(x[t], st["wg"][e], st["sg"][e]), case["act"])
                h = (h * _exact_product(x[t], st["wu"][e], st["su"][e])).to(dt)
                out[t] += share[t][:, None] * _exact_product(_exact_rows(h), st["wd"][e], st["sd"][e])
        return out
    x = st["x"].double() * st["xs"].double()[:, None] if case["x8"] else _exact_rows(st["x"])
    got = []
    for side in ("g", "u") if case["op"] == "gated" else ("",):
        v = _exact_product(x, st["w" + side], st["s" + side])
        got.append(v if st["b" + side] is None else v + st["b" + side].double())
    v = _exact_act(got[0], case["act"])
    if case["op"] == "gated":
        return v * got[1]
    return v if st["r"] is None else v + st["r"].double()
