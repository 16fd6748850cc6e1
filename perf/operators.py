"""The operators of a language model's feed-forward half whose speed is measured.

Three operators, in the order in which a block uses them:

  norm    residual_norm_out: h = x + scale * act(gate) * post_norm(y), out = pre_norm(h)
  linear  q4_gemm_out: act(x @ W + b), or x @ W + b + r, W in 4 bits with a scale (and a zero) for each group of k
  gated   q4_gated_out: act(x @ Wg + bg) * (x @ Wu + bu), both weights in 4 bits

A row is a token: one when a single sequence is being answered, tens when a batch is, thousands
when prompts are read.  W[k, n] = s[k // group, n] * (q[k, n] - z[k // group, n]), with z = 8
where a weight has no zeros; word [i, n] of the packed weights holds q[8 i .. 8 i + 7, n], the
lowest k in the lowest bits.
"""
import math
import os
import sys

import torch

own = False  # whether run() calls the framework's operators, or computes them from elementary operations

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
NORM_EPS, POST_EPS = 1e-5, 1e-6


def listed():
    return [
        # One token of one sequence between two blocks: the norm after the block, the residual, the next block's norm.
        {"name": "norm_token", "op": "norm", "M": 1, "D": 4096, "dtype": "bf16", "post": "rms", "pre": "rms",
         "gate_rows": 0, "gate_act": "none", "scale": 1.0, "affine": True},
        # A batch of sequences being answered, one gate value for each channel.
        {"name": "norm_batch", "op": "norm", "M": 128, "D": 8192, "dtype": "fp16", "post": "none", "pre": "layer",
         "gate_rows": 1, "gate_act": "none", "scale": 0.5, "affine": True},
        # Prompts of many thousand tokens, both norms, a residual scale.
        {"name": "norm_prompts", "op": "norm", "M": 16384, "D": 4096, "dtype": "bf16", "post": "rms", "pre": "rms",
         "gate_rows": 0, "gate_act": "none", "scale": 0.70710678, "affine": True},
        # Thirty-two sequences of 509 tokens, a gate row for each, a width that no vector load divides.
        {"name": "norm_ragged", "op": "norm", "M": 32 * 509, "D": 1021, "dtype": "fp16", "post": "layer", "pre": "layer",
         "gate_rows": 32, "gate_act": "sigmoid", "scale": 1.0, "affine": True},

        # The second layer of a block for one token: deep and narrow, the residual added.
        {"name": "linear_token_down", "op": "linear", "M": 1, "K": 16384, "N": 4096, "group": 128, "zeros": False,
         "bias": False, "residual": True, "act": "none", "dtype": "bf16"},
        # A small model's layer for one token: the call is short, latency counts.
        {"name": "linear_token_small", "op": "linear", "M": 1, "K": 1024, "N": 1024, "group": 64, "zeros": True,
         "bias": True, "residual": False, "act": "gelu_tanh", "dtype": "fp16"},
        # Sixteen sequences being answered at once.
        {"name": "linear_batch", "op": "linear", "M": 16, "K": 8192, "N": 8192, "group": 128, "zeros": True,
         "bias": False, "residual": False, "act": "none", "dtype": "bf16"},
        # Sizes that no tile divides, a last group that is not whole.
        {"name": "linear_ragged", "op": "linear", "M": 37, "K": 4072, "N": 4093, "group": 32, "zeros": True,
         "bias": True, "residual": True, "act": "none", "dtype": "fp16"},
        # Prompts: a product of the size of a training step's.
        {"name": "linear_prompts", "op": "linear", "M": 4096, "K": 4096, "N": 4096, "group": 128, "zeros": False,
         "bias": False, "residual": False, "act": "none", "dtype": "bf16"},

        # The first half of a gated block for one token: the largest weights of a layer.
        {"name": "gated_token", "op": "gated", "M": 1, "K": 4096, "N": 16384, "group": 128, "zeros": False,
         "bias": False, "act": "silu", "dtype": "bf16"},
        # A few sequences with a few guessed tokens each.
        {"name": "gated_batch", "op": "gated", "M": 48, "K": 2048, "N": 8192, "group": 64, "zeros": True,
         "bias": True, "act": "gelu_tanh", "dtype": "fp16"},
        # One sequence's prompt through the first half of a BERT-large sized block.
        {"name": "gated_prompt", "op": "gated", "M": 509, "K": 1024, "N": 4096, "group": 128, "zeros": False,
         "bias": True, "act": "silu", "dtype": "fp16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "gated"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "norm":
        D = _spread(rng, 64, 8192)
        if rng.random() < 0.6:
            D = max(64, D // 8 * 8)
        M = _spread(rng, 1, min(16384, 16384 * 4096 // D))
        gates = [0, 1, M] + [d for d in (2, 3, 4, 8, 16, 32) if M % d == 0]
        gate_rows = rng.choice(gates)
        return {"op": op, "M": M, "D": D, "dtype": dtype, "post": rng.choice(["none", "rms", "layer"]),
                "pre": rng.choice(["rms", "layer"]), "gate_rows": gate_rows,
                "gate_act": rng.choice(["none", "sigmoid", "silu"]) if gate_rows else "none",
                "scale": rng.choice([1.0, 0.5, 0.125, 1.5]), "affine": rng.random() < 0.8}
    K = max(64, _spread(rng, 64, 16384) // 8 * 8)
    if rng.random() < 0.6:
        K = max(128, K // 128 * 128)
    N = _spread(rng, 64, 16384)
    if rng.random() < 0.7:
        N = max(64, N // 64 * 64)
    both = 2 if op == "gated" else 1
    while both * K * N > 2 ** 27:
        N = N // 2
    M = _spread(rng, 1, max(1, min(4096, 2 ** 36 // (both * K * N))))
    case = {"op": op, "M": M, "K": K, "N": N, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
            "bias": rng.random() < 0.5, "dtype": dtype}
    if op == "gated":
        return {**case, "act": rng.choice(["silu", "gelu_tanh", "sigmoid", "relu"])}
    residual = rng.random() < 0.5
    return {**case, "residual": residual, "act": "none" if residual else rng.choice(["none", "relu", "gelu_tanh", "silu"])}


def _weight(case, gen, dt):
    """A weight in 4 bits: packed words, scales, zeros.  q is spread as the quantised values of a normal weight
    are, the scales such that the weight's standard deviation is about 1 / sqrt(K)."""
    K, N, G = case["K"], case["N"], case["group"]
    groups = -(-K // G)
    z = None
    q = torch.randn(K, N, generator=gen, device=DEV).mul_(2.4)
    if case["zeros"]:
        z = torch.randint(5, 11, (groups, N), generator=gen, device=DEV)
        q += z.repeat_interleave(G, 0)[:K]
        z = z.to(dt)
    else:
        q += 8
    q = q.round_().clamp_(0, 15).to(torch.int32).view(K // 8, 8, N)
    wq = q[:, 0].clone()
    for i in range(1, 8):
        wq |= q[:, i] << (4 * i)
    s = (0.5 + torch.rand(groups, N, generator=gen, device=DEV)) / (2.4 * math.sqrt(K))
    return wq, s.to(dt), z


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, generator=gen, device=DEV).mul_(std).add_(mean).to(dt)

    st = {"case": case}
    M = case["M"]
    if case["op"] == "norm":
        D = case["D"]
        st["x"], st["y"] = normal(M, D, std=2.0), normal(M, D, mean=0.1)
        st["gate"] = normal(case["gate_rows"], D, std=0.7) if case["gate_rows"] else None
        aff = case["affine"]
        for side in ("post", "pre"):
            st[side + "_gamma"] = normal(D, mean=1.0, std=0.2) if aff and case[side] != "none" else None
            st[side + "_beta"] = normal(D, std=0.2) if aff and case[side] == "layer" else None
        return st
    K, N = case["K"], case["N"]
    st["x"] = normal(M, K)
    st["x"][:, :: max(1, K // 5)] *= 8  # a few channels of activations are much larger than the others
    for side in ("g", "u") if case["op"] == "gated" else ("",):
        st["w" + side], st["s" + side], st["z" + side] = _weight(case, gen, dt)
        st["b" + side] = normal(N, std=0.5) if case["bias"] else None
    if case.get("residual"):
        st["r"] = normal(M, N)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    x = st["x"]
    if case["op"] == "norm":
        st["h"], st["out"] = torch.empty_like(x), torch.empty_like(x)
    else:
        st["out"] = torch.empty((case["M"], case["N"]), dtype=x.dtype, device=DEV)
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
    if case["op"] == "norm":
        return gp.residual_norm_out(st["x"], st["y"], gate=st["gate"], gate_act=case["gate_act"], scale=case["scale"],
                                    post=case["post"], post_gamma=st["post_gamma"], post_beta=st["post_beta"],
                                    post_eps=POST_EPS, norm=case["pre"], gamma=st["pre_gamma"], beta=st["pre_beta"],
                                    eps=NORM_EPS, h=st["h"], out=st["out"])
    if case["op"] == "linear":
        return gp.q4_gemm_out(st["x"], st["w"], st["s"], st["z"], b=st["b"], r=st.get("r"), act=case["act"],
                              group=case["group"], out=st["out"])
    return gp.q4_gated_out(st["x"], st["wg"], st["sg"], st["zg"], st["wu"], st["su"], st["zu"], bg=st["bg"], bu=st["bu"],
                           act=case["act"], group=case["group"], out=st["out"])


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


def _norm(v, kind, gamma, beta, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + eps)
    if gamma is not None:
        v = v * gamma.float()
    if beta is not None:
        v = v + beta.float()
    return v


def _dequantised(wq, s, z, group):
    """The weight [K, N] in 32 bits."""
    shifts = torch.arange(0, 32, 4, device=wq.device, dtype=torch.int32)
    q = ((wq[:, None, :] >> shifts[:, None]) & 15).reshape(-1, wq.shape[1]).float()
    K = q.shape[0]
    q -= 8.0 if z is None else z.float().repeat_interleave(group, 0)[:K]
    return q * s.float().repeat_interleave(group, 0)[:K]


def _run_plain(st):
    case = st["case"]
    dt = st["x"].dtype
    x = st["x"].float()
    if case["op"] == "norm":
        v = _norm(st["y"].float(), case["post"], st["post_gamma"], st["post_beta"], POST_EPS)
        if st["gate"] is not None:
            g = _act(st["gate"].float(), case["gate_act"])
            v = (v.view(g.shape[0], -1, v.shape[1]) * g[:, None, :]).view_as(x)
        h = x + case["scale"] * v
        return h.to(dt), _norm(h, case["pre"], st["pre_gamma"], st["pre_beta"], NORM_EPS).to(dt)
    got = []
    for side in ("g", "u") if case["op"] == "gated" else ("",):
        v = torch.matmul(x, _dequantised(st["w" + side], st["s" + side], st["z" + side], case["group"]))
        if st["b" + side] is not None:
            v += st["b" + side].float()
        got.append(v)
    if case["op"] == "gated":
        return (_act(got[0], case["act"]) * got[1]).to(dt)
    v = _act(got[0], case["act"])
    if case["residual"]:
        v = v + st["r"].float()
    return v.to(dt)


def work(case):
    M = case["M"]
    if case["op"] == "norm":
        D = case["D"]
        params = D * ((case["affine"] and case["post"] != "none") + (case["affine"] and case["post"] == "layer")
                      + (case["affine"]) + (case["affine"] and case["pre"] == "layer"))
        values = 4 * M * D + case["gate_rows"] * D + params
        flops = M * D * (3 + 7 * (case["post"] != "none") + 7)
        return {"bytes": 2 * values, "flops": flops}
    K, N = case["K"], case["N"]
    both = 2 if case["op"] == "gated" else 1
    groups = -(-K // case["group"])
    weight = K * N // 2 + 2 * groups * N * (2 if case["zeros"] else 1) + (2 * N if case["bias"] else 0)
    data = 2 * M * K + 2 * M * N * (2 if case.get("residual") else 1)
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


def _exact_norm(v, kind, gamma, beta, eps):
    """Row by row from its moments: sum(v) and sum(v^2) in 64 bits."""
    if kind == "none":
        return v
    n = v.shape[1]
    mean = v.sum(1, keepdim=True) / n if kind == "layer" else torch.zeros_like(v[:, :1])
    var = torch.linalg.vector_norm(v - mean, dim=1, keepdim=True) ** 2 / n
    v = (v - mean) / torch.sqrt(var + eps)
    return (v if gamma is None else v * gamma.double()) + (0 if beta is None else beta.double())


def _exact_product(x, wq, s, z, group):
    """Sum over the groups of s_g * (x_g @ (q_g - z_g)), the 4-bit values taken out of the words one place at a time."""
    K, N = 8 * wq.shape[0], wq.shape[1]
    words = wq.long() & 0xFFFFFFFF
    out = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    rows = max(group, 1024 // group * group)  # whole groups, about a thousand k at a time
    for k0 in range(0, K, rows):
        k = torch.arange(k0, min(K, k0 + rows), device=x.device)
        w = torch.div(words[k // 8], (16 ** (k % 8))[:, None], rounding_mode="floor").remainder(16).double()
        at = k // group
        w = (w - (8.0 if z is None else z.double()[at])) * s.double()[at]
        out += x[:, k] @ w
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    x = st["x"].double()
    if case["op"] == "norm":
        v = _exact_norm(st["y"].double(), case["post"], st["post_gamma"], st["post_beta"], POST_EPS)
        if st["gate"] is not None:
            rows = torch.arange(case["M"], device=x.device) // (case["M"] // case["gate_rows"])
            v = v * _exact_act(st["gate"].double(), case["gate_act"])[rows]
        h = x + case["scale"] * v
        return h, _exact_norm(h, case["pre"], st["pre_gamma"], st["pre_beta"], NORM_EPS)
    got = []
    for side in ("g", "u") if case["op"] == "gated" else ("",):
        v = _exact_product(x, st["w" + side], st["s" + side], st["z" + side], case["group"])
        got.append(v if st["b" + side] is None else v + st["b" + side].double())
    if case["op"] == "gated":
        return _exact_act(got[0], case["act"]) * got[1]
    v = _exact_act(got[0], case["act"])
    return v + st["r"].double() if case["residual"] else v
