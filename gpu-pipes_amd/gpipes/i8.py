"""Weights in 8 bits for gpipes.i8_gemm_out, i8_gated_out and i8_experts_out: packing, and rounding
to nearest.  Done once for a weight, with torch operations on whatever device it is on.  Every
function takes one weight [K, N], or the weights of E experts [E, K, N]."""
import torch


def packed_shape(K, N):
    """The shape of a packed weight [K, N]: blocks of 16 columns by 64 k."""
    return (-(-N // 16), -(-K // 64), 1024)


def pack(q):
    """q [(E,) K, N], whole numbers -128 .. 127 -> int8 [(E,) ceil(N / 16), ceil(K / 64), 1024]: byte
    256 g + 16 j + i of block [a, b] is q[64 b + 16 g + i, 16 a + j]; zeros behind K and N."""
    if q.dim() not in (2, 3) or 0 in q.shape:
        raise RuntimeError("q must be [K, N] or [E, K, N]")
    if q.dtype != torch.int8:
        v = q.to(torch.int64)
        if q.is_complex() or not bool(((v >= -128) & (v <= 127) & (v == q)).all()):
            raise RuntimeError("q must be whole numbers in -128 .. 127")
        q = v.to(torch.int8)
    if q.dim() == 3:
        out = torch.empty((q.shape[0], *packed_shape(*q.shape[1:])), dtype=torch.int8, device=q.device)
        for to, one in zip(out, q):
            to.copy_(pack(one))
        return out
    K, N = q.shape
    N16, K64, _ = packed_shape(K, N)
    v = torch.zeros((K64 * 64, N16 * 16), dtype=torch.int8, device=q.device)
    v[:K, :N] = q
    return v.view(K64, 4, 16, N16, 16).permute(3, 0, 1, 4, 2).reshape(N16, K64, 1024)


def unpack(wq, K, N):
    """The int8 q [(E,) K, N] of a packed weight."""
    if wq.dtype != torch.int8 or wq.dim() not in (3, 4) or tuple(wq.shape[-3:]) != packed_shape(K, N):
        raise RuntimeError(f"the packed weight must be int8 [(E,) {', '.join(map(str, packed_shape(K, N)))}]")
    N16, K64, _ = packed_shape(K, N)
    v = wq.reshape(-1, N16, K64, 4, 16, 16).permute(0, 2, 3, 5, 1, 4).reshape(-1, K64 * 64, N16 * 16)[:, :K, :N]
    return v if wq.dim() == 4 else v[0]


def dequantize(wq, scales, K):
    """The weight [(E,) K, N] in fp32: scales[(e,) n] * q[(e,) k, n]."""
    return unpack(wq, K, scales.shape[-1]).float() * scales[..., None, :]


def quantize(w):
    """w [(E,) K, N] float16, bfloat16 or float32 -> (packed, scales), rounded to nearest: a column spans
    -127 .. 127 steps of max|w| / 127.  scales float32 [(E,) N]; a column of zeros has scale 0."""
    if w.dim() not in (2, 3) or 0 in w.shape or w.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise RuntimeError("w must be float16, bfloat16 or float32 [K, N] or [E, K, N]")
    if not bool(torch.isfinite(w).all()):
        raise RuntimeError("w must be finite")
    top = w.abs().amax(-2).float()
    q = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    for to, one, t in zip(q.view(-1, *w.shape[-2:]), w.reshape(-1, *w.shape[-2:]), top.view(-1, w.shape[-1])):
        # in 64 bits, where neither 127 w nor the quotient's distance from a half is lost
        to.copy_(torch.where(t > 0, torch.round(127 * one.double() / t.double()), 0))
    return pack(q), (top.double() / 127).float()


def quantize_rows(x):
    """x [M, K] float16 or bfloat16 -> (q int8 [M, K], scales float32 [M]): the whole numbers and scales that the
    products make of a row of 16-bit x themselves, round(127 x / max|x|) and max|x| / 127."""
    if x.dim() != 2 or x.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("x must be float16 or bfloat16 [M, K]")
    v = x.double()
    top = v.abs().amax(1, keepdim=True)
    ok = (top > 0) & torch.isfinite(top)
    q = torch.where(ok, torch.round(127 * v / top), 0).to(torch.int8)
    scales = (top / 127).float()[:, 0]  # in 64 bits: torch divides by a number through its reciprocal
    return q, torch.where(torch.isfinite(top[:, 0]), scales, torch.nan)
