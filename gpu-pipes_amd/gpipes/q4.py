"""Weights in 4 bits for gpipes.q4_gemm_out and gpipes.q4_gated_out: packing, and rounding to
nearest.  Done once for a weight, with torch operations on whatever device it is on."""
import torch

GROUPS = (32, 64, 128)


def pack(q):
    """q [K, N], whole numbers 0 .. 15, K a multiple of 8 -> int32 words [K / 8, N], the lowest k in the lowest bits."""
    if q.dim() != 2 or q.shape[0] % 8:
        raise RuntimeError("q must be [K, N] with K a multiple of 8")
    v = q.to(torch.int64)
    if not bool(((v >= 0) & (v <= 15) & (v == q)).all()):  # a fraction, a NaN or an infinity is no longer what it was
        raise RuntimeError("q must be whole numbers in 0 .. 15")
    v = v.contiguous().view(-1, 8, q.shape[1])
    w = v[:, 0].clone()
    for i in range(1, 8):
        w |= v[:, i] << (4 * i)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def unpack(wq):
    """The int32 q [K, N] of packed words."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=wq.device)
    return ((wq[:, None, :] >> shifts[:, None]) & 15).reshape(-1, wq.shape[1])


def dequantize(wq, scales, zeros=None, group=128):
    """The weight [K, N] in fp32: scales * (q - zeros), zeros None: 8."""
    q = unpack(wq).float()
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, 0)[:q.shape[0]]
    return scales.float().repeat_interleave(group, 0)[:q.shape[0]] * (q - z)


def quantize(w, group=128, zeros=False):
    """w [K, N] float16 or bfloat16 -> (wq, scales, zeros), rounded to nearest in groups of `group` k (the last may
    be short).  Without zeros a group spans -7 .. 7 steps of max|w| / 7 (zeros None: 8); with them, 0 .. 15 steps
    from its least value, or zero, to its greatest, or zero, and the zero is a whole number."""
    if w.dim() != 2 or w.shape[0] % 8 or w.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("w must be float16 or bfloat16 [K, N] with K a multiple of 8")
    if group not in GROUPS:
        raise RuntimeError(f"group must be 32, 64 or 128 (got {group})")
    if not bool(torch.isfinite(w).all()):
        raise RuntimeError("w must be finite")
    K, N = w.shape
    groups = -(-K // group)
    v = torch.zeros((groups * group, N), dtype=torch.float32, device=w.device)
    v[:K] = w
    v = v.view(groups, group, N)
    if zeros:
        lo, hi = v.amin(1).clamp(max=0), v.amax(1).clamp(min=0)
        s = (hi / 15 - lo / 15).to(w.dtype)
        z = torch.where(s > 0, torch.round(-lo / s.float()), 0 * lo).clamp(0, 15)
    else:
        s = (v.abs().amax(1) / 7).to(w.dtype)
        z = torch.full_like(s, 8, dtype=torch.float32)
    q = torch.where(s[:, None] > 0, torch.round(v / s.float()[:, None]), 0 * v) + z[:, None]
    q = q.clamp(0, 15).view(-1, N)[:K]
    return pack(q), s, z.to(w.dtype) if zeros else None
