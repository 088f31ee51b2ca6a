"""The language models' attention in 64 bits, and how far a kernel's outputs may be from it.

``bounds`` counts the roundings: a bf16 value is off by at most half a step, HALF = 2^-8 relative. The kernels round
  * every output once,
  * the probabilities once before they multiply v (forward) or do (backward), and ds once before it multiplies k or q,
  * o once, which enters the backward pass through delta = do . o.
Everything else is in fp32. There the exponentials are the largest error: relative 8.6e-5 for the polynomial that takes a share of them, and
the score in front of one is a sum of up to 128 products of size 1 to 6 in fp32, times log2(e), so below 32: off by less than 128 * 2^-24 * 6 +
32 * 2^-23 = 5e-5. The sums over 2000 keys of positive terms add 2000 * 2^-24 = 1.2e-4 at most. FINE = 4e-4 covers numerator and divisor.
"""
import math

import torch

HALF = torch.finfo(torch.bfloat16).eps / 2
FINE = 4e-4


def seen_by(Sq, Skv, B, window=None, sinks=0, kv_len=None, q_start=0, causal=True):
    seen = torch.zeros(B, Sq, Skv, dtype=torch.bool)
    for b in range(B):
        start = int(q_start[b]) if isinstance(q_start, torch.Tensor) else q_start
        length = Skv if kv_len is None else min(Skv, int(kv_len[b]))
        for i in range(Sq):
            p = start + i
            if not causal:
                seen[b, i, :max(length, 0)] = True
                continue
            end = max(0, min(p + 1, length))
            seen[b, i, :end] = True
            if window is not None:
                seen[b, i, min(end, sinks):max(min(end, sinks), min(end, p - window + 1))] = False
    return seen


def bucket(rel, num_buckets, max_distance):
    side, n = num_buckets // 2, abs(rel)
    single = side // 2
    if n >= single:
        m = side - single
        n = single + sum(n ** m * single ** k >= max_distance ** k * single ** m for k in range(1, m))
    return n + (side if rel > 0 else 0)


def oracle(q, k, v, scale, seen, grad=None, sink=None, table=None, max_distance=128):
    """Outputs and bounds as dicts of fp64 tensors: out, and with ``grad`` dq, dk, dv, dsink, dtable."""
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    dev = q.device
    B, Sq, H, D = q.shape
    Skv, G = k.shape[1], k.shape[2]
    rep = H // G
    seen = seen.to(dev)
    used = seen.any(1)[:, :, None, None]
    k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)
    kh, vh = k.repeat_interleave(rep, 2), v.repeat_interleave(rep, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, kh) * scale
    which = None
    if table is not None:
        which = torch.tensor([[bucket(j - i, table.shape[0], max_distance) for j in range(Skv)] for i in range(Sq)], device=dev)
        s = s + table.detach().double().t()[:, which]
    s = s.masked_fill(~seen[:, None], -math.inf)
    last = torch.full((H,), -math.inf, dtype=torch.float64, device=dev) if sink is None else sink.detach().double()
    s = torch.cat((s, last[None, :, None, None].expand(B, H, Sq, 1)), -1)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    p_sink, p = p[..., -1], p[..., :-1]
    o = torch.einsum("bhij,bjhd->bihd", p, vh)
    mass = torch.einsum("bhij,bjhd->bihd", p, vh.abs())
    value, bound = dict(out=o), dict(out=HALF * o.abs() + (HALF + FINE) * mass)
    if grad is None:
        return value, bound
    d = grad.detach().double()
    fold = lambda t: t.reshape(B, Skv, G, rep, D).sum(3)
    delta = torch.einsum("bihd,bihd->bhi", d, o)[..., None]
    off = torch.einsum("bihd,bihd->bhi", d.abs(), HALF * o.abs() + (HALF + FINE) * mass)[..., None]        # of delta
    dp = torch.einsum("bihd,bjhd->bhij", d, vh)
    ds = p * (dp - delta)
    ds_off = p * off + FINE * (ds.abs() + p * (dp.abs() + delta.abs()))                                     # before ds is rounded
    ds_off16 = ds_off + HALF * ds.abs()
    value |= dict(dq=torch.einsum("bhij,bjhd->bihd", ds, kh) * scale, dk=fold(torch.einsum("bhij,bihd->bjhd", ds, q)) * scale,
                  dv=fold(torch.einsum("bhij,bihd->bjhd", p, d)))
    bound |= dict(dq=HALF * value["dq"].abs() + scale * torch.einsum("bhij,bjhd->bihd", ds_off16, kh.abs()),
                  dk=HALF * value["dk"].abs() + scale * fold(torch.einsum("bhij,bihd->bjhd", ds_off16, q.abs())),
                  dv=HALF * value["dv"].abs() + (HALF + FINE) * fold(torch.einsum("bhij,bihd->bjhd", p, d.abs())))
    if sink is not None:
        last_off = HALF if sink.dtype == torch.bfloat16 else 2.0 ** -24
        value["dsink"] = -(p_sink[..., None] * delta).sum((0, 2, 3))
        bound["dsink"] = last_off * value["dsink"].abs() + (p_sink[..., None] * (off + FINE * delta.abs())).sum((0, 2, 3))
    if table is not None:
        last_off = HALF if table.dtype == torch.bfloat16 else 2.0 ** -24
        add = lambda t: torch.zeros(H, table.shape[0], dtype=torch.float64, device=dev).index_add_(1, which.reshape(-1), t.sum(0).reshape(H, -1)).t()
        value["dtable"] = add(ds)
        bound["dtable"] = last_off * value["dtable"].abs() + add(ds_off)
    return value, bound


def check(got, value, bound, name):
    """Every element of every output within its bound (1e-30: sums of nothing)."""
    for key, t in got.items():
        assert torch.isfinite(t).all(), f"{name}: {key} has values that are not finite"
        off = (t.detach().double() - value[key]).abs() - bound[key]
        worst = float(off.max()) if off.numel() else 0.0
        assert worst <= 1e-30, f"{name}: {key} is {worst:.3g} outside its bound (largest value {float(value[key].abs().max()):.3g})"
