"""Packed sequences: each by itself in 64 bits, with the bounds of ``text_attention_oracle``; rows of no sequence are zero."""
import torch

from text_attention_oracle import oracle, seen_by


def packed_oracle(q, k, v, cu, scale, window=None, grad=None, sink=None):
    value = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v)) if grad is not None or n == "out"}
    bound = {n: torch.zeros_like(t) for n, t in value.items()}
    if grad is not None and sink is not None:
        value["dsink"], bound["dsink"] = (torch.zeros(q.shape[1], dtype=torch.float64, device=q.device) for _ in range(2))
        last = 2.0 ** -8 if sink.dtype == torch.bfloat16 else 2.0 ** -24
    for lo, hi in zip(cu[:-1], cu[1:]):
        if hi == lo:
            continue
        part = lambda t: None if t is None else t[None, lo:hi]
        a, b = oracle(part(q), part(k), part(v), scale, seen_by(hi - lo, hi - lo, 1, window), part(grad), sink)
        for n in value:
            if n == "dsink":
                value[n] += a[n]
                bound[n] += b[n] - last * a[n].abs()          # rounded once, at the end
            else:
                value[n][lo:hi], bound[n][lo:hi] = a[n][0], b[n][0]
    if "dsink" in value:
        bound["dsink"] += last * value["dsink"].abs()
    return value, bound
