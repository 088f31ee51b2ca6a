"""The paged cache in 64 bits, and how far the results may be from it.

Rounding to a type is off by at most half a step: HALF16 = 2^-8 relative for bf16; HALF8 = 2^-4 relative for e4m3, and half of its least step, 2^-10, below 2^-6.
Before that, in fp32: the mean of up to 128 squares in sums of 16 and a tree of 3 (19 roundings of positive terms, and the square's own), the root (off by 2 units), three
products and the two products and the sum of the rotation: less than 32 * 2^-24 = FINE of the sizes of the two products.
"""
import torch

HALF16, HALF8, FINE = 2.0 ** -8, 2.0 ** -4, 2.0 ** -19


def pool(pages, G, P, D, eight, device, seed):
    """Pages with values in use, and their scales or None."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, G, P, D, generator=g)
    if not eight:
        return x.to(torch.bfloat16).to(device), None
    return (x * 128).clamp(-448, 448).to(torch.float8_e4m3fn).to(device), torch.randint(118, 123, (pages, G), generator=g, dtype=torch.uint8).to(device)


def table_of(lengths, P, pages, width, seed=0):
    """int32 [B, width]: pages of its own for every sequence, anywhere in the pool; the rest of a row names no page."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, at = torch.full((len(lengths), width), -7, dtype=torch.int32), 0
    for b, n in enumerate(lengths):
        used = -(-n // P)
        table[b, :used] = order[at:at + used]
        at += used
    assert at <= pages
    return table


def values(pages, scale):
    return pages.double() if scale is None else pages.double() * (2.0 ** (scale.double() - 127))[:, :, None, None]


def angles(positions, D, device, base=1e4):
    a = torch.arange(positions, dtype=torch.float64)[:, None] / base ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    return a.cos().float().to(device), a.sin().float().to(device)


def turned(x, w, cos, sin, eps):
    """(values, sizes of the products that each is a sum of) of x [rows, heads, D]."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    (a, b), c, s = x.chunk(2, -1), cos.double()[:, None], sin.double()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1), torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)


def check_append(before, after, q_out, k, v, q, table, start, cu, cos, sin, q_norm, k_norm, eps, name="", k_out=None):
    """``before`` / ``after``: (k_pages, v_pages, k_scale, v_scale) as they were and are. Sequences without pages of their own are not for here."""
    P = before[0].shape[2]
    untouched = [torch.ones(t.shape[:3], dtype=torch.bool) for t in before[:2]]
    kept_scale = torch.ones(before[0].shape[:2], dtype=torch.bool)
    ends = cu if cu is not None else list(range(len(start) + 1))
    if q_out is not None:
        value, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, first in enumerate(start):
        lo, hi = ends[b], ends[b + 1]
        if hi == lo:
            continue
        c, s = cos[first:first + hi - lo].cpu(), sin[first:first + hi - lo].cpu()
        if q_out is not None:
            value[lo:hi], size[lo:hi] = turned(q[lo:hi].cpu(), q_norm, c, s, eps)
        if k_out is not None:
            y, fine = turned(k[lo:hi].cpu(), k_norm, c, s, eps)
            assert float(((k_out[lo:hi].cpu().double() - y).abs() - (HALF16 * y.abs() + FINE * fine)).max()) <= 0, f"{name}: keys"
        for i, (x, w) in enumerate(((k, k_norm), (v, None))):
            y, fine = turned(x[lo:hi].cpu(), w, c, s, eps) if i == 0 else (x[lo:hi].cpu().double(), torch.zeros(1, dtype=torch.float64).expand(x[lo:hi].shape))
            was, now = before[i].cpu(), after[i].cpu()
            scale_was, scale_now = (before[2 + i].cpu(), after[2 + i].cpu()) if before[2] is not None else (None, None)
            done = 0
            while done < hi - lo:
                page, slot = int(table[b, (first + done) // P]), (first + done) % P
                n = min(P - slot, hi - lo - done)
                part, off = y[done:done + n].transpose(0, 1), FINE * fine[done:done + n].transpose(0, 1)
                untouched[i][page, :, slot:slot + n] = False
                got = now[page, :, slot:slot + n].double()
                odd = ~torch.isfinite(part)
                if scale_was is None:
                    assert torch.equal(torch.nan_to_num(got[odd], 0.0, 1.0, -1.0), torch.nan_to_num(part[odd], 0.0, 1.0, -1.0)), name
                    room = HALF16 * part.abs() + off
                else:
                    assert torch.isnan(got[odd]).all(), f"{name}: what is not finite must be NaN"
                    most = torch.where(odd, 0.0, part.abs()).amax((1, 2))
                    bytes_now = scale_now[page].to(torch.int64)
                    for h in range(part.shape[0]):
                        least = 1
                        kept = int(scale_was[page, h]) if slot else 1
                        while float(most[h]) * (1 + FINE) > 448 * 2.0 ** (least - 127):
                            least += 1
                        under = least - 1 if least > 1 and float(most[h]) * (1 - FINE) <= 448 * 2.0 ** (least - 128) else least       # so near that rounding decides
                        assert int(bytes_now[h]) in (max(least, kept), max(under, kept)), f"{name}: scale {int(bytes_now[h])}, expected {max(least, kept)}"
                        if slot:
                            ratio = 2.0 ** float(kept - int(bytes_now[h]))
                            held = (was[page, h, :slot].float() * ratio).to(torch.float8_e4m3fn)
                            assert torch.equal(torch.nan_to_num(held.float(), nan=999.0), torch.nan_to_num(now[page, h, :slot].float(), nan=999.0)), f"{name}: what the page held before"
                            untouched[i][page, h, :slot] = False
                    kept_scale[page] = False
                    unit = (2.0 ** (bytes_now.double() - 127))[:, None, None]
                    got = got * unit
                    room = torch.maximum(HALF8 * part.abs(), 2.0 ** -10 * unit) + off
                far = torch.where(odd, 0.0, (got - part).abs() - room)
                assert float(far.max()) <= 0, f"{name}: {'kv'[i]} of sequence {b} is {float(far.max()):.3g} outside its bound"
                done += n
    for i in range(2):
        mask = untouched[i]
        assert torch.equal(before[i].cpu().view(torch.uint8 if before[2] is not None else torch.int16)[mask], after[i].cpu().view(torch.uint8 if before[2] is not None else torch.int16)[mask]), f"{name}: a slot that no token goes to"
        if before[2] is not None:
            assert torch.equal(before[2 + i].cpu()[kept_scale], after[2 + i].cpu()[kept_scale]), f"{name}: a scale that no token goes to"
    if k_out is not None:
        assert not k_out[ends[-1]:].any()
    if q_out is not None:
        far = (q_out.cpu().double() - value).abs() - (HALF16 * value.abs() + FINE * size)
        assert float(far.max()) <= 0, f"{name}: q is {float(far.max()):.3g} outside its bound"


def dense(pages, scale, table, lengths, width):
    """[B, width, G, D] in 64 bits; zeros behind the ends."""
    P, G, D = pages.shape[2], pages.shape[1], pages.shape[3]
    out = torch.zeros(len(lengths), width, G, D, dtype=torch.float64, device=pages.device)
    for b, n in enumerate(lengths):
        if n > 0:
            mine = table[b, :-(-n // P)].long().to(pages.device)
            x = values(pages[mine], None if scale is None else scale[mine])
            out[b, :n] = x.transpose(1, 2).reshape(-1, G, D)[:n]
    return out
