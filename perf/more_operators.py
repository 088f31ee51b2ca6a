"""Serving many prompts of a language model at once: one pass each through the operators, in plain torch or in kernels.

* ``paged_append``: keys and values of new tokens go into the pages of their sequences, normalised per head and rotated on the way, as bf16 or in
  8 bits (e4m3) with a power of two per page and head; the queries of the same tokens are normalised and rotated with them.
* ``paged_attention``: a token each, a few drafted tokens, or a part of a prompt attends to all of its sequence in the pages.
* ``packed_attention``: causal attention over prompts of different lengths that lie one behind the other, without padding; and its gradient.

Queries, keys, values and gradients are unit normal, scores have a variance of about one, as normalised queries and keys give; all is drawn on the
GPU from the seed. The lengths belong to the case; the seed shuffles them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BF16, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
F8_MAX = 448.0


# ---- the cases -------------------------------------------------------------------------------------------------------------
# batch sequences with lengths from `shortest` to `longest`; most are short, as prompts are. op: append / attention / packed
def listed():
    return [
        # a token of one sequence, in a stack of 16 / 8 heads that normalises queries and keys: latency
        _append("append_token", batch=1, heads=16, kv_heads=8, dim=128, page=64, eight=True, norm=True, shortest=1, longest=1, before=300, spare=0),
        # a token each of 128 sequences, most of them inside a page
        _append("append_tokens", batch=128, heads=32, kv_heads=8, dim=128, page=64, eight=True, norm=True, shortest=1, longest=1, before=4000, spare=0),
        # sixteen prompts, some of which go on behind a cached beginning
        _append("append_prompts", batch=16, heads=32, kv_heads=8, dim=128, page=64, eight=True, norm=False, shortest=5, longest=2048, before=500, spare=3),
        # the same kind of work into bf16 pages, heads of 64
        _append("append_prompts_bf16", batch=7, heads=28, kv_heads=4, dim=64, page=32, eight=False, norm=True, shortest=77, longest=1531, before=0, spare=0),
        # one token over a prompt of a few hundred: latency
        _attention("paged_token", batch=1, q=1, heads=16, kv_heads=8, dim=128, page=64, eight=True, shortest=300, longest=300),
        # a token each of 32 sequences of very different lengths, one of them not in use
        _attention("paged_tokens", batch=32, q=1, heads=32, kv_heads=8, dim=128, page=64, eight=True, shortest=0, longest=16384),
        # a token each over long caches: the memory's rate
        _attention("paged_tokens_long", batch=4, q=1, heads=32, kv_heads=8, dim=128, page=64, eight=True, shortest=70001, longest=131072),
        # five drafted tokens each over bf16 pages, eight heads to a key head
        _attention("paged_drafts_bf16", batch=8, q=5, heads=64, kv_heads=8, dim=64, page=16, eight=False, shortest=17, longest=4091),
        # the next part of two prompts whose beginnings are in the pages
        _attention("paged_chunk", batch=2, q=777, heads=28, kv_heads=4, dim=128, page=64, eight=True, shortest=2000, longest=6000),
        # captions for the 64-head text encoder with its learned sink logits and a window
        _packed("packed_captions", train=False, batch=16, heads=64, kv_heads=8, dim=64, shortest=7, longest=300, window=128, logits=True, spare=0),
        # prompts and documents together
        _packed("packed_prompts", train=False, batch=6, heads=32, kv_heads=8, dim=128, shortest=301, longest=4096, window=0, logits=False, spare=5),
        # a training step on packed captions of all lengths
        _packed("packed_train", train=True, batch=9, heads=32, kv_heads=8, dim=128, shortest=20, longest=1531, window=0, logits=False, spare=0),
    ]


def _append(name, **c):
    return dict(name=name, op="append", **c)


def _attention(name, **c):
    return dict(name=name, op="attention", **c)


def _packed(name, **c):
    return dict(name=name, op="packed", **c)


def _between(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append token", "append prompt", "token", "token", "drafts", "chunk", "packed", "packed train"])
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 8, 128), (28, 4, 128), (64, 8, 64), (20, 4, 64), (12, 12, 64), (12, 4, 128)])
    page, eight = rng.choice([16, 32, 64, 64, 128]), rng.random() < 0.7
    if kind.startswith("append"):
        batch = _between(rng, 1, 128)
        longest = 1 if kind == "append token" else _between(rng, 2, max(2, 16384 // batch))
        c = _append("", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page, eight=eight, norm=rng.random() < 0.5,
                    shortest=1 if longest == 1 else rng.randint(0, longest), longest=longest, before=rng.choice([0, _between(rng, 1, 4000)]),
                    spare=0 if longest == 1 else rng.choice([0, rng.randint(1, 20)]))
    elif kind in ("token", "drafts"):
        batch, q = _between(rng, 1, 64), 1 if kind == "token" else rng.randint(2, 8)
        longest = _between(rng, 1, 250000 // batch)
        c = _attention("", batch=batch, q=q, heads=heads, kv_heads=kv_heads, dim=dim, page=page, eight=eight,
                       shortest=rng.randint(1 if batch == 1 else 0, longest), longest=longest)      # a batch may have places that are not in use
    elif kind == "chunk":
        q = _between(rng, 20, 1000)
        longest = q + _between(rng, 1, 6000)
        c = _attention("", batch=rng.randint(1, 2), q=q, heads=heads, kv_heads=kv_heads, dim=dim, page=page, eight=eight,
                       shortest=rng.randint(q, longest), longest=longest)
    else:
        train = kind == "packed train"
        batch = _between(rng, 1, 32)
        longest = _between(rng, 2, max(2, min(1500 if train else 3000, (6000 if train else 12000) // batch)))
        c = _packed("", train=train, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, shortest=rng.randint(1, longest), longest=longest,
                    window=rng.choice([0, 0, _between(rng, 1, 1024)]), logits=rng.random() < 0.4, spare=rng.choice([0, rng.randint(1, 20)]))
    del c["name"]
    return c


def _lengths(case):
    """The lengths of a case, from `longest` down to `shortest`, more of the short ones."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [round(lo + (hi - lo) * (1 - i / max(n - 1, 1)) ** 2) for i in range(n)]


def _befores(case):
    """What each sequence of an append has in its pages already: nothing for every third one of several prompts."""
    n, most = case["batch"], case["before"]
    return [0 if case["longest"] > 1 and n > 1 and i % 3 == 1 else most * (n - i) // n for i in range(n)]


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(BF16)
    whole = lambda values: torch.tensor(values, dtype=torch.int32, device=DEV)
    H, G, D, B = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    lengths = _lengths(case)
    order = random.Random(seed).sample(range(B), B)
    lengths = [lengths[i] for i in order]
    st = dict(case, lengths=lengths, cu=whole([sum(lengths[:i]) for i in range(B + 1)]), scale=D ** -0.5)
    if case["op"] != "attention":
        # the views that a projection to queries, keys and values leaves
        T = sum(lengths) + case["spare"]
        st["q"], st["k"], st["v"] = normal(T, (H + 2 * G) * D).view(T, H + 2 * G, D).split([H, G, G], 1)
    if case["op"] == "packed":
        st["sink_logits"] = normal(H) if case["logits"] else None
        if case["train"]:
            st["q"], st["k"], st["v"] = (st[n].contiguous().requires_grad_() for n in ("q", "k", "v"))
            if case["logits"]:
                st["sink_logits"].requires_grad_()
            st["grad"] = normal(T, H, D)
        return st
    # pages: each sequence has its own, anywhere in the pool; those in use hold values of all sizes that 8 bits have
    P = case["page"]
    if case["op"] == "append":
        befores = [_befores(case)[i] for i in order]
        filled = [b + n for b, n in zip(befores, lengths)]
        st["start"] = whole(befores)
        st["q_norm"], st["k_norm"] = (1 + 0.1 * normal(D), 1 + 0.1 * normal(D)) if case["norm"] else (None, None)
        angles = torch.arange(max(filled) + 9, device=DEV, dtype=torch.float64)[:, None] / 1e6 ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        st["cos"], st["sin"] = angles.cos().float(), angles.sin().float()
    else:
        filled = lengths
        st["kv_len"] = whole(lengths)
        st["q"] = normal(B, case["q"], H, D)
    width = max(1, -(-max(filled) // P)) + 1
    pages = sum(-(-n // P) for n in filled) + 3
    places = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table, at = torch.zeros(B, width, dtype=torch.int32), 0
    for b, n in enumerate(filled):
        table[b, :-(-n // P)] = torch.arange(at, at - (-n // P))
        at -= -n // P
    st["table"] = places[table.to(DEV).long()]
    for name in ("k", "v"):
        pool = normal(pages, G, P, D)
        if case["eight"]:
            st[name + "_pages"] = (pool.float() * 128).clamp(-F8_MAX, F8_MAX).to(F8)
            st[name + "_scale"] = torch.randint(119, 122, (pages, G), generator=g, device=DEV, dtype=torch.uint8)      # 2^-8 to 2^-6
        else:
            st[name + "_pages"], st[name + "_scale"] = pool, None
    return st


def run(st):
    if own:
        return _kernels(st)
    with torch.no_grad():
        return {"append": _plain_append, "attention": _plain_attention, "packed": _plain_packed}[st["op"]](st)


def _kernels(st):
    from mojodiffusion_b200 import ops

    if st["op"] == "append":
        cu = None if st["longest"] == 1 else st["cu"]                     # a token each
        q = ops.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["start"], st["cos"], st["sin"], cu_seqlens=cu,
                             k_scale=st["k_scale"], v_scale=st["v_scale"], q=st["q"], q_norm=st["q_norm"], k_norm=st["k_norm"])
        return _appended(st, q)
    if st["op"] == "attention":
        return ops.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_len"], k_scale=st["k_scale"], v_scale=st["v_scale"], max_len=st["longest"])
    call = lambda: ops.packed_attention(st["q"], st["k"], st["v"], st["cu"], window=st["window"] or None, sink_logits=st["sink_logits"])
    if not st["train"]:
        with torch.no_grad():
            return call()
    out = call()
    names = [n for n in ("q", "k", "v", "sink_logits") if st[n] is not None]
    grads = torch.autograd.grad(out, [st[n] for n in names], st["grad"])
    return dict({"out": out.detach()}, **dict(zip(["d_" + n for n in names], grads)))


def _appended(st, q):
    """The rotated queries and the pool. Scales are bytes that stand for powers of two."""
    found = dict(q=q, k_pages=st["k_pages"], v_pages=st["v_pages"])
    if st["eight"]:
        found.update(k_scale=st["k_scale"].view(E8), v_scale=st["v_scale"].view(E8))
    return found


# ---- the plain form ----------------------------------------------------------------------------------------------------------
def _sequence_of(cu, T):
    """For each row its sequence (the last one's number behind the end), its place in it, and whether it belongs to one."""
    row = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous().long(), row, right=True)
    inside = seq < cu.numel() - 1
    seq = seq.clamp(max=cu.numel() - 2)
    return seq, row - cu.long()[seq], inside


def _plain_append(st):
    P, D, T = st["page"], st["dim"], st["k"].shape[0]
    seq, place, inside = _sequence_of(st["cu"], T)
    at = (st["start"].long()[seq] + place).clamp(max=st["cos"].shape[0] - 1)
    cos, sin = st["cos"][at][:, None], st["sin"][at][:, None]

    def turned(x, norm):
        x = x.float()
        if norm is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * norm.float()
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q = turned(st["q"], st["q_norm"]).to(BF16) * inside[:, None, None]
    page, slot = st["table"].long()[seq, (at // P).clamp(max=st["table"].shape[1] - 1)], at % P
    n = T - st["spare"]
    page, slot = page[:n], slot[:n]                                     # rows behind the last sequence go nowhere
    for name, x in (("k", turned(st["k"], st["k_norm"])), ("v", st["v"].float())):
        x, pool = x[:n], st[name + "_pages"]
        if st["eight"]:
            x = _to_pool_scale(st, name, x, page)
        pool[page, :, slot] = x.to(pool.dtype)
    return _appended(st, q)


def _to_pool_scale(st, name, x, page):
    """Gives the pages that x goes to their scales, brings what they hold already to them, and returns x in units of them."""
    P, pool, scale = st["page"], st[name + "_pages"], st[name + "_scale"]
    N, G = scale.shape
    most = torch.zeros(N, G, device=DEV).scatter_reduce_(0, page[:, None].expand(-1, G), x.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(most / F8_MAX)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(min=-126) + 127
    touched = torch.zeros(N, dtype=torch.bool, device=DEV).index_fill_(0, page, True)
    # the pages that sequences began before: the last one of each, where that is not full
    begun = st["start"].long() % P
    last = st["table"].long().gather(1, (st["start"].long() // P)[:, None])[:, 0]
    kept = torch.zeros(N, dtype=torch.long, device=DEV).index_add_(0, last, begun) * touched
    before = scale.long()
    now = torch.where(kept[:, None] > 0, torch.maximum(exponent, before), exponent)
    scale.copy_(torch.where(touched[:, None], now, before).to(torch.uint8))
    less = torch.ldexp(torch.ones((), device=DEV), (before - now)[last])                      # [B, G]
    held = (pool[last].float() * less[:, :, None, None]).to(F8)
    mine = (torch.arange(P, device=DEV) < kept[last][:, None])[:, None, :, None]
    pool[last] = torch.where(mine, held.float(), pool[last].float()).to(F8)
    return torch.ldexp(x, (127 - scale.to(torch.int32))[page][:, :, None])


def _plain_attention(st):
    q = st["q"].transpose(1, 2).float()
    B, H, n, D = q.shape
    G, P, width = st["kv_heads"], st["page"], max(1, -(-st["longest"] // st["page"]))
    table = st["table"][:, :width].long()

    def held(name):
        x = st[name + "_pages"][table].float()                                              # [B, width, G, P, D]
        if st["eight"]:
            x = torch.ldexp(x, (st[name + "_scale"][table].to(torch.int32) - 127)[..., None, None])
        return x.transpose(1, 2).reshape(B, G, width * P, D)

    grouped = lambda t: t.reshape(B, G, (H // G) * n, -1)
    s = (grouped(q) @ held("k").transpose(-1, -2)).reshape(B, H, n, -1) * st["scale"]
    key = torch.arange(width * P, device=DEV)
    at = (st["kv_len"].long() - n)[:, None] + torch.arange(n, device=DEV)
    hidden = key > at[:, :, None]
    s = s.masked_fill_(hidden[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (grouped(e) @ held("v")).reshape(B, H, n, D) / total.masked_fill(total == 0, 1.0)
    return o.transpose(1, 2).to(BF16)


def _plain_packed(st):
    T, H, D = st["q"].shape
    G, B, M = st["kv_heads"], st["batch"], max(st["lengths"])
    seq, place, inside = _sequence_of(st["cu"], T)
    start = st["cu"].long()
    i = torch.arange(M, device=DEV)
    rows = (start[:-1, None] + i).clamp(max=T - 1)                                          # [B, M]
    padded = lambda x: x[rows].transpose(1, 2).float()                                      # [B, heads, M, D]
    back = lambda x: (x.transpose(1, 2)[seq, place.clamp(max=M - 1)] * inside[:, None, None]).to(BF16)
    q, k, v = (padded(st[n]) for n in ("q", "k", "v"))
    grouped = lambda t: t.reshape(B, G, (H // G) * M, -1)
    heads = lambda t: t.reshape(B, H, M, -1)
    s = heads(grouped(q) @ k.transpose(-1, -2)).mul_(st["scale"])
    hidden = i > i[:, None]
    if st["window"]:
        hidden = hidden | (i[:, None] - i >= st["window"])
    s = s.masked_fill_(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    sink = st["sink_logits"]
    if sink is not None:
        sink = sink.float()[None, :, None, None]
        top = torch.maximum(top, sink)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    p = p.div_(total)
    o = heads(grouped(p) @ v)
    if not st["train"]:
        return back(o)
    used = i < (start[1:] - start[:-1])[:, None]
    d = padded(st["grad"]) * used[:, None, :, None]
    delta = (d * o).sum(-1, keepdim=True)
    ds = p * (heads(grouped(d) @ v.transpose(-1, -2)) - delta)
    found = dict(out=back(o), d_q=back(heads(grouped(ds) @ k) * st["scale"]), d_k=back(grouped(ds).transpose(-1, -2) @ grouped(q) * st["scale"]),
                 d_v=back(grouped(p).transpose(-1, -2) @ grouped(d)))
    if sink is not None:
        found["d_sink_logits"] = -(torch.exp(sink - top) / total * delta).sum((0, 2, 3), dtype=torch.float64).to(BF16)
    return found


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    T = sum(lengths)
    size = 1 if case.get("eight") else 2
    if case["op"] == "append":
        # q, k and v once in, q out, keys and values in the pages' type, a row of either table for each token
        return {"bytes": T * (2 * (2 * H + 2 * G) * D + 2 * size * G * D + 4 * D), "flops": T * (H + G) * D * (7 if case["norm"] else 3)}
    if case["op"] == "attention":
        n = case["q"]
        pairs = sum(max(length - n + 1 + i, 0) for length in lengths for i in range(n))
        return {"bytes": 2 * size * T * G * D + 4 * case["batch"] * n * H * D, "flops": 4 * pairs * H * D}
    near = lambda p: min(p + 1, case["window"]) if case["window"] else p + 1
    pairs = sum(near(p) for n in lengths for p in range(n))
    flops, moved = 4 * pairs * H * D, 4 * T * (H + G) * D
    if case["train"]:
        flops, moved = flops * 3.5, 2 * moved                         # five products of the backward pass to two of the forward; the four gradients
    return {"bytes": moved, "flops": flops}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "packed": _exact_packed}[case["op"]](st)


def _exact_append(st):
    """Values in the pages are those before their rounding, in units of the scales."""
    P, D = st["page"], st["dim"]
    found = dict(q=torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV), k_pages=st["k_pages"].double(), v_pages=st["v_pages"].double())
    if st["eight"]:
        found.update(k_scale=2.0 ** (st["k_scale"].double() - 127), v_scale=2.0 ** (st["v_scale"].double() - 127))

    def rotated(x, norm, positions):
        x = x.double()
        if norm is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * norm.double()
        z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * torch.complex(st["cos"].double(), st["sin"].double())[positions][:, None]
        return torch.cat((z.real, z.imag), -1)

    row = 0
    for b, n in enumerate(st["lengths"]):
        first = int(st["start"][b])
        positions = torch.arange(first, first + n, device=DEV)
        found["q"][row:row + n] = rotated(st["q"][row:row + n], st["q_norm"], positions)
        new = {"k": rotated(st["k"][row:row + n], st["k_norm"], positions), "v": st["v"][row:row + n].double()}
        row += n
        done = 0
        while done < n:
            page, slot = int(st["table"][b, (first + done) // P]), (first + done) % P
            count = min(P - slot, n - done)
            for name, x in new.items():
                x, pool = x[done:done + count], found[name + "_pages"]
                if st["eight"]:
                    scale = found[name + "_scale"]
                    needed = 2.0 ** torch.ceil(torch.log2(x.abs().amax((0, 2)) / F8_MAX))
                    now = torch.maximum(needed, scale[page]) if slot else needed
                    pool[page, :, :slot] *= (scale[page] / now)[:, None, None]
                    scale[page] = now
                    x = x / now[None, :, None]
                pool[page, :, slot:slot + count] = x.transpose(0, 1)
            done += count
    return found


def _exact_attention(st):
    n, H, G, P = st["q"].shape[1], st["heads"], st["kv_heads"], st["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    for b, length in enumerate(st["lengths"]):
        pages = st["table"][b, :-(-length // P)].long()
        if not length:
            continue
        for g in range(G):
            k, v = (st[name + "_pages"][pages, g].double() * (2.0 ** (st[name + "_scale"][pages, g].double() - 127))[:, None, None] if st["eight"]
                    else st[name + "_pages"][pages, g].double() for name in ("k", "v"))
            k, v = k.flatten(0, 1)[:length], v.flatten(0, 1)[:length]
            mine = slice(g * (H // G), (g + 1) * (H // G))
            s = torch.einsum("ihd,jd->hij", st["q"][b, :, mine].double(), k) * st["scale"]
            i, j = torch.arange(length - n, length, device=DEV)[:, None], torch.arange(length, device=DEV)
            p = torch.softmax(s.masked_fill(j > i, float("-inf")), -1)
            out[b, :, mine] = torch.einsum("hij,jd->ihd", p.masked_fill(i < 0, 0.0), v)
    return out


def _exact_packed(st):
    T, H, D = st["q"].shape
    G = st["kv_heads"]
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    sink = st["sink_logits"].detach().double() if st["sink_logits"] is not None else None
    d_sink = torch.zeros_like(sink) if sink is not None else None
    row = 0
    for n in st["lengths"]:
        rows = slice(row, row + n)
        row += n
        j = torch.arange(n, device=DEV)
        hidden = (j > j[:, None]) | (j[:, None] - j >= (st["window"] or n))
        for h in range(H):
            leaf = [t.clone().requires_grad_() for t in (q[rows, h], k[rows, h * G // H], v[rows, h * G // H])] + ([sink[h].clone().requires_grad_()] if sink is not None else [])
            with torch.enable_grad():
                s = (leaf[0] @ leaf[1].t() * st["scale"]).masked_fill(hidden, float("-inf"))
                if sink is not None:
                    s = torch.cat((s, leaf[3].expand(n, 1)), 1)
                o = torch.softmax(s, 1)[:, :n] @ leaf[2]
                out[rows, h] = o.detach()
                if st["train"]:
                    got = torch.autograd.grad(o, leaf, st["grad"][rows, h].double())
            if st["train"]:
                dq[rows, h] = got[0]
                dk[rows, h * G // H] += got[1]
                dv[rows, h * G // H] += got[2]
                if sink is not None:
                    d_sink[h] += got[3]
    if not st["train"]:
        return out
    found = dict(out=out, d_q=dq, d_k=dk, d_v=dv)
    if sink is not None:
        found["d_sink_logits"] = d_sink
    return found
