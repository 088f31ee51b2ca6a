"""Attention of the language models beside the diffusion models: one pass each through the operators, in plain torch or in kernels.

* ``window_attention``: causal grouped-query attention in which a query sees the last ``window`` keys and the first ``sinks`` ones, with
  an optional learned logit per head that takes part in the softmax and carries no value. Prompts, parts of prompts behind a cache,
  single tokens and a few drafted tokens over a cache, training steps.
* ``relative_attention``: attention over a whole prompt with a learned bias for buckets of relative positions, and its gradient.

Scores have unit variance, as normalised and rotated queries and keys give; values and gradients are unit normal. All is drawn on
the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16


# ---- the cases -------------------------------------------------------------------------------------------------------------
# op: window / relative; way: step (a few tokens over a cache), prompt, chunk (a part of a prompt behind a cache), train
def listed():
    return [
        # one token of one sequence, sliding layer of a 64-head stack with learned sink logits: latency
        _step("window_step_1", batch=1, q=1, heads=64, kv_heads=8, dim=64, cache=512, shortest=300, longest=300, window=128, sinks=0, logits=True),
        # a token each for sixteen sequences of different lengths that keep their first four tokens
        _step("window_step_batch", batch=16, q=1, heads=32, kv_heads=8, dim=128, cache=16384, shortest=1, longest=16384, window=4096, sinks=4, logits=False),
        # a token each over long caches without a window: the memory's rate
        _step("causal_step_long", batch=4, q=1, heads=32, kv_heads=8, dim=128, cache=131072, shortest=70001, longest=131072, window=0, sinks=0, logits=False),
        # five drafted tokens at once
        _step("window_step_drafts", batch=8, q=5, heads=32, kv_heads=8, dim=128, cache=4096, shortest=17, longest=4091, window=1024, sinks=4, logits=False),
        # a prompt through a sliding layer of the 64-head text encoder
        _prompt("window_prompt", batch=1, length=300, heads=64, kv_heads=8, dim=64, window=128, sinks=0, logits=True, ragged=False),
        # a long document
        _prompt("window_prompt_long", batch=1, length=8192, heads=32, kv_heads=8, dim=128, window=1024, sinks=4, logits=False, ragged=False),
        # the next part of two prompts whose beginnings are in the cache
        _chunk("window_chunk", batch=2, q=777, cache=6000, heads=28, kv_heads=4, dim=128, window=2048, sinks=4, logits=False),
        # training with a window, and with learned sink logits at an odd length
        _train("window_train", batch=2, length=2048, heads=32, kv_heads=8, dim=128, window=512, sinks=4, logits=False, ragged=False),
        _train("window_train_odd", batch=1, length=1531, heads=64, kv_heads=8, dim=64, window=128, sinks=0, logits=True, ragged=False),
        # a caption of 77 tokens, a padded batch of prompts of the 64-head encoder, and a training step on padded prompts
        _relative("relative_prompt_short", way="prompt", batch=1, length=77, heads=64, dim=64, buckets=32, distance=128, ragged=False),
        _relative("relative_prompt_batch", way="prompt", batch=8, length=512, heads=64, dim=64, buckets=32, distance=128, ragged=True),
        _relative("relative_train", way="train", batch=4, length=512, heads=64, dim=64, buckets=32, distance=128, ragged=True),
    ]


def _step(name, **c):
    return dict(name=name, op="window", way="step", **c)


def _prompt(name, **c):
    return dict(name=name, op="window", way="prompt", **c)


def _chunk(name, **c):
    return dict(name=name, op="window", way="chunk", **c)


def _train(name, **c):
    return dict(name=name, op="window", way="train", **c)


def _relative(name, **c):
    return dict(name=name, op="relative", **c)


def _between(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["step", "step", "prompt", "chunk", "train", "relative", "relative train"])
    heads, kv_heads, dim = rng.choice([(64, 8, 64), (32, 8, 128), (28, 4, 128), (16, 16, 64), (20, 4, 64), (12, 4, 128)])
    logits = rng.random() < 0.4
    sinks = rng.choice([0, 0, 1, 4, 4, rng.randint(2, 200)])
    if kind == "step":
        batch, q = rng.randint(1, 16), rng.choice([1, 1, 2, rng.randint(3, 8)])
        longest = _between(rng, 1, 250000 // batch)
        shortest = rng.randint(1 if batch == 1 else 0, longest)      # a batch may have places that are not in use
        c = _step("", batch=batch, q=q, heads=heads, kv_heads=kv_heads, dim=dim, cache=longest + rng.randint(0, 99), shortest=shortest,
                  longest=longest, window=rng.choice([0, _between(rng, 1, 8192)]), sinks=sinks, logits=logits)
    elif kind == "prompt":
        batch = rng.randint(1, 4)
        c = _prompt("", batch=batch, length=_between(rng, 1, 4096 // batch), heads=heads, kv_heads=kv_heads, dim=dim, window=rng.choice([0, _between(rng, 1, 2048)]),
                    sinks=sinks, logits=logits, ragged=rng.random() < 0.5)
    elif kind == "chunk":
        q = _between(rng, 20, 2000)
        c = _chunk("", batch=rng.randint(1, 2), q=q, cache=q + _between(rng, 1, 6000), heads=heads, kv_heads=kv_heads, dim=dim,
                   window=rng.choice([0, _between(rng, 1, 4096)]), sinks=sinks, logits=logits)
    elif kind == "train":
        batch = rng.randint(1, 4)
        c = _train("", batch=batch, length=_between(rng, 8, 3000 // batch), heads=heads, kv_heads=kv_heads, dim=dim, window=rng.choice([0, _between(rng, 16, 1024)]),
                   sinks=sinks, logits=logits, ragged=rng.random() < 0.5)
    else:
        heads, dim = rng.choice([(64, 64), (12, 64), (16, 128), (6, 64)])
        batch, train = rng.randint(1, 8), kind != "relative"
        buckets = rng.choice([32, 32, 32, 16, 64])
        c = _relative("", way="train" if train else "prompt", batch=batch, length=_between(rng, 8 if train else 1, min(1024, (2048 if train else 4096) // batch)), heads=heads, dim=dim,
                      buckets=buckets, distance=rng.choice([128, 128, rng.randint(buckets, 256)]), ragged=rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(BF16)
    whole = lambda lo, hi: torch.randint(lo, hi + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    B, H, D = case["batch"], case["heads"], case["dim"]
    G = case.get("kv_heads", H)
    st = dict(case, kv_len=None, q_start=0, sink_logits=None, table=None)
    if case["way"] == "step":
        # caches [batch, kv_heads, positions, dim], as the decoder keeps them
        T, n = case["cache"], case["q"]
        st["k"], st["v"] = (normal(B, G, T, D).transpose(1, 2) for _ in range(2))
        st["kv_len"] = whole(case["shortest"], case["longest"])
        st["q_start"] = st["kv_len"] - n
    elif case["way"] == "chunk":
        T, n = case["cache"], case["q"]
        st["k"], st["v"] = (normal(B, G, T, D).transpose(1, 2) for _ in range(2))
        st["q_start"] = whole(0, T - n)
        st["kv_len"] = st["q_start"] + n
    else:
        n = case["length"]
        st["k"], st["v"] = normal(B, n, G, D), normal(B, n, G, D)
        if case["ragged"]:
            st["kv_len"] = whole((n + 1) // 2, n)
    st["q"] = normal(B, n, H, D)
    if case["op"] == "relative":
        st["q"] = (st["q"].float() * D ** -0.5).to(BF16)      # these encoders train without a scale in the attention
        st["table"] = normal(case["buckets"], H)
        st["scale"] = 1.0
    else:
        st["scale"] = D ** -0.5
        if case["logits"]:
            st["sink_logits"] = normal(H)
    if case["way"] == "train":
        d = normal(B, n, H, D)
        if st["kv_len"] is not None:                          # the loss leaves padded rows out
            d = d * (torch.arange(n, device=DEV)[None, :] < st["kv_len"][:, None])[:, :, None, None]
        st["grad"] = d
        for name in ("q", "k", "v", "table", "sink_logits"):
            if st[name] is not None:
                st[name].requires_grad_()
    return st


def run(st):
    if own:
        return _kernels(st)
    with torch.no_grad():
        return _plain(st)


def _kernels(st):
    from mojodiffusion_b200 import ops

    if st["op"] == "window":
        call = lambda: ops.window_attention(st["q"], st["k"], st["v"], window=st["window"] or None, sinks=st["sinks"], kv_len=st["kv_len"],
                                            q_start=st["q_start"], sink_logits=st["sink_logits"])
    else:
        call = lambda: ops.relative_attention(st["q"], st["k"], st["v"], st["table"], max_distance=st["distance"], scale=st["scale"], kv_len=st["kv_len"])
    if st["way"] != "train":
        with torch.no_grad():
            return call()
    out = call()
    names = [n for n in ("q", "k", "v", "table", "sink_logits") if st[n] is not None]
    grads = torch.autograd.grad(out, [st[n] for n in names], st["grad"])
    return dict({"out": out.detach()}, **dict(zip(["d_" + n for n in names], grads)))


# ---- the plain form ----------------------------------------------------------------------------------------------------------
def _plain(st):
    q, k, v = (st[n].transpose(1, 2).float() for n in ("q", "k", "v"))
    B, H, n, D = q.shape
    G, T = k.shape[1], k.shape[2]
    rep = H // G
    grouped = lambda t: t.reshape(B, G, rep * n, -1)          # the query heads of a key head, one below the other
    heads = lambda t: t.reshape(B, H, n, -1)
    kT, vT = k.transpose(-1, -2), v.transpose(-1, -2)
    s = heads(grouped(q) @ kT) * st["scale"]
    key = torch.arange(T, device=q.device)
    if st["op"] == "window":
        at = torch.arange(n, device=q.device)
        at = st["q_start"][:, None] + at if isinstance(st["q_start"], torch.Tensor) else (st["q_start"] + at)[None]
        seen = key <= at[:, :, None]
        if st["window"]:
            seen = seen & ((at[:, :, None] - key < st["window"]) | (key < st["sinks"]))
    else:
        which = _bucket(key[None, :] - torch.arange(n, device=q.device)[:, None], st["buckets"], st["distance"])
        s = s + st["table"].float().t()[:, which]
        seen = torch.ones(1, n, T, dtype=torch.bool, device=q.device)
    if st["kv_len"] is not None:
        seen = seen & (key < st["kv_len"][:, None, None])
    s = s.masked_fill(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    sink = st["sink_logits"]
    if sink is not None:
        sink = sink.float()[None, :, None, None]
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == -math.inf, 0.0)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    share = 1.0 / total.masked_fill(total == 0, 1.0)
    p = e * share
    o = heads(grouped(p) @ v)
    back = lambda t: t.transpose(1, 2).to(BF16)
    if st["way"] != "train":
        return back(o)
    d = st["grad"].transpose(1, 2).float()
    delta = (d * o).sum(-1, keepdim=True)
    ds = p * (heads(grouped(d) @ vT) - delta)
    found = dict(out=back(o), d_q=back(heads(grouped(ds) @ k) * st["scale"]), d_k=back(grouped(ds).transpose(-1, -2) @ grouped(q) * st["scale"]),
                 d_v=back(grouped(p).transpose(-1, -2) @ grouped(d)))
    if st["table"] is not None:
        sums = torch.zeros(H, st["buckets"], dtype=torch.float64, device=q.device)
        sums.index_add_(1, which.reshape(-1), ds.sum(0, dtype=torch.float64).reshape(H, -1))
        found["d_table"] = sums.t().to(BF16)
    if sink is not None:
        found["d_sink_logits"] = -(torch.exp(sink - top) * share * delta).sum((0, 2, 3), dtype=torch.float64).to(BF16)
    return found


def _bucket(rel, buckets, distance):
    """Half of the buckets for each direction; of them half for single distances, the rest for distances that grow by equal factors up
    to ``distance``. The borders are found in whole numbers: n is in the k-th of m such buckets when (n / exact)^m >= (distance / exact)^k."""
    half = buckets // 2
    exact = half // 2
    m = half - exact
    borders = [next(n for n in range(exact, distance + 1) if n ** m * exact ** k >= distance ** k * exact ** m) for k in range(1, m)]
    n = rel.abs()
    far = exact + torch.bucketize(n, torch.tensor(borders, device=rel.device), right=True)
    return torch.where(rel > 0, half, 0) + torch.where(n < exact, n, far)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    B, H, D = case["batch"], case["heads"], case["dim"]
    G = case.get("kv_heads", H)
    if case["way"] == "step":
        n, length = case["q"], (case["shortest"] + case["longest"]) / 2
        sees = min(length, case["window"] + case["sinks"] + (n - 1) / 2) if case["window"] else length
        pairs, rows = B * n * sees, B * (min(length, sees + n - 1) if case["window"] else length)
    elif case["way"] == "chunk":
        n, T = case["q"], case["cache"]
        start = (T - n) // 2                                   # the middle of the places where a part may begin
        pairs = B * _pairs(start, n, case["window"], case["sinks"])
        rows = B * min(start + n, n + case["window"] + case["sinks"] if case["window"] else start + n)
    else:
        n = case["length"]
        mean = (((n + 1) // 2) + n) / 2 / n if case["ragged"] else 1.0
        pairs, rows = B * (_pairs(0, n, case["window"], case["sinks"]) if case["op"] == "window" else n * n * mean), B * n * mean
    flops = 4 * pairs * H * D
    moved = 2 * (2 * B * n * H * D + 2 * rows * G * D)          # q and the output, keys and values
    if case["way"] == "train":
        flops *= 3.5                                           # five products of the backward pass to two of the forward
        moved += 2 * (2 * B * n * H * D + 2 * rows * G * D)     # the output's gradient, dq, dk and dv
    if case["op"] == "relative":
        moved += 2 * case["buckets"] * H * (2 if case["way"] == "train" else 1)
    return {"bytes": moved, "flops": flops}


def _pairs(start, n, window, sinks):
    """Keys that n queries from position ``start`` see, together."""
    near = lambda p: min(p + 1, window) if window else p + 1
    return sum(near(p) + min(sinks, p + 1 - near(p)) for p in range(start, start + n))


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    train = case["way"] == "train"
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    B, n, H, D = q.shape
    T, G = k.shape[1], k.shape[2]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    table = st["table"].detach().double() if st["table"] is not None else None
    sink = st["sink_logits"].detach().double() if st["sink_logits"] is not None else None
    d_table = torch.zeros_like(table) if table is not None else None
    d_sink = torch.zeros_like(sink) if sink is not None else None
    index = torch.tensor([_place(r, case["buckets"], case["distance"]) for r in range(1 - n, n)], device=q.device) if table is not None else None
    for b in range(B):
        length = T if st["kv_len"] is None else int(st["kv_len"][b])
        start = int(st["q_start"][b]) if isinstance(st["q_start"], torch.Tensor) else st["q_start"]
        i = torch.arange(n, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None, :]
        hidden = torch.zeros(n, length, dtype=torch.bool, device=q.device)
        if case["op"] == "window":
            hidden |= j > i + start
            if case["window"]:
                hidden |= (j <= i + start - case["window"]) & (j >= case["sinks"])
        for h in range(H):
            leaf = [t.clone().requires_grad_() for t in (q[b, :, h], k[b, :length, h * G // H], v[b, :length, h * G // H])]
            extra = [t.clone().requires_grad_() for t in ([table[:, h]] if table is not None else []) + ([sink[h]] if sink is not None else [])]
            with torch.enable_grad():
                s = torch.einsum("id,jd->ij", leaf[0], leaf[1]) * st["scale"]
                if table is not None:
                    s = s + extra[0][index[(j - i) + (n - 1)]]
                s = s.masked_fill(hidden, float("-inf"))
                last = extra[-1].expand(n, 1) if sink is not None else torch.full((n, 1), -1e300, dtype=s.dtype, device=s.device)
                p = torch.softmax(torch.cat((s, last), 1), 1)[:, :length]            # -1e300: a row without keys comes out as zeros
                p = p.masked_fill(hidden, 0.0)
                o = p @ leaf[2]
                out[b, :, h] = o.detach()
                if train:
                    got = torch.autograd.grad(o, leaf + extra, st["grad"][b, :, h].double())
            if train:
                dq[b, :, h] = got[0]
                dk[b, :length, h * G // H] += got[1]
                dv[b, :length, h * G // H] += got[2]
                if table is not None:
                    d_table[:, h] += got[3]
                if sink is not None:
                    d_sink[h] += got[-1]
    if not train:
        return out
    found = dict(out=out, d_q=dq, d_k=dk, d_v=dv)
    if table is not None:
        found["d_table"] = d_table
    if sink is not None:
        found["d_sink_logits"] = d_sink
    return found


def _place(rel, buckets, distance):
    """The bucket of one relative position, in whole numbers."""
    per_side, n = buckets // 2, abs(rel)
    single = per_side // 2
    if n >= single:
        steps = per_side - single
        n = single + sum((n ** steps) * single ** k >= distance ** k * single ** steps for k in range(1, steps))
    return n + (per_side if rel > 0 else 0)
