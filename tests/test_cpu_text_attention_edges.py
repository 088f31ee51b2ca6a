"""The language models' attention at its edges, as far as a CPU shows it."""
import re
import subprocess
from pathlib import Path

import pytest
import torch

import mojodiffusion_b200
from mojodiffusion_b200 import ops as O

CSRC = Path(mojodiffusion_b200.__file__).parent / "csrc"


def _some_order_ends_in_a_deadlock(places, tiles=7):
    """All orders of the three parties that pass the staged queries of the dk / dv kernel with one score buffer: the warp that stages, another warp of its
    group, and the issuer of the products. A barrier is the number of phases that it has behind it; waiting for phase n, a warp sees only whether the
    phase that now runs has another parity than n, as mbarrier.try_wait.parity tells."""
    stager, other, issuer = [], [], [("end", "scores", 0)]
    for i in range(tiles):
        wait = [("wait", f"staged{i % places}", i // places), ("wait", "scores", i), ("arrive", "probabilities", i)]
        stager += [("end", f"staged{i % places}", i // places)] + wait
        other += wait
        issuer += [("wait", "probabilities", i)] + ([("end", "scores", i + 1)] if i + 1 < tiles else [])
    programs = (stager, other, issuer)
    start = ((0, 0, 0), (("probabilities", 0), ("scores", 0), *((f"staged{p}", 0) for p in range(places))), 0)
    todo, known = [start], {start}
    while todo:
        at, barriers, arrived = todo.pop()
        moved = False
        for w, program in enumerate(programs):
            if at[w] == len(program):
                continue
            do, name, n = program[at[w]]
            phases, here = dict(barriers), arrived
            if do == "wait" and phases[name] % 2 == n % 2:
                continue
            if do == "end":
                phases[name] += 1
            elif do == "arrive":
                here = (here + 1) % 2
                phases[name] += here == 0
            moved = True
            after = (tuple(p + (v == w) for v, p in enumerate(at)), tuple(sorted(phases.items())), here)
            if after not in known:
                known.add(after)
                todo.append(after)
        if not moved and any(at[w] < len(program) for w, program in enumerate(programs)):
            return True
    return False


def test_the_model_of_the_staged_queries():
    assert _some_order_ends_in_a_deadlock(1) and not _some_order_ends_in_a_deadlock(2)


def test_staged_queries_cannot_lose_a_warp():
    """Heads of 64 have one score buffer: the barriers per warpgroup that the kernel declares leave no order in which its warps wait for ever."""
    text = (CSRC / "text_attention_bwd.cu").read_text()
    declared = re.search(r"\blv_full\[2\](?:\[(\w+)\])?", text).group(1)
    given = re.search(r"constexpr int PLACES = 3 - BUFS;", text) if declared == "PLACES" else None
    assert not _some_order_ends_in_a_deadlock(2 if given else 1)


@pytest.mark.parametrize("stages", [2, 3])
def test_a_prompt_that_gives_up_waits_for_all_its_copies(stages, tmp_path):
    """The forward kernel's loop behind a wait that ran out, compiled for the host with barriers that write down who waits for them: the last copy of Q and
    the last one into every place of K and V, whatever the number of copies so far (K and V of a key tile in turn, one Q per item)."""
    text = (CSRC / "text_attention_fwd.cu").read_text()
    loop = re.search(r"\n( +)for \(int j = max\(loads.*?\n\1}\n", text, re.S)
    assert loop, "the loop over the copies on the way"
    source, program = tmp_path / "landing.cpp", tmp_path / "landing"
    source.write_text("""
#include <algorithm>
#include <cstdint>
#include <cstdio>
using std::max;
constexpr int STAGES = %d;
uint64_t q_full, k_full[STAGES], v_full[STAGES];
uint64_t globaltimer_ns() { return 0; }
bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  if (bar == &q_full) printf(" q,0,%%u", parity);
  else if (bar >= k_full && bar < k_full + STAGES) printf(" k,%%d,%%u", (int)(bar - k_full), parity);
  else printf(" v,%%d,%%u", (int)(bar - v_full), parity);
  return true;
}
int main() {
  for (int loads = 0; loads <= 6 * STAGES + 1; ++loads)
    for (int n_items = 0; n_items <= 4; ++n_items) {
      printf("%%d %%d", loads, n_items);
%s
      printf("\\n");
    }
}
""" % (stages, loop.group(0)))
    subprocess.run(["g++", "-std=c++17", "-o", str(program), str(source)], check=True)
    lines = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == (6 * stages + 2) * 5
    for line in lines:
        loads, items, *waits = line.split()
        want = {("q", 0): (int(items) - 1) % 2} if int(items) else {}
        for j in range(int(loads)):
            want["kv"[j % 2], j // 2 % stages] = j // 2 // stages % 2
        got = {(kind, int(place)): int(parity) for kind, place, parity in (w.split(",") for w in waits)}
        assert len(waits) == len(got) and got == want, line


def _t5(per_layer):
    from mojodiffusion_b200.models.text.t5 import T5Config, T5Encoder

    torch.manual_seed(0)
    return T5Encoder(T5Config(vocab_size=50, d_model=16, d_kv=8, d_ff=24, num_layers=3, num_heads=2, relative_attention_num_buckets=8, relative_attention_max_distance=10,
                              per_layer_bias=per_layer))


@pytest.mark.parametrize("per_layer", [False, True])
def test_t5_with_fused_attention_calls_what_is_hooked_or_replaced(per_layer, monkeypatch):
    """Attention modules and tables with hooks, forwards of their own or other classes run as with the separate operations, and change the result as there."""
    ids = torch.randint(0, 50, (3, 23), generator=torch.Generator().manual_seed(1))
    mask = (torch.arange(23)[None] < torch.tensor([23, 7, 15])[:, None]).long()
    kept = mask.bool()
    fused = []
    monkeypatch.setattr(O, "relative_attention", lambda *a, _f=O.relative_attention, **k: fused.append(1) or _f(*a, **k))

    def both(enc):
        enc.cfg.fused_attention = False
        want = enc(ids, mask)
        enc.cfg.fused_attention = True
        del fused[:]
        got = enc(ids, mask)
        assert float((got - want)[kept].abs().max()) < 1e-5
        return want, len(fused)

    enc = _t5(per_layer)
    plain, count = both(enc)
    assert count == 3
    attention = [b.layer[0].SelfAttention for b in enc.encoder.block]
    tables = [a.relative_attention_bias for a in attention if hasattr(a, "relative_attention_bias")]
    seen = []
    for place, change in (("hook", lambda: attention[1].register_forward_hook(lambda m, a, out: seen.append(len(a)) or out * 2)),
                          ("pre-hook", lambda: attention[1].register_forward_pre_hook(lambda m, a: (a[0] * 2, *a[1:]))),
                          ("table", lambda: tables[0].register_forward_hook(lambda m, a, out: out * 3))):
        handle = change()
        other, count = both(enc)
        assert float((other - plain)[kept].abs().max()) > 1e-3
        assert count == (2 if place != "table" or per_layer else 0)
        handle.remove()
    assert seen == [2, 2]
    forward = attention[2].forward
    attention[2].forward = lambda x, bias: forward(x, bias) + 1
    other, count = both(enc)
    assert count == 2 and float((other - plain)[kept].abs().max()) > 1e-3
    del attention[2].forward
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: None)
    try:
        assert both(enc)[1] == 0
    finally:
        handle.remove()
    assert both(enc)[1] == 3


@pytest.mark.parametrize("fused", [False, True])
def test_gpt_oss_attention_that_is_hooked_or_replaced(fused):
    """The attention's arguments stay x, cos, sin and the mask for whoever looks at them or takes its place."""
    from mojodiffusion_b200.models.text.gpt_oss import GptOssConfig, GptOssEncoder

    torch.manual_seed(0)
    cfg = GptOssConfig(vocab_size=50, hidden_size=16, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=8, intermediate_size=16, num_local_experts=4,
                       num_experts_per_tok=2, sliding_window=5)
    enc = GptOssEncoder(cfg)
    ids = torch.randint(0, 50, (2, 17), generator=torch.Generator().manual_seed(1))
    mask = (torch.arange(17)[None] < torch.tensor([17, 6])[:, None]).long()
    want = enc(ids, mask)
    cfg.fused_attention = fused
    close = lambda: float((enc(ids, mask) - want)[mask.bool()].abs().max()) < 1e-5
    args = []
    handle = enc.layers[0].self_attn.register_forward_pre_hook(lambda m, a: args.append(len(a)))
    assert close() and args == [4]
    handle.remove()
    att = enc.layers[1].self_attn
    forward = att.forward
    att.forward = lambda x, cos, sin, key_mask: forward(x, cos, sin, key_mask)
    assert close()
    del att.forward
    assert close()


@pytest.mark.parametrize("start", [2**30 - 1, 2**30, 2**31 - 10, -2**31, -2**30])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_no_window_at_far_positions(start, as_tensor):
    """Without a window, and with one beyond 32 bits, every earlier key is seen wherever the queries stand; none before the first key."""
    q, k, v = (torch.randn(1, s, 2, 8, generator=torch.Generator().manual_seed(s)) for s in (3, 20, 21))
    v = v[:, :20]
    at = torch.tensor([start], dtype=torch.int32) if as_tensor else start
    want = O.window_attention(q, k, v, q_start=20) if start > 0 else torch.zeros_like(q)
    for window in (None, 1 << 40):
        assert torch.equal(O.window_attention(q, k, v, window, q_start=at), want)
    assert torch.equal(O.window_attention(q, k, v, 7, q_start=at), torch.zeros_like(q))
    # other keys beside the two seen: another order of the 8 products of a score, 8 * 2^-24 * 20 of it and as much of a probability, over values up to 4
    first = O.window_attention(q, k[:, :2], v[:, :2], q_start=20) if start > 0 else torch.zeros_like(q)
    assert float((O.window_attention(q, k, v, 7, 2, q_start=at) - first).abs().max()) < 4 * 2 * 8 * 2.0 ** -24 * 20
