"""What the rotary / ragged-batch KV-cache calls promise beside their results, on the GPU: buffers that are one, error codes,
workspaces, accuracy where a lost tile or term would show.

Tolerances are bounds, stated beside their use (u = 2^-24, half a step of fp32)."""
import os
import subprocess
import sys

import pytest
import torch

import rope_kv_ref as ref
from conftest import ROOT
from test_gpu_rope_kv import U, attend_case, gen, ints, randn, run_attend, unaligned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,H,Hkv,dk", [(1, 3, 2, 1, 2), (1, 50, 4, 2, 4), (2, 300, 8, 2, 64), (4, 700, 16, 8, 128), (1, 5, 2, 2, 33)])
def test_one_gradient_buffer_for_both_norm_weights(engine, B, S, H, Hkv, dk):
    """gq is gk and dgq is dgk (one weight for queries and keys): the buffer receives both sums, every time the same bits."""
    g = gen(dk)
    qkv, w, start = randn(g, B * S, (H + 2 * Hkv) * dk), 1 + 0.2 * randn(g, dk), randn(g, dk)
    grads = [randn(g, B * h, S, dk) for h in (H, Hkv, Hkv)]
    freq = torch.tensor(ref.frequencies(dk // 2 * 2), dtype=torch.float64).cuda()
    how = dict(qkv=qkv, gq=w, gk=w, freq=freq)
    dqkv, alone = torch.empty_like(qkv), [torch.zeros(dk, device="cuda") for _ in range(2)]
    engine.qkv_norm_rope_bwd(*grads, dqkv, B, dgq=alone[0], dgk=alone[1], **how)
    first = None
    for _ in range(20):
        both, again = start.clone(), torch.empty_like(qkv)
        engine.qkv_norm_rope_bwd(*grads, again, B, dgq=both, dgk=both, **how)
        first = both if first is None else first
        assert torch.equal(both, first) and torch.equal(again, dqkv)
    # the sums over CTAs are 64-bit: each of the two alone is rounded once, and so is the result
    want = start.double() + alone[0].double() + alone[1].double()
    room = U * (alone[0].abs() + alone[1].abs() + first.abs()).double() * 1.001
    assert bool(((first.double() - want).abs() <= room).all())


def test_every_kind_of_refusal_is_reported(engine):
    """Two calls that each refuse a sequence, one reading after the other: neither report hides the other."""
    B, T, H, Hkv, dk, max_seq = 2, 3, 2, 1, 32, 16
    g = gen(3)
    K, V, Q = randn(g, B * Hkv, max_seq, dk), randn(g, B * Hkv, max_seq, dk), randn(g, B * H, T, dk)
    qkv = randn(g, B * T, (H + 2 * Hkv) * dk)
    assert engine.device_error() == 0
    for rows_first in (True, False):
        for rows in (rows_first, not rows_first):
            if rows:
                engine.kv_cache_extend(qkv, Q, K, V, ints([2, 15]))
            else:
                engine.kv_cache_compact(K, V, ints([[0, 1, 0], [1, 0, 0]]), ints([2, 2]), ints([2, 2]))
        engine.synchronize()
        assert [engine.device_error() for _ in range(3)] == [101, 102, 0]
    assert "ascending" in engine.last_error()


def test_binding_refuses_a_host_workspace(engine):
    """Large enough, but its address means nothing to a kernel: refused before anything is launched."""
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    ws = torch.zeros(engine.attention_workspace_bytes(), dtype=torch.uint8)
    before = engine.launch_count()
    for w in (ws, ws.pin_memory()):
        with pytest.raises(ValueError, match="engine's device"):
            engine.kv_cache_attend_tree(z(2, 8, 16), z(2, 8, 16), z(2, 3, 16), z(2, 3, 16), ints([2]), 1.0, workspace=w)
    assert engine.launch_count() == before


FIRST_CALL = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from axiom_b200.engine import Engine, EngineError
from test_gpu_rope_kv import attend_case, check_attend, run_attend
eng = Engine(0)
s = attend_case((3, 1, 8, 2, 128, [63, 64, 700], False, None), 7)
torch.cuda.synchronize()
side, refused = torch.cuda.Stream(), 0
for mode in ("relaxed", "global"):
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.stream(side):
            graph.capture_begin(capture_error_mode=mode)
            try:
                if {own}:
                    eng.set_stream(side.cuda_stream)
                eng.kv_cache_attend_tree(s["K"], s["V"], s["Q"], s["out"], s["lens"], s["scale"])
            except EngineError as e:
                refused += 1
                assert "workspace" in str(e), e
            finally:
                eng.set_stream(0)
                graph.capture_end()
    except (RuntimeError, torch.AcceleratorError):
        pass                      # a capture that the refused call spoilt
    del graph
assert refused == 2, refused
check_attend(s, run_attend(eng, s))
check_attend(s, run_attend(eng, s))
assert eng.device_error() == 0
print("served")
"""


@pytest.mark.parametrize("own", [False, True], ids=["another-stream", "the-engines-stream"])
def test_a_first_call_under_a_capture_leaves_no_workspace_behind(own):
    """The engine's workspace cannot be made while a stream is captured: the call is refused, and the next one, outside, makes it
    with its counters at zero and is served."""
    code = FIRST_CALL.format(root=ROOT, tests=os.path.join(ROOT, "tests"), own=own)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "served" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------------- accuracy, lost tiles and lost terms

# B, T, H, Hkv, dk, lens, mask
NORM = [
    (3, 1, 8, 2, 128, [63, 64, 700], None),
    (1, 4, 2, 1, 128, [40000], "tree"),
    (2, 16, 4, 4, 64, [9000, 77], "tree"),
    (2, 7, 4, 1, 96, [5000, 31], None),
    (1, 8, 4, 1, 128, [12000], "tree"),
    (1, 16, 4, 1, 100, [20000], "tree"),
    (2, 16, 8, 2, 128, [3000, 1500], "shared"),
    (1, 40, 2, 1, 64, [30000], "tree"),
    (1, 300, 2, 1, 96, [200], None),
    (2, 5, 3, 3, 50, [9, 2000], "tree"),
    (1, 40, 2, 1, 128, [3000], "tree"),
]


@pytest.mark.parametrize("shift", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("case", NORM, ids=lambda c: "-".join(map(str, c[:5])) + f"-{c[6]}-{max(c[5])}")
def test_attention_error_of_a_head_in_the_norm(engine, case, shift):
    """||got - want|| <= 5e-6 ||want|| over the tokens of every head of every sequence.

    For normal q, k, v and scale 1/sqrt(dk), scores s have deviation 1.  A score's sum of dk/8 products on the tensor core loses up to
    2^-23 of itself at each, always towards zero: a factor of at most 1 - 16 * 2^-23 on s (dk = 128); with weights p = exp(s)/sum that
    moves the output by 2^-19 * sqrt(E_{p^2}(s - E_p s)^2) = 2^-19 * sqrt(2) of its norm, 2.7e-6 (the two small products are 2^-10 of
    it).  What the splits drop (lo.lo below 2^-20, lo rounded at 2^-21) is independent over products: below 4e-7 of a
    score's deviation, and as much again in P.V.  P.V's six accumulations lose 6 * 2^-23 = 7e-7, the folds in fp32 sqrt(100) u = 6e-7.
    Together 4.8e-6.  One tf32 product in the place of three is off by 2^-11 an operand, 3e-4; a lost tile of 32 keys of 40,000 by
    sqrt(32 / 40000) = 3e-2."""
    B, T, H, Hkv, dk, lens, kind = case
    s = attend_case((B, T, H, Hkv, dk, lens, False, kind), 141)
    if shift:
        s["K"] = unaligned(s["K"])
    got = run_attend(engine, s, shift=shift)
    want, _, _ = ref.attend_tree(s["K"], s["V"], s["Q"], s["out"], s["lens"], s["scale"], None, s["mask"])
    err = (got.double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    assert float(err.max()) <= 5e-6


# a token's result is one key's value row when that key's score stands far above all others: p V / p of one key, in three products
# (2^-20 lo.lo, 2 * 2^-21 the lo parts' roundings), at most 6 * 2^-23 lost in their sum, and some 12 roundings of u in folds,
# merges and the division: 3.4e-6 of an element
ONE_KEY = 4e-6

# B, T, H, Hkv, dk, lens: one item over many CTAs, in every variant; many items
DOMINATED = [
    (1, 1, 4, 1, 128, [40000]),
    (1, 2, 4, 1, 64, [9000]),
    (1, 4, 4, 1, 64, [9000]),
    (2, 4, 4, 1, 128, [5000, 700]),
    (1, 8, 4, 1, 64, [6000]),
    (2, 16, 8, 2, 128, [9000, 130]),
    (1, 16, 4, 1, 64, [9000]),
    (2, 40, 8, 2, 64, [9000, 1000]),
    (1, 40, 4, 1, 128, [5000]),
    (70, 2, 4, 2, 96, list(range(20, 720, 10))),
    (1, 2, 2, 1, 50, [3000]),
]


@pytest.mark.parametrize("case", DOMINATED, ids=lambda c: "-".join(map(str, c[:5])) + f"-{max(c[5])}")
def test_a_dominating_key_in_every_tile(engine, case):
    """One key of each (sequence, key head) scores 60 where the others stay below 10: its value row is every token's result, wherever
    it lies.  A tile or a piece that is lost, counted twice at the wrong weight, or read from another's slot changes the result by
    the size of a value."""
    B, T, H, Hkv, dk, lens = case
    g, group, max_seq = gen(151), H // Hkv, max(lens) + T + 3
    K, V, u = randn(g, B * Hkv, max_seq, dk), randn(g, B * Hkv, max_seq, dk), randn(g, B * Hkv, 1, dk)
    u *= dk ** 0.5 / u.norm(dim=-1, keepdim=True)
    Q = (u + 0.1 * randn(g, B * Hkv, group * T, dk)).view(B * H, T, dk).contiguous()
    top = 60 * u[:, 0] / dk ** 0.5
    L, at, item = ints(lens).repeat_interleave(Hkv).long(), torch.arange(B * Hkv, device="cuda"), 32 * torch.arange(B * Hkv, device="cuda")
    out, worst = torch.empty_like(Q), torch.zeros((), device="cuda")
    for n in range((max(lens) + 32) // 32):
        j = (item + 32 * n + (n * 13) % 32) % (L + 1)          # a cached row or the first new one: every token sees it
        held = K[at, j].clone()
        K[at, j] = top
        engine.kv_cache_attend_tree(K, V, Q, out, ints(lens), dk ** -0.5)
        want = V[at, j].view(B, Hkv, 1, 1, dk)
        worst = torch.maximum(worst, ((out.view(B, Hkv, group, T, dk) - want).abs() / want.abs().clamp_min(1e-3)).max())
        K[at, j] = held
    # (the others' weight: 40000 exp(10 - 54) is nothing; the score itself is at least 60 (1 - 0.1 * 4 * sqrt(1/dk)) > 54)
    assert float(worst) <= ONE_KEY


@pytest.mark.parametrize("T,H,dk", [(1, 2, 64), (4, 4, 64), (16, 8, 64), (40, 4, 128), (4, 4, 50)])
def test_large_scores_with_a_clear_winner(engine, T, H, dk):
    """Scores of several thousand: rows whose best score is 40 above the next, and more than twice a score's error, are one value row."""
    s = attend_case((2, T, H, 2, dk, [100, 333], False, "tree" if T > 1 else None), 161)
    s["Q"] *= 100
    s["scale"] = -1.0
    got = run_attend(engine, s).view(2, H, T, dk)
    K, V, Q = (s[x].double().view(2, -1, s[x].shape[1], dk) for x in "KVQ")
    rows = won = 0
    for b in range(2):
        see = torch.cat((torch.ones(T, int(s["lens"][b]), dtype=torch.bool), ref.visible(b, T, T, s["mask"])), 1).cuda()
        for h in range(H):
            k, v = K[b, h // (H // 2), :see.shape[1]], V[b, h // (H // 2), :see.shape[1]]
            score = (-(Q[b, h] @ k.T)).masked_fill(~see, -torch.inf)
            error = float((Q[b, h].abs() @ k.abs().T).max()) * (3 * 2.0 ** -20 + 3 * dk / 8 * 2.0 ** -23)
            best = score.topk(2, -1)
            clear = best.values[:, 0] - best.values[:, 1] > 40 + 2 * error
            rows, won = rows + T, won + int(clear.sum())
            want = v[best.indices[:, 0]][clear]
            assert bool(((got[b, h].double()[clear] - want).abs() <= ONE_KEY * want.abs() + 1e-12).all())
    assert won > rows / 2


@pytest.mark.parametrize("B,S,H,Hkv,dk,rot,pairing", [(5, 1000, 8, 4, 64, 64, "half"), (1, 4096, 12, 4, 80, 32, "interleaved"), (2, 700, 6, 2, 50, 50, "half"),
                                                      (1, 262144, 16, 8, 128, 128, "half")])
def test_norm_gradients_in_the_norm(engine, B, S, H, Hkv, dk, rot, pairing):
    """||dg - want|| <= 4e-6 ||want||.  Terms d * u carry some 5 u of independent error each (angle, sine and cosine, rotation,
    reciprocal root, products), 3e-7 of the sum's norm; a lane's n sequential fp32 additions of terms of either sign add
    u sqrt(n / 6): 6.5e-7 for the 708 of the longest case; the rest is 64-bit.  Below 1.2e-6, four deviations of
    which would be 4e-6.  One token lost of 262,144 is off by 2e-3."""
    if B * S > 1 << 17 and torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 20 GB")
    g = gen(171)
    qkv, w = randn(g, B * S, (H + 2 * Hkv) * dk), [1 + 0.3 * randn(g, dk) for _ in range(2)]
    grads = [randn(g, B * h, S, dk) for h in (H, Hkv, Hkv)]
    freq = torch.tensor(ref.frequencies(rot), dtype=torch.float64).cuda()
    dg, dqkv = [torch.zeros(dk, device="cuda") for _ in range(2)], torch.empty_like(qkv)
    engine.qkv_norm_rope_bwd(*grads, dqkv, B, qkv=qkv, gq=w[0], gk=w[1], freq=freq, pairing=pairing, amplitude=1.25, dgq=dg[0], dgk=dg[1])
    x, pos = qkv.view(B, S, H + 2 * Hkv, dk), torch.arange(S, device="cuda")
    for got, d, first, heads in ((dg[0], grads[0], 0, H), (dg[1], grads[1], H, Hkv)):
        want = torch.zeros(dk, dtype=torch.float64, device="cuda")
        for b in range(B):
            for h in range(heads):
                xh = x[b, :, first + h].double()
                unit = xh * torch.rsqrt((xh * xh).mean(-1, keepdim=True) + 1e-6)
                turned = ref.rope_head(d[b * heads + h].double(), None, 0.0, -pos, freq, pairing, 1.25)      # the transposed rotation
                want += (turned * unit).sum(0)
        assert float((got.double() - want).norm() / want.norm()) <= 4e-6


def test_norm_gradients_of_many_tokens_keep_their_accuracy(engine):
    """A lane's chain of fp32 additions does not grow with the batch: 262,144 tokens of 16 + 2*8 heads of 128 make at most 142 additions
    of query terms a lane (283 steps, every second one of query heads), u sqrt(142 / 6) = 2.9e-7 of the sum's norm at most, and the
    terms' own errors add 0.8e-7 in square: 3.0e-7.  (A chain of all 708 that one set of CTAs makes is at 4.6e-7.)"""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 20 GB")
    S, H, Hkv, dk = 262144, 16, 8, 128
    g = gen(181)
    qkv, w, dg = randn(g, S, (H + 2 * Hkv) * dk), 1 + 0.3 * randn(g, dk), torch.zeros(dk, device="cuda")
    grads = [randn(g, h, S, dk) for h in (H, Hkv, Hkv)]
    freq, pos = torch.tensor(ref.frequencies(dk), dtype=torch.float64).cuda(), torch.arange(S, device="cuda")
    engine.qkv_norm_rope_bwd(*grads, torch.empty_like(qkv), 1, qkv=qkv, gq=w, gk=w, freq=freq, dgq=dg)
    want = torch.zeros(dk, dtype=torch.float64, device="cuda")
    for h in range(H):
        xh = qkv.view(S, -1, dk)[:, h].double()
        want += (ref.rope_head(grads[0][h].double(), None, 0.0, -pos, freq, "half", 1.0) * xh * torch.rsqrt((xh * xh).mean(-1, keepdim=True) + 1e-6)).sum(0)
    assert float((dg.double() - want).norm() / want.norm()) <= 3.5e-7


@pytest.mark.parametrize("T,H,dk", [(1, 2, 64), (5, 4, 50), (16, 8, 128), (40, 8, 64)])
def test_infinities_that_a_token_sees(engine, T, H, dk):
    """A cached key with an infinity is, for every row, an infinite score as the formula has it, or NaN (its two parts, as operands of
    the products, meet zeros); a cached value with one makes its column infinite or NaN; the other key head's and the other
    sequence's results keep their bits."""
    s = attend_case((2, T, H, 2, dk, [90, 200], False, None), 191)
    clean = run_attend(engine, s).view(2, 2, -1, dk)          # [sequence][key head][rows]
    for x, row in (("K", 33), ("V", 77)):
        bad = {**s, x: s[x].clone()}
        bad[x].view(2, 2, -1, dk)[1, 0, row, 5] = float("inf")
        got = run_attend(engine, bad).view(2, 2, -1, dk)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1, 1], clean[1, 1])
        if x == "K":
            k, v = (bad[w].view(2, 2, -1, dk)[1, 0, :200 + T].double() for w in "KV")
            score = s["scale"] * s["Q"].view(2, 2, -1, dk)[1, 0].double() @ k.T
            token = torch.arange(score.shape[0], device="cuda") % T
            p = torch.softmax(score.masked_fill(torch.arange(200 + T, device="cuda") > 200 + token[:, None], -torch.inf), -1)
            want, nan = p @ v, got[1, 0].isnan().all(-1)
            assert bool((nan | want.isfinite().all(-1)).all())                       # +inf: nothing but NaN
            assert float((got[1, 0].double() - want)[~nan].norm()) <= 5e-6 * float(want[~nan].norm())
        else:
            assert not bool(got[1, 0, :, 5].isfinite().any())
            assert torch.equal(got[1, 0, :, :5], clean[1, 0, :, :5]) and torch.equal(got[1, 0, :, 6:], clean[1, 0, :, 6:])


def test_a_failed_allocation_is_not_the_next_calls_error(engine):
    """The runtime keeps the error of a call that failed; it has been reported, and the launches behind it are not to blame."""
    H, dk = 2, 32
    qkv, out = torch.randn(3, 3 * H * dk, device="cuda"), [torch.zeros(H, 3, dk, device="cuda") for _ in range(3)]
    for _ in range(2):
        assert engine.lib.axb_storage_alloc(1 << 50) is None and "storage_alloc" in engine.last_error()
        engine.qkv_norm_rope(qkv, *out, 1)
    assert torch.equal(out[2], qkv.view(3, 3, H, dk)[:, 2].transpose(0, 1))
