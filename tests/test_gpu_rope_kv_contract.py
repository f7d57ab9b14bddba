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
from test_gpu_rope_kv import U, gen, ints, randn

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
