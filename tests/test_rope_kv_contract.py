"""What the rotary / ragged-batch KV-cache calls promise beside their results, without a GPU: refusals of buffers that meet, counters
that every launch leaves at zero."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import ROOT
from test_rope_kv_host import INVALID_SHAPE, P, attend_call, bwd_call, compact_call, eng, extend_call, rope_call  # noqa: F401


@pytest.mark.parametrize("override", [dict(dgk=P[9] + 64), dict(dgq=P[10] + 252), dict(dgq=P[8] + 128), dict(dgk=P[8]), dict(dgk=P[8] + 4 * (2 * 8 * 64 - 1))])
def test_norm_gradients_that_overlap_are_refused(eng, override):  # noqa: F811
    assert eng.lib.axb_qkv_norm_rope_bwd(*bwd_call(**override)) == INVALID_SHAPE
    assert "two outputs overlap" in eng.last_error()


@pytest.mark.parametrize("override", [dict(dgk=P[9]), dict(dgk=P[9] + 256), dict(dgq=P[8] + 4 * 2 * 8 * 64), dict(dgq=None), dict(dgk=None)])
def test_norm_gradients_side_by_side_or_in_one_buffer_are_not(eng, override):  # noqa: F811
    """A call that passes every check of its arguments ends at the missing device here (never run with one: the addresses are made up)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    assert eng.lib.axb_qkv_norm_rope_bwd(*bwd_call(**override)) != INVALID_SHAPE
    assert "no CUDA device" in eng.last_error()


@pytest.fixture(scope="module")
def line(tmp_path_factory):
    here, root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kv_tree_line_host"), ROOT
    so = str(tmp_path_factory.mktemp("line") / "line.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-shared", "-fPIC", "-I", here, "-I", os.path.join(root, "axiom_b200", "csrc"), "-I",
                    os.path.join(root, "include"), os.path.join(here, "line.cpp"), "-o", so], check=True)
    return C.CDLL(so)


# block_rows, tile_keys, min_stretch, gap: the warp-level kernel's lines
@pytest.mark.parametrize("how", [(8, 32, 4, 5), (16, 32, 4, 5), (32, 32, 4, 8)])
@pytest.mark.parametrize("give_up", [0, 3, 50, 100])
def test_the_work_line_and_its_counters(line, how, give_up):
    """The kernels' own division of a batch: every tile once, at most two shared pieces a CTA, and counters at zero after a launch
    in which CTAs gave up at any of their pieces (a counter left behind would make a later call add up pieces too early)."""
    left, would_stay = C.c_int(), 0
    for seed in range(60):
        B, T, per, Hkv, max_seq, ctas = [(1, 1, 4, 1, 3000, 148), (3, 7, 2, 2, 900, 148), (40, 3, 4, 3, 700, 148), (9, 16, 1, 2, 5000, 148),
                                         (2, 40, 3, 1, 333, 20), (300, 2, 4, 1, 90, 148)][seed % 6]
        assert line.line_check(1000 * give_up + seed, B, T, per, Hkv, max_seq, *how, ctas, give_up, C.byref(left)) == 0, seed
        would_stay += left.value
    assert (would_stay > 0) == (give_up > 0)      # without the arrivals of those that gave up, counters would stay behind


def test_a_refusal_does_not_hide_a_kernel_that_gave_up(line):
    for words, first in (([0, 0, 0], -1), ([94, 101, 102], 0), ([94, 0, 0], 0), ([0, 101, 102], 1), ([0, 0, 102], 2)):
        assert line.next_error((C.c_int * 3)(*words), 3) == first


class OtherGpusTensor:
    """What the binding asks of a tensor, of one that lies on GPU 1."""
    is_cuda, device = True, "cuda:1"

    def __init__(self, host):
        self.host, self.dtype, self.shape = host, host.dtype, host.shape

    def __getattr__(self, name):
        return getattr(self.host, name)

    def get_device(self):
        return 1


@pytest.fixture
def eng_on_0():
    from axiom_b200.engine import Engine
    e = Engine()
    e._on(0)            # as init(0) leaves it, where there is a device
    return e


def test_binding_refuses_a_workspace_elsewhere(eng, eng_on_0):  # noqa: F811
    import torch
    host = torch.zeros(1 << 25, dtype=torch.uint8)
    for e, ws in ((eng, host), (eng_on_0, host), (eng_on_0, OtherGpusTensor(host))):
        with pytest.raises(ValueError, match="engine's device"):
            e._workspace(ws)
    assert eng._workspace(None) is None and eng._workspace(4096) == 4096


def test_binding_refuses_another_gpus_tensors(eng_on_0):
    import torch
    z = lambda *s, dtype=torch.float32: OtherGpusTensor(torch.zeros(*s, dtype=dtype))  # noqa: E731
    lens, k = z(2, dtype=torch.int32), z(4, 32, 16)
    with pytest.raises(ValueError, match="engine's device is wanted, got cuda:1"):
        eng_on_0.kv_cache_attend_tree(k, k, z(8, 3, 16), z(8, 3, 16), lens, 1.0)
    with pytest.raises(ValueError, match="engine's device"):
        eng_on_0.qkv_norm_rope(z(6, 128), z(8, 3, 16), z(4, 3, 16), z(4, 3, 16), 2)
    with pytest.raises(ValueError, match="engine's device"):
        eng_on_0.kv_cache_compact(k, k, z(2, 5, dtype=torch.int32), lens, lens)


# every input that a call reads while it writes, met by an output at its first or last bytes
MEETS = (
    [("axb_qkv_norm_rope", rope_call, dict(bqkv=P[5], gq=P[6], gk=P[7], pos=P[8]), o) for o in [
        dict(Q=P[5] + 4 * 511), dict(K=P[6] + 252), dict(V=P[7] - 4 * (2 * 2 * 64 - 1)), dict(Q=P[1] + 252), dict(K=P[8] + 4), dict(V=P[8] - 4)]] +
    [("axb_qkv_norm_rope_bwd", bwd_call, dict(bqkv=P[5], pos=P[11]), o) for o in [
        dict(dqkv=P[5] + 4 * 511), dict(dqkv=P[6] + 252), dict(dqkv=P[7]), dict(dqkv=P[1] + 252), dict(dqkv=P[11] + 4)]] +
    [("axb_kv_cache_extend", extend_call, dict(bqkv=P[6], gq=P[7], gk=P[8], pos=P[9], n_new=P[10]), o) for o in [
        dict(Q=P[6]), dict(K=P[7] + 252), dict(V=P[8]), dict(Q=P[1]), dict(K=P[9] + 4), dict(V=P[5]), dict(Q=P[10])]] +
    [("axb_kv_cache_attend_tree", attend_call, dict(mask=P[5], n_new=P[6]), o) for o in [
        dict(out=P[5] + 8), dict(out=P[3]), dict(out=P[6]), dict(out=P[5] + 24, per_seq=1, B=2)]] +
    [("axb_kv_cache_compact", compact_call, dict(), o) for o in [
        dict(K=P[2] + 28), dict(V=P[3] + 4), dict(K=P[4]), dict(lens_out=P[0] + 64), dict(lens_out=P[1] + 4 * (2 * 2 * 128 * 64 - 1))]])


@pytest.mark.parametrize("name,call,base,override", MEETS, ids=lambda v: v if isinstance(v, str) else None)
def test_outputs_that_meet_any_input_are_refused(eng, name, call, base, override):  # noqa: F811
    assert getattr(eng.lib, name)(*call(**{**base, **override})) == INVALID_SHAPE
    assert "overlap" in eng.last_error() or "lies in" in eng.last_error()


@pytest.mark.parametrize("name,call,base", sorted({(n, c, tuple(sorted(b.items()))) for n, c, b, _ in MEETS}, key=lambda v: v[0]), ids=lambda v: v if isinstance(v, str) else None)
def test_outputs_beside_their_inputs_are_not(eng, name, call, base):  # noqa: F811
    import torch
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    beside = {"axb_qkv_norm_rope": dict(Q=P[5] + 4 * 512, V=P[8] + 8), "axb_qkv_norm_rope_bwd": dict(dqkv=P[6] + 256),
              "axb_kv_cache_extend": dict(Q=P[7] + 256, K=P[9] + 8), "axb_kv_cache_attend_tree": dict(out=P[5] + 16),
              "axb_kv_cache_compact": dict(K=P[2] + 32, lens_out=P[1] + 4 * 2 * 2 * 128 * 64)}[name]
    assert getattr(eng.lib, name)(*call(**{**dict(base), **beside})) != INVALID_SHAPE
    assert "no CUDA device" in eng.last_error()


def test_a_scale_that_is_infinite_in_the_kernels_domain_is_refused(eng):  # noqa: F811
    """Scores are taken to base 2: scale / ln 2 has to be finite as well."""
    import torch
    for scale in (2.4e38, -3e38, float("inf"), float("nan")):
        assert eng.lib.axb_kv_cache_attend_tree(*attend_call(scale=scale)) == INVALID_SHAPE and "scale" in eng.last_error()
    if not torch.cuda.is_available():
        for scale in (2.3e38, -2.3e38, 1e-45, 0.0):
            assert eng.lib.axb_kv_cache_attend_tree(*attend_call(scale=scale)) != INVALID_SHAPE
