"""Rotary / ragged-batch KV-cache entry points without a GPU: frequencies, refusals of arguments, the float64 restatement."""
import ctypes as C

import pytest
import torch

import rope_kv_ref as ref


@pytest.fixture(scope="module")
def eng():
    from axiom_b200 import build
    from axiom_b200.engine import Engine
    build.build()
    return Engine()          # loads the library, touches no device


@pytest.mark.parametrize("rot", [0, 2, 48, 64, 128, 256])
@pytest.mark.parametrize("how", [dict(), dict(base=500000.0), dict(scaling="linear", factor=4.0),
                                 dict(scaling="turns", factor=8.0, low=1.0, high=4.0, original_len=8192),
                                 dict(scaling="index", factor=16.0, low=1.0, high=32.0, original_len=4096),
                                 dict(scaling="index", factor=2.0, low=0.5, high=10000.0, original_len=128)])
def test_frequencies(eng, rot, how):
    got, want = eng.rope_frequencies(rot, **how), ref.frequencies(rot, **how)
    assert len(got) == rot // 2
    for g, w in zip(got, want):
        assert abs(g - w) <= 1e-13 * abs(w)       # a few roundings of 64-bit pow, log and a blend


@pytest.mark.parametrize("how", [dict(rot=3), dict(rot=-2), dict(rot=8, base=0.0), dict(rot=8, base=float("inf")),
                                 dict(rot=8, scaling="linear", factor=0.0), dict(rot=8, scaling="turns", factor=2.0, low=4.0, high=4.0, original_len=10),
                                 dict(rot=8, scaling="index", factor=2.0, low=1.0, high=4.0, original_len=0),
                                 dict(rot=8, base=1.0, scaling="index", factor=2.0, low=1.0, high=4.0, original_len=100)])
def test_frequencies_refuse(eng, how):
    from axiom_b200.engine import EngineError
    with pytest.raises(EngineError) as e:
        eng.rope_frequencies(**how)
    assert e.value.status == 6


NULL_ARG, INVALID_SHAPE, NOT_IMPLEMENTED = 1, 6, 10
P = [0x10000000 * (i + 1) for i in range(14)]      # distinct addresses that nobody reads: every call below is refused


def rope_call(**o):
    a = dict(qkv=P[0], bqkv=None, gq=None, gk=None, eps=1e-6, freq=P[1], rot=64, pairing=0, amplitude=1.0, pos=None, B=1, S=2, H=4, Hkv=2,
             dk=64, Q=P[2], K=P[3], V=P[4])
    a.update(o)
    return list(a.values())


def extend_call(**o):
    a = dict(qkv=P[0], bqkv=None, gq=None, gk=None, eps=1e-6, freq=P[1], rot=64, pairing=0, amplitude=1.0, pos=None, lens=P[5], n_new=None, B=1,
             T=2, H=4, Hkv=2, max_seq=128, dk=64, Q=P[2], K=P[3], V=P[4])
    a.update(o)
    return list(a.values())


def bwd_call(**o):
    a = dict(qkv=P[0], bqkv=None, gq=P[6], gk=P[7], eps=1e-6, freq=P[1], rot=64, pairing=0, amplitude=1.0, pos=None, dQ=P[2], dK=P[3], dV=P[4],
             B=1, S=2, H=4, Hkv=2, dk=64, dqkv=P[8], dgq=P[9], dgk=P[10], ws=None)
    a.update(o)
    return list(a.values())


def attend_call(**o):
    a = dict(K=P[0], V=P[1], Q=P[2], mask=None, per_seq=0, lens=P[3], n_new=None, out=P[4], B=1, H=4, Hkv=2, T=2, max_seq=128, dk=64, scale=0.125,
             ws=None)
    a.update(o)
    return list(a.values())


def compact_call(**o):
    a = dict(K=P[0], V=P[1], keep=P[2], n_keep=P[3], lens=P[4], lens_out=P[5], B=2, Hkv=2, T=4, max_seq=128, dk=64)
    a.update(o)
    return list(a.values())


SHARED = [(dict(freq=None), NULL_ARG), (dict(rot=66), INVALID_SHAPE), (dict(rot=7), INVALID_SHAPE), (dict(rot=-2), INVALID_SHAPE),
          (dict(pairing=2), INVALID_SHAPE), (dict(eps=-1.0), INVALID_SHAPE), (dict(eps=float("nan")), INVALID_SHAPE), (dict(H=5), INVALID_SHAPE),
          (dict(H=0), INVALID_SHAPE), (dict(Hkv=0), INVALID_SHAPE), (dict(B=-1), INVALID_SHAPE), (dict(dk=0), INVALID_SHAPE),
          (dict(dk=260), NOT_IMPLEMENTED), (dict(H=65536, Hkv=1), INVALID_SHAPE), (dict(B=1 << 31), INVALID_SHAPE), (dict(B=1 << 20, S=1 << 20), INVALID_SHAPE),
          (dict(qkv=None), NULL_ARG)]
REFUSED = (
    [("axb_qkv_norm_rope", rope_call, o, st) for o, st in SHARED] +
    [("axb_qkv_norm_rope", rope_call, o, st) for o, st in [(dict(Q=None), NULL_ARG), (dict(V=None), NULL_ARG), (dict(S=-1), INVALID_SHAPE),
                                                           (dict(K=P[0] + 64), INVALID_SHAPE), (dict(V=P[3]), INVALID_SHAPE), (dict(K=P[2] + 256), INVALID_SHAPE)]] +
    [("axb_qkv_norm_rope_bwd", bwd_call, o, st) for o, st in SHARED] +
    [("axb_qkv_norm_rope_bwd", bwd_call, o, st) for o, st in [(dict(gq=None), NULL_ARG), (dict(gk=None), NULL_ARG), (dict(dqkv=None), NULL_ARG),
                                                              (dict(dqkv=P[0]), INVALID_SHAPE), (dict(dqkv=P[3]), INVALID_SHAPE)]] +
    [("axb_kv_cache_extend", extend_call, {("T" if k == "S" else k): v for k, v in o.items()}, st) for o, st in SHARED] +
    [("axb_kv_cache_extend", extend_call, o, st) for o, st in [(dict(lens=None), NULL_ARG), (dict(K=None), NULL_ARG), (dict(max_seq=0), INVALID_SHAPE),
                                                               (dict(max_seq=1 << 31), INVALID_SHAPE), (dict(V=P[0]), INVALID_SHAPE), (dict(V=P[3] + 512), INVALID_SHAPE),
                                                               (dict(Q=P[4]), INVALID_SHAPE)]] +
    [("axb_kv_cache_attend_tree", attend_call, o, st) for o, st in [
        (dict(K=None), NULL_ARG), (dict(V=None), NULL_ARG), (dict(Q=None), NULL_ARG), (dict(lens=None), NULL_ARG), (dict(out=None), NULL_ARG),
        (dict(B=-1), INVALID_SHAPE), (dict(T=-1), INVALID_SHAPE), (dict(H=5), INVALID_SHAPE), (dict(Hkv=0), INVALID_SHAPE), (dict(dk=0), INVALID_SHAPE),
        (dict(dk=129), NOT_IMPLEMENTED), (dict(max_seq=0), INVALID_SHAPE), (dict(max_seq=1 << 31), INVALID_SHAPE), (dict(scale=float("inf")), INVALID_SHAPE),
        (dict(T=1 << 30), INVALID_SHAPE), (dict(max_seq=(1 << 30) + 1), INVALID_SHAPE), (dict(max_seq=1 << 30, B=64), INVALID_SHAPE),
        (dict(B=1 << 30), INVALID_SHAPE), (dict(out=P[2]), INVALID_SHAPE), (dict(out=P[0]), INVALID_SHAPE)]] +
    [("axb_kv_cache_compact", compact_call, o, st) for o, st in [
        (dict(K=None), NULL_ARG), (dict(keep=None), NULL_ARG), (dict(n_keep=None), NULL_ARG), (dict(lens=None), NULL_ARG), (dict(Hkv=0), INVALID_SHAPE),
        (dict(T=-1), INVALID_SHAPE), (dict(max_seq=0), INVALID_SHAPE), (dict(dk=0), INVALID_SHAPE), (dict(lens_out=P[4]), INVALID_SHAPE),
        (dict(lens_out=P[4] + 4), INVALID_SHAPE), (dict(lens_out=P[3]), INVALID_SHAPE), (dict(lens_out=P[2] + 8), INVALID_SHAPE), (dict(V=P[0]), INVALID_SHAPE)]])


@pytest.mark.parametrize("name,call,override,status", REFUSED, ids=lambda v: v if isinstance(v, str) else None)
def test_refusals(eng, name, call, override, status):
    """Refused before anything is launched or read, with a message."""
    assert getattr(eng.lib, name)(*call(**override)) == status
    assert name[4:] in eng.last_error()


def test_binding_refuses_wrong_tensors(eng):
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    lens = z(2, dtype=torch.int32)
    q, k = z(8, 3, 16), z(4, 32, 16)
    ok = dict(K_cache=k, V_cache=k.clone(), Q=q, out=z(8, 3, 16), lens=lens, scale=1.0)
    for bad in (dict(lens=lens.long()), dict(Q=q.transpose(0, 1).contiguous().transpose(0, 1)), dict(out=z(8, 2, 16)), dict(mask=z(2, 3, 2, dtype=torch.int64)),
                dict(mask=z(2, 3, 1, dtype=torch.int32)), dict(n_new=z(3, dtype=torch.int32)), dict(V_cache=z(4, 31, 16)), dict(Q=q.double())):
        with pytest.raises(ValueError):
            eng.kv_cache_attend_tree(**{**ok, **bad})
    with pytest.raises(ValueError):
        eng.qkv_norm_rope(z(6, 100), z(8, 3, 16), z(4, 3, 16), z(4, 3, 16), 2)
    with pytest.raises(ValueError):
        eng.kv_cache_compact(k, k.clone(), z(2, 5, dtype=torch.int64), lens, lens)


def test_binding_refuses_host_tensors(eng):
    k = torch.zeros(4, 32, 16)
    with pytest.raises(ValueError, match="engine's device"):
        eng.kv_cache_attend_tree(k, k.clone(), torch.zeros(8, 3, 16), torch.zeros(8, 3, 16), torch.zeros(2, dtype=torch.int32), 1.0)


def test_restated_gradient_against_differences():
    """The float64 restatement's gradient (autograd) agrees with central differences."""
    torch.manual_seed(3)
    B, T, H, Hkv, dk, rot = 1, 3, 2, 1, 6, 4
    x = torch.randn(B * T, (H + 2 * Hkv) * dk, dtype=torch.float64)
    gq, gk = torch.rand(dk, dtype=torch.float64) + 0.5, torch.rand(dk, dtype=torch.float64) + 0.5
    freq = torch.tensor(ref.frequencies(rot), dtype=torch.float64)
    weights = [torch.randn(B, h, T, dk, dtype=torch.float64) for h in (H, Hkv, Hkv)]

    def value(x, gq, gk, pairing):
        return sum((y * w).sum() for y, w in zip(ref.qkv_norm_rope(x, B, H, Hkv, dk, None, gq, gk, 1e-5, freq, pairing, 1.3), weights))

    for pairing in ("half", "interleaved"):
        leaves = [t.clone().requires_grad_() for t in (x, gq, gk)]
        grads = torch.autograd.grad(value(*leaves, pairing), leaves)
        for which, (t, grad) in enumerate(zip((x, gq, gk), grads)):
            for i in range(0, t.numel(), 5):
                step = torch.zeros_like(t).view(-1)
                step[i] = 1e-6
                args = [x, gq, gk]
                up, down = list(args), list(args)
                up[which], down[which] = t + step.view_as(t), t - step.view_as(t)
                diff = (value(*up, pairing) - value(*down, pairing)) / 2e-6
                assert abs(float(diff - grad.view(-1)[i])) < 1e-7 * (1 + abs(float(diff)))
