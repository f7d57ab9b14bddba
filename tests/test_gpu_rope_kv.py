"""Rotary positions, per-head norms and the ragged-batch KV cache on the GPU, through the C ABI, against float64.

Tolerances are bounds, stated beside their use (u = 2^-24, half a step of fp32)."""
import math

import numpy as np
import pytest
import torch

import rope_kv_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def ints(v):
    return torch.as_tensor(v, dtype=torch.int32).cuda()


def unaligned(t):
    """The same values at an address that is not a multiple of 16 bytes."""
    base = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)
    out = base[1:].view(t.shape)
    out.copy_(t)
    return out


# --------------------------------------------------------------------------------------------- rope, forward and backward

# B, S, H, Hkv, dk, rot, pairing, normed (q, k), bias, positions
ROPE = [
    (1, 1, 1, 1, 64, 64, "half", (1, 1), True, "none"),
    (2, 37, 4, 2, 64, 64, "half", (0, 0), False, "none"),
    (2, 37, 4, 2, 64, 64, "interleaved", (1, 1), True, "far"),
    (1, 130, 8, 4, 128, 128, "half", (1, 0), False, "far"),
    (3, 19, 6, 1, 80, 32, "interleaved", (0, 1), True, "none"),
    (1, 7, 5, 5, 96, 48, "half", (1, 1), False, "negative"),
    (2, 11, 3, 3, 50, 50, "half", (1, 1), True, "far"),
    (2, 11, 6, 2, 50, 24, "interleaved", (1, 1), False, "none"),
    (1, 9, 2, 1, 33, 32, "interleaved", (1, 1), True, "none"),
    (1, 9, 2, 1, 33, 2, "half", (0, 0), True, "none"),
    (1, 3, 2, 2, 256, 256, "half", (1, 1), False, "none"),
    (1, 3, 2, 2, 256, 64, "interleaved", (1, 1), False, "none"),
    (1, 5, 3, 3, 252, 8, "half", (1, 1), False, "none"),
    (1, 4, 2, 1, 255, 254, "interleaved", (1, 1), True, "none"),
    (1, 4, 2, 1, 1, 0, "half", (1, 1), True, "none"),
    (1, 4, 2, 1, 4, 4, "interleaved", (0, 0), False, "none"),
    (1, 4, 2, 1, 2, 2, "half", (0, 0), False, "none"),
    (1, 300, 40, 8, 72, 72, "half", (1, 1), False, "none"),
    (5, 1000, 8, 4, 64, 64, "half", (1, 1), False, "none"),
]


def rope_inputs(case, seed, shift):
    B, S, H, Hkv, dk, rot, pairing, normed, bias, where = case
    g = gen(seed)
    width = (H + 2 * Hkv) * dk
    s = dict(qkv=randn(g, B * S, width) * torch.exp(randn(g, width)), bias=randn(g, width) if bias else None,
             gq=1 + 0.3 * randn(g, dk) if normed[0] else None, gk=1 + 0.3 * randn(g, dk) if normed[1] else None, eps=1e-5, pairing=pairing,
             amplitude=1.25, freq=torch.tensor(ref.frequencies(rot), dtype=torch.float64).cuda() if rot else None, pos=None)
    if where != "none":
        lo, hi = (0, 1 << 20) if where == "far" else (-5000, 0)
        s["pos"] = torch.randint(lo, hi, (B, S), device="cuda", generator=g, dtype=torch.int32)
    if shift:
        for k in ("qkv", "bias", "gq", "gk"):
            s[k] = None if s[k] is None else unaligned(s[k])
    return s


def reference_of(s, case):
    B, S, H, Hkv, dk = case[:5]
    return ref.qkv_norm_rope(s["qkv"], B, H, Hkv, dk, s["bias"], s["gq"], s["gk"], s["eps"], s["freq"], s["pairing"], s["amplitude"], s["pos"])


def row_error(got, want, floor):
    """Largest error of a head row relative to the row's largest value (or floor, where that is larger)."""
    scale = torch.maximum(want.abs().amax(-1, keepdim=True), floor)
    return float(((got.double() - want).abs() / scale.clamp_min(1e-300)).max())


@pytest.mark.parametrize("shift", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c[:7])))
def test_qkv_norm_rope(engine, case, shift):
    B, S, H, Hkv, dk = case[:5]
    s = rope_inputs(case, 11, shift)
    out = [torch.full((B * h, S, dk), float("nan"), device="cuda") for h in (H, Hkv, Hkv)]
    if shift:
        out = [unaligned(o) for o in out]
    engine.qkv_norm_rope(s["qkv"], *out, B, **{k: v for k, v in s.items() if k != "qkv"})
    # Of a value, with the pair's larger element as the scale: bias 1 rounding (of the sum), the norm's factor
    # (sum of squares: at most 8 sequential and 5 tree additions, halved by the root: 8; rsqrt 2 ulp = 4; mean, eps: 2) and
    # its 2 products, cosine and sine to 2 ulp of 1 and the amplitude (5 together, for each of the pair's two terms), the
    # angle's own rounding to fp32 turns (2 pi half a step of 1/2: 4, on each term), 3 roundings of the rotation, twice the
    # pair's size at most: below 60 u.  The bias can cancel: the scale is then the larger summand.
    raw = s["qkv"].double().view(B, S, H + 2 * Hkv, dk).transpose(1, 2)
    if s["bias"] is not None:
        raw = raw.abs() + s["bias"].double().abs().view(H + 2 * Hkv, 1, dk)
    summed = reference_of({**s, "freq": None, "gq": None, "gk": None}, case)
    for i, (got, want) in enumerate(zip(out, reference_of(s, case))):
        lo, hi = (0, H, H + Hkv)[i], (H, H + Hkv, H + 2 * Hkv)[i]
        # what cancelled in the bias sum, carried through norm and amplitude
        cancel = raw[:, lo:hi].abs().amax(-1, keepdim=True) / summed[i].abs().amax(-1, keepdim=True).clamp_min(1e-300)
        floor = want.abs().amax(-1, keepdim=True) * cancel.clamp_min(1.0)
        assert row_error(got.view(B, -1, S, dk), want, floor) < 60 * U


def test_plain_pass_is_the_layout_pass(engine):
    """Without norm and rotation: bit for bit what head_interleave_qkv_split gives."""
    B, S, H, dk = 2, 33, 5, 48
    g = gen(1)
    qkv, bias = randn(g, B * S, 3 * H * dk), randn(g, 3 * H * dk)
    a, b = ([torch.empty(B * H, S, dk, device="cuda") for _ in range(3)] for _ in range(2))
    engine.qkv_norm_rope(qkv, *a, B, bias=bias)
    engine.head_interleave_qkv_split(qkv, bias, *b, B, S, H, dk)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_tokens_nan_stays_with_it(engine):
    B, S, H, Hkv, dk = 1, 20, 4, 2, 64
    g = gen(2)
    qkv = randn(g, S, (H + 2 * Hkv) * dk)
    freq = torch.tensor(ref.frequencies(dk), dtype=torch.float64).cuda()
    gq = torch.ones(dk, device="cuda")
    clean = [torch.empty(h, S, dk, device="cuda") for h in (H, Hkv, Hkv)]
    dirty = [torch.empty_like(x) for x in clean]
    engine.qkv_norm_rope(qkv, *clean, B, gq=gq, gk=gq, freq=freq)
    qkv[7, 3 * dk + 5] = float("nan")            # head 3 of token 7
    engine.qkv_norm_rope(qkv, *dirty, B, gq=gq, gk=gq, freq=freq)
    assert bool(torch.isnan(dirty[0][3, 7]).all())
    dirty[0][3, 7] = clean[0][3, 7]
    assert all(torch.equal(x, y) for x, y in zip(clean, dirty))


@pytest.mark.parametrize("shift", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c[:7])))
def test_qkv_norm_rope_bwd(engine, case, shift):
    B, S, H, Hkv, dk = case[:5]
    s = rope_inputs(case, 21, shift)
    g = gen(5)
    grads = [randn(g, B * h, S, dk) for h in (H, Hkv, Hkv)]
    start = [randn(g, dk) if s[k] is not None else None for k in ("gq", "gk")]
    dqkv = torch.full_like(s["qkv"], float("nan"))
    if shift:
        grads, dqkv = [unaligned(x) for x in grads], unaligned(dqkv)
    how = {k: v for k, v in s.items()}
    got_g = [None if x is None else x.clone() for x in start]
    engine.qkv_norm_rope_bwd(*grads, dqkv, B, dgq=got_g[0], dgk=got_g[1], **how)

    leaves = [s["qkv"].double().requires_grad_()] + [s[k].double().requires_grad_() if s[k] is not None else None for k in ("gq", "gk")]
    y = reference_of({**s, "qkv": leaves[0], "gq": leaves[1], "gk": leaves[2]}, case)
    used = [x for x in leaves if x is not None]
    want = iter(torch.autograd.grad(y, used, [d.double().view(v.shape) for d, v in zip(grads, y)], allow_unused=True))
    dx = next(want)
    # Scale of a head row's gradient: the largest |d g r| before the mean's part is taken off (that part is at most as large in
    # the 2-norm, so the difference can cancel).  Errors of d: 20 u (rotation, angles); of r: 14 u; of the two sums: 13 additions,
    # 3 products each; x itself one rounding of the bias sum, whose cancellation grows it: below 100 u of that scale times the
    # bias sum's cancellation.
    x = s["qkv"].double()
    xb = x if s["bias"] is None else x + s["bias"].double()
    big = (x.abs() if s["bias"] is None else x.abs() + s["bias"].double().abs()).view(B * S, -1, dk)
    cancel = (big.amax(-1, keepdim=True) / xb.view(B * S, -1, dk).abs().amax(-1, keepdim=True).clamp_min(1e-300)).clamp_min(1.0)
    rms = torch.sqrt((xb.view(B * S, -1, dk) ** 2).mean(-1, keepdim=True) + s["eps"])
    flat = torch.cat([d.view(B, -1, S, dk).transpose(1, 2).reshape(B * S, -1, dk) for d in grads], 1).double()
    scale = flat.abs().amax(-1, keepdim=True) * 2 * s["amplitude"]
    for k, lo, hi in (("gq", 0, H), ("gk", H, H + Hkv)):
        if s[k] is not None:
            scale[:, lo:hi] = scale[:, lo:hi] * s[k].double().abs().max() / rms[:, lo:hi] * math.sqrt(dk)
    err = (dqkv.double() - dx).abs().view(B * S, -1, dk) / scale / cancel
    assert float(err.max()) < 100 * U
    for k, held, got, d, lo, hi in (("gq", start[0], got_g[0], grads[0], 0, H), ("gk", start[1], got_g[1], grads[1], H, H + Hkv)):
        if held is None:
            continue
        add = next(want)
        # every term to 60 u of sqrt(dk) * 2 * amplitude * max |d| (|u| <= sqrt(dk)); at most 64 fp32 additions in a lane and 32 over
        # groups before the sums go on in 64 bits; one rounding of the result
        terms = float(d.double().abs().amax(-1).sum()) * 2 * s["amplitude"] * math.sqrt(dk) * float(cancel[:, lo:hi].max())
        assert float((got.double() - (held.double() + add)).abs().max()) < 160 * U * terms + U * float((held.double() + add).abs().max())


def test_norm_gradients_are_optional_and_repeatable(engine):
    case = (2, 500, 8, 4, 64, 64, "half", (1, 1), False, "none")
    B, S, H, Hkv, dk = case[:5]
    s = rope_inputs(case, 3, False)
    g = gen(4)
    grads = [randn(g, B * h, S, dk) for h in (H, Hkv, Hkv)]
    seen = []
    ws = torch.zeros(engine.attention_workspace_bytes(), dtype=torch.uint8, device="cuda")
    for dgq, dgk, w in ((1, 1, None), (1, 1, ws), (1, 0, None), (0, 1, None), (0, 0, None)):
        d = [torch.zeros(dk, device="cuda") if x else None for x in (dgq, dgk)]
        dqkv = torch.empty_like(s["qkv"])
        engine.qkv_norm_rope_bwd(*grads, dqkv, B, dgq=d[0], dgk=d[1], workspace=w, **s)
        seen.append((dqkv, *d))
    for dqkv, dgq, dgk in seen[1:]:
        assert torch.equal(dqkv, seen[0][0])
        assert dgq is None or torch.equal(dgq, seen[0][1])
        assert dgk is None or torch.equal(dgk, seen[0][2])


def test_rotation_only_backward_needs_no_activations(engine):
    B, S, H, dk = 1, 21, 3, 32
    g = gen(6)
    freq = torch.tensor(ref.frequencies(dk), dtype=torch.float64).cuda()
    grads = [randn(g, B * H, S, dk) for _ in range(3)]
    a, b = (torch.empty(B * S, 3 * H * dk, device="cuda") for _ in range(2))
    engine.qkv_norm_rope_bwd(*grads, a, B, freq=freq)
    engine.qkv_norm_rope_bwd(*grads, b, B, qkv=randn(g, B * S, 3 * H * dk), freq=freq)
    assert torch.equal(a, b)
    # the transposed rotation undoes the rotation: 20 u for each way
    back = [torch.empty_like(x) for x in grads]
    engine.qkv_norm_rope(a, *back, B, freq=freq)
    for x, y in zip(grads, back):
        assert float((x - y).abs().max()) < 40 * U * 2 * float(x.abs().max())


# ------------------------------------------------------------------------------------------------------------ extend

EXTEND = [
    (1, 1, 4, 2, 64, 64, "half", 16, False),
    (3, 5, 6, 2, 80, 32, "interleaved", 40, True),
    (4, 16, 8, 1, 128, 128, "half", 64, True),
    (2, 3, 2, 2, 50, 50, "interleaved", 9, True),
    (33, 2, 4, 4, 32, 32, "half", 17, True),
]


@pytest.mark.parametrize("tree_pos", [False, True])
@pytest.mark.parametrize("case", EXTEND, ids=lambda c: "-".join(map(str, c)))
def test_kv_cache_extend(engine, case, tree_pos):
    """Written rows match the head-major form of the same pass bit for bit; every other row keeps its bits."""
    B, T, H, Hkv, dk, rot, pairing, max_seq, ragged = case
    s = rope_inputs((B, T, H, Hkv, dk, rot, pairing, (1, 1), True, "none"), 31, False)
    rng = np.random.RandomState(B + T)
    n = rng.randint(0, T + 1, B) if ragged else np.full(B, T)
    lens = np.array([rng.randint(0, max_seq - k + 1) for k in n])
    lens[0], n[0] = max_seq - T, T                      # up to the last row
    pos = torch.as_tensor(lens[:, None] + (rng.randint(0, T, (B, T)) if tree_pos else np.arange(T)), dtype=torch.int32).cuda()
    g = gen(7)
    K, V = (randn(g, B * Hkv, max_seq, dk) for _ in range(2))
    K0, V0, Q0 = K.clone(), V.clone(), randn(g, B * H, T, dk)
    Q = Q0.clone()
    how = {k: v for k, v in s.items() if k not in ("qkv", "pos")}
    engine.kv_cache_extend(s["qkv"], Q, K, V, ints(lens), n_new=ints(n) if ragged else None, pos=pos if tree_pos else None, **how)
    want = [torch.empty(B * h, T, dk, device="cuda") for h in (H, Hkv, Hkv)]
    engine.qkv_norm_rope(s["qkv"], *want, B, pos=pos, **how)
    for b in range(B):
        Q0.view(B, H, T, dk)[b, :, :n[b]] = want[0].view(B, H, T, dk)[b, :, :n[b]]
        for held, new in ((K0, want[1]), (V0, want[2])):
            held.view(B, Hkv, max_seq, dk)[b, :, lens[b]:lens[b] + n[b]] = new.view(B, Hkv, T, dk)[b, :, :n[b]]
    assert torch.equal(Q, Q0) and torch.equal(K, K0) and torch.equal(V, V0)


def test_lengths_that_do_not_fit_are_refused_on_the_device(engine):
    """Sequences whose rows leave the cache are left alone, the others are served, and the error word says so."""
    B, T, H, Hkv, dk, max_seq = 6, 4, 2, 2, 32, 20
    g = gen(8)
    qkv = randn(g, B * T, (H + 2 * Hkv) * dk)
    lens, n = ints([3, -1, 17, 5, 16, 2 ** 31 - 1]), ints([4, 4, 4, 5, 4, 4])      # good, negative, too long, more than T, good, huge
    good = [0, 4]
    K, V = (randn(g, B * Hkv, max_seq, dk) for _ in range(2))
    Q = randn(g, B * H, T, dk)
    before = [x.clone() for x in (Q, K, V)]
    assert engine.device_error() == 0
    engine.kv_cache_extend(qkv, Q, K, V, lens, n_new=n)
    assert engine.device_error() == 101 and "do not fit" in engine.last_error() and engine.device_error() == 0
    for x, y in zip((Q, K, V), before):
        same = (x == y).view(B, -1).all(1).tolist()
        assert [b for b in range(B) if not same[b]] == good
    out = torch.full((B * H, T, dk), 5.0, device="cuda")
    engine.kv_cache_attend_tree(K, V, Q, out, lens, 0.2, n_new=n)
    assert engine.device_error() == 101
    want, smag, vmag = ref.attend_tree(K, V, Q, out * 0 + 5, ints([3, 0, 0, 0, 16, 0]), 0.2, n_new=ints([4, 0, 0, 0, 4, 0]))
    assert float((out.double() - want).abs().max()) < ref.attend_bound(smag, vmag, dk)


# ------------------------------------------------------------------------------------------------------------ attend

def tree_masks(rng, B, T):
    """Ancestor bits of random trees, int64 [B, T, words]."""
    words = (T + 63) // 64
    m = np.zeros((B, T, words), np.uint64)
    for b in range(B):
        for t in range(T):
            p = rng.randint(-1, t) if t else -1
            if p >= 0:
                m[b, t] = m[b, p]
            m[b, t, t // 64] |= np.uint64(1 << (t % 64))
    return torch.from_numpy(m.view(np.int64)).cuda()


# B, T, H, Hkv, dk, lens, ragged n_new, mask
ATTEND = [
    (1, 1, 1, 1, 64, [0], False, None),
    (1, 1, 4, 4, 64, [1], False, None),
    (3, 1, 8, 2, 128, [63, 64, 700], False, None),
    (4, 1, 8, 1, 32, [0, 62, 127, 128], False, None),
    (2, 4, 4, 4, 96, [60, 61], False, None),
    (2, 4, 4, 4, 96, [60, 61], False, "tree"),
    (5, 16, 2, 2, 128, [0, 5, 48, 300, 1111], True, "tree"),
    (3, 8, 8, 2, 64, [0, 130, 511], True, "tree"),
    (2, 7, 10, 2, 80, [64, 250], True, "shared"),
    (2, 16, 8, 2, 128, [99, 1500], False, "tree"),
    (2, 64, 6, 2, 64, [1, 321], True, "tree"),
    (1, 65, 3, 1, 72, [70], False, "tree"),
    (2, 130, 2, 1, 40, [10, 0], True, "tree"),
    (1, 100, 2, 2, 112, [37], False, None),
    (2, 5, 3, 3, 50, [9, 77], True, "tree"),
    (1, 3, 2, 1, 33, [65], False, "tree"),
    (1, 2, 1, 1, 1, [4], False, None),
    (1, 9, 2, 2, 6, [100], False, "tree"),
    (40, 2, 2, 1, 64, list(range(0, 400, 10)), True, "tree"),
    (1, 4, 2, 1, 128, [40000], False, "tree"),
    (7, 3, 16, 8, 64, [5000, 0, 1, 2, 3, 64, 4000], True, None),
    # more rows to a key head than the warp-level kernel takes: up to 64 of them ...
    (2, 6, 8, 2, 128, [700, 64], True, "tree"),
    (3, 8, 8, 2, 96, [0, 130, 4097], True, "tree"),
    (2, 5, 12, 3, 72, [63, 1], False, "shared"),
    (1, 17, 1, 1, 128, [47], False, "tree"),             # the new tokens end with a block
    (2, 16, 8, 2, 64, [900, 127], True, "tree"),
    (4, 9, 14, 2, 36, [0, 2000, 119, 5], True, "tree"),
    (70, 3, 16, 2, 128, list(range(0, 700, 10)), True, "tree"),
    (1, 16, 4, 1, 100, [20000], False, "tree"),          # one item over every CTA
    # ... and more
    (2, 1, 64, 1, 64, [300, 1000], False, None),
    (2, 3, 12, 1, 32, [0, 129], True, "tree"),
    (3, 33, 2, 2, 128, [63, 64, 0], True, "tree"),
    (1, 40, 2, 1, 64, [30000], False, "tree"),           # one item over every CTA
    (1, 40, 1, 1, 128, [12000], False, "shared"),
    (1, 300, 2, 1, 96, [200], False, None),
    (1, 200, 6, 2, 64, [0], False, None),
    (5, 17, 8, 4, 100, [1, 500, 0, 77, 128], True, "tree"),
    (3, 64, 4, 2, 128, [4000, 10, 900], True, "shared"),
    (1, 513, 1, 1, 64, [100], False, None),
]


def attend_case(case, seed, extra=3):
    B, T, H, Hkv, dk, lens, ragged, kind = case
    rng = np.random.RandomState(seed)
    g = gen(seed)
    max_seq = max(lens) + T + extra
    n = rng.randint(0, T + 1, B) if ragged else np.full(B, T)
    if ragged:
        n[0] = T
    mask = tree_masks(rng, B, T) if kind == "tree" else tree_masks(rng, 1, T)[0].contiguous() if kind == "shared" else None
    return dict(K=randn(g, B * Hkv, max_seq, dk), V=randn(g, B * Hkv, max_seq, dk), Q=randn(g, B * H, T, dk), out=randn(g, B * H, T, dk),
                lens=ints(lens), n_new=ints(n) if ragged else None, mask=mask, scale=1.0 / math.sqrt(dk))


def run_attend(engine, s, **more):
    out = s["out"].clone() if not more.pop("shift", False) else unaligned(s["out"])
    engine.kv_cache_attend_tree(s["K"], s["V"], s["Q"], out, s["lens"], s["scale"], n_new=s["n_new"], mask=s["mask"], **more)
    return out


def check_attend(s, got, magnitudes=None):
    want, smag, vmag = ref.attend_tree(s["K"], s["V"], s["Q"], s["out"], s["lens"], s["scale"], s["n_new"], s["mask"])
    err, bound = float((got.double() - want).abs().max()), ref.attend_bound(smag, vmag, s["Q"].shape[-1])
    assert err <= bound
    B, T = s["lens"].numel(), s["Q"].shape[1]
    if s["n_new"] is not None:         # rows behind the last token keep their bits
        behind = (torch.arange(T, device="cuda")[None, :] >= s["n_new"][:, None])[:, None, :, None].expand(B, s["Q"].shape[0] // B, T, s["Q"].shape[2])
        assert torch.equal(got.view(behind.shape)[behind], s["out"].view(behind.shape)[behind])


@pytest.mark.parametrize("shift", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[:5])) + f"-{c[7]}-{max(c[5])}")
def test_attend_tree(engine, case, shift):
    s = attend_case(case, 41)
    if shift:
        s["K"] = unaligned(s["K"])
    got = run_attend(engine, s, shift=shift)
    check_attend(s, got)
    assert torch.equal(got, run_attend(engine, s, shift=shift))      # bitwise repeatable


def test_attend_tree_is_kv_cache_attend_for_one_token(engine):
    """T = 1, equal lengths, no sharing: the single-token entry point's result (both to fp32 accuracy)."""
    g = gen(9)
    BH, max_seq, dk, L = 6, 300, 64, 257
    K, V, q = randn(g, BH, max_seq, dk), randn(g, BH, max_seq, dk), randn(g, BH, dk)
    a, b = torch.empty(BH, dk, device="cuda"), torch.empty(BH, 1, dk, device="cuda")
    engine.kv_cache_attend(K, V, q, a, L, 0.125)
    engine.kv_cache_attend_tree(K, V, q.view(BH, 1, dk), b, ints([L - 1]), 0.125)
    want, smag, vmag = ref.attend_tree(K, V, q.view(BH, 1, dk), b, ints([L - 1]), 0.125)
    assert float((a - b.view(BH, dk)).abs().max()) < 2 * ref.attend_bound(smag, vmag, dk)


@pytest.mark.parametrize("lens", [[0, 0], [0, 70]])
def test_rows_that_see_nothing_are_zero(engine, lens):
    B, T, H, Hkv, dk = 2, 5, 2, 1, 64
    s = attend_case((B, T, H, Hkv, dk, lens, False, "tree"), 51)
    s["mask"][:, 2] = 0
    s["mask"][:, 4] = 1 << 40          # a bit behind the last token counts for nothing
    got = run_attend(engine, s)
    check_attend(s, got)
    if lens[0] == 0:
        assert bool((got.view(B, H, T, dk)[0, :, 2] == 0).all() and (got.view(B, H, T, dk)[0, :, 4] == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).max])
@pytest.mark.parametrize("case", [(2, 6, 4, 2, 64, [59, 130], False, "tree"), (2, 40, 4, 2, 128, [59, 130], True, "tree"), (1, 20, 2, 1, 50, [3], False, "tree"),
                                  (2, 40, 4, 2, 64, [59, 130], True, "tree"), (1, 140, 2, 2, 96, [200], False, "tree")],
                         ids=["few", "many", "scalar", "many64", "blocks"])
def test_values_in_unseen_rows_reach_nobody(engine, case, bad):
    """Anything in cache rows behind the last token and in new rows that a token does not see leaves its result alone, bit for
    bit; a token that does see such a row becomes non-finite (or huge) in the columns concerned."""
    B, T, H, Hkv, dk, lens, ragged, _ = case
    s = attend_case(case, 61, extra=70)
    seen_by = lambda b, j: ((s["mask"][b, :, j // 64] >> (j % 64)) & 1).bool()  # noqa: E731
    clean = run_attend(engine, s)
    n = s["n_new"].tolist() if ragged else [T] * B
    Kc, Vc = (s[x].view(B, Hkv, -1, dk) for x in "KV")
    poisoned = []
    for b in range(B):
        Kc[b, :, lens[b] + n[b]:] = bad
        Vc[b, :, lens[b] + n[b]:] = bad
        j = n[b] - 2
        if j >= 1:
            Kc[b, :, lens[b] + j, 3] = bad
            Vc[b, :, lens[b] + j, 7] = bad
            poisoned.append((b, j))
    got = run_attend(engine, s)
    same = (got == clean).view(B, H, T, dk)
    for b in range(B):
        mine = [j for bb, j in poisoned if bb == b]
        for t in range(T):
            sees = t < n[b] and any(bool(seen_by(b, j)[t]) for j in mine)
            assert sees or bool(same[b, :, t].all()), (b, t)
    # the same values in V alone: a finite score row, a non-finite value
    if not math.isfinite(bad):
        s2 = attend_case(case, 61, extra=70)
        for b, j in poisoned:
            s2["V"].view(B, Hkv, -1, dk)[b, :, lens[b] + j, 7] = bad
        got = run_attend(engine, s2).view(B, H, T, dk)
        for b, j in poisoned:
            for t in range(n[b]):
                hit = bool(seen_by(b, j)[t])
                assert bool(torch.isfinite(got[b, :, t, 7]).all()) != hit
                rest = torch.cat((got[b, :, t, :7], got[b, :, t, 8:]), -1)
                assert torch.equal(rest, torch.cat((clean.view(B, H, T, dk)[b, :, t, :7], clean.view(B, H, T, dk)[b, :, t, 8:]), -1))


@pytest.mark.parametrize("case", [(2, 3, 4, 2, 64, [100, 333], True, "tree"), (2, 12, 8, 2, 128, [100, 333], True, "tree"),
                                  (2, 12, 8, 2, 64, [300, 20], True, "tree"), (1, 140, 2, 1, 64, [200], False, "tree"),
                                  (1, 140, 1, 1, 96, [64], False, None)], ids=lambda c: "-".join(map(str, c[:5])))
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0])
def test_scales(engine, case, scale):
    """A negative scale turns the order of the scores round, zero gives the mean of the rows seen."""
    s = attend_case(case, 73)
    s["scale"] = scale
    check_attend(s, run_attend(engine, s))


def test_many_short_sequences(engine):
    """More sequences than CTAs, than threads of a CTA: the work line is found in steps of 32 sequences."""
    rng = np.random.RandomState(5)
    for T, H, dk in ((1, 2, 32), (5, 8, 68)):
        B, g = 1300, gen(75)
        lens, n = rng.randint(0, 50, B), rng.randint(0, T + 1, B)
        s = dict(K=randn(g, B, 60, dk), V=randn(g, B, 60, dk), Q=randn(g, B * H, T, dk), out=randn(g, B * H, T, dk), lens=ints(lens), n_new=ints(n),
                 mask=None, scale=0.2)
        check_attend(s, run_attend(engine, s))


@pytest.mark.parametrize("case", [(4, 2, 8, 2, 128, [3000, 5, 700, 64], True, "tree"), (3, 4, 16, 4, 128, [2000, 900, 0], True, "tree"),
                                  (3, 16, 16, 4, 128, [4000, 300, 64], True, "tree"), (3, 16, 16, 4, 64, [4000, 300, 64], True, "tree"),
                                  (2, 64, 12, 4, 64, [2500, 1000], True, "tree"), (2, 40, 8, 2, 112, [1500, 100], True, "tree")],
                         ids=lambda c: "-".join(map(str, c[:5])))
def test_the_same_call_many_times(engine, case):
    """Loads, products and partial results land in a different order every time; the result has the same bits."""
    s = attend_case(case, 77)
    first = run_attend(engine, s)
    out = s["out"].clone()
    for _ in range(150):
        engine.kv_cache_attend_tree(s["K"], s["V"], s["Q"], out, s["lens"], s["scale"], n_new=s["n_new"], mask=s["mask"])
        assert torch.equal(out, first)
    assert engine.device_error() == 0


def test_large_scores(engine):
    """Scores of several thousand (a soft-max that is one key) stay finite and exact."""
    s = attend_case((2, 4, 4, 2, 64, [100, 333], False, "tree"), 71)
    s["Q"] *= 100
    s["scale"] = -1.0                      # a negative scale is a scale like any other
    got = run_attend(engine, s)
    want, smag, _ = ref.attend_tree(s["K"], s["V"], s["Q"], s["out"], s["lens"], s["scale"], None, s["mask"])
    assert bool(torch.isfinite(got).all())
    # rows whose two best scores are further apart than the scores' error bound and 20 give one key's value
    err = smag * (3 * 2.0 ** -20 + 24 * 2.0 ** -23)
    close = (got.double() - want).abs().amax(-1) < 1e-5 * 5 + 2 * math.expm1(min(2 * err, 1.0)) * 5
    assert bool(close.all())


def test_binding_refuses_wrong_types_and_strides(engine):
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    lens, keep = z(2, dtype=torch.int32), z(2, 5, dtype=torch.int32)
    ok = dict(K_cache=z(4, 32, 16), V_cache=z(4, 32, 16), Q=z(8, 3, 16), out=z(8, 3, 16), lens=lens, scale=1.0)
    for bad, what in ((dict(lens=lens.long()), "int32"), (dict(Q=z(3, 8, 16).transpose(0, 1)), "contiguous"), (dict(Q=z(8, 3, 16).double()), "float32"),
                      (dict(mask=z(2, 3, 1, dtype=torch.int32)), "int64"), (dict(mask=z(3, 2, dtype=torch.int64)), "mask"),
                      (dict(out=z(8, 2, 16)), "out"), (dict(V_cache=z(4, 31, 16)), "head-major"), (dict(n_new=z(3, dtype=torch.int32)), "n_new"),
                      (dict(workspace=z(64)), "workspace")):
        with pytest.raises(ValueError, match=what):
            engine.kv_cache_attend_tree(**{**ok, **bad})
    with pytest.raises(ValueError, match="float64"):
        engine.qkv_norm_rope(z(6, 128), z(8, 3, 16), z(4, 3, 16), z(4, 3, 16), 2, freq=z(8))
    with pytest.raises(ValueError, match="int32"):
        engine.kv_cache_compact(ok["K_cache"], ok["V_cache"], keep.long(), lens, lens.clone())
    assert engine.device_error() == 0


def test_empty_calls(engine):
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    lens0, lens = ints([]), ints([2])
    before = engine.launch_count()
    engine.qkv_norm_rope(z(0, 96), z(0, 0, 16), z(0, 0, 16), z(0, 0, 16), 0)
    engine.kv_cache_attend_tree(z(0, 8, 16), z(0, 8, 16), z(0, 2, 16), z(0, 2, 16), lens0, 1.0)
    engine.kv_cache_attend_tree(z(2, 8, 16), z(2, 8, 16), z(2, 0, 16), z(2, 0, 16), lens, 1.0)
    engine.kv_cache_compact(z(0, 8, 16), z(0, 8, 16), z(0, 2).int(), lens0, lens0)
    assert engine.launch_count() == before
    out = z(2, 3, 16) + 4
    engine.kv_cache_attend_tree(z(2, 8, 16), z(2, 8, 16), z(2, 3, 16), out, lens, 1.0, n_new=ints([0]))
    lens_out = ints([-5])
    engine.kv_cache_compact(z(2, 8, 16), z(2, 8, 16), z(1, 0).int(), ints([0]), lens, lens_out)
    assert bool((out == 4).all()) and lens_out.tolist() == [2]


def test_other_stream_own_workspace_and_graphs(engine):
    """Two captured graphs with a workspace each, replayed side by side on two streams, and eager calls between: the bits of
    one call alone."""
    cases = [attend_case((3, 8, 8, 2, 64, [100, 900, 3000], True, "tree"), 81), attend_case((2, 16, 8, 1, 128, [2500, 64], False, "tree"), 82)]
    want = [run_attend(engine, s) for s in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs, outs, spaces = [], [], []
    for s, st in zip(cases, streams):
        outs.append(s["out"].clone())
        spaces.append(torch.zeros(engine.attention_workspace_bytes(), dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            engine.set_stream(torch.cuda.current_stream().cuda_stream)
            try:
                engine.kv_cache_attend_tree(s["K"], s["V"], s["Q"], outs[-1], s["lens"], s["scale"], n_new=s["n_new"], mask=s["mask"],
                                            workspace=spaces[-1])
            finally:
                engine.set_stream(0)
        graphs.append(gr)
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        eager = run_attend(engine, cases[0])
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0]) and all(torch.equal(x, y) for x, y in zip(outs, want))


def test_captured_steps(engine):
    """A serving step (extend, attend, compact) and a training pass (forward, backward with the norms' gradients), each captured
    on a stream of its own and replayed, give the bits of the eager calls; the gradients of norm weights add up over replays."""
    g = gen(95)
    B, T, H, Hkv, dk, max_seq = 3, 6, 8, 2, 128, 400
    lens, n_new, keep, n_keep = ints([5, 300, 64]), ints([6, 2, 4]), ints([[0, 2, 5, 0, 0, 0], [1, 0, 0, 0, 0, 0], [0, 1, 3, 0, 0, 0]]), ints([3, 1, 3])
    mask = tree_masks(np.random.RandomState(95), B, T)
    freq = torch.tensor(ref.frequencies(dk), dtype=torch.float64, device="cuda")
    gq, gk, bias = randn(g, dk), randn(g, dk), randn(g, (H + 2 * Hkv) * dk)
    qkv, K0, V0 = randn(g, B * T, (H + 2 * Hkv) * dk), randn(g, B * Hkv, max_seq, dk), randn(g, B * Hkv, max_seq, dk)
    grads = [randn(g, B * h, T, dk) for h in (H, Hkv, Hkv)]

    def serve(K, V, Q, out, lens_out):
        engine.kv_cache_extend(qkv, Q, K, V, lens, n_new=n_new, bias=bias, gq=gq, gk=gk, freq=freq)
        engine.kv_cache_attend_tree(K, V, Q, out, lens, dk ** -0.5, n_new=n_new, mask=mask)
        engine.kv_cache_compact(K, V, keep, n_keep, lens, lens_out)

    def train(Q, K, V, dqkv, dgq, dgk):
        engine.qkv_norm_rope(qkv, Q, K, V, B, bias=bias, gq=gq, gk=gk, freq=freq, pairing="interleaved")
        engine.qkv_norm_rope_bwd(*grads, dqkv, B, qkv=qkv, bias=bias, gq=gq, gk=gk, freq=freq, pairing="interleaved", dgq=dgq, dgk=dgk)

    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    state = lambda: [K0.clone(), V0.clone(), z(B * H, T, dk), z(B * H, T, dk), ints([0] * B)]  # noqa: E731
    outputs = lambda: [*(z(B * h, T, dk) for h in (H, Hkv, Hkv)), torch.zeros_like(qkv), z(dk), z(dk)]  # noqa: E731
    for step, make in ((serve, state), (train, outputs)):
        want, got = make(), make()
        step(*want)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=torch.cuda.Stream()):
            engine.set_stream(torch.cuda.current_stream().cuda_stream)
            try:
                step(*got)
            finally:
                engine.set_stream(0)
        for x, y in zip(got, make()):
            x.copy_(y)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        if step is train:
            gr.replay()
            torch.cuda.synchronize()
            for x, y in zip(got[4:], want[4:]):                # the second sum starts from the first: two roundings
                assert float((x - 2 * y).abs().max()) <= 2 * 2.0 ** -23 * float(y.abs().max())
        del gr
    assert engine.device_error() == 0


def test_more_than_32_bits_of_elements(engine):
    """Queries, keys and values of 2^31 elements and more: the last tokens' rows have the bits of a call of their own."""
    S, H, Hkv, dk = 840016, 16, 2, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 27 GB")
    W, last = (H + 2 * Hkv) * dk, 5
    assert S * W > 1 << 31
    freq = torch.tensor(ref.frequencies(dk), dtype=torch.float64, device="cuda")
    g = gen(97)
    gq, gk = randn(g, dk), randn(g, dk)
    qkv = torch.empty(S, W, device="cuda").fill_(0.5)
    qkv[-last:] = randn(g, last, W)
    big = [torch.empty(h, S, dk, device="cuda") for h in (H, Hkv, Hkv)]
    engine.qkv_norm_rope(qkv, *big, 1, gq=gq, gk=gk, freq=freq)
    small = [torch.empty(h, last, dk, device="cuda") for h in (H, Hkv, Hkv)]
    pos = ints(range(S - last, S))
    engine.qkv_norm_rope(qkv[-last:].contiguous(), *small, 1, gq=gq, gk=gk, freq=freq, pos=pos)
    assert all(torch.equal(x[:, -last:], y) for x, y in zip(big, small))
    dqkv, few = torch.empty(S, W, device="cuda"), torch.empty(last, W, device="cuda")
    engine.qkv_norm_rope_bwd(*big, dqkv, 1, qkv=qkv, gq=gq, gk=gk, freq=freq)
    engine.qkv_norm_rope_bwd(*small, few, 1, qkv=qkv[-last:].contiguous(), gq=gq, gk=gk, freq=freq, pos=pos)
    assert torch.equal(dqkv[-last:], few)
    del qkv, big, dqkv
    torch.cuda.empty_cache()


def test_cache_beyond_32_bit_offsets(engine):
    """Head 2 of a cache of 2^23 rows starts 2^31 elements (8 GiB) in; rows at both ends of it."""
    Hkv, dk, max_seq, T = 3, 128, (1 << 23) + 64, 4
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 26 GB for the caches")
    K, V = (torch.empty(Hkv, max_seq, dk, device="cuda") for _ in range(2))
    g = gen(91)
    qkv, Q = randn(g, T, 3 * Hkv * dk), torch.empty(Hkv, T, dk, device="cuda")
    for L in (200, max_seq - T):
        lo = max(0, L - 300)
        for x in (K, V):
            x[:, lo:L] = randn(g, Hkv, L - lo, dk)
            x[:, L:L + T] = 0
        engine.kv_cache_extend(qkv, Q, K, V, ints([L]))
        flat = qkv.view(T, 3, Hkv, dk).permute(1, 2, 0, 3)
        assert torch.equal(Q, flat[0]) and torch.equal(K[:, L:L + T], flat[1]) and torch.equal(V[:, L:L + T], flat[2])
        keep = ints([[1, 3, 0, 0]])
        engine.kv_cache_compact(K, V, keep, ints([2]), ints([L]))
        assert torch.equal(K[:, L:L + 2], flat[1][:, [1, 3]]) and torch.equal(V[:, L:L + 2], flat[2][:, [1, 3]])
        assert torch.equal(K[:, L + 2:L + T], flat[1][:, 2:])
        if L == 200:
            wide = randn(g, 10 * Hkv, T, dk)      # 40 rows to a key head: the tensor-memory kernel
            got = torch.empty_like(wide)
            engine.kv_cache_attend_tree(K, V, wide, got, ints([L]), 0.1)
            short = [x[:, :L + T].contiguous() for x in (K, V)]
            want, smag, vmag = ref.attend_tree(*short, wide, got, ints([L]), 0.1)
            assert float((got.double() - want).abs().max()) < ref.attend_bound(smag, vmag, dk)
            out = torch.empty_like(Q)
            engine.kv_cache_attend_tree(K, V, Q, out, ints([L]), 0.1)
            short = [x[:, :L + T].contiguous() for x in (K, V)]
            want, smag, vmag = ref.attend_tree(*short, Q, out, ints([L]), 0.1)
            assert float((out.double() - want).abs().max()) < ref.attend_bound(smag, vmag, dk)
    del K, V
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------------------ compact

@pytest.mark.parametrize("shift", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("B,T,Hkv,dk", [(1, 1, 1, 64), (4, 16, 2, 64), (3, 40, 5, 50), (9, 130, 8, 128), (2, 7, 1, 1), (2, 5, 3, 300)])
def test_kv_cache_compact(engine, B, T, Hkv, dk, shift):
    rng = np.random.RandomState(T)
    max_seq = T + 20
    g = gen(T)
    K, V = (randn(g, B * Hkv, max_seq, dk) for _ in range(2))
    if shift:
        K = unaligned(K)
    lens = rng.randint(0, 21, B)
    n = rng.randint(0, T + 1, B)
    n[0] = T                                          # the identity: nothing moves
    keep = np.full((B, T), -7, np.int32)              # entries behind n_keep are not read as indices
    for b in range(B):
        keep[b, :n[b]] = np.sort(rng.permutation(T)[:n[b]])
    want = [K.clone(), V.clone()]
    for b in range(B):
        for x in want:
            x = x.view(B, Hkv, max_seq, dk)
            x[b, :, lens[b]:lens[b] + n[b]] = x[b][:, (lens[b] + keep[b, :n[b]]).tolist()].clone()
    lens_out = ints(np.zeros(B))
    engine.kv_cache_compact(K, V, ints(keep), ints(n), ints(lens), lens_out)
    assert torch.equal(K, want[0]) and torch.equal(V, want[1]) and lens_out.tolist() == (lens + n).tolist()


def test_kv_cache_compact_refuses_bad_lists(engine):
    B, T, Hkv, dk, max_seq = 8, 4, 2, 32, 24
    g = gen(12)
    K, V = (randn(g, B * Hkv, max_seq, dk) for _ in range(2))
    K0, V0 = K.clone(), V.clone()
    keep = ints([[0, 2, 3, 0], [1, 1, 0, 0], [3, 2, 0, 0], [-1, 0, 0, 0], [1, 4, 0, 0], [1, 2, 3, 0], [0, 1, 2, 3], [2, 0, 0, 0]])
    n = ints([3, 2, 2, 1, 2, 5, -1, 1])               # good, twice the same, falling, negative, beyond T, too many, negative count, row outside
    lens = ints([2, 2, 2, 2, 2, 2, 2, 22])
    lens_out = torch.zeros_like(lens)
    engine.kv_cache_compact(K, V, keep, n, lens, lens_out)
    assert engine.device_error() == 102 and "ascending" in engine.last_error()
    assert lens_out.tolist() == [5, 2, 2, 2, 2, 2, 2, 22]
    for x, x0 in ((K, K0), (V, V0)):
        x0.view(B, Hkv, max_seq, dk)[0, :, 2:5] = x0.view(B, Hkv, max_seq, dk)[0][:, [2, 4, 5]].clone()
        assert torch.equal(x, x0)


# ------------------------------------------------------------------------------------------------------------ together

def test_drafted_decode_from_end_to_end(engine):
    """A prompt as a chain, then rounds of drafted trees whose accepted branch is compacted: every round's attention matches
    float64 attention over the accepted tokens and the branch, recomputed from the tokens' projections alone."""
    B, H, Hkv, dk, max_seq, prompt, T = 3, 4, 2, 64, 128, 21, 12
    width = (H + 2 * Hkv) * dk
    g, rng = gen(101), np.random.RandomState(5)
    gq, gk = 1 + 0.2 * randn(g, dk), 1 + 0.2 * randn(g, dk)
    freq = torch.tensor(engine.rope_frequencies(dk, scaling="turns", factor=8.0, low=1.0, high=4.0, original_len=64), dtype=torch.float64).cuda()
    how = dict(gq=gq, gk=gk, freq=freq)
    K, V = (torch.full((B * Hkv, max_seq, dk), float("nan"), device="cuda") for _ in range(2))
    story = [[] for _ in range(B)]                    # accepted tokens' projections
    lens, lens_out = ints([0] * B), ints([0] * B)

    def expect(b, rows):
        """Float64 attention of the last token of rows [n, width] over all of them."""
        q, k, v = ref.qkv_norm_rope(torch.stack(rows), 1, H, Hkv, dk, None, gq, gk, 1e-6, freq)
        k, v = (x[0].repeat_interleave(H // Hkv, 0) for x in (k, v))
        p = torch.softmax((q[0, :, -1:] @ k.transpose(1, 2)) * 0.125, -1)
        return (p @ v)[:, 0]

    def step(T, pos, mask, n):
        qkv = randn(g, B * T, width)
        Q, out = torch.empty(B * H, T, dk, device="cuda"), torch.zeros(B * H, T, dk, device="cuda")
        engine.kv_cache_extend(qkv, Q, K, V, lens, n_new=n, pos=pos, **how)
        engine.kv_cache_attend_tree(K, V, Q, out, lens, 0.125, n_new=n, mask=mask)
        return qkv.view(B, T, width), out.view(B, H, T, dk)

    # tolerance: inputs of the attention to 60 u of values of at most ~8 (rope test), scores of |q||k| <= 64 * 8 * 8 / 8 at the very most
    # would be 512; these normed heads stay under 30: e = 30 * (120 u + bound's 1e-5) -> 2.2 e |v| + 1e-5 |v|, |v| < 6
    tol = 6 * (2.2 * 30 * (120 * U + 1.3e-5) + 1e-5)
    n = ints([prompt, prompt - 5, 1])
    qkv, out = step(prompt, None, None, n)
    for b in range(B):
        story[b] = list(qkv[b, :int(n[b])])
        for t in (0, int(n[b]) - 1):
            assert float((out[b, :, t].double() - expect(b, story[b][:t + 1])).abs().max()) < tol
    lens = lens + n
    for _ in range(4):
        parent = np.array([[rng.randint(-1, t) if t else -1 for t in range(T)] for _ in range(B)])
        depth, mask = np.zeros((B, T), int), np.zeros((B, T, 1), np.int64)
        for b in range(B):
            for t in range(T):
                p = parent[b, t]
                depth[b, t] = 0 if p < 0 else depth[b, p] + 1
                mask[b, t, 0] = (0 if p < 0 else mask[b, p, 0]) | (1 << t)
        pos = (lens[:, None] + ints(depth)).contiguous()
        n = ints([T, T - 3, T - 1])
        qkv, out = step(T, pos, torch.from_numpy(mask).cuda(), n)
        keep, n_keep = np.zeros((B, T), int), np.zeros(B, int)
        for b in range(B):
            leaf = rng.randint(0, int(n[b]))
            path = [j for j in range(T) if (mask[b, leaf, 0] >> j) & 1]
            rows = story[b] + [qkv[b, j] for j in path]
            assert float((out[b, :, leaf].double() - expect(b, rows)).abs().max()) < tol
            keep[b, :len(path)], n_keep[b] = path, len(path)
            story[b] = rows
        engine.kv_cache_compact(K, V, ints(keep), ints(n_keep), lens, lens_out)
        lens = lens_out.clone()
    assert lens.tolist() == [len(x) for x in story]


def test_training_pass_from_end_to_end(engine):
    """Projection -> norm and rotation -> causal attention -> gradients back to the projection and the norm weights, against
    float64 autograd."""
    B, S, H, dk = 2, 160, 3, 64
    g = gen(111)
    qkv = randn(g, B * S, 3 * H * dk)
    gq, gk = 1 + 0.2 * randn(g, dk), 1 + 0.2 * randn(g, dk)
    freq = torch.tensor(engine.rope_frequencies(dk), dtype=torch.float64).cuda()
    how = dict(gq=gq, gk=gk, freq=freq, pairing="interleaved")
    q, k, v, o, dq, dk_, dv = (torch.empty(B * H, S, dk, device="cuda") for _ in range(7))
    L, do = torch.empty(B * H, S, device="cuda"), randn(g, B * H, S, dk)
    engine.qkv_norm_rope(qkv, q, k, v, B, **how)
    engine.sdpa_fwd(q, k, v, o, L, 0.125, True)
    engine.sdpa_bwd(q, k, v, o, do, L, dq, dk_, dv, 0.125, True)
    dqkv, dgq, dgk = torch.empty_like(qkv), torch.zeros(dk, device="cuda"), torch.zeros(dk, device="cuda")
    engine.qkv_norm_rope_bwd(dq, dk_, dv, dqkv, B, qkv=qkv, dgq=dgq, dgk=dgk, **how)
    leaves = [x.double().requires_grad_() for x in (qkv, gq, gk)]
    Q, K, V = ref.qkv_norm_rope(leaves[0], B, H, H, dk, None, leaves[1], leaves[2], 1e-6, freq, "interleaved")
    P = torch.softmax((Q @ K.transpose(2, 3) * 0.125).masked_fill(torch.ones(S, S, device="cuda").triu(1).bool(), -math.inf), -1)
    want = torch.autograd.grad((P @ V * do.double().view(B, H, S, dk)).sum(), leaves)
    # the attention's own parity bar is 1e-5 of the largest value; this pass adds 100 u
    for got, ref_ in zip((dqkv, dgq, dgk), want):
        assert float((got.double() - ref_).abs().max()) <= 2e-5 * float(ref_.abs().max())
