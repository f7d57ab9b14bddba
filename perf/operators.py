"""Measured cases of the operators around rotary positions and the contiguous KV cache.

Everything is fp32, the element type of this library's dense entry points:

  rope, rope_grad  q | k | v of a projection, flat [B*S, (H + 2*Hkv)*dk], -> head-major q, k, v with an optional bias, an
                   optional RMS norm of every q and k head and the position rotation; and the gradients of that pass.
  extend           the same pass for up to T new tokens of every sequence of a decode batch: keys and values go to the
                   cache rows lens[b] ... lens[b] + n_new[b] - 1 of sequence b.
  attend           attention of those tokens (a chain, or a tree of drafted tokens) over the cache and one another.
  compact          the accepted tokens of a drafted tree move to the front of the drafted rows of the cache.

The plain forms are elementary torch operations in 32 bits (angles and long sums in 64); `exact` restates each in 64 bits.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a training step's layer pass: biased projection, neighbouring pairs on part of the head, a length of no power of two
        dict(name="rope_train_partial", op="rope", B=8, S=1000, H=12, Hkv=4, dk=80, rot=32, pairing="interleaved", norm=False, bias=True,
             scaling="none", far=False),
        # prefill of one long prompt: shared key heads, normed heads, frequencies stretched for a long context, far positions
        dict(name="rope_long_prompt", op="rope", B=1, S=16384, H=32, Hkv=8, dk=128, rot=128, pairing="half", norm=True, bias=False,
             scaling="turns", far=True),
        # gradients of a training batch with normed heads (the norm weights' gradients are added to what is there)
        dict(name="rope_grad_norm", op="rope_grad", B=4, S=2048, H=16, Hkv=8, dk=128, rot=128, pairing="half", norm=True, bias=False,
             scaling="none", far=False),
        # gradients of one fine-tuning sequence of odd length, rotation only
        dict(name="rope_grad_odd", op="rope_grad", B=1, S=999, H=12, Hkv=4, dk=96, rot=48, pairing="half", norm=False, bias=False,
             scaling="none", far=False),
        # one user's next token: latency
        dict(name="extend_one", op="extend", B=1, T=1, H=32, Hkv=8, dk=128, rot=128, pairing="half", norm=True, bias=False,
             scaling="none", max_seq=4096, ragged=False),
        # a serving batch that verifies up to 16 drafted tokens for each sequence
        dict(name="extend_batch", op="extend", B=48, T=16, H=32, Hkv=8, dk=128, rot=128, pairing="half", norm=True, bias=False,
             scaling="linear", max_seq=512, ragged=True),
        # one token of one sequence over a short cache: latency
        dict(name="attend_one_short", op="attend", B=1, T=1, H=16, Hkv=8, dk=64, max_seq=1024, low=0.5, tree=False, ragged=False),
        # token-by-token decode of a batch of very different lengths, four heads to a key head
        dict(name="attend_decode_batch", op="attend", B=32, T=1, H=32, Hkv=8, dk=128, max_seq=4096, low=0.1, tree=False, ragged=False),
        # up to 16 drafted tokens for each sequence of a batch with long contexts
        dict(name="attend_tree16", op="attend", B=8, T=16, H=32, Hkv=8, dk=128, max_seq=8192, low=0.25, tree=True, ragged=True),
        # wide trees: 64 drafted tokens of four heads share each key head
        dict(name="attend_tree64", op="attend", B=8, T=64, H=24, Hkv=6, dk=64, max_seq=4096, low=0.25, tree=True, ragged=False),
        # the accepted branches of a batch's trees
        dict(name="compact_batch", op="compact", B=32, T=64, Hkv=8, dk=128, max_seq=512),
        # one sequence's accepted branch: latency
        dict(name="compact_one", op="compact", B=1, T=16, Hkv=8, dk=64, max_seq=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    Hkv, group = rng.choice((1, 2, 3, 4, 5, 8, 16)), rng.choice((1, 1, 2, 3, 4, 6, 8))
    return Hkv * group, Hkv, rng.choice((32, 40, 50, 64, 64, 72, 80, 96, 112, 128, 128))


def draw(rng):
    op = rng.choice(("rope", "rope_grad", "extend", "attend", "attend", "compact"))
    H, Hkv, dk = _heads(rng)
    width = (H + 2 * Hkv) * dk
    rope = dict(rot=rng.choice((dk, dk, dk // 2 // 2 * 2)), pairing=rng.choice(("half", "interleaved")), norm=rng.random() < 0.5,
                bias=rng.random() < 0.3, scaling=rng.choice(("none", "linear", "turns", "index")))
    if op in ("rope", "rope_grad"):
        B = _log(rng, 1, 16)
        most = (80 if op == "rope" else 24) * 1000000 // (width * B)
        return dict(op=op, B=B, S=_log(rng, 1, max(1, min(16384, most))), H=H, Hkv=Hkv, dk=dk, far=rng.random() < 0.5, **rope)
    if op == "extend":
        B, T = _log(rng, 1, 48), _log(rng, 1, 64)
        T = max(1, min(T, 6000000 // (width * B)))
        return dict(op=op, B=B, T=T, H=H, Hkv=Hkv, dk=dk, max_seq=T + _log(rng, 1, 1000), ragged=rng.random() < 0.7, **rope)
    if op == "attend":
        B, T = _log(rng, 1, 32), rng.choice((1, 1, _log(rng, 2, 96)))
        rows = B * Hkv * dk
        by_work = 2500000000 // (B * H * T * dk)       # keys that keep a pass under the largest listed one's operations
        return dict(op=op, B=B, T=T, H=H, Hkv=Hkv, dk=dk, max_seq=T + _log(rng, 1, max(1, min(60000, by_work, 60000000 // rows))),
                    low=rng.choice((0.0, 0.1, 0.5, 1.0)), tree=T > 1 and rng.random() < 0.7, ragged=rng.random() < 0.6)
    B, T = _log(rng, 1, 48), _log(rng, 1, 96)
    return dict(op=op, B=B, T=T, Hkv=Hkv, dk=dk, max_seq=T + _log(rng, 1, max(1, 40000000 // (B * Hkv * dk))))


# ----------------------------------------------------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n whole numbers spread evenly over lo .. hi (their middle for one)."""
    return [(lo + hi + 1) // 2] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(c):
    most = c["max_seq"] - c["T"]
    return _spread(int(c.get("low", 0.25) * most), most, c["B"])


def _counts(c):
    return _spread(1, c["T"], c["B"]) if c.get("ragged") else [c["T"]] * c["B"]


def _frequencies(rot, scaling, base=10000.0):
    """Radians per position of every pair, in 64 bits."""
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2.0 * i / max(rot, 1))
    if scaling == "linear":
        return f / 4.0
    if scaling == "turns":     # pairs that turn often over the original context keep their frequency
        keep = np.clip((8192 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return f * (keep + (1.0 - keep) / 8.0)
    if scaling == "index":     # the same ramp, linear in the pair's index
        at = lambda turns: rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        slow = np.clip((i - first) / max(last - first, 1e-3), 0.0, 1.0)
        return f * (1.0 - slow) + f / 16.0 * slow
    return f


def _rope_inputs(c, rng, g):
    width = (c["H"] + 2 * c["Hkv"]) * c["dk"]
    # outlier channels, as projections of trained models have them
    spread = torch.exp(0.5 * torch.randn(width, device="cuda", generator=g))
    s = {"width": width, "qkv": torch.randn(c["B"] * c.get("S", c.get("T")), width, device="cuda", generator=g) * spread,
         "bias": torch.randn(width, device="cuda", generator=g) if c["bias"] else None, "gq": None, "gk": None,
         "freq": torch.from_numpy(_frequencies(c["rot"], c["scaling"])).cuda(),
         "amplitude": 0.1 * math.log(16.0) + 1.0 if c["scaling"] == "index" else 1.0, "pos": None}
    if c["norm"]:
        s["gq"] = 1.0 + 0.2 * torch.randn(c["dk"], device="cuda", generator=g)
        s["gk"] = 1.0 + 0.2 * torch.randn(c["dk"], device="cuda", generator=g)
    if c.get("far"):
        at = rng.randint(0, 1000000, c["B"])[:, None] + np.arange(c["S"])[None, :]
        s["pos"] = torch.from_numpy(at.astype(np.int32)).cuda()
    return s


def _tree(c, rng):
    """Parents (-1: hangs on the context), depths and the ancestor bits of every token, [B, T] and [B, T, words]."""
    B, T = c["B"], c["T"]
    words = (T + 63) // 64
    parent, depth = np.full((B, T), -1, np.int64), np.zeros((B, T), np.int64)
    bits = np.zeros((B, T, words), np.uint64)
    every = np.arange(B)
    for t in range(T):
        if t:
            parent[:, t] = rng.randint(max(-1, t - 8), t, B)
            has = parent[:, t] >= 0
            bits[has, t] = bits[every[has], parent[has, t]]
            depth[has, t] = depth[every[has], parent[has, t]] + 1
        bits[:, t, t // 64] |= np.uint64(1 << (t % 64))
    return depth, bits


def prepare(case, seed):
    c = dict(case)
    rng = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    ints = lambda v: torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).cuda()  # noqa: E731
    s = {"case": c}
    if c["op"] in ("rope", "rope_grad", "extend"):
        s.update(_rope_inputs(c, rng, g))
    if c["op"] in ("rope", "rope_grad"):
        shape = lambda heads: (c["B"] * heads, c["S"], c["dk"])  # noqa: E731
        if c["op"] == "rope":
            s["out"] = [torch.empty(shape(h), device="cuda") for h in (c["H"], c["Hkv"], c["Hkv"])]
        else:
            s["grads"] = [rand(*shape(h)) for h in (c["H"], c["Hkv"], c["Hkv"])]
            s["dqkv"] = torch.empty_like(s["qkv"])
            s["dgq"], s["dgk"] = (rand(c["dk"]), rand(c["dk"])) if c["norm"] else (None, None)
        return s
    s["lens"] = ints(rng.permutation(_lens(c)))
    if c["op"] in ("extend", "attend"):
        s["n_new"] = ints(rng.permutation(_counts(c))) if c["ragged"] else None
    s["K"], s["V"] = (rand(c["B"] * c["Hkv"], c["max_seq"], c["dk"]) for _ in range(2))
    if c["op"] == "extend":
        depth, _ = _tree(c, rng)
        s["pos"] = (s["lens"][:, None] + ints(depth)) if c["T"] > 1 else None
        s["q"] = rand(c["B"] * c["H"], c["T"], c["dk"])
    elif c["op"] == "attend":
        s["q"], s["out"] = (rand(c["B"] * c["H"], c["T"], c["dk"]) for _ in range(2))
        s["mask"] = torch.from_numpy(_tree(c, rng)[1].view(np.int64)).cuda() if c["tree"] else None
    else:
        # a root-to-leaf path of a random tree, three tokens at the least where there are so many
        n = rng.permutation(_spread(min(3, c["T"]), max(1, c["T"] // 4), c["B"]))
        keep = np.zeros((c["B"], c["T"]), np.int32)
        for b in range(c["B"]):
            keep[b, : n[b]] = np.sort(rng.permutation(c["T"])[: n[b]])
        s["keep"], s["n_keep"], s["lens_out"] = ints(keep), ints(n), torch.empty_like(s["lens"])
    return s


# ------------------------------------------------------------------------------------------------------ plain forms

def _turn(x, cos, sin, pairing):
    """Rotates the leading 2 * cos.shape[-1] elements of every head of x [rows, heads, dk]; cos, sin [rows, 1, pairs]."""
    half = cos.shape[-1]
    if half == 0:
        return x
    if pairing == "half":
        a, b = x[..., :half], x[..., half: 2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _angles(s, T):
    c = s["case"]
    if s["pos"] is not None:
        pos = s["pos"].reshape(-1)
    elif c["op"] == "extend":
        pos = (s["lens"][:, None] + torch.arange(T, device="cuda")).reshape(-1)
    else:
        pos = torch.arange(T, device="cuda").repeat(c["B"])
    a = pos.double()[:, None, None] * s["freq"]
    return (a.cos() * s["amplitude"]).float(), (a.sin() * s["amplitude"]).float()


def _split(s, flat):
    c = s["case"]
    return flat.view(flat.shape[0], -1, c["dk"]).split((c["H"], c["Hkv"], c["Hkv"]), 1)


def _projected(s):
    return _split(s, s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"])


EPS = 1e-6


def _normed(x, g):
    return x if g is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * g


def _rotated(s, T):
    """q, k, v as [B*T, heads, dk]."""
    cos, sin = _angles(s, T)
    q, k, v = _projected(s)
    pairing = s["case"]["pairing"]
    return _turn(_normed(q, s["gq"]), cos, sin, pairing), _turn(_normed(k, s["gk"]), cos, sin, pairing), v


def _head_major(x, B):
    return x.view(B, -1, *x.shape[1:]).transpose(1, 2)


def _plain_rope(s):
    c = s["case"]
    for out, x in zip(s["out"], _rotated(s, c["S"])):
        out.view(c["B"], -1, c["S"], c["dk"]).copy_(_head_major(x, c["B"]))
    return s["out"]


def _plain_rope_grad(s):
    c = s["case"]
    cos, sin = _angles(s, c["S"])
    flat = [g.view(c["B"], -1, c["S"], c["dk"]).transpose(1, 2).reshape(c["B"] * c["S"], -1, c["dk"]) for g in s["grads"]]
    x = _projected(s)
    parts = []
    for d, x0, g, dg in zip(flat[:2], x[:2], (s["gq"], s["gk"]), (s["dgq"], s["dgk"])):
        d = _turn(d, cos, -sin, c["pairing"])
        if g is not None:
            r = torch.rsqrt((x0 * x0).mean(-1, keepdim=True) + EPS)
            unit = x0 * r
            dg += (d * unit).sum((0, 1), dtype=torch.float64).float()
            d = d * g
            d = r * (d - unit * (d * unit).mean(-1, keepdim=True))
        parts.append(d)
    torch.cat([p.reshape(p.shape[0], -1) for p in parts + flat[2:]], 1, out=s["dqkv"])
    return [s["dqkv"], s["dgq"], s["dgk"]]


def _plain_extend(s):
    c = s["case"]
    B, T = c["B"], c["T"]
    q, k, v = (_head_major(x, B) for x in _rotated(s, T))
    at = torch.arange(T, device="cuda")
    n = s["n_new"] if s["n_new"] is not None else torch.full((B,), T, device="cuda")
    valid = (at[None, :] < n[:, None])[:, None, :, None]
    rows = (s["lens"][:, None] + at[None, :]).long()[:, None, :, None]
    held = s["q"].view(B, -1, T, c["dk"])
    held.copy_(torch.where(valid, q, held))
    for cache, new in ((s["K"], k), (s["V"], v)):
        cache = cache.view(B, -1, c["max_seq"], c["dk"])
        rows_of = rows.expand(-1, new.shape[1], -1, c["dk"])
        cache.scatter_(2, rows_of, torch.where(valid, new, cache.gather(2, rows_of)))
    return [s["q"], s["K"], s["V"]]


def _seen(s):
    """[B, T, max_seq]: which cache rows a token attends to."""
    c = s["case"]
    B, T, N = c["B"], c["T"], c["max_seq"]
    j = torch.arange(N, device="cuda")[None, :] - s["lens"][:, None]                     # index among the new tokens, < 0: cached
    n = s["n_new"][:, None] if s["n_new"] is not None else T
    new = (j >= 0) & (j < n)
    t = torch.arange(T, device="cuda")
    if s["mask"] is None:
        mine = t[None, :, None] >= j[:, None, :]
    else:
        jc = j.clamp(0, T - 1)
        words = s["mask"].gather(2, (jc // 64)[:, None, :].expand(-1, T, -1))
        mine = ((words >> (jc % 64)[:, None, :]) & 1).bool()
    return (j < 0)[:, None, :] | (new[:, None, :] & mine)


def _plain_attend(s):
    c = s["case"]
    B, T, N, dk, Hkv = c["B"], c["T"], c["max_seq"], c["dk"], c["Hkv"]
    q = s["q"].view(B, Hkv, -1, dk)
    K, V = (s[x].view(B, Hkv, N, dk) for x in "KV")
    scores = torch.matmul(q, K.transpose(2, 3)).view(B, Hkv, -1, T, N) * (1.0 / math.sqrt(dk))
    scores = scores.masked_fill(~_seen(s)[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    y = torch.matmul(p.view(B, Hkv, -1, N), V).view(B, c["H"], T, dk)
    out = s["out"].view(B, c["H"], T, dk)
    if s["n_new"] is not None:
        y = torch.where((torch.arange(T, device="cuda")[None, :] < s["n_new"][:, None])[:, None, :, None], y, out)
    out.copy_(y)
    return s["out"]


def _plain_compact(s):
    c = s["case"]
    B, T, dk = c["B"], c["T"], c["dk"]
    at = torch.arange(T, device="cuda")
    kept = (at[None, :] < s["n_keep"][:, None])[:, None, :, None]
    to = (s["lens"][:, None] + at[None, :]).long()[:, None, :, None]
    come = (s["lens"][:, None] + s["keep"]).long()[:, None, :, None]
    for cache in (s["K"], s["V"]):
        cache = cache.view(B, c["Hkv"], c["max_seq"], dk)
        wide = (-1, c["Hkv"], -1, dk)
        held = cache.gather(2, to.expand(wide))
        cache.scatter_(2, to.expand(wide), torch.where(kept, cache.gather(2, come.expand(wide)), held))
    torch.add(s["lens"], s["n_keep"], out=s["lens_out"])
    return [s["K"], s["V"], s["lens_out"]]


# ------------------------------------------------------------------------------------------------- one pass, the work

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rope": _plain_rope, "rope_grad": _plain_rope_grad, "extend": _plain_extend, "attend": _plain_attend,
                "compact": _plain_compact}[c["op"]](s)
    from axiom_b200.engine import get_engine
    eng = get_engine()
    if c["op"] in ("rope", "rope_grad", "extend"):
        how = dict(bias=s["bias"], gq=s["gq"], gk=s["gk"], eps=EPS, freq=s["freq"], pairing=c["pairing"], amplitude=s["amplitude"],
                   pos=s["pos"])
    if c["op"] == "rope":
        eng.qkv_norm_rope(s["qkv"], *s["out"], c["B"], **how)
        return s["out"]
    if c["op"] == "rope_grad":
        eng.qkv_norm_rope_bwd(*s["grads"], s["dqkv"], c["B"], qkv=s["qkv"], dgq=s["dgq"], dgk=s["dgk"], **how)
        return [s["dqkv"], s["dgq"], s["dgk"]]
    if c["op"] == "extend":
        eng.kv_cache_extend(s["qkv"], s["q"], s["K"], s["V"], s["lens"], n_new=s["n_new"], **how)
        return [s["q"], s["K"], s["V"]]
    if c["op"] == "attend":
        eng.kv_cache_attend_tree(s["K"], s["V"], s["q"], s["out"], s["lens"], 1.0 / math.sqrt(c["dk"]), n_new=s["n_new"],
                                 mask=s["mask"])
        return s["out"]
    eng.kv_cache_compact(s["K"], s["V"], s["keep"], s["n_keep"], s["lens"], s["lens_out"])
    return [s["K"], s["V"], s["lens_out"]]


def work(case):
    c = case
    dk, Hkv = c["dk"], c["Hkv"]
    if c["op"] == "compact":
        kept = sum(_spread(min(3, c["T"]), max(1, c["T"] // 4), c["B"]))
        return {"bytes": 16.0 * kept * Hkv * dk + 16.0 * c["B"], "flops": 0}
    H = c["H"]
    if c["op"] == "attend":
        lens, counts = _lens(c), sorted(_counts(c))
        # which count meets which length is drawn: the mean of the best and the worst pairing
        pairs = (sum(x * y for x, y in zip(lens, counts)) + sum(x * y for x, y in zip(lens, counts[::-1]))) / 2
        return {"bytes": 8.0 * Hkv * dk * (sum(lens) + sum(counts)) + 8.0 * H * dk * sum(counts),
                "flops": 4.0 * H * dk * (pairs + sum(counts))}
    width = (H + 2 * Hkv) * dk
    rows = sum(_counts(c)) if c["op"] == "extend" else c["B"] * c["S"]
    if c["op"] == "rope_grad":
        moved = 2 * width + ((H + Hkv) * dk if c["norm"] else 0)
        return {"bytes": 4.0 * rows * moved, "flops": rows * (H + Hkv) * (3.0 * c["rot"] + (10.0 * dk if c["norm"] else 0))}
    return {"bytes": 8.0 * rows * width, "flops": rows * (H + Hkv) * (3.0 * c["rot"] + (4.0 * dk if c["norm"] else 0))}


# ------------------------------------------------------------------------------------------------ the same in 64 bits

def _exact_head(x, g, where, freq, amplitude, pairing):
    """One tensor of heads [..., tokens, dk] in 64 bits at positions `where` [..., tokens] by complex multiplication."""
    if g is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * g
    pairs = len(freq)
    if pairs == 0:
        return x
    turn = torch.polar(torch.full_like(where, amplitude)[..., None].expand(*where.shape, pairs), where[..., None] * freq)
    if pairing == "half":
        z = torch.complex(x[..., :pairs], x[..., pairs: 2 * pairs]) * turn
        y = torch.cat((z.real, z.imag), -1)
    else:
        z = torch.view_as_complex(x[..., : 2 * pairs].reshape(*x.shape[:-1], pairs, 2)) * turn
        y = torch.view_as_real(z).reshape(*x.shape[:-1], 2 * pairs)
    return torch.cat((y, x[..., 2 * pairs:]), -1)


def _exact_rope(s, qkv, gq, gk):
    c = s["case"]
    B, T, H, Hkv, dk = c["B"], c.get("S", c.get("T")), c["H"], c["Hkv"], c["dk"]
    if s["bias"] is not None:
        qkv = qkv + s["bias"].double()
    start = s["lens"].double()[:, None] if c["op"] == "extend" else 0.0
    where = s["pos"].double() if s["pos"] is not None else (torch.arange(T, device="cuda").double() + start).expand(B, T)
    where = where[:, None, :]
    heads = qkv.reshape(B, T, H + 2 * Hkv, dk).permute(0, 2, 1, 3)
    how = (s["freq"], s["amplitude"], c["pairing"])
    return (_exact_head(heads[:, :H], gq, where.expand(B, H, T), *how),
            _exact_head(heads[:, H: H + Hkv], gk, where.expand(B, Hkv, T), *how), heads[:, H + Hkv:])


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    dbl = lambda x: None if x is None else x.double()  # noqa: E731
    if c["op"] == "rope":
        return [x.reshape(-1, c["S"], c["dk"]) for x in _exact_rope(s, s["qkv"].double(), dbl(s["gq"]), dbl(s["gk"]))]
    if c["op"] == "rope_grad":
        leaves = [s["qkv"].double().requires_grad_()] + [s[k].double().requires_grad_() for k in ("gq", "gk") if s[k] is not None]
        gq, gk = leaves[1:] if c["norm"] else (None, None)
        y = _exact_rope(s, leaves[0], gq, gk)
        grads = torch.autograd.grad(y, leaves, [d.double().view(x.shape) for d, x in zip(s["grads"], y)])
        more = [s["dgq"].double() + grads[1], s["dgk"].double() + grads[2]] if c["norm"] else [None, None]
        return [grads[0]] + more
    B, N, dk, Hkv, T = c["B"], c["max_seq"], c["dk"], c["Hkv"], c["T"]
    lens = s["lens"].tolist()
    K, V = (s[x].double().view(B, Hkv, N, dk) for x in "KV")
    if c["op"] == "compact":
        n_keep, keep = s["n_keep"].tolist(), s["keep"].tolist()
        for b in range(B):
            come = [lens[b] + k for k in keep[b][: n_keep[b]]]
            for cache in (K, V):
                cache[b, :, lens[b]: lens[b] + n_keep[b]] = cache[b][:, come].clone()
        return [K.view(-1, N, dk), V.view(-1, N, dk), s["lens"] + s["n_keep"]]
    counts = s["n_new"].tolist() if s["n_new"] is not None else [T] * B
    if c["op"] == "extend":
        q, k, v = _exact_rope(s, s["qkv"].double(), dbl(s["gq"]), dbl(s["gk"]))
        Q = s["q"].double().view(B, -1, T, dk)
        for b in range(B):
            n = counts[b]
            Q[b, :, :n] = q[b, :, :n]
            K[b, :, lens[b]: lens[b] + n] = k[b, :, :n]
            V[b, :, lens[b]: lens[b] + n] = v[b, :, :n]
        return [Q.view(-1, T, dk), K.view(-1, N, dk), V.view(-1, N, dk)]
    out = s["out"].double().view(B, c["H"], T, dk)
    group = c["H"] // Hkv
    bits = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint64)
    for b in range(B):
        n, rows = counts[b], lens[b] + counts[b]
        shown = np.tril(np.ones((n, n), bool))
        if bits is not None:
            shown = np.array([[(int(bits[b, t, j // 64]) >> (j % 64)) & 1 for j in range(n)] for t in range(n)], bool)
        hide = torch.cat((torch.zeros(n, lens[b], dtype=torch.bool, device="cuda"), ~torch.from_numpy(shown).cuda()), 1)
        for h in range(c["H"]):
            z = (s["q"].view(B, -1, T, dk)[b, h, :n].double() @ K[b, h // group, :rows].T) / math.sqrt(dk)
            out[b, h, :n] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ V[b, h // group, :rows]
    return out.view(-1, T, dk)
