"""Float64 restatements (torch, CPU or GPU) of the rotary / per-head-norm pass and of the ragged-batch KV-cache calls.
Test infrastructure only."""
import math

import torch


def frequencies(rot, base=10000.0, scaling="none", factor=1.0, low=1.0, high=32.0, original_len=0):
    out = []
    if scaling == "index":
        index_of = lambda turns: rot * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(index_of(high)), 0), min(math.ceil(index_of(low)), rot - 1)
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "none":
            keep = 1.0
        elif scaling == "linear":
            keep = 0.0
        elif scaling == "turns":
            keep = (original_len * f / (2 * math.pi) - low) / (high - low)
        else:
            keep = 1.0 - (i - first) / max(last - first, 1e-3)
        keep = min(max(keep, 0.0), 1.0)
        out.append(f if scaling == "none" else f * keep + f / factor * (1.0 - keep))
    return out


def rope_head(x, g, eps, pos, freq, pairing, amplitude):
    """x [..., tokens, dk] float64, pos [..., tokens]."""
    if g is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * g
    if freq is None or len(freq) == 0:
        return x
    n = len(freq)
    t = pos[..., None].double() * freq
    c, s = torch.cos(t) * amplitude, torch.sin(t) * amplitude
    y = x.clone()
    ia = torch.arange(n, device=x.device) if pairing == "half" else 2 * torch.arange(n, device=x.device)
    ib = ia + n if pairing == "half" else ia + 1
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def qkv_norm_rope(qkv, B, H, Hkv, dk, bias=None, gq=None, gk=None, eps=1e-6, freq=None, pairing="half", amplitude=1.0, pos=None):
    """-> q [B, H, T, dk], k, v [B, Hkv, T, dk] in float64; pos [B, T] or None."""
    x = qkv.double()
    if bias is not None:
        x = x + bias.double()
    T = x.shape[0] // max(B, 1)
    x = x.view(B, T, H + 2 * Hkv, dk).transpose(1, 2)
    if pos is None:
        pos = torch.arange(T, device=x.device).expand(B, T)
    pos = pos.view(B, 1, T).double()
    d = lambda g: None if g is None else g.double()  # noqa: E731
    f = None if freq is None else freq.double()
    return (rope_head(x[:, :H], d(gq), eps, pos, f, pairing, amplitude), rope_head(x[:, H:H + Hkv], d(gk), eps, pos, f, pairing, amplitude),
            x[:, H + Hkv:])


def visible(b, T, n, mask):
    """[n, n] truth values: new token t sees new token j; mask int64 words [B, T, W], [T, W] or None."""
    if mask is None:
        return torch.ones(n, n, dtype=torch.bool).tril()
    m = mask[b] if mask.dim() == 3 else mask
    m = m.cpu()
    j = torch.arange(n)
    return ((m[:n][:, j // 64] >> (j % 64)) & 1).bool()


def attend_tree(K, V, Q, out, lens, scale, n_new=None, mask=None):
    """Float64 result with `out`'s own values in rows behind n_new; K, V [B*Hkv, max_seq, dk], Q [B*H, T, dk].  Also returns
    the largest scale * sum |q||k| of a visible pair and the largest visible |v| (the error bound's magnitudes)."""
    B = lens.numel()
    BH, T, dk = Q.shape
    H, Hkv = BH // B, K.shape[0] // B
    y = out.double().clone().view(B, H, T, dk)
    smag, vmag = 0.0, 0.0
    for b in range(B):
        L, n = int(lens[b]), int(n_new[b]) if n_new is not None else T
        if n == 0:
            continue
        see = torch.cat((torch.ones(n, L, dtype=torch.bool), visible(b, T, n, mask)), 1).to(Q.device)
        for h in range(H):
            k = K.view(B, Hkv, -1, dk)[b, h // (H // Hkv), :L + n].double()
            v = V.view(B, Hkv, -1, dk)[b, h // (H // Hkv), :L + n].double()
            q = Q.view(B, H, T, dk)[b, h, :n].double()
            for t in range(n):
                idx = see[t].nonzero().flatten()
                if idx.numel() == 0:
                    y[b, h, t] = 0.0
                    continue
                s = (k[idx] * q[t]).sum(-1) * scale
                y[b, h, t] = torch.softmax(s, -1) @ v[idx]
                smag = max(smag, float((k[idx] * q[t]).abs().sum(-1).max()) * abs(scale))
                vmag = max(vmag, float(v[idx].abs().max()))
    return y.view(BH, T, dk), smag, vmag


def attend_bound(smag, vmag, dk):
    """Error bound of the three-product tf32 evaluation.  A product of two fp32 values cut to 10 mantissa bits (hi) with
    remainders cut likewise (lo): the dropped lo.lo is below 2^-20 of it, each cut of a lo operand below 2^-20, so 3 * 2^-20;
    the 3 * dk / 8 accumulations of a score may each lose 2^-23 of the running sum.  That error e of a score changes a
    probability by a factor of up to exp(2e) ~ 1 + 2e (numerator and denominator); 2^x and the sums add about 2^-21 per
    step of the merges (at most 8 here); P.V loses 3 * 2^-20 of sum p |v| <= max |v| again."""
    e = smag * (3 * 2.0 ** -20 + 3 * dk / 8 * 2.0 ** -23 + 2.0 ** -22)
    return vmag * (2.2 * e + 3 * 2.0 ** -20 + 10 * 2.0 ** -21)
