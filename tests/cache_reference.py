"""The key/value cache and the 4-bit weights in 64 bits, from their definitions (include/ns2.h)."""

import math

import torch

GROUP = 32


def nibbles(codes):
    """uint8 [..., n] -> [..., 2n], the low four bits first."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def i4_weight(codes, scale, group):
    """[N, K] float64 that 4-bit codes [N, K/2] and fp16 scales [N, K/group] stand for."""
    return (nibbles(codes).double() - 8) * scale.double().repeat_interleave(group, 1)


def i4_codes(w, group):
    """The codes and scales of a weight [N, K] whose values are exact in fp32, as ns2_quantize_i4 defines them."""
    g = w.float().unflatten(1, (-1, group))
    scale = (g.abs().amax(-1) / 7).half()
    s = scale.float().unsqueeze(-1)
    q = (torch.where(s > 0, (g / s).round().clamp(-7, 7), 0.0) + 8).to(torch.uint8).flatten(1)
    return q[:, 0::2] | (q[:, 1::2] << 4), scale


def cache_codes(x):
    """The codes [..., D/2] and groups [..., D/32, 2] (step, offset) of fp32 values [..., D]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    step, off = ((hi - lo) / 15).half(), lo.half()
    s, o = step.float().unsqueeze(-1), off.float().unsqueeze(-1)
    q = torch.where(s > 0, ((g - o) / s).round().clamp(0, 15), 0.0).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([step, off], -1)


def cache_values(codes, groups):
    """float64 [..., D]: half(offset + code * step)."""
    q = nibbles(codes).double().unflatten(-1, (-1, GROUP))
    return (q * groups[..., 0:1].double() + groups[..., 1:2].double()).flatten(-2).half().double()


def rope_table(rows, D, theta=1e4):
    a = torch.arange(rows, dtype=torch.float64)[:, None] / theta ** (torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    return torch.cat([a.cos().reshape(-1), a.sin().reshape(-1)]).float()


def head_norm(x, w, cs, pos, rope_rows, eps):
    """x [rows, heads, D] float64, positions [rows] -> normed (w given) and rotated (cs given) heads."""
    D = x.shape[-1]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cs is None:
        return x
    cos, sin = (t.reshape(-1, D // 2).double() for t in cs.chunk(2))
    at = pos.long().clamp(0, cos.shape[0] - 1)
    turned = (pos >= 0) & (pos < rope_rows)
    c = torch.where(turned[:, None], cos[at], 1.0)[:, None]
    s = torch.where(turned[:, None], sin[at], 0.0)[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attention(q, pos, k, v, window, sinks, scale):
    """q [B, L, H, D], pos [B, L], k and v [B, cap, KH, D], all float64; rows without a key are NaN. Only visible
    values are touched. Returns the outputs and, per output, bounds of what roundings can do to it:
    max|v| of the visible keys, max over them of scale * sum |q||k|, their number."""
    B, L, H, D = q.shape
    KH, cap = k.shape[2], k.shape[1]
    o = torch.full_like(q, math.nan)
    vmax, smax, n = (torch.zeros(B, L, H, 1, dtype=torch.float64, device=q.device) for _ in range(3))
    for b in range(B):
        for i in range(L):
            p = int(pos[b, i])
            if p < 0 or p >= cap:
                continue
            j = torch.arange(p + 1, device=q.device)
            if window:
                j = j[(j < sinks) | (j > p - window)]
            for g in range(KH):
                h = slice(g * (H // KH), (g + 1) * (H // KH))
                kk, vv = k[b, j, g], v[b, j, g]
                s = scale * (q[b, i, h] @ kk.t())
                o[b, i, h] = torch.softmax(s, -1) @ vv
                vmax[b, i, h] = vv.abs().max()
                smax[b, i, h] = scale * (q[b, i, h].abs() @ kk.abs().t()).amax(-1, keepdim=True)
                n[b, i, h] = len(j)
    return o, vmax, smax, n


def attention_bound(o, vmax, smax, n, D, fp16):
    """How far a kernel's output may be from o. A score is a sum of D products, each off by 2^-21 of itself (two
    operands split into fp16 parts that keep 22 bits: 2^-22 each; fp16 operands are exact), summed in fp32 in
    any order (D 2^-24): off by at most d = smax (2^-21 + D 2^-24), and so are exponent (2^-23 relative of |s|,
    below smax, times log2 e) and maximum. Weights and their sum change by a factor within e^(2 (d + 2 smax 2^-23))
    and 2^-20 for exp2; a sum over n keys by n 2^-24, twice. fp16 weights are off by 2^-11 of themselves or, below
    2^-14, by 2^-25, and the output is rounded to fp16 (2^-11). The fp32 form splits weights: 2^-22."""
    d = smax * (2.0**-21 + D * 2.0**-24 + 2 * 2.0**-23)
    t = (torch.expm1(4 * d) + n * 2.0**-23 + 2.0**-20) * vmax
    if fp16:
        return t + vmax * (2.0**-11 + n * 2.0**-25) + o.abs() * 2.0**-11 + 2.0**-24
    return t + vmax * (2.0**-21 + n * 2.0**-36) + o.abs() * 2.0**-23


def gemma_hidden(W, ids, window, sinks, cache_bits, device):
    """The text encoder (17 layers of 640, 4 heads of 256 on one key/value head) with the sliding window of its local
    layers and keys and values as a cache holds them, in float64. W: name -> tensor."""
    H, D = 4, 256

    def w(name):
        return W[name].double().to(device)

    def rms(x, name):
        return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (w(name) + 1)

    def held(x):
        if cache_bits == 16:
            return x.half().double()
        return cache_values(*cache_codes(x.float()))

    x = w("model.embed_tokens.weight")[torch.tensor(ids, device=device)] * math.sqrt(640)
    L = len(ids)
    p = torch.arange(L, device=device)
    for i in range(17):
        n = f"model.layers.{i}."
        every = (i + 1) % 6 == 0
        a = p[:, None].double() / (1e6 if every else 1e4) ** (torch.arange(D // 2, dtype=torch.float64, device=device) * 2 / D)

        def turn(t):
            u, v = t.chunk(2, -1)
            c, s = a.cos()[:, None], a.sin()[:, None]
            return torch.cat([u * c - v * s, v * c + u * s], -1)

        h = rms(x, n + "input_layernorm.weight")
        q = turn(rms((h @ w(n + "self_attn.q_proj.weight").t()).reshape(L, H, D), n + "self_attn.q_norm.weight"))
        k = held(turn(rms((h @ w(n + "self_attn.k_proj.weight").t()).reshape(L, 1, D), n + "self_attn.k_norm.weight"))[:, 0])
        v = held(h @ w(n + "self_attn.v_proj.weight").t())
        seen = p <= p[:, None]
        if not every:
            seen = seen & ((p > p[:, None] - window) | (p < sinks))
        s = torch.where(seen, (q.transpose(0, 1) @ k.t()) / math.sqrt(D), -math.inf)
        o = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(L, H * D)
        x = x + rms(o @ w(n + "self_attn.o_proj.weight").t(), n + "post_attention_layernorm.weight")
        h = rms(x, n + "pre_feedforward_layernorm.weight")
        g = h @ w(n + "mlp.gate_proj.weight").t()
        g = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g**3))) * (h @ w(n + "mlp.up_proj.weight").t())
        x = x + rms(g @ w(n + "mlp.down_proj.weight").t(), n + "post_feedforward_layernorm.weight")
    return rms(x, "model.norm.weight")
