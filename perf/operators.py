"""The text encoder's operators over a key/value cache and on 4-bit weights, as timed cases.

Each case is a dict of plain values whose "kind" names the operator:

  linear     y = act(x W^T + bias) on 4-bit weights with group scales: W[n, k] = scale[n, k / group] (code[n, k] - 8)
  write      new tokens enter a cache: q and k heads RMS-normed and rotated to their positions, q written out, k and v
             stored at their positions as fp16 or as 4-bit codes with an fp16 step and offset per 32 values
  attention  grouped-query attention of queries at given positions over such a cache: key j is visible to position p if
             j <= p and (j < sinks or window == 0 or j > p - window)

Tokens of a batch are rows b * L + i; pos holds each row's position, -1 for the padding behind a shorter sequence, whose
outputs stay as they were. Cache rows behind a sequence's last position hold whatever was there before (here also
infinities and NaN). A 4-bit cache stands for the fp16 values half(offset + code * step).

Where `own` is false, run() computes the operators from elementary torch operations in 32 bits; where it is true, it
calls the framework. Widths are those of the text encoder (640, 4 heads of 256 on one key/value head, window 512) and of
the image model (1536, heads of 96), with generic ones of 64 and 128 beside them.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
GROUP = 32  # cache values per 4-bit step and offset


# ---- the cases ------------------------------------------------------------------------------

def listed():
    return [
        # one token's q|k|v projection in the text encoder: the smallest call, all latency
        _linear("linear_qkv_1", 1, 1536, 640, 32, "f32", False, "none"),
        # the logits of one token against the tied 262144-row embedding table
        _linear("linear_logits_1", 1, 262144, 640, 64, "f16", False, "none"),
        # an image model's MLP projection for a few conditioning rows
        _linear("linear_w12_5", 5, 8192, 1536, 128, "f32", True, "silu"),
        # a short prompt through the encoder's gate/up projection
        _linear("linear_gate_up_77", 77, 4096, 640, 32, "f16", False, "gelu_tanh"),
        # one token of one sequence enters an fp16 cache
        _write("write_step_f16", 1, 1, 4, 1, 256, 1024, 700, "f16", "f32", False),
        # a batch of prompts of unequal lengths enters a 4-bit cache
        _write("write_prompts_i4", 8, 300, 4, 1, 256, 2048, 0, "i4", "f32", True),
        # a long document at generic widths enters an fp16 cache
        _write("write_document_f16", 1, 8191, 16, 4, 128, 8192, 0, "f16", "f16", False),
        # the next token of one sequence in a window layer of the encoder: latency
        _attention("step_window_f16", 1, 1, 4, 1, 256, 1024, 700, 512, 4, "f16", "f32", False),
        # a batch of sequences of unequal lengths, next token, global layer, 4-bit cache
        _attention("step_batch_i4", 32, 1, 4, 1, 256, 16384, 16000, 0, 0, "i4", "f16", True),
        # a batch at generic widths, next token, all keys of an fp16 cache
        _attention("step_batch_f16", 16, 1, 16, 4, 128, 16384, 16383, 0, 0, "f16", "f16", False),
        # a long prompt through a window layer of the encoder, first tokens kept visible
        _attention("prompt_window_f16", 1, 4096, 4, 1, 256, 4096, 0, 512, 4, "f16", "f16", False),
        # prompts that continue cached ones, odd lengths, all keys of a 4-bit cache
        _attention("prompt_continued_i4", 2, 3001, 16, 4, 128, 8192, 1003, 0, 0, "i4", "f32", True),
    ]


def _linear(name, M, N, K, group, io, bias, act):
    return {"name": name, "kind": "linear", "M": M, "N": N, "K": K, "group": group, "io": io, "bias": bias, "act": act}


def _write(name, batch, L, H, KH, D, cap, start, kv, io, ragged):
    return {"name": name, "kind": "write", "batch": batch, "L": L, "H": H, "KH": KH, "D": D, "cap": cap, "start": start,
            "kv": kv, "io": io, "ragged": ragged}


def _attention(name, batch, L, H, KH, D, cap, start, window, sinks, kv, io, ragged):
    return {"name": name, "kind": "attention", "batch": batch, "L": L, "H": H, "KH": KH, "D": D, "cap": cap, "start": start,
            "window": window, "sinks": sinks, "kv": kv, "io": io, "ragged": ragged}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "write", "attention", "attention", "attention"])
    if kind == "linear":
        group = rng.choice([32, 64, 128])
        K = group * _log_int(rng, max(1, 128 // group), 6144 // group)
        c = _linear("", _log_int(rng, 1, 300), _log_int(rng, 64, 65536), K, group, rng.choice(["f32", "f16"]),
                    rng.random() < 0.5, rng.choice(["none", "silu", "gelu_tanh"]))
        if c["M"] * c["N"] > 1 << 23:
            c["N"] = max(64, (1 << 23) // c["M"])
    else:
        H, KH, D = rng.choice([(4, 1, 256), (16, 16, 96), (16, 4, 128), (8, 2, 64), (6, 2, 128), (5, 1, 64)])
        kv, io, ragged = rng.choice(["f16", "i4"]), rng.choice(["f32", "f16"]), rng.random() < 0.5
        if kind == "write":
            cap = _log_int(rng, 64, 8192)
            L = _log_int(rng, 1, cap)
            batch = _log_int(rng, 1, max(1, min(32, 16384 // L)))
            c = _write("", batch, L, H, KH, D, cap, rng.randint(0, cap - L), kv, io, ragged)
        else:
            cap = _log_int(rng, 64, 16384)
            L = 1 if rng.random() < 0.4 else _log_int(rng, 2, min(cap, 2000))
            batch = _log_int(rng, 1, max(1, min(24, 2000 // L, (1 << 26) // (cap * KH * D))))
            c = _attention("", batch, L, H, KH, D, cap, rng.randint(0, cap - L), rng.choice([0, _log_int(rng, 1, 2048)]),
                           rng.choice([0, rng.randint(1, 40)]), kv, io, ragged)
    del c["name"]
    return c


def _spans(c):
    """(first position, tokens) of each sequence, by the case alone."""
    rng = random.Random("%d %d %d %d" % (c["batch"], c["L"], c["cap"], c["start"]))
    spans = []
    for b in range(c["batch"]):
        full = not c["ragged"] or b == 0
        s = c["start"] if full else int(c["start"] * (0.3 + 0.7 * rng.random()))
        n = c["L"] if full else max(1, int(c["L"] * (0.3 + 0.7 * rng.random())))
        spans.append((s, n))
    return spans


# ---- what a pass has to move and compute ------------------------------------------------------

def work(case):
    c = case
    io = 4 if c["io"] == "f32" else 2
    if c["kind"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": N * K // 2 + N * K // c["group"] * 2 + M * K * io + M * N * 4 + (N * 4 if c["bias"] else 0),
                "flops": 2 * M * N * K}
    H, KH, D = c["H"], c["KH"], c["D"]
    per = 2.0 if c["kv"] == "f16" else 0.5 + 4.0 / GROUP  # bytes of a cached value
    tokens = sum(n for _, n in _spans(c))
    if c["kind"] == "write":
        return {"bytes": int(tokens * ((H + 2 * KH) * D * 4 + H * D * io + 2 * KH * D * per + D * 4)),
                "flops": tokens * (H + KH) * D * 8}
    w, sinks, keys, pairs = c["window"], c["sinks"], 0, 0
    for s, n in _spans(c):
        last = s + n - 1
        lo = 0 if w == 0 else max(0, s - w + 1)
        keys += last + 1 - lo + min(sinks, lo)
        for p in range(s, s + n):
            lo = 0 if w == 0 else max(0, p - w + 1)
            pairs += p + 1 - lo + min(sinks, lo)
    return {"bytes": int(keys * KH * D * 2 * per + tokens * H * D * io * 2), "flops": 4 * pairs * H * D}


# ---- inputs ---------------------------------------------------------------------------------

def _io(c):
    return torch.float32 if c["io"] == "f32" else torch.float16


def _positions(c):
    pos = torch.full((c["batch"], c["L"]), -1, dtype=torch.int32)
    for b, (s, n) in enumerate(_spans(c)):
        pos[b, :n] = torch.arange(s, s + n, dtype=torch.int32)
    return pos.to(DEV)


def _quantized(x):
    """fp32 values [..., D] -> 4-bit codes [..., D / 2] and fp16 (step, offset) [..., D / 32, 2]."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    step, lo = ((hi - lo) / 15).half(), lo.half()
    s, o = step.float().unsqueeze(-1), lo.float().unsqueeze(-1)
    q = torch.where(s > 0, ((g - o) / s).round().clamp(0, 15), torch.zeros_like(g)).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([step, lo], -1)


def _nibbles(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, groups):
    """What 4-bit codes [..., D / 2] and groups [..., D / 32, 2] stand for, as fp16 values in 32 bits."""
    q = _nibbles(codes).float().unflatten(-1, (-1, GROUP))
    return (q * groups[..., 0].float().unsqueeze(-1) + groups[..., 1].float().unsqueeze(-1)).flatten(-2).half().float()


def _rope(cap, D):
    """cos [cap][D / 2], then sin, of position times 1 / 10000^(2 i / D)."""
    a = torch.arange(cap, dtype=torch.float64).reshape(-1, 1) / 1e4 ** (torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    return torch.cat([a.cos().reshape(-1), a.sin().reshape(-1)]).float().to(DEV)


def _prepare_linear(c, normal):
    M, N, K = c["M"], c["N"], c["K"]
    x = normal(M, K)
    x[:, normal(K) > 2.5] *= 8  # activations have a few strong columns
    # weights as a quantizer leaves them: normal values, their group's largest magnitude on code 1 or 15
    w = normal(N, K // c["group"], c["group"])
    big = w.abs().amax(-1, keepdim=True)
    q = ((w / big * 7).round() + 8).to(torch.uint8).reshape(N, K)
    return {"x": x.to(_io(c)), "codes": q[:, 0::2] | (q[:, 1::2] << 4), "scale": (big.squeeze(-1) / 7 / math.sqrt(K)).half(),
            "bias": normal(N) * 0.1 if c["bias"] else None, "y": torch.empty(M, N, device=DEV)}


def _prepare_write(c, normal):
    B, L, H, KH, D, cap = (c[n] for n in ("batch", "L", "H", "KH", "D", "cap"))
    s = {"x": normal(B * L, (H + 2 * KH) * D) * 3, "wq": 1 + 0.1 * normal(D), "wk": 1 + 0.1 * normal(D), "cs": _rope(cap, D),
         "pos": _positions(c), "q": torch.zeros(B * L, H * D, dtype=_io(c), device=DEV)}
    rows = torch.arange(B, device=DEV).repeat_interleave(L) * cap + s["pos"].flatten()
    s["new"] = (s["pos"].flatten() >= 0).nonzero().flatten()  # the token rows that are no padding,
    s["at"] = rows[s["new"]]  # and their cache rows
    if c["kv"] == "f16":
        s["k"], s["v"] = (torch.zeros(B, cap, KH, D, dtype=torch.float16, device=DEV) for _ in "kv")
    else:
        s["k"], s["v"] = (torch.zeros(B, cap, KH, D // 2, dtype=torch.uint8, device=DEV) for _ in "kv")
        s["kg"], s["vg"] = (torch.zeros(B, cap, KH, D // GROUP, 2, dtype=torch.float16, device=DEV) for _ in "kv")
    return s


def _prepare_attention(c, normal):
    B, L, H, KH, D, cap = (c[n] for n in ("batch", "L", "H", "KH", "D", "cap"))
    s = {"pos": _positions(c), "q": normal(B * L, H * D).to(_io(c)), "o": torch.zeros(B * L, H * D, dtype=_io(c), device=DEV)}
    for name in "kv":
        if c["kv"] == "f16":
            s[name] = torch.cat([normal(cap, KH, D).half() for _ in range(B)]).reshape(B, cap, KH, D)
        else:
            parts = [_quantized(normal(cap, KH, D)) for _ in range(B)]
            s[name], s[name + "g"] = (torch.stack(p) for p in zip(*parts))
        # rows behind the last token: whatever an earlier sequence, or nobody, left there
        for b, (p, n) in enumerate(_spans(c)):
            tail = s[name if c["kv"] == "f16" else name + "g"][b, p + n:]
            tail[0::3], tail[1::3] = math.inf, math.nan
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = _PREPARE[case["kind"]](case, lambda *shape: torch.randn(*shape, generator=g, device=DEV))
    state["case"] = case
    return state


# ---- the plain forms ----------------------------------------------------------------------------

def _activated(y, act):
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(s):
    c = s["case"]
    w = (_nibbles(s["codes"]).float() - 8).unflatten(-1, (-1, c["group"])) * s["scale"].float().unsqueeze(-1)
    y = s["x"].float() @ w.flatten(-2).t()
    return _activated(y if s["bias"] is None else y + s["bias"], c["act"])


def _normed(x, w, cos, sin):
    """Per-head RMS norm of x [rows, heads, D], then the split-half rotation by cos, sin [rows, 1, D / 2]."""
    x = x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    c = s["case"]
    H, KH, D = c["H"], c["KH"], c["D"]
    new, at = s["new"], s["at"]
    cos, sin = (t.reshape(-1, 1, D // 2)[at % c["cap"]] for t in s["cs"].chunk(2))
    q, k, v = s["x"][new].unflatten(-1, (-1, D)).split([H, KH, KH], 1)
    s["q"][new] = _normed(q, s["wq"], cos, sin).flatten(1).to(s["q"].dtype)
    for name, t in (("k", _normed(k, s["wk"], cos, sin)), ("v", v)):
        if c["kv"] == "f16":
            s[name].flatten(0, 1)[at] = t.half()
        else:
            codes, groups = _quantized(t)
            s[name].flatten(0, 1)[at] = codes
            s[name + "g"].flatten(0, 1)[at] = groups
    return _written(s)


def _written(s):
    """The queries and the cache: all of an fp16 one, of a 4-bit one the values that the new rows stand for."""
    if s["case"]["kv"] == "f16":
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    out = {"q": s["q"]}
    for name in "kv":
        out[name] = _values(s[name].flatten(0, 1)[s["at"]], s[name + "g"].flatten(0, 1)[s["at"]]).half()
    return out


def _plain_attention(s):
    c = s["case"]
    B, L, H, KH, D, w = (c[n] for n in ("batch", "L", "H", "KH", "D", "window"))
    pos = s["pos"].long()
    used = max(p + n for p, n in _spans(c))
    j = torch.arange(used, device=DEV)
    held = (j <= pos.amax(1, keepdim=True))[:, :, None, None]
    k, v = (s[n][:, :used].float() if c["kv"] == "f16" else _values(s[n][:, :used], s[n + "g"][:, :used]) for n in "kv")
    k, v = (torch.where(held, t, 0.0).permute(0, 2, 1, 3) for t in (k, v))
    q = s["q"].float().reshape(B, L, KH, H // KH, D).permute(0, 2, 3, 1, 4).reshape(B, KH, -1, D)
    seen = j <= pos[..., None]
    if w:
        seen &= (j > pos[..., None] - w) | (j < c["sinks"])
    score = ((q / math.sqrt(D)) @ k.transpose(2, 3).contiguous()).reshape(B, KH, H // KH, L, used)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = e.sum(-1, keepdim=True)
    o = (e.reshape(B, KH, -1, used) @ v.contiguous()).reshape(B, KH, H // KH, L, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B * L, H * D).to(s["o"].dtype)
    return torch.where(pos.reshape(-1, 1) >= 0, o, s["o"])


# ---- the framework's calls ------------------------------------------------------------------------

def _lib():
    pkg = os.path.join(os.getcwd(), "nanosaur2-web_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ns2

    lib = ns2.load(0)
    lib.set_stream(torch.cuda.current_stream().cuda_stream)
    return lib


def _own_linear(s):
    c, lib = s["case"], _lib()
    lib.linear_i4(s["x"], int(c["io"] == "f16"), c["K"], s["codes"], s["scale"], s["y"], c["M"], c["N"], c["K"], c["group"],
                  bias=s["bias"], act=c["act"])
    return s["y"]


def _cache_view(c):
    return dict(batch=c["batch"], L=c["L"], H=c["H"], KH=c["KH"], D=c["D"], cap=c["cap"], ldkv=c["KH"] * c["D"],
                kvBatch=c["cap"] * c["KH"] * c["D"], ldq=c["H"] * c["D"], q_fmt=int(c["io"] == "f16"))


def _own_write(s):
    c, lib = s["case"], _lib()
    lib.head_norm_cache(s["x"], s["pos"], s["q"], s["k"], s["v"], ldx=(c["H"] + 2 * c["KH"]) * c["D"], w_q=s["wq"], w_k=s["wk"],
                        cs=s["cs"], sin_off=c["cap"] * c["D"] // 2, rope_rows=c["cap"], eps=EPS, k_groups=s.get("kg"),
                        v_groups=s.get("vg"), **_cache_view(c))
    return _written(s)


def _own_attention(s):
    c, lib = s["case"], _lib()
    if "work" not in s:
        need = lib.attention_cache_bytes(c["batch"], c["L"], c["H"], c["KH"], c["D"], c["cap"], c["window"], c["sinks"])
        s["work"] = torch.empty(need, dtype=torch.uint8, device=DEV) if need else None
    lib.attention_cache(s["q"], s["pos"], s["k"], s["v"], s["o"], ldo=c["H"] * c["D"], window=c["window"], sinks=c["sinks"],
                        k_groups=s.get("kg"), v_groups=s.get("vg"), work=s["work"], **_cache_view(c))
    return s["o"]


_PREPARE = {"linear": _prepare_linear, "write": _prepare_write, "attention": _prepare_attention}
_PLAIN = {"linear": _plain_linear, "write": _plain_write, "attention": _plain_attention}
_OWN = {"linear": _own_linear, "write": _own_write, "attention": _own_attention}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---- 64 bits, from the definitions ------------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"linear": _exact_linear, "write": _exact_write, "attention": _exact_attention}[c["kind"]](c, s)


def _exact_values(codes, groups):
    d = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=DEV)
    d[..., 0::2], d[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    at = torch.arange(d.shape[-1], device=DEV) // GROUP
    return (groups[..., at, 1].double() + d * groups[..., at, 0].double()).half().double()


def _exact_linear(c, s):
    y = torch.empty(c["M"], c["N"], dtype=torch.float64, device=DEV)
    x = s["x"].double()
    at = torch.arange(c["K"], device=DEV) // c["group"]
    for n in range(0, c["N"], 4096):
        codes = s["codes"][n:n + 4096]
        w = torch.empty(codes.shape[0], c["K"], dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
        y[:, n:n + 4096] = x @ (w * s["scale"][n:n + 4096].double()[:, at]).t()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if c["act"] == "silu":
        return y * torch.sigmoid(y)
    if c["act"] == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y**3))
    return y


def _exact_write(c, s):
    H, KH, D = c["H"], c["KH"], c["D"]
    pos = s["pos"].flatten()[s["new"]].long()
    x = s["x"].double()[s["new"]].reshape(-1, H + 2 * KH, D)
    turn = torch.complex(*(t.reshape(-1, D // 2)[pos].double() for t in s["cs"].chunk(2)))[:, None]

    def turned(t, w):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(t[..., : D // 2], t[..., D // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    q = s["q"].double()
    q[s["new"]] = turned(x[:, :H], s["wq"]).reshape(-1, H * D)
    out = {"q": q}
    for name, t in (("k", turned(x[:, H:H + KH], s["wk"])), ("v", x[:, H + KH:])):
        if c["kv"] == "f16":
            out[name] = s[name].double()
            out[name].reshape(-1, KH, D)[s["at"]] = t
        else:
            g = t.reshape(*t.shape[:-1], -1, GROUP)
            lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            step, lo = ((hi - lo) / 15).half().double(), lo.half().double()
            out[name] = (lo + ((g - lo) / step).round().clamp(0, 15) * step).reshape(t.shape).half().double()
    return out


def _exact_attention(c, s):
    B, L, H, KH, D, w = (c[n] for n in ("batch", "L", "H", "KH", "D", "window"))
    o = s["o"].double().reshape(B, L, H, D)
    q = s["q"].double().reshape(B, L, H, D)
    for b, (p0, n) in enumerate(_spans(c)):
        used = p0 + n
        j = torch.arange(used, device=DEV)
        p = torch.arange(p0, used, device=DEV)[:, None]
        seen = (j <= p) & ((j > p - w) | (j < c["sinks"]) if w else j >= 0)
        for g in range(KH):
            k, v = (s[m][b, :used, g].double() if c["kv"] == "f16" else _exact_values(s[m][b, :used, g], s[m + "g"][b, :used, g])
                    for m in "kv")
            for h in range(g * (H // KH), (g + 1) * (H // KH)):
                score = q[b, :n, h] @ k.t() / math.sqrt(D)
                o[b, :n, h] = torch.softmax(torch.where(seen, score, -math.inf), -1) @ v
    return o.reshape(B * L, H * D)
