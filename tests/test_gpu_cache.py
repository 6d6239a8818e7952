"""Tokens entering a key/value cache and attention over it (ns2_head_norm_cache, ns2_attention_cache) against their
definitions in 64 bits: head layouts, fp16 and 4-bit caches, fp32 and fp16 queries, windows, sinks, lengths from one
token on, padding rows, stale cache rows, strides, refusals, graphs and streams."""

import math

import pytest
import torch

import cache_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


def gen(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device=DEV)


def positions(spans, L):
    pos = torch.full((len(spans), L), -1, dtype=torch.int32)
    for b, (s, n) in enumerate(spans):
        pos[b, :n] = torch.arange(s, s + n, dtype=torch.int32)
    return pos.to(DEV)


# ---- attention ----------------------------------------------------------------------------------

class Cache:
    """A cache of `batch` sequences with its own strides; values as float64, stale rows poisoned."""

    def __init__(self, rnd, batch, cap, KH, D, i4, pad_row=0, pad_seq=0):
        self.batch, self.cap, self.KH, self.D, self.i4 = batch, cap, KH, D, i4
        self.ldkv, self.kvBatch = KH * D + pad_row, cap * (KH * D + pad_row) + pad_seq
        size = batch * self.kvBatch
        self.raw, self.groups, self.value = {}, {"k": None, "v": None}, {}
        for name in "kv":
            x = rnd(batch, cap, KH, D)
            if i4:
                self.raw[name] = torch.zeros(size // 2, dtype=torch.uint8, device=DEV)
                self.groups[name] = torch.zeros(size // 32, 2, dtype=torch.float16, device=DEV)
                codes, groups = R.cache_codes(x)
                self.view(self.raw[name], 2).copy_(codes)
                self.group_view(name).copy_(groups)
                self.value[name] = R.cache_values(codes, groups)
            else:
                self.raw[name] = torch.zeros(size, dtype=torch.float16, device=DEV)
                self.view(self.raw[name], 1).copy_(x.half())
                self.value[name] = x.half().double()

    def view(self, t, per):
        return torch.as_strided(t, (self.batch, self.cap, self.KH, self.D // per),
                                (self.kvBatch // per, self.ldkv // per, self.D // per, 1))

    def group_view(self, name):
        return torch.as_strided(self.groups[name], (self.batch, self.cap, self.KH, self.D // 32, 2),
                                (self.kvBatch // 16, self.ldkv // 16, self.D // 16, 2, 1))

    def poison(self, b, rows):
        """What an earlier sequence may have left in rows nobody sees."""
        for name in "kv":
            t = self.group_view(name)[b, rows] if self.i4 else self.view(self.raw[name], 1)[b, rows]
            t[0::3], t[1::3], t[2::3] = math.inf, math.nan, -65504.0

    def args(self):
        return dict(cap=self.cap, ldkv=self.ldkv, kvBatch=self.kvBatch, KH=self.KH, D=self.D, batch=self.batch,
                    k_groups=self.groups["k"], v_groups=self.groups["v"])


def attend(lib, cache, q, pos, window, sinks, fp16, pad=0, scale=None, o=None):
    """q [B, L, H, D] float; returns o [B, L, H, D] (rows of padding keep 7)."""
    B, L, H, D = q.shape
    ld = H * D + pad
    dt = torch.float16 if fp16 else torch.float32
    qb = torch.full((B * L, ld), 3.0, dtype=dt, device=DEV)
    qb[:, : H * D] = q.reshape(B * L, H * D).to(dt)
    ob = torch.full((B * L + 2, ld), 7.0, dtype=dt, device=DEV)
    need = lib.attention_cache_bytes(B, L, H, cache.KH, D, cache.cap, window, sinks)
    work = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    a = cache.args()
    a["batch"] = B
    lib.attention_cache(qb, pos, cache.raw["k"], cache.raw["v"], ob, L=L, H=H, ldq=ld, ldo=ld, window=window, sinks=sinks,
                        scale=scale, q_fmt=int(fp16), work=work[:need] if need else None, **a)
    torch.cuda.synchronize()
    assert (work[need:] == 255).all(), "bytes behind the work memory were written"
    assert (ob[:, H * D:] == 7).all() and (ob[B * L:] == 7).all(), "values outside the rows were written"
    return ob[: B * L, : H * D].reshape(B, L, H, D)


def check(got, q, pos, cache, window, sinks, fp16, what, scale=None):
    D = q.shape[-1]
    qd = (q.half() if fp16 else q.float()).double()
    ref, vmax, smax, n = R.attention(qd, pos, cache.value["k"], cache.value["v"], window, sinks, scale or 1 / math.sqrt(D))
    live = (pos >= 0) & (pos < cache.cap)
    bound = R.attention_bound(ref, vmax, smax, n, D, fp16)[live]
    assert (got[~live] == 7).all(), f"{what}: padding rows were written"
    err = (got[live].double() - ref[live]).abs()
    print(f"[parity] {what}: largest error / bound {(err / bound).max().item():.3f}", flush=True)
    assert torch.isfinite(got[live]).all() and (err <= bound).all(), what


HEADS = [(4, 1, 256), (16, 16, 96), (8, 2, 128), (6, 2, 64), (5, 1, 64), (3, 1, 128), (20, 1, 96), (1, 1, 256), (40, 2, 64)]


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("H,KH,D", HEADS)
def test_single_tokens(ns2lib, H, KH, D, i4, fp16):
    """One token per sequence: the first token of all, ends of tiles, a full cache, a padding row, one past the cache."""
    pos = torch.tensor([[0], [1], [15], [31], [32], [63], [64], [199], [-1], [200], [130]], dtype=torch.int32, device=DEV)
    rnd = gen(H * D)
    for window, sinks in ((0, 0), (1, 0), (1, 2), (33, 4), (64, 0), (150, 70), (500, 500)):
        cache = Cache(rnd, len(pos), 200, KH, D, i4)
        for b in range(len(pos)):
            p = int(pos[b])
            cache.poison(b, slice(max(0, p + 1), None))
            if window and p - window + 1 > sinks:
                cache.poison(b, slice(sinks, p - window + 1))
        q = rnd(len(pos), 1, H, D)
        check(attend(ns2lib, cache, q, pos, window, sinks, fp16), q, pos, cache, window, sinks, fp16,
              f"step {H}/{KH}x{D} i4={i4} fp16={fp16} window {window} sinks {sinks}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("H,KH,D", HEADS)
@pytest.mark.parametrize("L,start", [(2, 0), (17, 3), (70, 0), (129, 61)])
def test_prompts(ns2lib, H, KH, D, i4, fp16, L, start):
    """Several tokens at once, unequal lengths with padding rows, keys before them in the cache."""
    spans = [(start, L), (start // 2, max(1, L // 3)), (start, L - 1)]
    pos = positions(spans, L)
    rnd = gen(L + H * D)
    for window, sinks in ((0, 0), (7, 2), (64, 1), (40, 100)):
        cache = Cache(rnd, 3, 200, KH, D, i4)
        for b, (s, n) in enumerate(spans):
            cache.poison(b, slice(s + n, None))
            if window and s - window + 1 > sinks:
                cache.poison(b, slice(sinks, s - window + 1))
        q = rnd(3, L, H, D)
        check(attend(ns2lib, cache, q, pos, window, sinks, fp16), q, pos, cache, window, sinks, fp16,
              f"prompt {L} from {start} {H}/{KH}x{D} i4={i4} fp16={fp16} window {window} sinks {sinks}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_later_tokens_do_not_reach_earlier_ones(ns2lib, D, i4, fp16):
    """Infinities and NaN in one token's key and value: rows before it, and rows whose window has passed it, are
    those of a cache without them, in the same call."""
    L, bad, window = 150, 70, 30
    pos = positions([(0, L)], L)
    rnd = gen(D)
    cache = Cache(rnd, 1, 160, 2, D, i4)
    q = rnd(1, L, 8, D)
    clean = attend(ns2lib, cache, q, pos, window, 2, fp16)
    cache.poison(0, slice(bad, bad + 2))
    got = attend(ns2lib, cache, q, pos, window, 2, fp16)
    far = torch.ones(L, dtype=torch.bool, device=DEV)
    far[bad: bad + 1 + window] = False
    check(torch.where(far[None, :, None, None], got, clean), q, pos, cache, window, 2, fp16, f"D={D} i4={i4} fp16={fp16}")
    assert not torch.isfinite(got[0, bad: bad + window]).any(-1).any(), "a visible NaN was lost"


def attend64(q, pos, cache, window, sinks):
    """R.attention over whole batches; what nobody sees has no part in cache.value."""
    B, L, H, D = q.shape
    p, j = pos.long()[:, :, None], torch.arange(cache.cap, device=DEV)
    seen = (j <= p) & (p < cache.cap)
    if window:
        seen = seen & ((j < sinks) | (j > p - window))
    k, v = (cache.value[n].permute(0, 2, 1, 3) for n in "kv")  # [B, KH, cap, D]
    qg = q.reshape(B, L, cache.KH, H // cache.KH, D).permute(0, 2, 3, 1, 4)
    m = seen[:, None, None]

    def back(t):
        return t.permute(0, 3, 1, 2, 4).reshape(B, L, H, -1)

    s = torch.where(m, qg @ k[:, :, None].transpose(-1, -2).contiguous() / math.sqrt(D), -math.inf)
    size = torch.where(m, qg.abs() @ k[:, :, None].abs().transpose(-1, -2).contiguous() / math.sqrt(D), 0.0).amax(-1, keepdim=True)
    o = torch.softmax(s, -1) @ v[:, :, None]
    vmax = v.abs().amax((2, 3))[:, :, None, None, None].expand_as(size)
    return back(o), back(vmax), back(size), seen.sum(-1)[:, :, None, None].double()


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("B,L,H,KH,D", [(8, 140, 16, 16, 96), (16, 300, 8, 2, 64), (20, 270, 6, 2, 128), (43, 70, 4, 1, 256), (24, 150, 16, 8, 96)])
def test_batches_of_prompts(ns2lib, B, L, H, KH, D, i4, fp16):
    """Enough columns for every block size; sequences of unequal lengths, some without a token, rows nobody sees poisoned."""
    cap = L + 90
    spans = [((37 * b) % 90, (L, L - 1, 0, 1, 64, L // 2)[b % 6]) for b in range(B)]
    pos = positions(spans, L)
    rnd = gen(B + D)
    q = rnd(B, L, H, D)
    qd = (q.half() if fp16 else q).double()
    for window, sinks in ((0, 0), (70, 3)):
        cache = Cache(rnd, B, cap, KH, D, i4)
        for b, (s, n) in enumerate(spans):
            cache.poison(b, slice(s + n, None))
            if window and s - window + 1 > sinks:
                cache.poison(b, slice(sinks, s - window + 1))
        got = attend(ns2lib, cache, q, pos, window, sinks, fp16)
        ref, vmax, smax, n = attend64(qd, pos, cache, window, sinks)
        live = (pos >= 0) & (pos < cap)
        assert (got[~live] == 7).all(), "padding rows were written"
        bound = R.attention_bound(ref, vmax, smax, n, D, fp16)[live]
        err = (got[live].double() - ref[live]).abs()
        print(f"[parity] {B}x{L} {H}/{KH}x{D} i4={i4} fp16={fp16}: largest error / bound {(err / bound).max().item():.3f}", flush=True)
        assert torch.isfinite(got[live]).all() and (err <= bound).all()
        # what enters at the token of row 50 shows in the rows that see it, and in no others
        for b, (s, n) in enumerate(spans):
            if n > 50:
                cache.poison(b, slice(s + 50, s + 53))
        bad = attend(ns2lib, cache, q, pos, window, sinks, fp16)
        row = torch.arange(L, device=DEV)
        far = row < 50
        if window:
            far = far | (row >= 52 + window)
        assert torch.equal(bad[:, far], got[:, far])
        hit = live & (row >= 52) & ((row < 51 + window) if window else True)  # (of rows 50 to 52, the third is finite)
        assert not torch.isfinite(bad[hit]).any()


@pytest.mark.parametrize("L", [3, 80])
@pytest.mark.parametrize("D", [64, 256])
def test_queries_of_any_magnitude(ns2lib, D, L):
    """fp32 queries far below and beyond fp16's range, each head with its own; the scale takes the large ones back."""
    rnd = gen(D + L)
    pos = positions([(60, L), (0, L)], L)
    cache = Cache(rnd, 2, 160, 2, D, False)
    q = rnd(2, L, 4, D)
    for h, f in ((0, 1e-20), (1, 1e-3), (2, 1.0), (3, 1e4)):
        q[:, :, h] *= f
    for scale, f in ((1 / math.sqrt(D), 1.0), (1e-25, 1e24), (1e20, 1e-21)):
        check(attend(ns2lib, cache, q * f, pos, 0, 0, False, scale=scale), q * f, pos, cache, 0, 0, False, f"D={D} x {f}", scale=scale)


@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("L", [1, 40])
def test_any_positions(ns2lib, L, i4):
    """Rows in any order, some at the same position, some of them padding."""
    g = torch.Generator().manual_seed(L)
    pos = torch.randint(-40, 330, (2, L), generator=g, dtype=torch.int32).to(DEV)
    rnd = gen(L)
    cache = Cache(rnd, 2, 300, 2, 64, i4)
    q = rnd(2, L, 4, 64)
    for window, sinks in ((0, 0), (50, 3)):
        check(attend(ns2lib, cache, q, pos, window, sinks, False), q, pos, cache, window, sinks, False, f"any {L} i4={i4}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("L", [1, 35])
def test_strides(ns2lib, L, i4, fp16):
    """Rows of q and o wider than the heads, gaps between cache rows and between sequences."""
    pos = positions([(90, L), (3, L)], L)
    rnd = gen(11)
    cache = Cache(rnd, 2, 140, 2, 96, i4, pad_row=32, pad_seq=64)
    q = rnd(2, L, 6, 96)
    check(attend(ns2lib, cache, q, pos, 60, 4, fp16, pad=8), q, pos, cache, 60, 4, fp16, f"strides {L} i4={i4} fp16={fp16}")


@pytest.mark.parametrize("L", [1, 33])
def test_one_cache_for_all(ns2lib, L):
    """kvBatch = 0: every sequence reads the same cached rows."""
    rnd = gen(12)
    cache = Cache(rnd, 1, 140, 1, 128, False)
    pos = positions([(100, L), (20, L), (0, L)], L)
    q = rnd(3, L, 4, 128)
    cache.kvBatch = 0
    got = attend(ns2lib, cache, q, pos, 0, 0, False)
    for name in "kv":
        cache.value[name] = cache.value[name].expand(3, -1, -1, -1)
    check(got, q, pos, cache, 0, 0, False, f"shared {L}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
def test_long_caches(ns2lib, i4, fp16):
    """Thousands of keys for one token and for a few."""
    for L, B, (H, KH, D) in ((1, 3, (4, 1, 256)), (5, 2, (8, 2, 128)), (1, 1, (16, 16, 96)), (66, 1, (2, 1, 64))):
        rnd = gen(D)
        cap = 6000
        spans = [(cap - L - 211 * b, L) for b in range(B)]
        pos = positions(spans, L)
        cache = Cache(rnd, B, cap, KH, D, i4)
        q = rnd(B, L, H, D)
        for window, sinks in ((0, 0), (3333, 100)):
            check(attend(ns2lib, cache, q, pos, window, sinks, fp16), q, pos, cache, window, sinks, fp16,
                  f"long {L} {H}/{KH}x{D} i4={i4} fp16={fp16} window {window}")


@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("L", [1, 20])
def test_offsets_past_32_bits(ns2lib, L, i4):
    """Cache rows more than 2^32 values into the buffer."""
    rnd = gen(13)
    ld, cap, D = 1 << 23, 600, 64
    small = Cache(rnd, 1, cap, 1, D, i4)
    big = Cache.__new__(Cache)
    big.__dict__.update(small.__dict__)
    big.ldkv, big.kvBatch, size = ld, cap * ld, (cap - 1) * ld + D
    big.raw, big.groups = {}, {"k": None, "v": None}
    for name in "kv":
        big.raw[name] = torch.empty(size // 2 if i4 else size, dtype=torch.uint8 if i4 else torch.float16, device=DEV)
        big.view(big.raw[name], 2 if i4 else 1).copy_(small.view(small.raw[name], 2 if i4 else 1))
        if i4:
            big.groups[name] = torch.empty(size // 32, 2, dtype=torch.float16, device=DEV)
            big.group_view(name).copy_(small.group_view(name))
    pos = positions([(cap - L, L)], L)
    q = rnd(1, L, 4, D)
    check(attend(ns2lib, big, q, pos, 0, 0, True), q, pos, big, 0, 0, True, f"far offsets {L} i4={i4}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("L", [1, 90])
def test_large_scores(ns2lib, L, fp16):
    """Scores of hundreds, rising and falling along the keys, and scores that are all -inf or equal."""
    rnd = gen(14)
    D, cap = 128, 400
    cache = Cache(rnd, 2, cap, 1, D, False)
    ramp = torch.linspace(-1, 1, cap, device=DEV)
    k = torch.zeros(2, cap, 1, D, device=DEV)
    k[0, :, 0, 0], k[1, :, 0, 0] = ramp, -ramp
    cache.view(cache.raw["k"], 1).copy_(k.half())
    cache.value["k"] = k.half().double()
    q = torch.zeros(2, L, 2, D, device=DEV)
    q[..., 0, 0], q[..., 1, 0] = 4096.0, 0.0
    pos = positions([(cap - L, L)] * 2, L)
    check(attend(ns2lib, cache, q, pos, 0, 0, fp16), q, pos, cache, 0, 0, fp16, f"large scores {L} fp16={fp16}")


def test_other_scale_and_repeated_calls(ns2lib):
    """A scale of one's own; the same call twice gives the same bits (long split sums included)."""
    rnd = gen(15)
    cache = Cache(rnd, 2, 3000, 2, 64, True)
    for L in (1, 100):
        pos = positions([(2800, L), (1500, L)], L)
        q = rnd(2, L, 8, 64)
        a = attend(ns2lib, cache, q, pos, 0, 0, False, scale=0.03)
        check(a, q, pos, cache, 0, 0, False, f"scale {L}", scale=0.03)
        assert torch.equal(a, attend(ns2lib, cache, q, pos, 0, 0, False, scale=0.03))


# ---- new tokens into a cache -----------------------------------------------------------------------

def write(lib, x, pos, H, KH, D, cap, *, i4, fp16, wq, wk, cs, rope_rows, fill, pad=0):
    """Returns q rows, and k, v, their groups as [B, cap, KH, ...] buffers that held `fill` before."""
    B, L = pos.shape
    ld = KH * D + pad
    size = B * cap * ld
    q = torch.full((B * L, H * D + 8), 7.0, dtype=torch.float16 if fp16 else torch.float32, device=DEV)
    out = {"q": q}
    for n in "kv":
        if i4:
            out[n] = torch.full((size // 2,), int(fill), dtype=torch.uint8, device=DEV)
            out[n + "g"] = torch.full((size // 32, 2), float(fill), dtype=torch.float16, device=DEV)
        else:
            out[n] = torch.full((size,), float(fill), dtype=torch.float16, device=DEV)
    lib.head_norm_cache(x, pos, q, out["k"], out["v"], batch=B, L=L, H=H, KH=KH, D=D, ldx=x.shape[1], ldq=H * D + 8, cap=cap,
                        ldkv=ld, kvBatch=cap * ld, w_q=wq, w_k=wk, cs=cs, sin_off=cs.numel() // 2 if cs is not None else 0,
                        rope_rows=rope_rows, eps=EPS, q_fmt=int(fp16), k_groups=out.get("kg"), v_groups=out.get("vg"))
    torch.cuda.synchronize()
    for n in "kv":
        if i4:
            out[n] = out[n].reshape(B, cap, -1)[..., : KH * D // 2].reshape(B, cap, KH, D // 2)
            out[n + "g"] = out[n + "g"].reshape(B, cap, -1, 2)[:, :, : KH * D // 32].reshape(B, cap, KH, D // 32, 2)
        else:
            out[n] = out[n].reshape(B, cap, ld)[..., : KH * D].reshape(B, cap, KH, D)
    return out


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("H,KH,D", HEADS)
def test_write(ns2lib, H, KH, D, i4, fp16):
    """Norm, rotation at the position and storage. fp32 arithmetic is off by at most 2^-20 of the head's largest
    magnitude (a D-term sum of squares in a square root, a few products); fp16 storage by 2^-11 of the value, 4-bit
    storage by half a step, plus the roundings of the offset (2^-11 |o|) and of the step (2^-11 of 15 steps)."""
    rnd = gen(H + D)
    cap, L = 90, 37
    spans = [(0, L), (50, L - 5), (cap - 3, 3)]
    pos = positions(spans, L)
    pos[1, 3] = cap  # past the cache: padding
    x = rnd(3 * L, (H + 2 * KH) * D + 4) * 3
    wq, wk = 1 + 0.2 * rnd(D), 1 + 0.2 * rnd(D)
    for norms, rows in (((wq, wk), cap), ((wq, None), 60), ((None, wk), 0)):
        cs = R.rope_table(cap, D).to(DEV) if rows else None
        got = write(ns2lib, x, pos, H, KH, D, cap, i4=i4, fp16=fp16, wq=norms[0], wk=norms[1], cs=cs, rope_rows=rows, fill=9,
                    pad=32)
        flat = pos.flatten()
        live = (flat >= 0) & (flat < cap)
        heads = x[:, : (H + 2 * KH) * D].double().reshape(3 * L, H + 2 * KH, D)
        ref = {"q": R.head_norm(heads[:, :H], norms[0], cs, flat, rows, EPS),
               "k": R.head_norm(heads[:, H: H + KH], norms[1], cs, flat, rows, EPS), "v": heads[:, H + KH:]}
        q = got["q"]
        assert (q[:, H * D:] == 7).all() and (q[~live] == 7).all(), "padding of q was written"
        qv = q[live, : H * D].double().reshape(-1, H, D)
        qr = ref["q"][live]
        slack = qr.abs().amax(-1, keepdim=True) * 2.0**-20
        assert ((qv - qr).abs() <= slack + (2.0**-11 * qr.abs() if fp16 else 0)).all(), "q"
        b = torch.arange(3, device=DEV).repeat_interleave(L)[live]
        at = flat[live].long()
        for n in "kv":
            r = ref[n][live]
            slack = r.abs().amax(-1, keepdim=True) * 2.0**-20
            untouched = torch.ones(3, cap, dtype=torch.bool, device=DEV)
            untouched[b, at] = False
            assert (got[n][untouched] == 9).all(), f"other rows of {n} were written"
            if i4:
                assert (got[n + "g"][untouched] == 9).all(), f"other groups of {n} were written"
                groups = got[n + "g"][b, at]
                step, off = (groups[..., i].double().repeat_interleave(32, -1) for i in (0, 1))
                val = R.cache_values(got[n][b, at], groups)
                bound = step / 2 + 2.0**-11 * (off.abs() + 15 * step + val.abs()) + slack
                assert ((val - r).abs() <= bound).all(), n
                assert (step <= (r.unflatten(-1, (-1, 32)).amax(-1) - r.unflatten(-1, (-1, 32)).amin(-1)).repeat_interleave(32, -1) / 15
                        * (1 + 2.0**-10) + slack).all(), f"steps of {n}"
            else:
                assert ((got[n][b, at].double() - r).abs() <= 2.0**-11 * r.abs() + slack + 2.0**-24).all(), n


def test_four_bit_codes_exactly(ns2lib):
    """Values that are not normed: codes and groups equal the definition, also for equal values, zeros, tiny and
    huge ranges and values on a border between two codes."""
    rnd = gen(21)
    D, L = 128, 64
    x = rnd(L, 3 * D)
    v = x[:, 2 * D:]
    v[0] = 0.0
    v[1] = 1.2345
    v[2] = torch.arange(D, device=DEV) % 32 * 0.5
    v[3] *= 1e-7
    v[4] *= 1e4
    v[5, ::2] = -3.0
    v[6] = v[6].abs() + 100
    pos = positions([(0, L)], L)
    got = write(ns2lib, x, pos, 1, 1, D, L, i4=True, fp16=False, wq=None, wk=None, cs=None, rope_rows=0, fill=1)
    for n, r in (("k", x[:, D: 2 * D]), ("v", v)):
        codes, groups = R.cache_codes(r.cpu().reshape(L, 1, D))
        assert torch.equal(got[n + "g"][0].cpu(), groups), n
        assert torch.equal(got[n][0].cpu(), codes), n


@pytest.mark.parametrize("H,KH,D", HEADS)
def test_four_bit_keys_exactly(ns2lib, H, KH, D):
    """Normed and rotated keys, and values: codes and groups are those of 64-bit arithmetic. (Its own error is below
    2^-45 of a value; one of the 10^5 values here lies as near to a border with a chance below 10^-7.)"""
    rnd = gen(24 + D)
    L, cap = 150, 160
    pos = positions([(5, L), (0, L - 20)], L)
    x = rnd(2 * L, (H + 2 * KH) * D) * 3
    w, cs = 1 + 0.1 * rnd(D), R.rope_table(cap, D).to(DEV)
    got = write(ns2lib, x, pos, H, KH, D, cap, i4=True, fp16=False, wq=w, wk=w, cs=cs, rope_rows=cap, fill=0)
    flat = pos.flatten()
    live = flat >= 0
    heads = x.double().reshape(2 * L, H + 2 * KH, D)
    b, at = torch.arange(2, device=DEV).repeat_interleave(L)[live], flat[live].long()
    for n, r in (("k", R.head_norm(heads[:, H: H + KH], w, cs, flat, cap, EPS)), ("v", heads[:, H + KH:])):
        g = r[live].unflatten(-1, (-1, 32))
        lo, hi = g.amin(-1), g.amax(-1)
        step, off = ((hi - lo) / 15).float().half(), lo.float().half()
        q = ((g - off.double().unsqueeze(-1)) / step.double().unsqueeze(-1)).round().clamp(0, 15)
        assert torch.equal(got[n + "g"][b, at], torch.stack([step, off], -1)), n
        assert torch.equal(R.nibbles(got[n][b, at]).double(), q.flatten(-2)), n


@pytest.mark.parametrize("i4", [False, True])
def test_values_that_are_not_numbers(ns2lib, i4):
    """A NaN or an infinity stays visible in its own group (or value) and nowhere else."""
    rnd = gen(22)
    D, L = 96, 5
    x = rnd(L, 3 * D)
    x[1, 2 * D + 40], x[2, 2 * D + 3], x[3, 2 * D + 95] = math.nan, math.inf, -math.inf
    got = write(ns2lib, x, positions([(0, L)], L), 1, 1, D, L, i4=i4, fp16=False, wq=None, wk=None, cs=None, rope_rows=0, fill=0)
    val = (R.cache_values(got["v"], got["vg"]) if i4 else got["v"].double())[0, :, 0]
    bad = torch.zeros(L, D, dtype=torch.bool, device=DEV)
    if i4:
        bad[1, 32:64], bad[2, 0:32], bad[3, 64:96] = True, True, True
    else:
        bad[1, 40], bad[2, 3], bad[3, 95] = True, True, True
    assert torch.equal(~torch.isfinite(val), bad)


def test_queries_in_place(ns2lib):
    """q may be X itself."""
    rnd = gen(23)
    H, KH, D, L = 4, 1, 256, 9
    x = rnd(L, (H + 2 * KH) * D)
    w = 1 + 0.1 * rnd(D)
    cs = R.rope_table(L, D).to(DEV)
    k, v = (torch.zeros(L, D, dtype=torch.float16, device=DEV) for _ in "kv")
    q = torch.zeros(L, H * D, device=DEV)
    y = x.clone()
    for src, dst, ld in ((x, q, H * D), (y, y, x.shape[1])):
        ns2lib.head_norm_cache(src, positions([(0, L)], L), dst, k, v, batch=1, L=L, H=H, KH=KH, D=D, ldx=x.shape[1], ldq=ld, cap=L,
                               ldkv=D, kvBatch=L * D, w_q=w, w_k=w, cs=cs, sin_off=cs.numel() // 2, rope_rows=L)
    torch.cuda.synchronize()
    assert torch.equal(y[:, : H * D], q) and torch.equal(y[:, H * D:], x[:, H * D:])


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("H,KH,D", [(8, 2, 64), (4, 4, 96), (6, 2, 128), (4, 1, 256)])
def test_long_documents(ns2lib, H, KH, D, i4, fp16):
    """Thousands of tokens in one call (several heads per lane group) hold what calls of 1000 tokens write, bit for bit;
    queries in place too."""
    heads, per = H + 2 * KH, 256 // D
    L = 65536 * per // (2 * heads) + 77
    cap = L + 9
    rnd = gen(D)
    x = rnd(2 * L, heads * D)
    pos = positions([(9, L), (0, L - 50)], L)
    w, cs = 1 + 0.2 * rnd(D), R.rope_table(cap, D).to(DEV)
    a = dict(i4=i4, fp16=fp16, wq=w, wk=w, cs=cs, rope_rows=cap - 5, fill=1)
    got = write(ns2lib, x, pos, H, KH, D, cap, **a)
    seq = x.reshape(2, L, -1)
    want = None
    for i in range(0, L, 1000):
        part = write(ns2lib, seq[:, i: i + 1000].reshape(-1, heads * D).contiguous(), pos[:, i: i + 1000].contiguous(), H, KH, D, cap, **a)
        if want is None:
            want = {n: t.clone() for n, t in part.items() if n != "q"}
        n = min(1000, L - i)
        assert torch.equal(got["q"].reshape(2, L, -1)[:, i: i + n], part["q"].reshape(2, n, -1))
        for b in range(2):
            at = pos[b, i: i + n].long()
            at = at[at >= 0]
            for name in want:
                want[name][b, at] = part[name][b, at]
    for name in want:
        assert torch.equal(got[name], want[name]), name
    if not fp16:
        y, k, v = x.clone(), *(torch.zeros(2, cap, KH * D, dtype=torch.float16, device=DEV) for _ in "kv")
        ns2lib.head_norm_cache(y, pos, y, k, v, batch=2, L=L, H=H, KH=KH, D=D, ldx=heads * D, ldq=heads * D, cap=cap, ldkv=KH * D,
                               kvBatch=cap * KH * D, w_q=w, w_k=w, cs=cs, sin_off=cs.numel() // 2, rope_rows=cap - 5)
        torch.cuda.synchronize()
        live = (pos >= 0).flatten()
        assert torch.equal(y[live, : H * D], got["q"][live, : H * D]) and torch.equal(y[:, H * D:], x[:, H * D:])
        assert torch.equal(y[~live], x[~live])


# ---- graphs, streams, refusals ----------------------------------------------------------------------

@pytest.mark.parametrize("i4", [False, True])
def test_recorded_steps(ns2lib, i4):
    """A step (write, then attention) recorded once and replayed for later positions, with eager work and
    synchronizations between the replays: each replay equals the eager calls on a cache of its own."""
    rnd = gen(31)
    B, H, KH, D, cap = 3, 4, 1, 256, 700
    stream = torch.cuda.Stream()
    ns2lib.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            caches = [Cache(gen(32), B, cap, KH, D, i4) for _ in range(2)]
            x = rnd(B, (H + 2 * KH) * D)
            pos = torch.tensor([[600], [20], [-1]], dtype=torch.int32, device=DEV)
            w = 1 + 0.1 * rnd(D)
            cs = R.rope_table(cap, D).to(DEV)
            need = ns2lib.attention_cache_bytes(B, 1, H, KH, D, cap, 512, 4)
            bufs = [(torch.zeros(B, H * D, dtype=torch.float16, device=DEV), torch.zeros(B, H * D, dtype=torch.float16, device=DEV),
                     torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)) for _ in range(2)]

            def step(i):
                q, o, work = bufs[i]
                c = caches[i]
                ns2lib.head_norm_cache(x, pos, q, c.raw["k"], c.raw["v"], L=1, H=H, ldx=x.shape[1], ldq=H * D, w_q=w, w_k=w, cs=cs,
                                       sin_off=cs.numel() // 2, rope_rows=cap, q_fmt=1, **c.args())
                ns2lib.attention_cache(q, pos, c.raw["k"], c.raw["v"], o, L=1, H=H, ldq=H * D, ldo=H * D, window=512, sinks=4, q_fmt=1,
                                       work=work, **c.args())

            stream.synchronize()
            ns2lib.graph_begin()
            step(0)
            graph = ns2lib.graph_end()
            for n in range(5):
                x.copy_(rnd(*x.shape))
                ns2lib.graph_launch(graph)
                step(1)
                stream.synchronize()
                assert torch.equal(bufs[0][1], bufs[1][1]), f"replay {n}"
                for name in "kv":
                    assert torch.equal(caches[0].raw[name], caches[1].raw[name])
                pos += (pos >= 0).int()
                _ = torch.randn(1000, 1000, device=DEV).sum().item()
            ns2lib.graph_destroy(graph)
            assert (bufs[0][1][2] == 0).all()
    finally:
        ns2lib.set_stream(torch.cuda.current_stream().cuda_stream)


BASE = dict(batch=1, L=1, H=4, KH=2, D=64, cap=64, ldkv=128, kvBatch=64 * 128, ldq=256)


@pytest.mark.parametrize("change", [dict(D=80), dict(D=32), dict(D=512), dict(H=3), dict(KH=0), dict(H=0), dict(cap=0), dict(ldq=255),
                                    dict(ldq=258), dict(ldkv=120), dict(ldkv=132), dict(kvBatch=-8), dict(kvBatch=8196), dict(q_fmt=2),
                                    dict(window=-1), dict(sinks=-1), dict(ldo=128), dict(ldo=257), dict(k=None), dict(v=None),
                                    dict(pos=None), dict(q=None), dict(o=None), dict(vg=None), dict(k=8), dict(q=4), dict(o=4), dict(cap=(1 << 30) + 1),
                                    dict(batch=1 << 22), dict(batch=1 << 30, L=1 << 30), dict(L=1 << 22)])
def test_attention_refusals(ns2lib, change):
    """Refused on the host, before any launch: the output keeps what it held."""
    import ns2

    t = {n: torch.zeros(64 * 128, device=DEV) for n in ("q", "k", "v", "o", "kg", "vg")}
    t["pos"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    a = dict(BASE, ldo=256, window=0, sinks=0, q_fmt=0, kg=None, vg=None)
    ptr = {n: t[n] for n in ("q", "pos", "k", "v", "o")}
    if "vg" in change:
        a["kg"] = t["kg"]
    for n, x in change.items():
        if n in ptr:
            ptr[n] = None if x is None else ptr[n].data_ptr() + x
        else:
            a[n] = x
    kg, vg = a.pop("kg"), a.pop("vg")
    need = ns2lib.attention_cache_bytes(1, 1, 4, 2, 64, 64, 0, 0)
    work = torch.zeros(max(need, 16), dtype=torch.uint8, device=DEV)
    with pytest.raises(ns2.NS2Error, match="ns2_attention_cache"):
        ns2lib.attention_cache(ptr["q"], ptr["pos"], ptr["k"], ptr["v"], ptr["o"], k_groups=kg, v_groups=vg, work=work, **a)
    torch.cuda.synchronize()
    assert (t["o"] == 0).all()


@pytest.mark.parametrize("change", [dict(D=48), dict(H=5), dict(ldx=500), dict(ldx=514), dict(x=4), dict(x=None), dict(wk=4), dict(cs=4),
                                    dict(sin_off=2), dict(sin_off=-4), dict(rope_rows=-1), dict(batch=2, kvBatch=64), dict(kvBatch=8196),
                                    dict(kg=None), dict(k=2), dict(ldq=250), dict(cap=(1 << 30) + 1),
                                    dict(batch=1 << 30, L=1 << 30, kvBatch=64 * 128)])
def test_write_refusals(ns2lib, change):
    import ns2

    t = {n: torch.zeros(128 * 128, device=DEV) for n in ("x", "q", "k", "v", "kg", "vg", "wk", "cs")}
    t["pos"] = torch.zeros(2, dtype=torch.int32, device=DEV)
    a = dict(BASE, ldx=512, sin_off=64, rope_rows=2, q_fmt=0)
    ptr = {n: t[n] for n in ("x", "pos", "q", "k", "v", "wk", "cs", "kg", "vg")}
    if not set(change) & {"kg"}:
        ptr["kg"] = ptr["vg"] = None
    for n, x in change.items():
        if n in ptr:
            ptr[n] = None if x is None else ptr[n].data_ptr() + x
        else:
            a[n] = x
    with pytest.raises(ns2.NS2Error, match="ns2_head_norm_cache"):
        ns2lib.head_norm_cache(ptr["x"], ptr["pos"], ptr["q"], ptr["k"], ptr["v"], w_k=ptr["wk"], cs=ptr["cs"], k_groups=ptr["kg"],
                               v_groups=ptr["vg"], **a)
    torch.cuda.synchronize()
    assert (t["q"] == 0).all() and (t["k"] == 0).all()


def test_work_memory_is_checked(ns2lib):
    """Too little work memory, or none where some is needed, is refused; nothing to do is no error."""
    import ns2

    a = dict(batch=1, L=1, H=4, KH=1, D=256, cap=65536, ldkv=256, kvBatch=65536 * 256)
    need = ns2lib.attention_cache_bytes(1, 1, 4, 1, 256, 65536, 0, 0)
    q, o, kv = torch.zeros(1024, device=DEV), torch.zeros(1024, device=DEV), torch.zeros(65536 * 256, dtype=torch.float16, device=DEV)
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    if need:
        for work in (None, torch.empty(need - 16, dtype=torch.uint8, device=DEV)):
            with pytest.raises(ns2.NS2Error, match="work memory"):
                ns2lib.attention_cache(q, pos, kv, kv, o, ldq=1024, ldo=1024, work=work, **a)
    a["batch"] = 0
    ns2lib.attention_cache(q, pos, kv, kv, o, ldq=1024, ldo=1024, **a)
    a.update(batch=1, L=0)
    ns2lib.attention_cache(q, pos, kv, kv, o, ldq=1024, ldo=1024, **a)


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.07])
def test_scales_that_are_not_positive(ns2lib, scale, fp16):
    """A scale of 0 weighs all visible keys alike, a negative one prefers the opposite keys; one that is no number is
    refused."""
    import ns2

    rnd = gen(41)
    cache = Cache(rnd, 2, 200, 2, 96, False)
    for L in (1, 70):
        pos = positions([(120, L), (3, L)], L)
        q = rnd(2, L, 8, 96)
        got = attend(ns2lib, cache, q, pos, 50, 3, fp16, scale=scale)
        qd = (q.half() if fp16 else q.float()).double()
        ref, vmax, smax, n = R.attention(qd, pos, cache.value["k"], cache.value["v"], 50, 3, scale)
        assert ((got.double() - ref).abs() <= R.attention_bound(ref, vmax, smax.abs(), n, 96, fp16)).all()
        with pytest.raises(ns2.NS2Error, match="scale"):
            attend(ns2lib, cache, q, pos, 50, 3, fp16, scale=math.nan)


@pytest.mark.parametrize("i4", [False, True])
def test_two_streams_at_once(ns2lib, i4):
    """Calls on two streams, each with work memory of its own, over one cache: the bits of the calls by themselves."""
    rnd = gen(51)
    H, KH, D, cap = 8, 2, 128, 5000
    cache = Cache(rnd, 2, cap, KH, D, i4)
    calls = []
    for L, start in ((1, 4900), (6, 3000), (130, 2000)):
        pos = positions([(start, L), (start // 3, L)], L)
        q = rnd(2, L, H, D).reshape(2 * L, H * D)
        need = ns2lib.attention_cache_bytes(2, L, H, KH, D, cap, 0, 0)
        works = [torch.empty(max(need, 16), dtype=torch.uint8, device=DEV) for _ in range(3)]
        outs = [torch.zeros(2 * L, H * D, device=DEV) for _ in range(3)]
        calls.append((L, pos, q, works, outs))
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]

    def run(i):
        for L, pos, q, works, outs in calls:
            ns2lib.attention_cache(q, pos, cache.raw["k"], cache.raw["v"], outs[i], L=L, H=H, ldq=H * D, ldo=H * D, work=works[i],
                                   **cache.args())

    try:
        run(0)
        torch.cuda.synchronize()
        for _ in range(5):
            for i in (1, 2):
                ns2lib.set_stream(streams[i].cuda_stream)
                run(i)
        torch.cuda.synchronize()
    finally:
        ns2lib.set_stream(streams[0].cuda_stream)
    for _, _, _, _, outs in calls:
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
def test_recorded_prompts(ns2lib, i4, fp16):
    """A piece of a prompt and a prompt of many columns recorded together, over work memory of the graph's own: each
    replay equals eager calls on other work memory, with eager work between the replays."""
    rnd = gen(52)
    H, KH, D, cap, dt = 4, 2, 64, 3000, torch.float16 if fp16 else torch.float32
    cache = Cache(rnd, 1, cap, KH, D, i4)
    stream = torch.cuda.Stream()
    ns2lib.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            bufs = []
            for L in (20, 300):
                pos = torch.zeros(1, L, dtype=torch.int32, device=DEV)
                q = torch.zeros(L, H * D, dtype=dt, device=DEV)
                need = ns2lib.attention_cache_bytes(1, L, H, KH, D, cap, 900, 5)
                bufs.append((L, pos, q, [torch.empty(max(need, 16), dtype=torch.uint8, device=DEV) for _ in range(2)],
                             [torch.zeros(L, H * D, dtype=dt, device=DEV) for _ in range(2)]))

            def calls(i):
                for L, pos, q, works, outs in bufs:
                    ns2lib.attention_cache(q, pos, cache.raw["k"], cache.raw["v"], outs[i], L=L, H=H, ldq=H * D, ldo=H * D, window=900,
                                           sinks=5, q_fmt=int(fp16), work=works[i], **cache.args())

            stream.synchronize()
            ns2lib.graph_begin()
            calls(0)
            graph = ns2lib.graph_end()
            for n in range(4):
                for L, pos, q, _, _ in bufs:
                    pos.copy_(positions([(600 * n + 7, L - n)], L))
                    q.copy_(rnd(L, H * D))
                ns2lib.graph_launch(graph)
                calls(1)
                stream.synchronize()
                for _, _, _, _, outs in bufs:
                    assert torch.equal(outs[0], outs[1]), f"replay {n}"
                _ = torch.randn(500, 500, device=DEV).sum().item()
            ns2lib.graph_destroy(graph)
    finally:
        ns2lib.set_stream(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("i4", [False, True])
def test_a_cache_of_one_position(ns2lib, i4):
    """The shortest cache: the one token that fits sees itself, whatever the window."""
    rnd = gen(53)
    for H, KH, D in HEADS:
        cache = Cache(rnd, 2, 1, KH, D, i4)
        pos = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
        q = rnd(2, 1, H, D)
        for window, sinks in ((0, 0), (1, 0), (2**31 - 1, 2**31 - 1)):
            check(attend(ns2lib, cache, q, pos, window, sinks, False), q, pos, cache, window, sinks, False, f"one {H}/{KH}x{D} i4={i4}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("L", [1, 5, 70, 300])
def test_values_that_are_all_alike(ns2lib, L, D, i4, fp16):
    """Where every visible key holds the same values, the output is these values, however the weights lie: some keys at
    the maximum and hundreds below it that share a score, so that roundings of their weight do not average out. Weights
    taken in 22 bits and two sums over n <= 1001 keys in fp32 leave 2^-21 + 2 n 2^-24 < 1.3e-4 of a value; an fp16
    output is then the value itself (its neighbours' borders are 2^-12 = 2.4e-4 away), also at fp16's largest."""
    cap, H, KH = 1001, 8, 2
    cache = Cache(gen(61), 1, cap, KH, D, i4)
    v = torch.linspace(-3, 3, D, device=DEV).half()
    v[::32], v[5::32] = 65504.0, -65504.0
    if i4:
        # one step of 0 per group: the group's value is its offset
        v = v[::32].repeat_interleave(32) * torch.where(torch.arange(D, device=DEV) % 64 < 32, 1.0, -1.0).half()
        cache.raw["v"].zero_()
        cache.group_view("v")[..., 0], cache.group_view("v")[..., 1] = 0.0, v[::32]
    else:
        cache.view(cache.raw["v"], 1).copy_(v)
    pos = positions([(cap - L, L)], L)
    q = torch.zeros(1, L, H, D, device=DEV)
    q[..., 3] = 1.0
    k = torch.zeros(1, cap, KH, D, device=DEV)
    k[0, :, :, 3] = -1.0
    k[0, ::16] = 0.0  # (in every tile, so that no part of the keys has the lower score as its own maximum)
    if i4:
        codes, groups = R.cache_codes(k)
        cache.view(cache.raw["k"], 2).copy_(codes)
        cache.group_view("k").copy_(groups)
    else:
        cache.view(cache.raw["k"], 1).copy_(k.half())
    # weights of the many about half way between two halves, just above or below, where one rounding is off most
    for m in (1 + 20.47 / 1024, 1 + 20.53 / 1024, 1 + 0.53 / 1024, 1.5 + 0.47 / 1024, 1.25 + 0.53 / 1024):
        score = -math.log(2) + math.log(m)
        got = attend(ns2lib, cache, q, pos, 0, 0, fp16, scale=-score)
        if fp16:
            assert torch.equal(got, v.expand_as(got)), f"weight {m}"
        else:
            # (and the output's own rounding)
            assert ((got.double() - v.double()).abs() <= v.double().abs() * (2.0**-21 + 2 * cap * 2.0**-24 + 2.0**-22)).all(), f"weight {m}"


def test_queries_over_other_rows_are_refused(ns2lib):
    """q may be X itself only where a lane overwrites no more than what it has read: fp32 at X's distance. Any other rows
    that share bytes with X's would be written before other blocks have read them."""
    import ns2

    H, KH, D, L = 4, 2, 64, 3
    width = (H + 2 * KH) * D
    x = torch.arange(4 * L * width, device=DEV, dtype=torch.float32)
    before = x.clone()
    k, v = (torch.zeros(L, KH * D, dtype=torch.float16, device=DEV) for _ in "kv")
    pos = positions([(0, L)], L)
    a = dict(batch=1, L=L, H=H, KH=KH, D=D, cap=L, ldkv=KH * D, kvBatch=L * KH * D)
    at = x.data_ptr() + 4 * L * width
    for off, ldq, q_fmt in ((0, width, 1), (0, 2 * width, 1), (0, H * D, 0), (0, width + 4, 0), (4 * D, width, 0), (-4 * D, width, 0),
                            (4 * width, width, 0), (-4 * width, width, 0), (4 * (width - D), width, 0), (4 * (H * D - 4), width, 0),
                            (4 * L * width - 16, H * D, 0), (-16, H * D, 1), (16 - 4 * H * D * L, H * D, 0)):
        with pytest.raises(ns2.NS2Error, match="q overlaps X"):
            ns2lib.head_norm_cache(at, pos, at + off, k, v, ldx=width, ldq=ldq, q_fmt=q_fmt, **a)
    torch.cuda.synchronize()
    assert torch.equal(x, before) and (k == 0).all() and (v == 0).all()


@pytest.mark.parametrize("fp16", [False, True])
def test_queries_beside_the_rows(ns2lib, fp16):
    """Rows of q between the rows of X in one buffer, right behind them and right before them, hold what rows of their own
    hold; X stays."""
    rnd = gen(62)
    H, KH, D, L = 4, 1, 96, 33
    width, per = (H + 2 * KH) * D, H * D // (2 if fp16 else 1)  # (floats of a row of q)
    w, cs, pos = 1 + 0.1 * rnd(D), R.rope_table(L, D).to(DEV), positions([(0, L)], L)
    data = rnd(L, width)
    dt = torch.float16 if fp16 else torch.float32
    a = dict(batch=1, L=L, H=H, KH=KH, D=D, cap=L, ldkv=KH * D, kvBatch=L * KH * D, w_q=w, w_k=w, cs=cs, sin_off=cs.numel() // 2,
             rope_rows=L, q_fmt=int(fp16))

    def caches():
        return [torch.zeros(L, KH * D, dtype=torch.float16, device=DEV) for _ in "kv"]

    own, want = torch.zeros(L, H * D, dtype=dt, device=DEV), caches()
    ns2lib.head_norm_cache(data, pos, own, *want, ldx=width, ldq=H * D, **a)
    for x0, q0, ld in ((0, width, width + per), (per, 0, width + per), (0, width + 8, width + per + 8), (0, L * width, 0), (L * per, 0, 0)):
        buf = torch.full((L * (width + per + 8),), 3.0, device=DEV)
        ldx, ldq = ld or width, ld or per
        x = torch.as_strided(buf, (L, width), (ldx, 1), x0)
        x.copy_(data)
        got = caches()
        ns2lib.head_norm_cache(buf.data_ptr() + 4 * x0, pos, buf.data_ptr() + 4 * q0, *got, ldx=ldx, ldq=ldq * (2 if fp16 else 1), **a)
        torch.cuda.synchronize()
        q = torch.as_strided(buf, (L, per), (ldq, 1), q0).contiguous().view(dt)
        assert torch.equal(q, own) and torch.equal(x, data) and all(torch.equal(m, n) for m, n in zip(got, want))


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("L", [1, 5, 70, 300])
def test_visible_infinities(ns2lib, L, D, i4, fp16):
    """What is not finite in keys and values that are visible does what it does in 64 bits: a value of +-inf makes that
    dimension +-inf, both of them or a NaN make it NaN, a key whose score is -inf weighs nothing, and the dimensions and
    rows that meet none of it stay within the usual bound."""
    cap, H, KH = 700, 4, 2
    rnd = gen(63 + D)
    cache = Cache(rnd, 1, cap, KH, D, i4)
    pos = positions([(cap - L - 20, L)], L)
    q = rnd(1, L, H, D)
    q[..., 7] = q[..., 7].abs() + 0.5

    def put(name, key, head, dim, x):
        if i4:  # the offset of the dimension's group
            cache.group_view(name)[0, key, head, dim // 32, 1] = x
            cache.value[name][0, key, head, dim // 32 * 32: dim // 32 * 32 + 32] = x
        else:
            cache.view(cache.raw[name], 1)[0, key, head, dim] = x
            cache.value[name][0, key, head, dim] = x

    late = cap - 20 - L // 2 - 1  # (seen by the later rows only)
    for key, head, dim, x in ((40, 0, 3, math.inf), (333, 1, 5, -math.inf), (100, 1, D - 1, math.inf), (200, 1, D - 2, -math.inf),
                              (late, 0, D - 3, math.nan), (late, 1, 5, -math.inf)):
        put("v", key, head, dim, x)
    if not i4:  # scores of -inf: one key far from the others, and eight in a row
        for key in (77, *range(160, 168)):
            put("k", key, 0, 7, -math.inf)
            put("k", key, 1, 7, -math.inf)
    for window, sinks in ((0, 0), (400, 90)):
        got = attend(ns2lib, cache, q, pos, window, sinks, fp16)[0].double()
        qd = (q.half() if fp16 else q).double()
        ref = R.attention(qd, pos, cache.value["k"], cache.value["v"], window, sinks, 1 / math.sqrt(D))[0][0]
        kinds = [torch.where(torch.isnan(t), 2.0, torch.where(torch.isinf(t), t.sign(), 0.0)) for t in (got, ref)]
        assert torch.equal(*kinds), f"window {window}: {(kinds[0] != kinds[1]).sum().item()} of {got.numel()} outputs of another kind"
        k, v = (torch.where(torch.isfinite(cache.value[n]), cache.value[n], 0.0) for n in "kv")
        _, vmax, smax, n = R.attention(qd, pos, k, v, window, sinks, 1 / math.sqrt(D))
        bound = R.attention_bound(torch.where(torch.isfinite(ref), ref, 0.0), vmax, smax, n, D, fp16)[0]
        fine = torch.isfinite(ref)
        assert ((got - ref).abs() <= bound)[fine].all()


@pytest.mark.parametrize("i4", [False, True])
@pytest.mark.parametrize("L", [3, 80])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_queries_of_each_magnitude(ns2lib, D, L, i4):
    """fp32 queries of one magnitude per call, far below and beyond fp16's range, with a scale that makes their scores
    those of ordinary queries: the bound is small beside the values (asserted), so that a wrong query shows."""
    rnd = gen(64 + D + L)
    pos = positions([(60, L), (0, L)], L)
    cache = Cache(rnd, 2, 160, 2, D, i4)
    base = rnd(2, L, 4, D)
    for f in (1e-30, 1e-20, 1e-7, 1e-3, 1.0, 3e2, 1e4, 1e12, 1e30):
        q, scale = base * f, 1 / (f * math.sqrt(D))
        got = attend(ns2lib, cache, q, pos, 0, 0, False, scale=scale)
        # (the scale as the call takes it, in 32 bits)
        ref, vmax, smax, n = R.attention(q.double(), pos, cache.value["k"], cache.value["v"], 0, 0, float(torch.tensor(scale, dtype=torch.float32)))
        bound = R.attention_bound(ref, vmax, smax, n, D, False)
        live = (pos >= 0)
        assert (bound[live] < 1e-2 * vmax[live]).all()
        err = (got[live].double() - ref[live]).abs()
        print(f"[parity] D={D} L={L} i4={i4} x {f}: largest error / bound {(err / bound[live]).max().item():.3f}", flush=True)
        assert (err <= bound[live]).all(), f


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("L", [1, 90])
def test_scores_that_are_all_minus_infinity(ns2lib, L, fp16):
    """A row all of whose scores are -inf has no softmax: NaN, in its own heads; where one key is left, the row is that
    key's value."""
    rnd = gen(65)
    D, cap = 128, 400
    cache = Cache(rnd, 2, cap, 2, D, False)
    k = cache.view(cache.raw["k"], 1)
    k[:, :, :, 0] = -math.inf
    k[1, 17, 0, 0] = 1.0  # (sequence 1, head 0: one key is left)
    q = rnd(2, L, 4, D)
    q[..., 0] = 1.0
    pos = positions([(cap - L, L)] * 2, L)
    got = attend(ns2lib, cache, q, pos, 0, 0, fp16)
    assert torch.isnan(got[0]).all() and torch.isnan(got[1, :, 2:]).all()
    want = cache.value["v"][1, 17, 0]
    err = (got[1, :, :2].double() - want).abs()
    # one weight in 21 bits over itself, two sums, the output's rounding
    assert (err <= want.abs() * (2.0**-21 + 2.0**-22 + (2.0**-11 if fp16 else 2.0**-23)) + 2.0**-24).all()
