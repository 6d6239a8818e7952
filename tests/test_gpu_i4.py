"""Linears on 4-bit weights (ns2_linear_i4) and their quantizer (ns2_quantize_i4) against the weights that the codes stand
for, in 64 bits: rows from one on, odd widths, groups, both activation types, every epilogue, strides, refusals."""

import math

import pytest
import torch

import cache_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return g, lambda *shape: torch.randn(*shape, generator=g, device=DEV)


def weight(g, N, K, group):
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scale = ((torch.rand(N, K // group, generator=g, device=DEV) + 0.5) / (4.6 * math.sqrt(K))).half()
    return codes, scale


def act64(y, act):
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))
    return y


def run(lib, x, codes, scale, group, *, fp16, K, bias=None, add=None, act="none", resid=False, gate=None, alpha=1.0, pad=0, cOff=0, gOff=0):
    """Output and its reference with the bound of its error. The products x code are exact but for the split of an fp32 x
    (2^-22); they and the scaled groups are summed in fp32 in any order (at most (K + 4) 2^-24 of the sum of magnitudes);
    the epilogue's few operations and its activation are off by 2^-20 of the terms; an activation's slope is at most 1.13."""
    M, N = x.shape[0], codes.shape[0]
    lda = x.shape[1]
    xd = x.half() if fp16 else x
    C = torch.full((M + 1, N + pad), 5.0, device=DEV).contiguous()
    C0 = C.clone()
    lib.linear_i4(xd, int(fp16), lda, codes, scale, C, M, N, K, group, bias=bias, add=add, ldc=N + pad, cOff=cOff, alpha=alpha, act=act,
                  resid=resid, gate=gate, gOff=gOff)
    torch.cuda.synchronize()
    W = R.i4_weight(codes, scale, group)
    xd = xd[:, :K].double()
    y = alpha * (xd @ W.t())
    size = abs(alpha) * (xd.abs() @ W.abs().t())
    bound = size * (2.0**-22 + (K + 4) * 2.0**-24)
    for t in (bias, add):
        if t is not None:
            y, size = y + t.double(), size + t.double().abs()
    bound = 1.13 * (bound + size * 2.0**-22) + 2.0**-20 * size
    y = act64(y, act)
    if resid:
        gt = gate[gOff: gOff + N].double() if gate is not None else 1.0
        y = 5.0 + gt * y
        bound = bound * (gt.abs() if gate is not None else 1.0) + 2.0**-22 * (5 + y.abs())
    flat, flat0 = C.flatten(), C0.flatten()
    mine = torch.zeros_like(flat, dtype=torch.bool)
    at = cOff + torch.arange(M, device=DEV)[:, None] * (N + pad) + torch.arange(N, device=DEV)
    mine[at.flatten()] = True
    assert torch.equal(flat[~mine], flat0[~mine]), "values outside the output were written"
    return flat[at], y, bound


def check(got, what):
    out, ref, bound = got
    err = (out.double() - ref).abs()
    print(f"[parity] {what}: largest error / bound {(err / bound.clamp(min=1e-30)).max().item():.3f}", flush=True)
    assert torch.isfinite(out).all() and (err <= bound).all(), what


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 128), (16, 128), (17, 256), (100, 640), (333, 1536), (64, 2048), (1000, 384), (48, 6144)])
def test_rows_and_widths(ns2lib, N, K, group, fp16):
    g, rnd = gen(N + K + group)
    codes, scale = weight(g, N, K, group)
    for M in (1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 130):
        check(run(ns2lib, rnd(M, K), codes, scale, group, fp16=fp16, K=K), f"{M}x{N}x{K} group {group} fp16={fp16}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("K", [32, 64, 96, 160, 224, 416, 1056, 2080])
def test_widths_of_one_group(ns2lib, K, fp16):
    """K any multiple of the group."""
    g, rnd = gen(K)
    codes, scale = weight(g, 37, K, 32)
    for M in (1, 6, 40):
        check(run(ns2lib, rnd(M, K), codes, scale, 32, fp16=fp16, K=K), f"{M}x37x{K} fp16={fp16}")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("M", [1, 7, 50])
@pytest.mark.parametrize("opts", [dict(bias=1), dict(bias=1, act="silu"), dict(add=1, act="gelu_tanh"), dict(resid=True),
                                  dict(resid=True, gate=1, gOff=5), dict(bias=1, add=1, resid=True, gate=1, alpha=-0.5, act="silu"),
                                  dict(pad=3, cOff=2), dict(pad=13, alpha=2.0)])
def test_epilogues(ns2lib, M, opts, fp16):
    g, rnd = gen(M)
    N, K = 147, 320
    codes, scale = weight(g, N, K, 64)
    o = dict(opts)
    for n, shape in (("bias", (N,)), ("add", (M, N)), ("gate", (N + 9,))):
        if n in o:
            o[n] = rnd(*shape)
    check(run(ns2lib, rnd(M, K), codes, scale, 64, fp16=fp16, K=K, **o), f"{M} {opts} fp16={fp16}")


@pytest.mark.parametrize("fp16", [False, True])
def test_strides_and_magnitudes(ns2lib, fp16):
    """Rows of A wider than K (what lies behind K is not read: NaN), every code, a few strong columns, tiny activations."""
    g, rnd = gen(5)
    N, K = 70, 1024
    codes, scale = weight(g, N, K, 128)
    for M in (1, 12, 20):
        x = torch.full((M, K + 16), math.nan, device=DEV)
        x[:, :K] = rnd(M, K)
        x[:, 5] *= 300
        x[0, 7:300] *= 2.0**-12
        check(run(ns2lib, x, codes, scale, 128, fp16=fp16, K=K), f"{M} strided fp16={fp16}")


def test_one_row_does_not_reach_another(ns2lib):
    """A NaN or an infinity in a row of A, or in a scale, stays in its row or column."""
    g, rnd = gen(6)
    M, N, K = 11, 40, 256
    codes, scale = weight(g, N, K, 32)
    for fp16 in (False, True):
        x = rnd(M, K)
        clean, _, _ = run(ns2lib, x, codes, scale, 32, fp16=fp16, K=K)
        y = x.clone()
        y[3, 100], y[8, 0] = math.nan, math.inf
        s = scale.clone()
        s[21, 2] = math.nan
        got, _, _ = run(ns2lib, y, codes, s, 32, fp16=fp16, K=K)
        rows = torch.tensor([3, 8], device=DEV)
        assert not torch.isfinite(got[rows]).any() and not torch.isfinite(got[:, 21]).any()
        keep = torch.ones(M, N, dtype=torch.bool, device=DEV)
        keep[rows], keep[:, 21] = False, False
        assert torch.equal(got[keep], clean[keep])


def test_many_columns(ns2lib):
    """A table of embeddings as the weight of the logits."""
    g, rnd = gen(7)
    codes, scale = weight(g, 50001, 640, 64)
    for M in (1, 3):
        check(run(ns2lib, rnd(M, 640), codes, scale, 64, fp16=True, K=640), f"{M}x50001")


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(130, 8200, 384), (33, 30011, 256), (17, 65537, 128), (48, 14003, 1408),  # many rows and columns
                                   (32, 65540, 256), (61, 33001, 1408), (115, 18003, 640), (300, 8001, 128), (48, 44003, 128),
                                   (1, 65553, 640), (4, 65600, 1152), (6, 65539, 256), (12, 65553, 384), (16, 66000, 128),  # a table
                                   (1, 8181, 640), (7, 8177, 1408), (16, 5003, 640), (40, 2050, 896),  # K over sixteen waves
                                   (1, 20003, 1664), (8, 20003, 640), (16, 10007, 512), (90, 3001, 640)])  # over four
def test_blocks_of_every_size(ns2lib, M, N, K, group, fp16):
    g, rnd = gen(M + N)
    codes, scale = weight(g, N, K, group)
    check(run(ns2lib, rnd(M, K), codes, scale, group, fp16=fp16, K=K, bias=rnd(N), act="silu", pad=1), f"{M}x{N}x{K} group {group} fp16={fp16}")


@pytest.mark.parametrize("M,N,K", [(9, 300, 1536), (5, 66000, 256), (40, 9000, 512)])
def test_rows_of_any_magnitude(ns2lib, M, N, K):
    """fp32 rows far below and beyond fp16's range, some of them changing their magnitude along the row, a row of zeros."""
    g, rnd = gen(N)
    codes, scale = weight(g, N, K, 64)
    x = rnd(M, K)
    for r, f in ((0, 1e-30), (1, 1e-12), (2, 1e6), (3, 1e30), (4, 0.0)):
        x[r] *= f
    x[1, K // 2:] *= 1e4
    check(run(ns2lib, x, codes, scale, 64, fp16=False, K=K), f"{M}x{N}x{K}")


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantizer(ns2lib, group):
    """Codes and scales equal the definition; zeros, one strong value, tiny groups, values on a border."""
    _, rnd = gen(8)
    N, K = 33, 384
    w = (rnd(N, K) * 0.05).to(torch.bfloat16)
    w[0] = 0
    w[1, ::7] = 3.5
    w[2] = 1e-30
    w[3] = (torch.arange(K, device=DEV) % 15 - 7).to(torch.bfloat16)
    w[4] = ((torch.arange(K, device=DEV) % 29 - 14) / 2).to(torch.bfloat16)
    w[5] *= 1e-4
    codes = torch.zeros(N, K // 2, dtype=torch.uint8, device=DEV)
    scale = torch.zeros(N, K // group, dtype=torch.float16, device=DEV)
    ns2lib.quantize_i4(w, codes, scale, N, K, group)
    torch.cuda.synchronize()
    rc, rs = R.i4_codes(w.cpu(), group)
    assert torch.equal(scale.cpu(), rs) and torch.equal(codes.cpu(), rc)
    err = (R.i4_weight(codes, scale, group) - w.double()).abs()
    step = scale.double().repeat_interleave(group, 1)
    # half a step, and at the ends the rounding of the step (2^-11 of 7 steps; below 2^-14 it is 2^-25 absolute)
    assert (err <= step / 2 + 7 * (step * 2.0**-11 + 2.0**-25)).all()
    w[7, 5] = math.inf
    ns2lib.quantize_i4(w, codes, scale, N, K, group)
    torch.cuda.synchronize()
    bad = torch.zeros_like(scale, dtype=torch.bool)
    bad[7, 5 // group] = True
    assert torch.equal(torch.isnan(scale), bad)


@pytest.mark.parametrize("change", [dict(group=16), dict(group=48), dict(K=80), dict(K=0), dict(N=0), dict(N=-1), dict(M=-1), dict(a_fmt=2),
                                    dict(lda=120), dict(lda=130), dict(ldc=30), dict(cOff=-1), dict(gOff=-1), dict(act=3), dict(N=(1 << 29) + 1, ldc=1 << 30), dict(M=1 << 20), dict(A=4),
                                    dict(W=8), dict(scale=1), dict(A=None), dict(W=None), dict(scale=None), dict(C=None)])
def test_refusals(ns2lib, change):
    import ns2

    t = {n: torch.zeros(8192, device=DEV) for n in ("A", "W", "scale", "C")}
    a = dict(a_fmt=0, lda=128, M=1, N=32, K=128, group=32, ldc=32, cOff=0, act=0, gOff=0)
    ptr = {n: x.data_ptr() for n, x in t.items()}
    for n, x in change.items():
        if n in ptr:
            ptr[n] = None if x is None else ptr[n] + x
        else:
            a[n] = x
    with pytest.raises(ns2.NS2Error, match="ns2_linear_i4"):
        ns2lib.call("ns2_linear_i4", ptr["A"], a["a_fmt"], a["lda"], ptr["W"], ptr["scale"], None, None, ptr["C"], a["M"], a["N"],
                    a["K"], a["group"], a["ldc"], a["cOff"], 1.0, a["act"], 0, None, a["gOff"])
    torch.cuda.synchronize()
    assert (t["C"] == 0).all()
    if "group" in change or change.get("K") == 80:
        with pytest.raises(ns2.NS2Error, match="ns2_quantize_i4"):
            ns2lib.quantize_i4(t["A"], t["W"], t["scale"], 32, a["K"], a["group"])


def infinite_classes(x, W):
    """0 where an output of x W^T is finite, 1 and -1 where it is an infinity, 2 where it is NaN, in 64 bits."""
    y = x.double() @ W.t()
    return torch.where(torch.isnan(y), 2, torch.where(torch.isinf(y), y.sign(), 0.0))


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 40, 256), (7, 40, 96), (16, 1030, 2080), (33, 30011, 256), (1, 66000, 640), (12, 66000, 128),
                                   (9, 20003, 1664), (40, 2050, 896), (20, 1040, 6144)])
def test_infinite_activations(ns2lib, M, N, K, fp16):
    """An infinity in a row of A makes each of the row's outputs the infinity that its weight's sign says, NaN where the
    weight is 0 or where two infinities meet with other signs; what is finite beside it decides nothing. Other rows are
    those of a call without it."""
    g, rnd = gen(M + N + K)
    codes, scale = weight(g, N, K, 32)
    W = R.i4_weight(codes, scale, 32)
    x = rnd(M, K)
    clean, _, _ = run(ns2lib, x, codes, scale, 32, fp16=fp16, K=K)
    y = x.clone()
    bad = torch.zeros(M, dtype=torch.bool, device=DEV)
    for r, put in ((0, {K // 3: math.inf}), (M // 2, {K - 1: -math.inf}), (M - 1, {1: math.inf, K // 2: -math.inf})):
        if bad[r]:
            continue
        bad[r] = True
        for k, v in put.items():
            y[r, k] = v
    if not fp16:
        y[0, K // 2 + 1] = 1e30  # (finite: beyond fp16's range)
    got, _, _ = run(ns2lib, y, codes, scale, 32, fp16=fp16, K=K)
    kinds = torch.where(torch.isnan(got), 2, torch.where(torch.isinf(got), got.sign(), 0.0)).double()
    assert torch.equal(kinds, infinite_classes(y, W))
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("a_fmt", [0, 1])
def test_widths_near_the_end_of_32_bits_are_refused(ns2lib, a_fmt):
    """K's last chunk of 128 columns would end past 2^31; refused before any launch."""
    import ns2

    C = torch.zeros(64, device=DEV)
    p = C.data_ptr()
    for K, group in (((1 << 31) - 32, 32), ((1 << 31) - 128, 128), ((1 << 30) + 32, 32)):
        with pytest.raises(ns2.NS2Error, match="ns2_linear_i4"):
            ns2lib.call("ns2_linear_i4", p, a_fmt, K, p, p, None, None, p, 1, 1, K, group, 1, 0, 1.0, 0, 0, None, 0)
    torch.cuda.synchronize()
    assert (C == 0).all()


@pytest.mark.parametrize("fp16", [False, True])
def test_a_wide_row(ns2lib, fp16):
    """K of millions: small whole numbers at a few places, the first and the last columns among them, whose sums are exact."""
    g, rnd = gen(9)
    K = 1 << 22
    for M, N in ((1, 3), (5, 17)):
        codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
        scale = torch.full((N, K // 128), 0.5, dtype=torch.float16, device=DEV)
        x = torch.zeros(M, K, device=DEV)
        at = torch.cat([torch.randint(0, K, (500,), generator=g, device=DEV), torch.tensor([0, 127, 128, K - 129, K - 128, K - 1], device=DEV)])
        x[:, at] = torch.randint(-8, 9, (M, len(at)), generator=g, device=DEV).float()
        C = torch.empty(M, N, device=DEV)
        ns2lib.linear_i4(x.half() if fp16 else x, int(fp16), K, codes, scale, C, M, N, K, 128)
        cols = torch.unique(at)
        byte = codes[:, cols // 2].long()
        w = torch.where(cols % 2 == 1, byte >> 4, byte & 15).double() - 8
        assert torch.equal(C.double(), x[:, cols].double() @ w.t() * 0.5)
