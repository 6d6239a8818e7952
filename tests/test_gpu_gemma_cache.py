"""The text encoder over a key/value cache, through the Node host (run_gemma.js --cache) and as a chain of the C ABI's
calls: tokens in pieces of any length, the local layers' window, sinks, 4-bit weights, 4-bit caches, recorded steps.

Tolerance of the 17 layers: 1e-2, as for whole prompts. A 4-bit cache makes steps of its inputs' small differences: where
products differ by 5e-4 of a value's spread, one code in 5e-4 / 0.27 falls on the other side of a border and is off by a
step (0.27 of the spread for normal values), a noise of sqrt(2e-3) * 0.27 = 1.2 % of the keys and values per layer, at
most 5e-2 after 17 layers that add up at random."""

import json
import os
import subprocess

import numpy as np
import pytest
import torch

import cache_reference as R
import gemma_fixture as G
from conftest import assert_close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "gemma_encode.npz")


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    z = np.load(GOLDEN, allow_pickle=False)
    meta = json.loads(bytes(z["meta"]).decode())
    d = tmp_path_factory.mktemp("gemma_cache")
    tensors = G.make_weights(seed=meta["weight_seed"])
    path = str(d / "gemma3_bf16.safetensors")
    G.save_weights(tensors, path)
    return tensors, path, d, z


def hidden(model, ids, *args):
    _, path, d, _ = model
    idf, out = str(d / "ids.json"), str(d / "h.f32")
    with open(idf, "w") as f:
        json.dump(ids, f)
    G.run_node(["--weights", path, "--ids", idf, "--out", out, *map(str, args)])
    return torch.from_numpy(np.fromfile(out, dtype=np.float32).reshape(len(ids), 640))


def four_bit(tensors, group=32):
    """The weights that the quantized linears stand for."""
    out = dict(tensors)
    for name, w in tensors.items():
        if "proj" in name:
            codes, scale = R.i4_codes(w.float(), group)
            out[name] = R.i4_weight(codes, scale, group)
    return out


@pytest.mark.parametrize("case,chunk", [("one", 1), ("short", 3), ("ragged", 1), ("ragged", 7)])
def test_pieces_of_a_prompt_match_the_golden(model, case, chunk):
    z = model[3]
    ids = [int(i) for i in z[f"{case}.ids"]]
    got = hidden(model, ids, "--cache", len(ids) + 5, "--chunk", chunk)
    assert_close(got, torch.from_numpy(z[f"{case}.out"]), 1e-2, f"{case} in pieces of {chunk}")


def test_a_prompt_longer_than_the_window(model):
    ids = G.make_ids(620, seed=46)
    ref = R.gemma_hidden(model[0], ids, 512, 4, 16, DEV)
    for chunk in (620, 111):
        got = hidden(model, ids, "--cache", 700, "--chunk", chunk, "--sinks", 4)
        assert_close(got, ref, 1e-2, f"620 tokens in pieces of {chunk}")


def test_four_bit_weights(model):
    ids = G.make_ids(60, seed=47)
    W = four_bit(model[0])
    ref = R.gemma_hidden(W, ids, 512, 0, 16, DEV)
    for chunk in (60, 1):
        got = hidden(model, ids, "--cache", 64, "--chunk", chunk, "--weight-bits", 4)
        assert_close(got, ref, 1e-2, f"4-bit weights in pieces of {chunk}")
    # the whole-prompt encoder takes them too
    assert_close(hidden(model, ids, "--weight-bits", 4), ref, 1e-2, "4-bit weights, whole prompt")


def test_four_bit_cache(model):
    ids = G.make_ids(90, seed=48)
    ref = R.gemma_hidden(model[0], ids, 512, 0, 4, DEV)
    whole = hidden(model, ids, "--cache", 96, "--cache-bits", 4)
    assert_close(whole, ref, 5e-2, "4-bit cache")
    pieces = hidden(model, ids, "--cache", 96, "--cache-bits", 4, "--chunk", 13)
    assert_close(pieces, whole, 5e-2, "4-bit cache, in pieces")


def test_recorded_steps_match_eager_ones(model):
    ids = G.make_ids(23, seed=49)
    for bits in (16, 4):
        args = ("--cache", 32, "--chunk", 1, "--weight-bits", 4, "--cache-bits", bits)
        assert torch.equal(hidden(model, ids, *args), hidden(model, ids, *args, "--graph")), bits


@pytest.mark.parametrize("i4cache", [False, True])
def test_chain_of_calls(ns2lib, i4cache):
    """q|k|v projection -> write -> attention -> output projection on 4-bit weights for two sequences: a prompt piece, a
    second one, single tokens. Each call is held to its definition on what the call before really wrote, and rows
    behind the shorter sequence stay as they were."""
    lib = ns2lib
    g = torch.Generator(device=DEV).manual_seed(50)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=DEV)

    B, H, KH, D, K, cap = 2, 4, 1, 256, 640, 300
    width = (H + 2 * KH) * D
    ws = {}
    for name, (N, k) in {"qkv": (width, K), "o": (K, H * D)}.items():
        w = (rnd(N, k) / k**0.5).to(torch.bfloat16)
        codes = torch.empty(N, k // 2, dtype=torch.uint8, device=DEV)
        scale = torch.empty(N, k // 32, dtype=torch.float16, device=DEV)
        lib.quantize_i4(w, codes, scale, N, k, 32)
        ws[name] = (codes, scale, R.i4_weight(codes, scale, 32))
    wq, wk, cs = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D), R.rope_table(cap, D).to(DEV)
    if i4cache:
        raw = {n: torch.zeros(B, cap, KH, D // 2, dtype=torch.uint8, device=DEV) for n in "kv"}
        groups = {n: torch.full((B, cap, KH, D // 32, 2), float("nan"), dtype=torch.float16, device=DEV) for n in "kv"}
    else:
        raw = {n: torch.full((B, cap, KH, D), float("nan"), dtype=torch.float16, device=DEV) for n in "kv"}
        groups = {"k": None, "v": None}
    lengths = [0, 0]
    for counts in ([120, 75], [40, 61], [1, 1], [1, 0], [1, 1]):
        L = max(counts)
        pos = torch.full((B, L), -1, dtype=torch.int32)
        for b, n in enumerate(counts):
            pos[b, :n] = torch.arange(lengths[b], lengths[b] + n)
            lengths[b] += n
        pos = pos.to(DEV)
        live = (pos >= 0).flatten()
        x = rnd(B * L, K)
        qkv = torch.empty(B * L, width, device=DEV)
        lib.linear_i4(x, 0, K, ws["qkv"][0], ws["qkv"][1], qkv, B * L, width, K, 32)
        q = torch.full((B * L, H * D), 7.0, dtype=torch.float16, device=DEV)
        a = dict(batch=B, L=L, H=H, KH=KH, D=D, cap=cap, ldkv=KH * D, kvBatch=cap * KH * D, ldq=H * D, q_fmt=1,
                 k_groups=groups["k"], v_groups=groups["v"])
        lib.head_norm_cache(qkv, pos, q, raw["k"], raw["v"], ldx=width, w_q=wq, w_k=wk, cs=cs, sin_off=cs.numel() // 2,
                            rope_rows=cap, **a)
        o = torch.full((B * L, H * D), 7.0, dtype=torch.float16, device=DEV)
        need = lib.attention_cache_bytes(B, L, H, KH, D, cap, 64, 4)
        lib.attention_cache(q, pos, raw["k"], raw["v"], o, ldo=H * D, window=64, sinks=4,
                            work=torch.empty(need, dtype=torch.uint8, device=DEV) if need else None, **a)
        y = torch.empty(B * L, K, device=DEV)
        lib.linear_i4(o, 1, H * D, ws["o"][0], ws["o"][1], y, B * L, K, H * D, 32)
        torch.cuda.synchronize()

        assert (q[~live] == 7).all() and (o[~live] == 7).all()
        xd = x.double()
        slack = (2.0**-21 + (K + 4) * 2.0**-24) * (xd.abs() @ ws["qkv"][2].abs().t())
        assert ((qkv.double() - xd @ ws["qkv"][2].t()).abs() <= slack).all()
        heads = qkv.double().reshape(B * L, H + 2 * KH, D)
        qr = R.head_norm(heads[:, :H], wq, cs, pos.flatten(), cap, 1e-6)[live].reshape(-1, H * D)
        assert ((q[live].double() - qr).abs() <= 2.0**-11 * qr.abs() + 2.0**-20 * qr.abs().max()).all()
        val = {n: R.cache_values(raw[n], groups[n]) if i4cache else raw[n].double() for n in "kv"}
        ref, vmax, smax, n = R.attention(q.double().reshape(B, L, H, D), pos, val["k"], val["v"], 64, 4, D**-0.5)
        bound = R.attention_bound(ref, vmax, smax, n, D, True).reshape(B * L, H * D)[live]
        assert ((o.double() - ref.reshape(B * L, H * D))[live].abs() <= bound).all()
        od = o.double()
        slack = (H * D + 4) * 2.0**-24 * (od.abs() @ ws["o"][2].abs().t())
        assert ((y.double() - od @ ws["o"][2].t()).abs() <= slack).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_calls_in_flight_and_steps_of_one_sequence(model, bits):
    """Two sequences: calls that do not wait for each other give the bits of calls one by one, and a recorded step that
    one sequence sits out those of an eager call."""
    script = os.path.join(os.path.dirname(os.path.abspath(__file__)), "js", "extend_overlap.mjs")
    p = subprocess.run(["node", script, model[1], str(bits)], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, p.stderr[-2000:]
    got = json.loads(p.stdout.strip().splitlines()[-1])
    assert got == {"overlap": 0, "recorded": 0, "lengths": [[6, 6], [6, 6], [9, 9], [9, 9]]}


@pytest.mark.parametrize("chunk", [1, 9])
def test_loras_over_a_cache(model, chunk):
    """LoRAs on the encoder's linears act on tokens in pieces as on the whole prompt (which is held to the goldens)."""
    from safetensors.torch import save_file

    lora = str(model[2] / "te_lora.safetensors")
    save_file(G.make_te_lora(), lora)
    ids = G.make_ids(21, seed=51)
    whole = hidden(model, ids, "--lora", lora + ":0.8")
    got = hidden(model, ids, "--cache", 32, "--chunk", chunk, "--lora", lora + ":0.8")
    assert_close(got, whole, 1e-2, f"LoRA in pieces of {chunk}")
    plain = hidden(model, ids, "--cache", 32, "--chunk", chunk)
    assert (got - plain).norm() > 1e-2 * plain.norm(), "the LoRA changes less than the tolerance"
