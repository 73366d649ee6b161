"""The Qwen3 emotion-text decoder with 4-bit weights (ITTS_QWEN_W4, ITTS_QWEN_W4_HEAD) on the MI355X.

One cached row: attention returns that row's V, so a prefill of one id is a chain of the public operators
(itts_ops) and equals it bit for bit.  Longer: against the FP32 oracle run on the weights that the 4 bits
stand for, whose only difference is the 8-bit rounding of the products' inputs.  A code is off by at most
half a step, uniformly: step / sqrt(12), with a step of max / 127 and a group's largest of 128 normal
values under 4 sigma (a share of 0.8 % lies over 4): 0.0091 of the values' size for each product.  L
layers put 4 L + 1 such roundings one after the other, which add as squares: a relative error of
0.0091 * sqrt(4 L + 1) = 0.027 for two layers.  The rounded inputs of an exact implementation are as far
off.  The bar is twice that.
"""
import os

import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import rel_err

pytestmark = pytest.mark.gpu
LAYERS, GROUP = 2, 128
BAR = 2 * 0.0091 * np.sqrt(4 * LAYERS + 1)
MATRICES = ("q_proj.weight", "k_proj.weight", "v_proj.weight", "o_proj.weight", "gate_proj.weight", "up_proj.weight", "down_proj.weight")


@pytest.fixture(scope="module")
def ops(itts):
    import itts_ops

    return itts_ops


@pytest.fixture(scope="module")
def qw(itts):
    return itts.make_synthetic_qwen_weights(layers=LAYERS, seed=17)


@pytest.fixture(scope="module")
def dec(itts, qw):
    d = itts.QwenDecoder(qw, layers=LAYERS, weight_bits=4)
    yield d
    d.close()


def ids_of(seed, n):
    return [int(x) for x in np.random.default_rng(seed).integers(0, 151936, n)]


def four_bits(w):
    q, s = ref.codes4(w.astype(np.float64), GROUP)
    return (q * np.repeat(s, GROUP, 1)[:, : w.shape[1]]).astype(np.float32)


@pytest.fixture(scope="module")
def rounded(oracle, qw):
    """The oracle on the layers' matrices as 4 bits have them (the tied embedding in full)."""
    return oracle.OracleQwen({k: four_bits(v) if k.endswith(MATRICES) else v for k, v in qw.items()}, layers=LAYERS)


@pytest.mark.parametrize("head_bits", [4, 32])
def test_one_id_is_the_operators_one_after_the_other(itts, ops, qw, dec, head_bits):
    d = dec if head_bits == 4 else itts.QwenDecoder(qw, layers=LAYERS, weight_bits=4, head_bits=32)
    t = {k: torch.from_numpy(v).cuda() for k, v in qw.items()}
    with torch.no_grad():
        for token in (0, 77, 151935):
            got = d.prefill([token])
            h = t["qwen.model.embed_tokens.weight"][token : token + 1].clone()
            for i in range(LAYERS):
                p = f"qwen.model.layers.{i}."
                m = lambda *n: torch.cat([t[p + x + ".weight"] for x in n])  # noqa: E731
                qkv = ops.q4_linear(h, ops.q4_pack(m("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), GROUP),
                                    norm_weight=t[p + "input_layernorm.weight"])
                att = qkv[:, -1024:].view(8, 1, 128).expand(8, 2, 128).reshape(1, 2048)
                h = ops.q4_linear(att, ops.q4_pack(m("self_attn.o_proj"), GROUP), residual=h)
                gu = torch.stack([t[p + "mlp.gate_proj.weight"], t[p + "mlp.up_proj.weight"]], 1).view(-1, 1024)
                ff = ops.q4_linear(h, ops.q4_pack(gu, GROUP), norm_weight=t[p + "post_attention_layernorm.weight"], swiglu=True)
                h = ops.q4_linear(ff, ops.q4_pack(m("mlp.down_proj"), GROUP), residual=h)
            e, last = t["qwen.model.embed_tokens.weight"], t["qwen.model.norm.weight"]
            if head_bits == 4:
                n = ops.rmsnorm_q8(h, last)
                want = ops.q4_matmul(n.q, n.scales, ops.q4_pack(e, GROUP))
                assert np.array_equal(got, want.cpu().numpy()[0])
            else:
                # the FP32 head's sums of 1024 products after its own norm: 2^-24 * 1024 of the terms' sizes at most
                x = ref.rms(ref.to64(h), ref.to64(last), 1e-6)
                want = ref.to64(e) @ x[0]
                size = np.abs(ref.to64(e)) @ np.abs(x[0])
                assert np.all(np.abs(got - want) <= 1100 * 2.0 ** -24 * size)
    if d is not dec:
        d.close()


@pytest.mark.parametrize("n_prompt", [2, 17, 64, 65, 200])
def test_prefill_and_steps_stay_within_the_rounding(itts, qw, rounded, n_prompt):
    d = itts.QwenDecoder(qw, layers=LAYERS, weight_bits=4, head_bits=32)
    p = ids_of(n_prompt, n_prompt + 4)
    got, want = [d.prefill(p[:n_prompt])], [rounded.prefill(p[:n_prompt])]
    for i in range(4):
        got.append(d.step(p[n_prompt + i]))
        want.append(rounded.step(p[n_prompt + i]))
    d.close()
    for i, (g, w) in enumerate(zip(got, want)):
        e = rel_err(g, w)
        print(f"{n_prompt} ids + {i}: {e:.4f} (bar {BAR:.4f})", flush=True)
        assert np.all(np.isfinite(g)) and e <= BAR, (i, e)


@pytest.mark.parametrize("n_prompt", [510, 2046])
def test_steps_merge_many_splits(itts, oracle, n_prompt):
    """One layer, caches of 8 and 9, and of 32 and 33 splits of 64 rows, which the output projection merges."""
    w = itts.make_synthetic_qwen_weights(layers=1, seed=23)
    d = itts.QwenDecoder(w, layers=1, weight_bits=4, head_bits=32)
    orc = oracle.OracleQwen({k: four_bits(v) if k.endswith(MATRICES) else v for k, v in w.items()}, layers=1)
    p, bar = ids_of(n_prompt, n_prompt + 5), 2 * 0.0091 * np.sqrt(5)
    print(f"{n_prompt} ids, one layer", flush=True)
    d.prefill(p[:n_prompt])
    orc.prefill(p[:n_prompt])
    for i in range(5):
        e = rel_err(d.step(p[n_prompt + i]), orc.step(p[n_prompt + i]))
        print(f"row {n_prompt + i}: {e:.4f} (bar {bar:.4f})", flush=True)
        assert e <= bar
    d.close()


def test_steps_continue_a_prefill(dec):
    """A prefill of n ids and steps, and one of n + 3: the same cache up to the 8-bit rounding's moves (as the bar)."""
    p = ids_of(5, 70)
    dec.prefill(p[:67])
    steps = [dec.step(t) for t in p[67:]][-1]
    assert rel_err(steps, dec.prefill(p)) <= BAR


def test_generate_is_greedy_steps(dec):
    p = ids_of(9, 30)
    logits, want = dec.prefill(p), []
    for _ in range(12):
        want.append(int(np.argmax(logits)))
        logits = dec.step(want[-1])
    got, eos = dec.generate_tokens(p, 12)
    assert got == want and not eos
    assert np.array_equal(dec.step(got[-1]), logits)
    # a longer prompt after the step was captured makes the prefill's buffers anew
    long = ids_of(10, 700)
    first, _ = dec.generate_tokens(long, 9)
    logits, again = dec.prefill(long), []
    for _ in range(9):
        again.append(int(np.argmax(logits)))
        logits = dec.step(again[-1])
    assert first == again
    assert dec.generate_tokens(p, 12)[0] == want


def test_generate_stops_at_eos(itts, qw, dec):
    for seed in range(11, 40):
        prompt = ids_of(seed, 12)
        toks, _ = dec.generate_tokens(prompt, 12)
        ks = [i for i in range(1, len(toks)) if toks[i] not in toks[:i]]
        if ks:
            break
    k, t = ks[0], toks[ks[0]]
    w = dict(qw)
    e = w["qwen.model.embed_tokens.weight"].copy()
    e[[t, itts.QWEN_EOS]] = e[[itts.QWEN_EOS, t]]
    w["qwen.model.embed_tokens.weight"] = e
    d = itts.QwenDecoder(w, layers=LAYERS, weight_bits=4)
    prompt = [itts.QWEN_EOS if x == t else x for x in prompt]
    assert d.generate(prompt, 12) == toks[:k] + [itts.QWEN_EOS]
    d.close()


def test_graph_replay_equals_eager(itts, qw, dec):
    os.environ["ITTS_QWEN_GRAPHS"] = "0"
    try:
        eager = itts.QwenDecoder(qw, layers=LAYERS, weight_bits=4)
    finally:
        del os.environ["ITTS_QWEN_GRAPHS"]
    p = ids_of(21, 40)
    assert np.array_equal(dec.prefill(p[:30]), eager.prefill(p[:30]))
    for t in p[30:]:
        assert np.array_equal(dec.step(t), eager.step(t))
    assert dec.generate_tokens(p[:9], 20) == eager.generate_tokens(p[:9], 20)
    eager.close()


def test_head_alone_in_four_bits(itts, oracle, qw):
    """FP32 layers with a 4-bit head, against the oracle with that head: one rounding to 8 bits."""
    d = itts.QwenDecoder(qw, layers=LAYERS, weight_bits=32, head_bits=4)
    full = itts.QwenDecoder(qw, layers=LAYERS)
    p = ids_of(31, 21)
    e = four_bits(qw["qwen.model.embed_tokens.weight"])
    full.prefill(p[:20])
    d.prefill(p[:20])
    got = d.step(p[20])
    want = full.step(p[20])
    # the state that the head reads, recovered from the full head's logits (4096 equations for 1024 numbers)
    x, *_ = np.linalg.lstsq(qw["qwen.model.embed_tokens.weight"][:4096].astype(np.float64), want[:4096].astype(np.float64), rcond=None)
    assert rel_err(got, e.astype(np.float64) @ x) <= 2 * 0.0091
    assert d.generate_tokens(p[:12], 6)[0][0] == int(np.argmax(d.prefill(p[:12])))
    d.close()
    full.close()


def test_bundle_gives_the_same_bits(itts, qw, dec, tmp_path):
    path = itts.write_mit2_bundle(tmp_path / "qwen.mit2", qw, single_file=True)
    b = itts.Bundle(path, require_model=False)
    d = itts.QwenDecoder.from_bundle(b, layers=LAYERS, weight_bits=4)
    b.close()
    p = ids_of(33, 24)
    assert np.array_equal(dec.prefill(p[:20]), d.prefill(p[:20]))
    assert np.array_equal(dec.step(p[20]), d.step(p[20]))
    d.close()
