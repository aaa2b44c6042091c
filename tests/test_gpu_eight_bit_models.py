"""Models whose projections' weights, or whose keys and values, are kept in 8 bits: through the engine, the generation loop and the command line, against the same model
written out in 64 bits with the same roundings to 8 bits."""
import dataclasses
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import plain_8bit
import plain_qwen3 as plain
from gpu_util import model_folder, oracle, random_tokens, run_whole
from qwen_triton_b200 import Engine, QwenB200ForCausalLM, StepEntry, load_preset, write_random_model
from qwen_triton_b200.weights import Checkpoint

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
BOTH = {"weight_format": "fp8", "cache_format": "fp8"}
FORMATS = [{"weight_format": "fp8"}, {"cache_format": "fp8"}, BOTH]


def _names(formats):
    return "+".join(sorted(formats))


def engine8(preset, dtype, formats, **kwargs):
    kwargs.setdefault("max_tokens", 4096)
    return Engine.from_pretrained(model_folder(preset, dtype), dtype=dtype, **formats, **kwargs)


def plain_logits8(preset, dtype, tokens, formats):
    """The model in float64 with the same roundings to 8 bits: one weight of [q; k; v], one of [gate; up], as the layers keep them in float32; a page's keys
    and values under the scale of its largest number."""
    raw, weights = oracle(preset, dtype)
    w = {name: t.double() for name, t in weights.items()}
    cfg = plain.read_config(raw)
    d, heads, kv_heads = cfg["head_dim"], cfg["heads"], cfg["kv_heads"]

    def linear(x, matrix, bias=None):
        y = plain_8bit.product(*plain_8bit.quantise_rows(x), *plain_8bit.quantise_weight(matrix))[0] if "weight_format" in formats else x @ matrix.T
        return y if bias is None else y + bias

    def held(rows):
        """[tokens, kv_heads, d] as the cache gives them back."""
        if "cache_format" not in formats:
            return rows
        out = rows.clone()
        for first in range(0, len(rows), 64):
            for h in range(kv_heads):
                part = rows[first:first + 64, h]
                scale = 2.0 ** plain_8bit.power_for(float(part.abs().max()))
                out[first:first + 64, h] = plain_8bit.as_e4m3(part / scale) * scale
        return out

    x = w["model.embed_tokens.weight"][torch.tensor(tokens)]
    cos, sin = plain.rope_tables(torch.arange(len(tokens)), cfg["rotary_dim"], cfg["theta"], torch.float64)
    for i in range(cfg["layers"]):
        p = f"model.layers.{i}"
        a = f"{p}.self_attn"
        h = plain.rms_norm(x, w[f"{p}.input_layernorm.weight"], cfg["eps"])
        bias = torch.cat([w[f"{a}.{n}_proj.bias"] for n in "qkv"]) if cfg["attention_bias"] else None
        qkv = linear(h, torch.cat([w[f"{a}.{n}_proj.weight"] for n in "qkv"]), bias).view(len(tokens), heads + 2 * kv_heads, d)
        q = plain.apply_rope(plain.rms_norm(qkv[:, :heads], w[f"{a}.q_norm.weight"], cfg["eps"]), cos, sin)
        k = plain.apply_rope(plain.rms_norm(qkv[:, heads:heads + kv_heads], w[f"{a}.k_norm.weight"], cfg["eps"]), cos, sin)
        out = plain.attention_scores(q, held(k), held(qkv[:, heads + kv_heads:]), d ** -0.5, None).reshape(len(tokens), heads * d)
        x = x + linear(out, w[f"{a}.o_proj.weight"], w[f"{a}.o_proj.bias"] if cfg["attention_bias"] else None)
        h = plain.rms_norm(x, w[f"{p}.post_attention_layernorm.weight"], cfg["eps"])
        gate, up = linear(h, torch.cat((w[f"{p}.mlp.gate_proj.weight"], w[f"{p}.mlp.up_proj.weight"]))).chunk(2, dim=1)
        x = x + linear(gate * torch.sigmoid(gate) * up, w[f"{p}.mlp.down_proj.weight"])
    x = plain.rms_norm(x, w["model.norm.weight"], cfg["eps"])
    return x @ (w["model.embed_tokens.weight"] if cfg["tied"] else w["lm_head.weight"]).T


def off(a, b):
    return float((a.double().cpu() - b.double().cpu()).norm() / b.double().cpu().norm())


# One layer in float32.  A number that float32 leaves within its error (some 2^-21 of it, of steps of 2^-4 to 2^-3) of a border between two 8-bit numbers may fall on the
# other side: of the some 10^5 numbers that 150 tokens bring to 8 bits in a layer, 10^5 * 2^-21 / 2^-4 = 0.8.  One that does moves its row of the product (K >= 64) by at most
# 2^-3 / sqrt(64) = 1.6 %, after which the row's later numbers cross borders too, until the row is off by two independent roundings in each of seven places (q, k, v's
# input, k, v, the output's, the MLP's, its product's two factors): sqrt(7 * 2 * 0.026^2) = 10 %.  Four such rows of 150 are sqrt(4 / 150) * 10 % = 1.6 % of the whole.
ONE_LAYER = 0.016


def off_after(layers):
    """Several layers, or other cuts of a prompt (a page's numbers held under a smaller scale first), or bfloat16: once any number has crossed a border, each crossing
    makes more: numbers d apart, relative to themselves, lie on two sides of a border in d / step of the cases, so their distance in the mean square grows from d^2 to
    d * step, up to two independent roundings (2 * 0.026^2).  That fixed point is reached within a layer or two from any start, so the distance is bounded by the
    roundings alone: seven places of a layer, as above, whose squares add up along the layers."""
    return (layers * 7 * 2 * 0.026 ** 2) ** 0.5


@pytest.mark.parametrize("formats", FORMATS, ids=_names)
@pytest.mark.parametrize("preset", ["tiny-a", "tiny-b", "tiny-d"])
def test_one_layer(preset, formats, tmp_path, monkeypatch):
    config = dataclasses.replace(load_preset(preset), num_hidden_layers=1, layer_types=load_preset(preset).layer_types[:1])
    write_random_model(tmp_path, config, 4, torch.float32)
    checkpoint = Checkpoint(tmp_path)
    weights = {name: checkpoint.read(name) for name in checkpoint.names()}
    monkeypatch.setitem(globals(), "oracle", lambda *args: (config.to_hf_dict(), weights))
    tokens = random_tokens(preset, 150, 1)
    want = plain_logits8(preset, "fp32", tokens, formats)
    logits = run_whole(Engine.from_pretrained(tmp_path, dtype="fp32", max_tokens=1024, **formats), tokens)
    assert off(logits, want) < ONE_LAYER
    rows = (logits.double().cpu() - want).norm(dim=1) / want.norm(dim=1)
    assert float(rows.median()) < 1e-3                                     # most rows meet no border at all


@pytest.mark.parametrize("formats", FORMATS, ids=_names)
@pytest.mark.parametrize("preset", ["tiny-a", "tiny-b", "tiny-d"])
def test_logits_are_those_of_the_model_in_8_bits(preset, formats):
    tokens = random_tokens(preset, 150, 1)
    logits = run_whole(engine8(preset, "fp32", formats), tokens)
    want = plain_logits8(preset, "fp32", tokens, formats)
    assert off(logits, want) < off_after(load_preset(preset).num_hidden_layers)
    # and not those of the model without: these are further off than float32's own error by far
    assert off(plain_logits8(preset, "fp32", tokens, {}), want) > 1e-3


@pytest.mark.parametrize("formats", FORMATS, ids=_names)
@pytest.mark.parametrize("preset", ["tiny-a", "tiny-b", "tiny-d"])
def test_logits_in_bfloat16(preset, formats):
    """Prompts and single tokens.  Here a weight's rows lie otherwise (gate and up in turns), so that its blocks' scales are others: four more roundings a layer,
    independent of the statement's; and bfloat16 itself, some ten roundings of 2^-9 a layer."""
    layers = load_preset(preset).num_hidden_layers
    close = (layers * 11 * 2 * 0.026 ** 2) ** 0.5 + (10 * layers) ** 0.5 * 2 ** -9
    tokens = random_tokens(preset, 80, 1)
    want = plain_logits8(preset, "bf16", tokens, formats)
    engine = engine8(preset, "bf16", formats)
    assert off(run_whole(engine, tokens), want) < close
    slot = engine.new_sequence()
    got = [engine.step([StepEntry(slot, tokens[:60], list(range(60)))]).cpu()]
    got += [engine.step([StepEntry(slot, [t], [0])]).cpu() for t in tokens[60:]]
    assert off(torch.cat(got), want) < close


@pytest.mark.parametrize("preset", ["tiny-a", "tiny-b", "tiny-d"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_steps_give_the_logits_of_whole_prompts(preset, dtype):
    """Prompts of unequal lengths in pieces, then single tokens across a page's end, launched, captured and replayed, beside a prompt by itself: but for the
    roundings to 8 bits the logits do not depend on the cuts."""
    close = off_after(load_preset(preset).num_hidden_layers)
    engine = engine8(preset, dtype, BOTH)
    tokens = [random_tokens(preset, n, i) for i, n in enumerate((110, 75, 140))]
    whole = [run_whole(engine, t) for t in tokens]
    slots = [engine.new_sequence() for _ in tokens]
    got = [[] for _ in tokens]
    done = [0, 0, 0]
    for count in (40, 20, 5):
        logits = engine.step([StepEntry(s, t[a:a + count], list(range(count))) for s, t, a in zip(slots, tokens, done)])
        for i in range(3):
            got[i].append(logits[i * count:(i + 1) * count].cpu())
            done[i] += count
    while any(a < len(t) for a, t in zip(done, tokens)):
        live = [i for i in range(3) if done[i] < len(tokens[i])]
        logits = engine.step([StepEntry(slots[i], [tokens[i][done[i]]], [0]) for i in live])
        for row, i in enumerate(live):
            got[i].append(logits[row:row + 1].cpu())
            done[i] += 1
    assert engine.graph_replays > 10
    for pieces, want in zip(got, whole):
        assert off(torch.cat(pieces), want) < close
    engine.check_kernels()


def test_slots_and_pages_are_used_again():
    """A page of a released sequence starts anew: a new sequence's logits are those of a fresh engine, whatever the page held."""
    fresh = engine8("tiny-a", "fp32", BOTH)
    used = engine8("tiny-a", "fp32", BOTH, max_tokens=256)
    for seed in range(4):
        run_whole(used, random_tokens("tiny-a", 250, seed))
    tokens = random_tokens("tiny-a", 200, 9)
    assert torch.equal(run_whole(used, tokens), run_whole(fresh, tokens))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_generation_and_shared_prefixes(dtype):
    """Greedy tokens alone and behind shared pages are the same; continuations run; what is kept is half as large or less."""
    model = QwenB200ForCausalLM.from_pretrained_hf(model_folder("tiny-b", dtype), dtype=dtype, max_tokens=4096, **BOTH)
    plain_model = QwenB200ForCausalLM.from_pretrained_hf(model_folder("tiny-b", dtype), dtype=dtype, max_tokens=4096)
    start = random_tokens("tiny-b", 130, 5)
    prompts = [start + random_tokens("tiny-b", n, n) for n in (3, 20, 7)]
    alone = [r.tokens for r in model.generate(prompts, max_new_tokens=6, ignore_eos=True)]
    shared = [r.tokens for r in model.generate(prompts, max_new_tokens=6, ignore_eos=True, share_prefix=True)]
    assert [len(t) for t in alone] == [6, 6, 6] and alone == shared
    assert len(model.continuations(start, 3, max_new_tokens=5, temperature=0.9, seed=2)) == 3
    small, large = model.engine.memory_report(), plain_model.engine.memory_report()
    size = 4 if dtype == "fp32" else 2
    assert small["cache"] < large["cache"] / size * 1.05 and small["weights"] < large["weights"]
    assert model.engine.cache.token_bytes() * size == plain_model.engine.cache.token_bytes()


def test_the_command_line_takes_the_formats():
    out = subprocess.run([sys.executable, "-m", "qwen_triton_b200.scripts.smoke", "--model-id", str(model_folder("tiny-a", "bf16")), "--prompt-ids", "5,17,3", "--prompt-ids", "9,1",
                          "--max-new-tokens", "4", "--weight-format", "fp8", "--cache-format", "fp8", "--compare-ref"], cwd=ROOT, capture_output=True, text=True, timeout=900)
    assert out.returncode == 0 and out.stdout.count("generated=") == 2 and "logit_max_abs_diff" in out.stdout


def test_refusals():
    folder = model_folder("tiny-a", "bf16")
    with pytest.raises(ValueError, match="neither None nor"):
        Engine.from_pretrained(folder, weight_format="int8")
    with pytest.raises(ValueError, match="8 bits goes with"):
        engine8("tiny-c", "bf16", {"cache_format": "fp8"})                 # a sliding window
    with pytest.raises(ValueError, match="8 bits goes with"):
        engine8("tiny-a", "bf16", {"cache_format": "fp8"}, page_tokens=16)
    with pytest.raises(ValueError, match="another layer"):
        Engine.from_config(load_preset("misudra-tiny-a"), cache_format="fp8")
    engine8("tiny-c", "bf16", {"weight_format": "fp8"})
