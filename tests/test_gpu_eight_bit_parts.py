"""A layer's attention and its feed-forward, each by itself, with weights (and keys and values) in 8 bits and bfloat16 activations: against 64 bits with every rounding where
the layer has it, gate and up in turns as the layer keeps them, and against the same without the roundings to 8 bits."""
import dataclasses

import pytest
import torch

import plain_8bit
import plain_qwen3 as plain
from gpu_util import random_tokens
from qwen_triton_b200 import Engine, StepEntry, load_preset, write_random_model
from qwen_triton_b200.ops import kernels
from qwen_triton_b200.weights import Checkpoint

pytestmark = pytest.mark.gpu
WEIGHTS, BOTH = {"weight_format": "fp8"}, {"weight_format": "fp8", "cache_format": "fp8"}
LOUDER = 16.0                 # the part under test outweighs the embedding that it is added to


def model(preset, part, folder):
    """(config, weights) of one layer in bfloat16, whose other part adds nothing."""
    config = dataclasses.replace(load_preset(preset), num_hidden_layers=1, layer_types=load_preset(preset).layer_types[:1])
    write_random_model(folder, config, 4, torch.bfloat16)
    checkpoint = Checkpoint(folder)
    weights = {name: checkpoint.read(name) for name in checkpoint.names()}
    quiet, loud = ("self_attn.o_proj", "mlp.down_proj") if part == "feed-forward" else ("mlp.down_proj", "self_attn.o_proj")
    for name in weights:
        if quiet in name:
            weights[name] = torch.zeros_like(weights[name])
        elif loud in name:
            weights[name] = weights[name] * LOUDER
    return config, weights


def statement(config, weights, tokens, formats, eight=True, work=torch.float64):
    """Logits.  ``eight`` False: the same without the roundings to 8 bits.  Products with a bias stay in float up to what reads them; all others are bfloat16."""
    w = {name: t.to(work) for name, t in weights.items()}
    cfg = plain.read_config(config.to_hf_dict())
    d, heads, kv_heads, biased = cfg["head_dim"], cfg["heads"], cfg["kv_heads"], cfg["attention_bias"]

    def kept(x):
        return x.to(torch.bfloat16).to(work)

    def linear(x, matrix, bias=None):
        if eight:
            y = plain_8bit.product(*plain_8bit.quantise_rows(x), *plain_8bit.quantise_weight(matrix))[0].to(work)
        else:
            y = x @ matrix.T
        return kept(y) if bias is None else y + bias

    def held(rows):
        if not eight or "cache_format" not in formats:
            return kept(rows)
        out = rows.clone()
        for first in range(0, len(rows), 64):
            for h in range(kv_heads):
                piece = rows[first:first + 64, h]
                scale = 2.0 ** plain_8bit.power_for(float(piece.abs().max()))
                out[first:first + 64, h] = plain_8bit.as_e4m3(piece / scale).to(work) * scale
        return out

    a, m = "model.layers.0.self_attn", "model.layers.0.mlp"
    x = w["model.embed_tokens.weight"][torch.tensor(tokens)]
    cos, sin = plain.rope_tables(torch.arange(len(tokens)), cfg["rotary_dim"], cfg["theta"], torch.float64)
    h = kept(plain.rms_norm(x, w["model.layers.0.input_layernorm.weight"], cfg["eps"]))
    bias = torch.cat([w[f"{a}.{n}_proj.bias"] for n in "qkv"]) if biased else None
    qkv = linear(h, torch.cat([w[f"{a}.{n}_proj.weight"] for n in "qkv"]), bias).view(len(tokens), heads + 2 * kv_heads, d)
    q = kept(plain.apply_rope(plain.rms_norm(qkv[:, :heads], w[f"{a}.q_norm.weight"], cfg["eps"]), cos.to(work), sin.to(work)))
    k = plain.apply_rope(plain.rms_norm(qkv[:, heads:heads + kv_heads], w[f"{a}.k_norm.weight"], cfg["eps"]), cos.to(work), sin.to(work))
    out = kept(plain.attention_scores(q, held(k), held(qkv[:, heads + kv_heads:]), d ** -0.5, None)).reshape(len(tokens), heads * d)
    x = x + linear(out, w[f"{a}.o_proj.weight"], w[f"{a}.o_proj.bias"] if biased else None)
    h = kept(plain.rms_norm(x, w["model.layers.0.post_attention_layernorm.weight"], cfg["eps"]))
    inter, hidden = cfg["intermediate"], cfg["hidden"]
    group = kernels.SWIGLU_GROUP if inter % kernels.SWIGLU_GROUP == 0 and hidden % 8 == 0 else 0
    gate_up = linear(h, kernels.interleave_gate_up(w[f"{m}.gate_proj.weight"], w[f"{m}.up_proj.weight"], group))
    gate, up = gate_up.view(len(tokens), -1, 2, group).unbind(2) if group else gate_up.chunk(2, dim=1)
    gate, up = gate.reshape(len(tokens), inter), up.reshape(len(tokens), inter)
    x = x + linear(kept(gate * torch.sigmoid(gate) * up), w[f"{m}.down_proj.weight"])
    x = kept(plain.rms_norm(x, w["model.norm.weight"], cfg["eps"]))
    return x @ (w["model.embed_tokens.weight"] if cfg["tied"] else w["lm_head.weight"]).T


def rows_off(a, b):
    return ((a.double() - b.double()).norm(dim=1) / b.double().norm(dim=1)).cpu()


# How far the layer may be from the statement, as a part of what the roundings to 8 bits amount to (0.05 for the feed-forward, 0.015 to 0.08 for attention, mean of rows).
# Feed-forward: float32's sums are off by some 2^-20 of a number, so that 2^-20 / 2^-8 of a row's 500 numbers fall on the other side of a border between bfloat16 numbers, one in
# eight rows; it moves by 2^-8, and in one of 16 cases across a border between 8-bit numbers, by 2^-3: of some 64 numbers of a row, 1/8 * (2^-8 + 2^-3 / 16) / 8 = 2e-4.
# Attention: its weights are halves, so that its results are off by up to 2^-12.  1/16 of them fall on the other side of a bfloat16 border, 1/256 on that of an 8-bit one, by
# 2^-3.5 in the mean square: sqrt(1 / 256) * 2^-3.5 = 0.0055 of the product, where the roundings in three places amount to sqrt(3) * 0.026, eight times that.
PART = {"feed-forward": 1 / 20, "attention": 1 / 5}


@pytest.mark.parametrize("part,formats", [("feed-forward", WEIGHTS), ("attention", WEIGHTS), ("attention", BOTH)], ids=lambda v: v if isinstance(v, str) else "+".join(sorted(v)))
@pytest.mark.parametrize("preset", ["tiny-a", "tiny-b", "tiny-d"])
def test_a_part_rounds_where_the_statement_does(preset, part, formats, tmp_path):
    """Whole prompts, and steps of one token behind a prompt."""
    config, weights = model(preset, part, tmp_path)
    tokens = random_tokens(preset, 150, 1)
    want, without = statement(config, weights, tokens, formats), statement(config, weights, tokens, formats, eight=False)
    effect = float(rows_off(without, want).mean())
    assert effect > 0.01

    def logits(**kwargs):
        engine = Engine(config.model_spec(), lambda name: weights[name], dtype="bf16", max_tokens=1024, **kwargs)
        slot = engine.new_sequence()
        whole = engine.step([StepEntry(slot, tokens, list(range(150)))]).cpu()
        engine.release(slot)
        slot = engine.new_sequence()
        steps = [engine.step([StepEntry(slot, tokens[:130], list(range(130)))]).cpu()]
        steps += [engine.step([StepEntry(slot, [t], [0])]).cpu() for t in tokens[130:]]
        engine.check_kernels()
        return whole, torch.cat(steps)

    for got in logits(**formats):
        assert float(rows_off(got, want).mean()) < PART[part] * effect
    for got in logits():                                   # what is asked above can be told from a layer in 16 bits
        assert float(rows_off(got, want).mean()) > effect / 2
