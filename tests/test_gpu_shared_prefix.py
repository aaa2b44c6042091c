"""Sequences that share cache pages through the engine, the sampler and the command line: the same logits and tokens as without."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_util import assert_close, make_engine, model_folder, plain_logits, random_tokens
from qwen_triton_b200 import QwenB200ForCausalLM, SamplingParams, StepEntry
from qwen_triton_b200.ops import kernels
from qwen_triton_b200.sampling import uniform_for
from qwen_triton_b200.sampling.sampler import Sampler

pytestmark = pytest.mark.gpu
PRESETS = ("tiny-a", "tiny-b", "tiny-d")


@pytest.fixture
def always_shared(monkeypatch):
    """One-token steps take the shared kernels however little is shared; the calls are counted."""
    calls = []
    real = kernels.attention_decode_shared
    monkeypatch.setattr(kernels, "sharing_pays", lambda *args: True)
    monkeypatch.setattr(kernels, "attention_decode_shared", lambda *args, **kw: (calls.append(1), real(*args, **kw))[1])
    return calls


@pytest.mark.parametrize("preset", PRESETS)
@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
def test_logits_of_sequences_that_share(preset, dtype, always_shared):
    """Two groups and a sequence by itself, stepped token by token (launched, captured and replayed), then after the one they took it from has ended."""
    engine = make_engine(preset, dtype, max_tokens=4096)
    prompts = [random_tokens(preset, 200, 1), random_tokens(preset, 70, 2), random_tokens(preset, 33, 3)]
    first = [engine.new_sequence() for _ in prompts]
    engine.step([StepEntry(s, p, []) for s, p in zip(first, prompts)])
    history = {s: list(p) for s, p in zip(first, prompts)}
    for source, tokens in ((0, 192), (0, 128), (1, 64)):
        slot = engine.new_sequence(first[source], tokens)
        history[slot] = prompts[source][:tokens]
    order = [first[1], *[s for s in history if s not in first], first[0], first[2]]
    for step in range(5):
        if step == 4:
            engine.release(first[0])
            order.remove(first[0])
        tokens = [random_tokens(preset, 1, 100 * step + i)[0] for i in range(len(order))]
        logits = engine.step([StepEntry(s, [t], [0]) for s, t in zip(order, tokens)]).cpu()
        for row, (slot, token) in enumerate(zip(order, tokens)):
            history[slot].append(token)
            assert_close(logits[row:row + 1], plain_logits(preset, dtype, history[slot])[-1:], dtype, f"{preset} {dtype} step {step} row {row}")
    assert always_shared
    engine.check_kernels()
    for slot in order:
        engine.release(slot)
    engine.cache.book.check()


@pytest.mark.parametrize("preset", PRESETS)
def test_generation_with_a_shared_prefix(preset, always_shared):
    """float32, greedy: the same tokens, with fewer pages and the prefix run once."""
    model = QwenB200ForCausalLM.from_pretrained_hf(model_folder(preset, "fp32"), dtype="fp32", max_tokens=4096)
    start = random_tokens(preset, 150, 7)
    prompts = [start + random_tokens(preset, 3 + 2 * i, 8 + i) for i in range(5)]
    plain = model.generate(prompts, max_new_tokens=6, ignore_eos=True)
    assert not always_shared
    shared = model.generate(prompts, max_new_tokens=6, ignore_eos=True, share_prefix=True)
    assert [r.tokens for r in shared] == [r.tokens for r in plain]
    assert always_shared
    assert not model.engine.cache.book.live_slots()
    model.engine.cache.book.check()


def test_models_that_cannot_share():
    """A windowed group: nothing is shared, and generation is what it is without asking."""
    model = QwenB200ForCausalLM.from_pretrained_hf(model_folder("tiny-c", "fp32"), dtype="fp32", max_tokens=2048)
    assert not model.engine.can_share
    slot = model.engine.new_sequence()
    model.engine.step([StepEntry(slot, random_tokens("tiny-c", 130, 1), [])])
    with pytest.raises(RuntimeError, match="pages"):
        model.engine.new_sequence(slot, 64)
    model.engine.release(slot)
    prompts = [random_tokens("tiny-c", 140, 2)] * 2
    assert [r.tokens for r in model.generate(prompts, max_new_tokens=4, share_prefix=True)] == [r.tokens for r in model.generate(prompts, max_new_tokens=4)]


def test_continuations_are_ranked_and_reproducible():
    model = QwenB200ForCausalLM.from_pretrained_hf(model_folder("tiny-b", "bf16"), dtype="bf16", max_tokens=8192)
    prompt = random_tokens("tiny-b", 300, 3)
    options = dict(max_new_tokens=8, temperature=0.9, seed=5, top_k=40, min_p=0.01, ignore_eos=True)
    results = model.continuations(prompt, 6, **options)
    means = [sum(r.logprobs) / len(r.logprobs) for r in results]
    assert means == sorted(means, reverse=True) and all(len(r.tokens) == len(r.logprobs) == 8 for r in results)
    assert len({tuple(r.tokens) for r in results}) > 1                       # each request has numbers of its own
    assert [r.tokens for r in model.continuations(prompt, 6, **options)] == [r.tokens for r in results]
    with pytest.raises(ValueError):
        model.continuations(prompt, 0)


def test_the_sampler_takes_parameters_of_each_row():
    """Against the choice formed here from the definition, with numbers far from every boundary left as they come."""
    gen = torch.Generator().manual_seed(3)
    logits = 3 * torch.randn((40, 503), generator=gen)
    params = [SamplingParams(temperature=(0.0, 0.7, 1.0, 1.4)[i % 4], seed=i, top_k=(0, 20)[i % 2], top_p=(1.0, 0.9)[i // 2 % 2], min_p=(0.0, 0.05)[i // 3 % 2],
                             logprobs=True) for i in range(40)]
    sampler = Sampler(torch.device("cuda:0"))
    for round_number in range(6):                                            # more rounds than there are buffers
        requests, steps = list(range(40)), [round_number] * 40
        pending = sampler.launch(logits.cuda(), params, requests, steps)
        tokens, logprobs = pending.tokens(), pending.logprobs()
        for row, p in enumerate(params):
            x = logits[row].double()
            if p.temperature == 0:
                assert tokens[row] == int(x.argmax()) and logprobs[row] == 0.0
                continue
            y = (x - x.max()) / p.temperature
            w = y.exp()
            order = x.argsort(descending=True)                               # no two logits are equal
            rank = torch.empty_like(order).scatter_(0, order, torch.arange(503))
            keep = rank < p.top_k if p.top_k else torch.ones(503, dtype=torch.bool)
            if p.top_p < 1:
                mass = torch.where(keep, w, 0.0)
                before = torch.empty_like(w).scatter_(0, order, mass[order].cumsum(0) - mass[order])
                keep &= before < p.top_p * mass.sum()
            keep &= w >= p.min_p
            running = torch.where(keep, w, 0.0).cumsum(0)
            target = uniform_for(p.seed, row, round_number) * running[-1]
            near = float(((running - target).abs() / running[-1]).min())
            if near < 1e-5:
                continue
            want = int((running > target).nonzero()[0])
            assert tokens[row] == want
            assert abs(logprobs[row] - float(y[want] - running[-1].log())) < 1e-4
    same = [SamplingParams(temperature=0.8, seed=4, top_k=7)] * 40           # alike and nothing new: the kernel that was there
    a = sampler.launch(logits.cuda(), same, list(range(40)), [0] * 40)
    b = sampler.launch(logits.cuda(), same[0], list(range(40)), [0] * 40)
    assert a.tokens() == b.tokens() and a.logprobs() is None
    with pytest.raises(ValueError, match="parameters"):
        sampler.launch(logits.cuda(), same[:3], list(range(40)), [0] * 40)


def test_command_line(capsys):
    from qwen_triton_b200.scripts import smoke
    smoke.main(["--preset", "tiny-b", "--random-weights", "--seed", "3", "--random-prompts", "150", "--samples", "3", "--temperature", "0.8", "--min-p", "0.02",
                "--max-new-tokens", "4", "--ignore-eos"])
    lines = [line for line in capsys.readouterr().out.splitlines() if line.startswith("generated=")]
    means = [float(line.rsplit("=", 1)[1]) for line in lines]
    assert len(lines) == 3 and means == sorted(means, reverse=True) and all(math.isfinite(m) for m in means)
