"""One-token steps over shared pages as the engine runs them: launched, captured and replayed, by the form that a step takes for itself."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from gpu_util import assert_close, make_engine, plain_logits, random_tokens
from qwen_triton_b200 import Engine, StepEntry, load_preset
from qwen_triton_b200.cache import CacheError
from qwen_triton_b200.ops import kernels

pytestmark = pytest.mark.gpu


@pytest.fixture
def plans(monkeypatch):
    """The plans of the shared calls that steps make."""
    seen = []
    real = kernels.attention_decode_shared
    monkeypatch.setattr(kernels, "attention_decode_shared", lambda *args: (seen.append(args[11]), real(*args))[1])
    return seen


@pytest.mark.parametrize("preset", ("tiny-a", "tiny-b", "tiny-d"))
def test_two_launches_in_a_captured_step(preset, plans, monkeypatch):
    """bfloat16 on the tensor cores, small sizes made to take the form of large ones: two groups and one sequence in seven rows, padded to eight."""
    monkeypatch.setattr(kernels, "sharing_pays", lambda *args: True)
    monkeypatch.setattr(kernels, "DIRECT_BYTES", 0)
    engine = make_engine(preset, "bf16", max_tokens=4096)
    prompts = [random_tokens(preset, 300, 1), random_tokens(preset, 70, 2), random_tokens(preset, 33, 3)]
    first = [engine.new_sequence() for _ in prompts]
    engine.step([StepEntry(s, p, []) for s, p in zip(first, prompts)])
    history = {s: list(p) for s, p in zip(first, prompts)}
    for source, tokens in ((0, 256), (0, 256), (0, 192), (1, 64)):
        history[engine.new_sequence(first[source], tokens)] = prompts[source][:tokens]
    order = [first[1], *[s for s in history if s not in first], first[0], first[2]]
    assert len(order) == 7
    for step in range(5):
        tokens = [random_tokens(preset, 1, 100 * step + i)[0] for i in range(len(order))]
        logits = engine.step([StepEntry(s, [t], [0]) for s, t in zip(order, tokens)]).cpu()
        for row, (slot, token) in enumerate(zip(order, tokens)):
            history[slot].append(token)
            assert_close(logits[row:row + 1], plain_logits(preset, "bf16", history[slot])[-1:], "bf16", f"{preset} step {step} row {row}")
    assert plans and all(plan.shared_ranges > 0 for plan in plans)
    assert engine.graph_replays >= 3
    engine.check_kernels()


def steps_of(engine, shared, members, alone, steps=4):
    """Logits of ``steps`` steps of ``members`` sequences that took ``shared`` tokens of the first, and of ``alone`` more by themselves."""
    preset = "tiny-d"
    first = engine.new_sequence()
    engine.step([StepEntry(first, random_tokens(preset, shared + 5, 1), [])])
    slots = [first] + [engine.new_sequence(first, shared) for _ in range(members - 1)]
    apart = [engine.new_sequence() for _ in range(alone)]
    if apart:
        engine.step([StepEntry(s, random_tokens(preset, 90 + i, 2 + i), []) for i, s in enumerate(apart)])
    out = []
    for step in range(steps):
        entries = [StepEntry(s, [random_tokens(preset, 1, 1000 * step + i)[0]], [0]) for i, s in enumerate(slots + apart)]
        out.append(engine.step(entries).cpu())
    shape = engine._plan_decode(slots + apart, True).key[3]
    for slot in slots + apart:
        engine.release(slot)
    engine.check_kernels()
    return out, shape


@pytest.mark.parametrize("dtype, heads, kv_heads, dim, shared, members, alone", [
    ("bf16", 5, 5, 64, 1920, 32, 0), ("bf16", 5, 5, 64, 1920, 30, 6), ("bf16", 8, 4, 128, 1856, 16, 3), ("fp32", 5, 5, 64, 1920, 32, 3), ("fp32", 4, 2, 128, 512, 3, 2)])
def test_a_step_shares_of_itself_where_it_pays(dtype, heads, kv_heads, dim, shared, members, alone, plans, monkeypatch):
    """The rule as it is: the step takes the shared form in two launches, and gives what it gives without."""
    config = dataclasses.replace(load_preset("tiny-d"), num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=dim)
    engine = Engine.from_config(config, seed=4, dtype=dtype, max_tokens=8192)
    got, shape = steps_of(engine, shared, members, alone)
    assert shape is not None and plans and all(plan.shared_ranges > 0 and plan.head_dim == dim for plan in plans)
    count = len(plans)
    monkeypatch.setattr(kernels, "sharing_pays", lambda *args: False)
    want, shape = steps_of(engine, shared, members, alone)
    assert shape is None and len(plans) == count
    for step, (a, b) in enumerate(zip(got, want)):
        assert_close(a, b, dtype, f"step {step}")


@pytest.mark.parametrize("shared, members, alone", [(64, 2, 14), (1920, 2, 30), (1920, 8, 56)])
def test_a_step_that_shares_little_is_a_step_like_any_other(shared, members, alone, plans):
    """No shared call, and no shape of groups under which a graph of its own would be kept."""
    engine = make_engine("tiny-d", "bf16", max_tokens=16384)
    _, shape = steps_of(engine, shared, members, alone, steps=2)
    assert shape is None and not plans


def test_a_position_that_is_planned_and_has_not_run_is_not_shared():
    """Its keys and values are not there yet."""
    engine = make_engine("tiny-d", "fp32")
    prompt = random_tokens("tiny-d", 127, 5)
    slot = engine.new_sequence()
    engine.step([StepEntry(slot, prompt, [])])
    plan = engine.plan_decode([slot])
    assert engine.length(slot) == 128
    with pytest.raises(CacheError, match="127 have run"):
        engine.new_sequence(slot, 128)
    early = engine.new_sequence(slot)
    assert engine.length(early) == 64
    plan = engine.plan_decode([slot], extend=False)               # planned again: still not run
    with pytest.raises(CacheError, match="127 have run"):
        engine.new_sequence(slot, 128)
    token = random_tokens("tiny-d", 1, 6)
    engine.run_planned(plan, token)
    late = engine.new_sequence(slot)
    assert engine.length(late) == 128
    logits = engine.step([StepEntry(early, prompt[64:100], [35]), StepEntry(late, [7, 9], [1])])
    assert_close(logits[:1], plain_logits("tiny-d", "fp32", prompt[:100])[-1:], "fp32", "taken before the step")
    assert_close(logits[1:], plain_logits("tiny-d", "fp32", prompt + token + [7, 9])[-1:], "fp32", "taken behind it")
    for s in (slot, early, late):
        engine.release(s)
    engine.plan_decode([again := engine.new_sequence()])
    engine.release(again)                                         # a slot's next sequence has nothing of a plan that never ran
    slot = engine.new_sequence()
    engine.step([StepEntry(slot, prompt[:64], [])])
    assert engine.length(engine.new_sequence(slot)) == 64
    engine.cache.book.check()


def test_a_batch_keeps_its_kernel_while_requests_end(monkeypatch):
    """Rows with parameters of their own go through one kernel, also when those that are left are alike."""
    from qwen_triton_b200 import SamplingParams
    from qwen_triton_b200.sampling.sampler import Sampler
    calls = []
    for name in ("argmax", "sample_keyed", "sample_filtered"):
        real = getattr(kernels, name)
        monkeypatch.setattr(kernels, name, lambda *args, _name=name, _real=real: (calls.append(_name), _real(*args))[1])
    logits = torch.randn((3, 500), generator=torch.Generator().manual_seed(1)).cuda()
    sampler = Sampler(torch.device("cuda:0"))
    alike, other = SamplingParams(temperature=0.8, top_p=0.9), SamplingParams()
    sampler.sample(logits, [alike, other, alike], [0, 1, 2], [0] * 3)
    sampler.sample(logits[:2], [alike, alike], [0, 2], [1] * 2)
    sampler.sample(logits[:1], [other], [1], [1])
    assert calls == ["sample_filtered"] * 3
    sampler.sample(logits, alike, [0, 1, 2], [0] * 3)               # one for all rows: as without a list
    sampler.sample(logits, other, [0, 1, 2], [0] * 3)
    assert calls[3:] == ["sample_keyed", "argmax"]
    assert sampler.sample(logits[:0], [], [], []) == []


def test_the_command_keeps_its_batch_size(monkeypatch, capsys):
    import importlib
    loop = importlib.import_module("qwen_triton_b200.engine.generate")
    from qwen_triton_b200.scripts import smoke
    batches = []
    real = loop.BatchRun
    monkeypatch.setattr(loop, "BatchRun", lambda *args, **kw: (batches.append(list(args[4])), real(*args, **kw))[1])
    smoke.main(["--preset", "tiny-b", "--random-weights", "--random-prompts", "150", "--samples", "5", "--max-batch-size", "2", "--temperature", "0.8",
                "--max-new-tokens", "3", "--ignore-eos"])
    assert batches == [[0, 1], [2, 3], [4]]
    assert sum(line.startswith("generated=") for line in capsys.readouterr().out.splitlines()) == 5


@pytest.mark.parametrize("asked, different", [([], True), (["--temperature", "0"], False)])
def test_the_command_draws_its_samples(asked, different, capsys):
    """Without a temperature, several samples are drawn at 1; none of them at 0."""
    from qwen_triton_b200.scripts import smoke
    smoke.main(["--preset", "tiny-b", "--random-weights", "--random-prompts", "90", "--samples", "4", "--max-new-tokens", "6", "--ignore-eos", *asked])
    lines = {line.split(" finish")[0] for line in capsys.readouterr().out.splitlines() if line.startswith("generated=")}
    assert len(lines) == (4 if different else 1)


def test_a_batch_step_by_step_has_the_options_of_generate():
    from gpu_util import model_folder
    from qwen_triton_b200 import QwenB200ForCausalLM
    model = QwenB200ForCausalLM.from_pretrained_hf(model_folder("tiny-b", "fp32"), dtype="fp32", max_tokens=4096)
    start = random_tokens("tiny-b", 150, 7)
    prompts = [start + random_tokens("tiny-b", 3 + i, 8 + i) for i in range(3)]
    options = dict(max_new_tokens=5, temperature=0.9, seed=3, min_p=0.02, logprobs=True, share_prefix=True, ignore_eos=True)
    want = model.generate(prompts, **options)
    run = model.start_batch(prompts, **options)
    try:
        run.start()
        first = model.engine.cache.book.pages(run.slot_of[0], 0)[:2]
        assert all(model.engine.cache.book.pages(run.slot_of[i], 0)[:2] == first for i in (1, 2))
        while not run.done:
            run.advance()
    finally:
        run.close()
    assert [r.tokens for r in run.results] == [r.tokens for r in want]
    assert [r.logprobs for r in run.results] == [r.logprobs for r in want] and all(len(r.logprobs) == 5 for r in want)
