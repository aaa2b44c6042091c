"""The step function: a model, its cache and its buffers on one GPU.

``Engine.step`` takes, for each sequence of a batch, the next tokens (a whole prompt, a chunk of
it, or one token) and the places whose logits are wanted; it runs exactly those tokens as one
packed batch from the cache that earlier steps left, and returns float logits.  Sequences have
their own lengths, nothing is padded, and the logits at a position do not depend on how the
tokens were cut into steps or on what else was in the batch, beyond rounding.

The reference's counterpart is ``QwenTritonForCausalLM.forward`` with ``past_key_values`` and
``logits_to_keep`` (qwen_triton/models/core.py:321-375): a rectangular batch with one shared
length (qwen_triton/modules/cache.py:21), correct for unequal lengths only in prefill.
"""
from __future__ import annotations

from collections import OrderedDict
from dataclasses import dataclass
from pathlib import Path
from typing import Sequence

import numpy as np
import torch

from ..cache import CacheError, SequenceCache
from ..config import load_config
from ..config.spec import ModelSpec
from ..ops import kernels
from ..parts.base import Runtime, Workspace
from ..weights import open_checkpoint, random_source
from .model import CausalLM, expected_tensors
from .step import StepContext, StepEntry, plan_passes, shared_shape, tokens_not_again

_DTYPES = {
    "bf16": torch.bfloat16, "bfloat16": torch.bfloat16, "fp32": torch.float32, "float32": torch.float32,
    torch.bfloat16: torch.bfloat16, torch.float32: torch.float32,
}


def parse_dtype(dtype) -> torch.dtype:
    """``bf16``/``bfloat16``/``fp32``/``float32`` (the reference also reads fp16 names,
    qwen_triton/models/core.py:29-44; half precision is not built here)."""
    key = dtype.lower() if isinstance(dtype, str) else dtype
    if key not in _DTYPES:
        raise ValueError(f"unsupported dtype {dtype!r}: this library runs bfloat16 or float32")
    return _DTYPES[key]


def require_gpu(device: torch.device) -> None:
    if device.type != "cuda" or not torch.cuda.is_available():
        raise RuntimeError("qwen_triton_b200 runs on a CUDA device (sm_100a) only; there is no host path")
    major, minor = torch.cuda.get_device_capability(device)
    if major != 10:
        raise RuntimeError(f"the kernels are built for sm_100a; device {device} is sm_{major}{minor}")


def check_formats(spec: ModelSpec, weight_format: str | None, cache_format: str | None) -> dict[str, str]:
    """What the parts are told of ``weight_format`` and ``cache_format``: None keeps the compute type, "fp8" the weights of attention's and the feed-forward's
    projections as 8-bit numbers with a scale for each block of 128 x 128 (their rows are brought to 8 bits too), or keys and values with a scale for each
    page and head (half the memory; steps of few sequences take as long as over a 16-bit cache or a little longer, the fused write being the latter's).  Models of dense
    attention and gated feed-forwards take them; parts that do not say so themselves.  ``cache_format`` also wants every layer call to have a cache entry of its own."""
    formats = {name: given for name, given in (("weight_format", weight_format), ("cache_format", cache_format)) if given is not None}
    for name, given in formats.items():
        if given != "fp8":
            raise ValueError(f"{name}={given!r} is neither None nor 'fp8'")
        for layer in spec.layers:
            if layer.block.kind != "pre_norm" or layer.mixer.kind != "attention" or layer.feed_forward is None or layer.feed_forward.kind != "gated_mlp":
                raise ValueError(f"{name}='fp8' is for models of dense attention and gated feed-forwards; {layer.prefix} of {spec.architecture} is another layer")
    if cache_format is not None and any(call.cache_of is not None for call in spec.schedule):
        raise ValueError("cache_format='fp8' is for models whose every layer call writes keys and values of its own; a call of this one reads another's")
    return formats


@dataclass
class PlannedDecode:
    """A one-token step that has been prepared up to the tokens' values (``Engine.plan_decode``)."""

    slots: tuple            # the sequences, in the order their tokens are given
    lengths: tuple          # their lengths once the step has run; checked again when it runs
    count: int              # sequences
    padded: int             # rows the step runs (a power of two up to 32, a multiple of 16 beyond)
    key: tuple              # shape the CUDA graph is kept under
    context: int            # bucket of the longest sequence
    prepared: object        # the packed metadata in pinned memory


class Engine:
    def __init__(self, spec: ModelSpec, source, *, dtype=torch.bfloat16, max_tokens: int = 8192,
                 max_seq_len: int | None = None, max_step_tokens: int = 4096, device: str | torch.device = "cuda:0",
                 page_tokens: int = 64, chunk_tokens: int = 256, options: dict | None = None, weight_format: str | None = None, cache_format: str | None = None,
                 cuda_graphs: bool = True, max_graph_batch: int = 256, max_graphs: int = 48) -> None:
        formats = check_formats(spec, weight_format, cache_format)
        self.device = torch.device(device)
        require_gpu(self.device)
        torch.cuda.set_device(self.device)
        self.dtype = parse_dtype(dtype)
        self.spec = spec
        max_tokens = max(int(max_tokens), page_tokens)
        self.max_seq_len = min(int(max_seq_len or spec.max_positions), spec.max_positions,
                               -(-max_tokens // page_tokens) * page_tokens)
        self.max_step_tokens = int(max_step_tokens)
        workspace = Workspace(self.device)
        self.runtime = Runtime(device=self.device, dtype=self.dtype, max_step_tokens=self.max_step_tokens,
                               max_positions=self.max_seq_len, workspace=workspace, page_tokens=page_tokens,
                               options={**(options or {}), **formats})
        self.model = CausalLM(spec, self.runtime)
        self.model.load(source)
        self.cache = SequenceCache(self.model.cache_requests(), [c.cache_of for c in spec.schedule],
                                   max_tokens=max_tokens, max_seq_len=self.max_seq_len, dtype=self.dtype,
                                   device=self.device, page_tokens=page_tokens, chunk_tokens=chunk_tokens)
        workspace.allocate()
        widths = [self.cache.max_blocks(g) for g in range(len(self.cache.groups))]
        max_seqs = self.max_step_tokens            # a pass never has more sequences than tokens (padded decode rows included)
        self._meta = torch.zeros(StepContext.meta_size(self.max_step_tokens, max_seqs, widths), dtype=torch.int32,
                                 device=self.device)
        self._ctx = StepContext(device=self.device, meta=self._meta)
        self.steps_run = 0
        # one-token steps are captured once per shape and replayed: the launches of a step cost more on the
        # host than they run on the device.  A part whose step only launches kernels says so (graph_safe = True;
        # a block answers for the parts it runs); one part that does not, or touches the host, and every step
        # launches its kernels one by one.
        stepped = [self.model.embedding, *self.model.entries, *self.model.blocks, self.model.final_norm, self.model.head]
        self._graphs_enabled = bool(cuda_graphs) and all(getattr(part, "graph_safe", False) for part in stepped)
        # captured steps by shape, least recently used first; at most ``max_graphs`` are kept (a long generation at
        # many batch sizes and context buckets would otherwise grow device memory without limit), and all of them
        # write their logits into one buffer, made at the first one-token step
        self._graphs: OrderedDict[tuple, object] = OrderedDict()
        self.max_graphs = max(1, int(max_graphs))
        self._graph_logits: torch.Tensor | None = None
        self._planned: set[int] = set()          # sequences whose last position is planned and has not run
        self._status_host = torch.zeros(4, dtype=torch.int32, pin_memory=True)
        self._status_event: torch.cuda.Event | None = None
        self.max_graph_batch = max_graph_batch
        self.graph_replays = 0
        self.last_meta_bytes = 0        # host-to-device bytes of the latest pass (its packed metadata)

    # ------------------------------------------------------------------ construction
    @classmethod
    def from_pretrained(cls, model_path: str | Path, **kwargs) -> "Engine":
        """Model folder with config.json and safetensors; the architecture is chosen by config.json."""
        config = load_config(model_path)
        spec = config.model_spec()
        engine = cls(spec, open_checkpoint(model_path, expected_tensors(spec)), **kwargs)
        engine.config = config
        return engine

    @classmethod
    def from_config(cls, config, seed: int = 0, weights_dtype=None, **kwargs) -> "Engine":
        """Seeded random weights drawn on the device (no model folder is written): the same values that
        ``write_random_model`` writes for this seed.  ``weights_dtype`` is the element type a model folder would
        store them in (by default the compute type): a float32 engine with ``weights_dtype="bf16"`` runs the very
        weights of the bfloat16 model in true 32-bit arithmetic."""
        spec = config.model_spec()
        dtype = parse_dtype(kwargs.get("dtype", torch.bfloat16))
        device = kwargs.get("device", "cuda:0")
        stored = parse_dtype(weights_dtype) if weights_dtype is not None else None
        engine = cls(spec, random_source(expected_tensors(spec), seed, dtype, device, stored), **kwargs)
        engine.config = config
        return engine

    # ------------------------------------------------------------------ properties
    @property
    def vocab_size(self) -> int:
        return self.spec.vocab_size

    @property
    def eos_token_ids(self) -> tuple[int, ...]:
        return tuple(self.spec.eos_token_ids)

    @property
    def page_tokens(self) -> int:
        return self.cache.page_tokens

    @property
    def total_pages(self) -> int:
        return self.cache.book.groups[0].num_pages if self.cache.book.groups else self.cache.num_slots

    @property
    def num_slots(self) -> int:
        return self.cache.num_slots

    # ------------------------------------------------------------------ sequences
    @property
    def can_share(self) -> bool:
        """Whether a sequence may start with another one's cached tokens."""
        return self.cache.can_share

    def new_sequence(self, prefix_of: int | None = None, tokens: int | None = None) -> int:
        """Take a slot for a sequence that starts at position 0, or with the first ``tokens`` (whole pages; default: all of its whole pages) of the sequence in
        ``prefix_of``, whose keys and values it then shares.  Captured one-token steps read sequences that share their first pages together where that is faster
        (``kernels.sharing_pays``).  A position that is planned (``plan_decode``) and has not run yet has no keys and values to share."""
        if prefix_of is None:
            return self.cache.alloc()
        length = self.length(prefix_of) - (prefix_of in self._planned)
        if tokens is None:
            tokens = length // self.page_tokens * self.page_tokens
        elif tokens > length:
            raise CacheError(f"slot {prefix_of}: {tokens} tokens of which {length} have run")
        return self.cache.alloc(prefix_of, tokens)

    def release(self, slot: int) -> None:
        """Give back the slot and every page the sequence holds."""
        self.cache.free(slot)
        self._planned.discard(slot)

    def length(self, slot: int) -> int:
        return self.cache.book.length(slot)

    def can_hold(self, lengths_by_slot: dict[int, int]) -> bool:
        return self.cache.book.can_hold(lengths_by_slot)

    accepts_chosen_tokens = True       # run_planned(plan, rows, chosen=...) takes token ids that are still on the device

    def check_kernels(self, wait: bool = True) -> None:
        """Raise if a bounded wait inside a tensor-core kernel ran out during a step (its results are then invalid).
        Every step ends with a copy of the status word into pinned memory; this waits for the latest of those
        copies and looks at the host's copy.  ``wait=False`` only looks: enough for a caller that has read a step's
        results (the copy of that step has then happened) and must not wait for a later step that is already queued."""
        if self._status_event is None:
            return
        if wait:
            self._status_event.synchronize()
        if int(self._status_host[0]) != 0:
            kernels.check_status(self.device)            # reads the word itself, clears it and raises with the role that gave up

    def _mirror_status(self) -> None:
        self._status_host.copy_(kernels.status_word(self.device), non_blocking=True)
        if self._status_event is None:
            self._status_event = torch.cuda.Event()
        self._status_event.record()

    # ------------------------------------------------------------------ the step
    def step(self, entries: Sequence[StepEntry]) -> torch.Tensor:
        """Run the given tokens; return float logits [sum of wanted places, vocab] in the order of
        the entries and, within an entry, of its ``want`` list."""
        entries = list(entries)
        if not entries:
            return torch.empty((0, self.spec.vocab_size), dtype=torch.float32, device=self.device)
        book = self.cache.book
        seen: set[int] = set()
        targets: dict[int, int] = {}
        for entry in entries:
            if entry.slot in seen:
                raise ValueError(f"slot {entry.slot} appears twice in one step")
            seen.add(entry.slot)
            if not book.is_live(entry.slot):
                raise ValueError(f"slot {entry.slot} is not in use")
            if not entry.tokens:
                raise ValueError(f"slot {entry.slot}: a step entry needs at least one token")
            low, high = min(entry.tokens), max(entry.tokens)
            if low < 0 or high >= self.spec.vocab_size:
                raise ValueError(f"slot {entry.slot}: token id {low if low < 0 else high} is outside 0..{self.spec.vocab_size - 1}")
            for place in entry.want:
                if not 0 <= place < len(entry.tokens):
                    raise ValueError(f"slot {entry.slot}: wanted place {place} is outside its {len(entry.tokens)} tokens")
            targets[entry.slot] = book.length(entry.slot) + len(entry.tokens)
            if targets[entry.slot] > self.max_seq_len:
                raise ValueError(f"slot {entry.slot}: {targets[entry.slot]} tokens exceed max_seq_len={self.max_seq_len}")
        if not book.can_hold(targets):
            raise RuntimeError("the cache cannot hold this step: too many tokens are live (raise max_tokens)")

        if (self._graphs_enabled and len(entries) <= min(self.max_graph_batch, self.max_step_tokens // 2)
                and all(len(e.tokens) == 1 and e.want == [0] for e in entries)):
            self.steps_run += 1
            logits = self._decode_step(entries)
            self._mirror_status()
            return logits

        n_want = sum(len(e.want) for e in entries)
        logits = torch.empty((n_want, self.spec.vocab_size), dtype=torch.float32, device=self.device)
        want_base = np.cumsum([0] + [len(e.want) for e in entries])
        chunk_limit = self.cache.chunk_tokens if self.cache.has_window else None
        passes = plan_passes([len(e.tokens) for e in entries], self.max_step_tokens, chunk_limit)
        for pieces in passes:
            slots, tokens, past, rows, final_rows, row0 = [], [], [], [], [], 0
            for piece in pieces:
                entry = entries[piece.entry]
                slots.append(entry.slot)
                tokens.append(entry.tokens[piece.begin:piece.end])
                past.append(book.length(entry.slot))
                for k, place in enumerate(entry.want):
                    if piece.begin <= place < piece.end:
                        rows.append(row0 + place - piece.begin)
                        final_rows.append(int(want_base[piece.entry]) + k)
                row0 += piece.end - piece.begin
                book.extend(entry.slot, past[-1] + piece.end - piece.begin)
            tables = []
            for group in range(len(self.cache.groups)):
                width = max(1, max(len(book.pages(s, group)) for s in slots))
                table = np.zeros((len(slots), width), dtype=np.int32)
                for i, s in enumerate(slots):
                    pages = book.pages(s, group)
                    table[i, :len(pages)] = pages
                tables.append(table)
            self._ctx.fill(slots, tokens, past, rows, tables)
            self.last_meta_bytes = self._ctx.meta_bytes
            direct = len(passes) == 1 or final_rows == list(range(final_rows[0], final_rows[0] + len(rows))) if rows else True
            if not rows:
                self.model.forward(self._ctx, self.cache, None)
            elif direct:
                self.model.forward(self._ctx, self.cache, logits[final_rows[0]:final_rows[0] + len(rows)])
            else:
                part = torch.empty((len(rows), self.spec.vocab_size), dtype=torch.float32, device=self.device)
                self.model.forward(self._ctx, self.cache, part)
                logits.index_copy_(0, torch.tensor(final_rows, device=self.device), part)
        self.steps_run += 1
        self._mirror_status()
        return logits

    def _decode_step(self, entries: list[StepEntry]) -> torch.Tensor:
        """One token per sequence, every logit wanted: plan and run in one go."""
        plan = self._plan_decode([e.slot for e in entries], extend=True)
        return self._run_planned(plan, [e.tokens[0] for e in entries])

    # ------------------------------------------------------------------ a one-token step in two halves
    def plan_decode(self, slots: Sequence[int], extend: bool = True) -> "PlannedDecode | None":
        """The half of a one-token step that does not depend on the tokens' values: checks, one more position for
        every sequence, page tables, the packed metadata in pinned memory.  A caller that waits for the device to
        hand over the previous step's tokens can do this meanwhile and call ``run_planned`` once it has them.

        ``extend=False`` plans again for sequences that an abandoned plan has already given their next position
        (a plan is abandoned by just not running it; sequences that end are released as usual).  Returns None
        where one-token steps are not run at a fixed shape (CUDA graphs off, or too many sequences): use ``step``.
        """
        slots = list(slots)
        if not slots or not self._graphs_enabled or len(slots) > min(self.max_graph_batch, self.max_step_tokens // 2):
            return None
        book = self.cache.book
        if len(set(slots)) != len(slots):
            raise ValueError("a slot appears twice in one step")
        targets = {}
        for slot in slots:
            if not book.is_live(slot):
                raise ValueError(f"slot {slot} is not in use")
            targets[slot] = book.length(slot) + (1 if extend else 0)
            if targets[slot] > self.max_seq_len:
                raise ValueError(f"slot {slot}: {targets[slot]} tokens exceed max_seq_len={self.max_seq_len}")
        if extend and not book.can_hold(targets):
            raise RuntimeError("the cache cannot hold this step: too many tokens are live (raise max_tokens)")
        return self._plan_decode(slots, extend)

    def run_planned(self, plan: "PlannedDecode", tokens: Sequence[int], chosen: torch.Tensor | None = None) -> torch.Tensor:
        """The other half: the tokens (one per planned sequence, in the plan's order) go in and the step runs.
        Returns float logits [sequences, vocab].

        With ``chosen`` (int32 on the device, as a sampling kernel leaves it) ``tokens`` are row numbers of it: the
        step is then queued behind that kernel without the host having seen the tokens."""
        tokens = [int(t) for t in tokens]
        if len(tokens) != plan.count:
            raise ValueError(f"{len(tokens)} tokens for a plan of {plan.count} sequences")
        low, high = min(tokens), max(tokens)
        if chosen is not None:
            if chosen.dtype != torch.int32 or chosen.device != self.device or low < 0 or high >= chosen.numel():
                raise ValueError("chosen tokens must be int32 on the engine's device, and every row number within them")
        elif low < 0 or high >= self.spec.vocab_size:
            raise ValueError(f"token id {low if low < 0 else high} is outside 0..{self.spec.vocab_size - 1}")
        book = self.cache.book
        for slot, length in zip(plan.slots, plan.lengths):
            if not book.is_live(slot) or book.length(slot) != length:
                raise ValueError(f"slot {slot} has changed since this step was planned (released, or stepped in between)")
        self.steps_run += 1
        logits = self._run_planned(plan, tokens, chosen)
        self._mirror_status()
        return logits

    def _plan_decode(self, slots: list[int], extend: bool) -> "PlannedDecode":
        """Fixed shape of a one-token step: batch padded to a power of two up to 32 and to a multiple of 16 beyond (the
        kernels' choices follow the padded count: 48 rows run 4 % shorter as 48 than as 64), page tables to a
        multiple of 16 pages, so that a captured CUDA graph can be replayed.  Padded rows read and write only the
        cache's spare page and spare state row, and their logits are dropped."""
        book, cache = self.cache.book, self.cache
        count = len(slots)
        padded = 1
        while padded < count and padded < 32:
            padded *= 2
        if padded < count:
            padded = -(-count // 16) * 16
        if extend:
            past = [book.length(s) for s in slots]
            for slot, before in zip(slots, past):
                book.extend(slot, before + 1)
            self._planned.update(slots)
        else:
            past = [book.length(s) - 1 for s in slots]
        widths, tables = [], []
        for group in range(len(cache.groups)):
            need = max(len(book.pages(s, group)) for s in slots)
            width = min(cache.max_blocks(group), -(-need // 16) * 16)
            table = np.full((padded, width), cache.dummy_page, dtype=np.int32)
            for i, s in enumerate(slots):
                pages = book.pages(s, group)
                table[i, :len(pages)] = pages
            widths.append(width)
            tables.append(table)
        context = -(-(max(past) + 1) // 1024) * 1024
        pad = padded - count
        groups, shape = book.shared_groups(slots), None
        # a shape of groups only where some layer takes it: every shape is a graph of its own
        pays = tuple(kind for kind in sorted(self.runtime.options.get("shared_attention", ()))
                     if kernels.sharing_pays(tokens_not_again(groups), *kind, self.dtype, self.page_tokens)) if groups else ()
        if not pays:
            groups = []
        if groups:
            if pad:                                              # padded rows: one token of their own
                if groups[-1][1]:
                    groups.append(([], 0))
                groups[-1][0].extend(range(count, padded))
            shape = shared_shape(groups, [p + 1 for p in past] + [1] * pad)
        prepared = self._ctx.prepare_decode(slots + [cache.dummy_slot] * pad, past + [0] * pad, tables, groups, shape, pays)
        return PlannedDecode(slots=tuple(slots), lengths=tuple(p + 1 for p in past), count=count, padded=padded,
                             key=(padded, tuple(widths), context, shape, pays), context=context, prepared=prepared)

    def _run_planned(self, plan: "PlannedDecode", tokens: list[int], chosen: torch.Tensor | None = None) -> torch.Tensor:
        cache, count, padded = self.cache, plan.count, plan.padded
        fill = -1 if chosen is not None else 0                  # padded rows: token 0 either way
        self._planned.difference_update(plan.slots)
        self._ctx.commit_decode(plan.prepared, tokens + [fill] * (padded - count), plan.context, chosen, self.spec.vocab_size)
        self.last_meta_bytes = self._ctx.meta_bytes
        key = plan.key
        if self._graph_logits is None:         # one buffer for every shape: a replay's rows are copied out of it anyway
            most = min(self.max_graph_batch, self.max_step_tokens // 2)
            rows = 1
            while rows < most:
                rows *= 2
            self._graph_logits = torch.empty((rows, self.spec.vocab_size), dtype=torch.float32, device=self.device)
        logits = self._graph_logits[:padded]
        state = self._graphs.get(key)
        if state is None:                      # first time at this shape: run the launches themselves
            self.model.forward(self._ctx, cache, logits)
            self._graphs[key] = "warm"
            while len(self._graphs) > self.max_graphs:
                self._graphs.popitem(last=False)
            return logits[:count].clone()
        self._graphs.move_to_end(key)
        if state == "warm":                    # second time: capture (nothing runs during capture), then replay
            graph = torch.cuda.CUDAGraph()
            before = kernels.launch_count()
            with torch.cuda.graph(graph):
                self.model.forward(self._ctx, cache, logits)
            state = (graph, kernels.launch_count() - before)
            self._graphs[key] = state
        graph, launches = state
        graph.replay()
        kernels.count_launches(launches)
        self.graph_replays += 1
        return logits[:count].clone()

    def memory_report(self) -> dict[str, int]:
        return {"weights": self.model.weight_bytes(), "cache": self.cache.bytes(),
                "workspace": self.runtime.workspace.bytes()}
