"""Next-token choice: greedy, or temperature sampling with a reproducible random stream.

The reference picks ``argmax`` of the last position and nothing else
(qwen_triton/models/core.py:405).  Temperature sampling here draws token
``softmax(logits / T)`` by inverse CDF in vocabulary order with one uniform number per
(seed, request, step), so a request's tokens do not depend on what else is in the batch.
``top_k`` and ``top_p`` (both off by default) leave only the most likely tokens to draw from:
the k largest logits, and of those the smallest set of the most likely whose renormalised
probabilities sum to ``top_p``; tokens that tie with the last one kept are kept as well, so that
the set does not depend on an order among equals.  ``min_p`` leaves, of these, the tokens at least so many times as likely as the
likeliest; ``logprobs`` asks for the log-probability with which each token was drawn.  Rows with either, or with parameters of their own, go through one kernel
for all of them (``kernels.sample_filtered``), with the same uniform numbers.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from ..ops import kernels

_MASK64 = (1 << 64) - 1


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0     # 0: greedy (ties go to the lowest token id)
    seed: int = 0
    top_k: int = 0               # > 0: only the k largest logits (with temperature > 0)
    top_p: float = 1.0           # < 1: only the most likely tokens that sum to this share (with temperature > 0)
    min_p: float = 0.0           # > 0: only tokens at least this many times as likely as the likeliest (with temperature > 0)
    logprobs: bool = False       # also the log-probability with which each token was drawn

    def __post_init__(self) -> None:
        if self.temperature < 0.0:
            raise ValueError("temperature must not be negative")
        if self.top_k < 0 or not 0.0 < self.top_p <= 1.0:
            raise ValueError("top_k must not be negative and top_p must lie in (0, 1]")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError("min_p must lie in [0, 1]")


def _mix64(value: int) -> int:
    value = (value + 0x9E3779B97F4A7C15) & _MASK64
    value = ((value ^ (value >> 30)) * 0xBF58476D1CE4E5B9) & _MASK64
    value = ((value ^ (value >> 27)) * 0x94D049BB133111EB) & _MASK64
    return value ^ (value >> 31)


def uniform_for(seed: int, request: int, step: int) -> float:
    """Uniform number in [0, 1) for the ``step``-th new token of request ``request``.  The sampling kernel computes
    the same number on the device; this host statement of it is what tests compare with."""
    state = _mix64(seed & _MASK64)
    state = _mix64(state ^ (request & _MASK64))
    state = _mix64(state ^ (step & _MASK64))
    return (state >> 40) / float(1 << 24)


def uniforms_for(seeds: np.ndarray, requests: np.ndarray, steps: np.ndarray) -> np.ndarray:
    """``uniform_for`` of many rows, as float32 (24 bits: exact)."""
    def mix(value):
        value = value + np.uint64(0x9E3779B97F4A7C15)
        value = (value ^ (value >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        value = (value ^ (value >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return value ^ (value >> np.uint64(31))
    with np.errstate(over="ignore"):
        state = mix(mix(mix(seeds.astype(np.uint64)) ^ requests.astype(np.uint64)) ^ steps.astype(np.uint64))
    return ((state >> np.uint64(40)).astype(np.float64) / float(1 << 24)).astype(np.float32)


class PendingTokens:
    """Token ids on their way to the host: ``tokens()`` waits for the copy and returns them, ``logprobs()`` what came with them."""

    def __init__(self, host: torch.Tensor, event: torch.cuda.Event, rows: int, device: torch.Tensor | None = None, with_logprobs: bool = False) -> None:
        self._host, self._event, self._rows, self._with_logprobs = host, event, rows, with_logprobs
        self.device = device        # the ids on the device (int32 [rows]), for a step that is queued before the host reads them

    def tokens(self) -> list[int]:
        self._event.synchronize()
        return self._host[:self._rows].tolist()

    def logprobs(self) -> list[float] | None:
        """The log-probability with which each token was drawn; None where nobody asked for it."""
        if not self._with_logprobs:
            return None
        self._event.synchronize()
        return self._host[self._rows:2 * self._rows].view(torch.float32).tolist()


class Sampler:
    """Chooses one token per logits row on the device and returns the ids to the host."""

    _RING = 4

    def __init__(self, device: torch.device) -> None:
        self.device = torch.device(device)
        self._hosts: list[torch.Tensor] = []     # pinned buffers the ids are copied into, used in turn
        self._keys: list[tuple] = []             # pinned (request, step) buffers, their events and the device copy
        self._numbers_used = 0
        self._numbers: list[tuple] = []          # pinned rows of parameters and numbers, their events and the device copy
        self._turn = 0

    def _keys_on_device(self, requests: list[int], steps: list[int]) -> torch.Tensor:
        """(request, step) per row as int32 [rows, 2] on the device, through a pinned buffer and an asynchronous
        copy: the host does not wait for the device and the device not for the host."""
        rows = len(requests)
        if not self._keys or self._keys[0][0].shape[0] < rows:
            size = max(rows, 64)
            self._keys = [(torch.empty((size, 2), dtype=torch.int32, pin_memory=True), torch.cuda.Event(),
                           torch.empty((size, 2), dtype=torch.int32, device=self.device)) for _ in range(self._RING)]
        host, event, device = self._keys[self._turn % self._RING]
        if self._turn >= self._RING:
            event.synchronize()                  # the copy that last used this buffer has happened
        pairs = host.numpy()
        pairs[:rows, 0] = requests
        pairs[:rows, 1] = steps
        device[:rows].copy_(host[:rows], non_blocking=True)
        event.record()
        return device[:rows]

    def _launch_filtered(self, logits: torch.Tensor, params: list[SamplingParams], requests: list[int], steps: list[int]) -> PendingTokens:
        """The choice with a row's own parameters: they and the rows' uniform numbers go to the device in one copy, ids and log-probabilities back in one."""
        rows = len(params)
        if not self._numbers or self._numbers[0][0].shape[1] < rows:
            size = max(rows, 64)
            self._numbers = [(torch.empty((5, size), dtype=torch.float32, pin_memory=True), torch.cuda.Event(),
                              torch.empty((5, size), dtype=torch.float32, device=self.device)) for _ in range(self._RING)]
            self._numbers_used = 0
        host, event, device = self._numbers[self._numbers_used % self._RING]
        if self._numbers_used >= self._RING:
            event.synchronize()                  # the copy that last used this buffer has happened
        self._numbers_used += 1
        flat = host.view(-1)[:5 * rows]
        numbers = flat.numpy().reshape(5, rows)
        numbers[0] = [p.temperature for p in params]
        numbers[1] = [p.top_p for p in params]
        numbers[2] = [p.min_p for p in params]
        numbers[3] = uniforms_for(np.array([p.seed & _MASK64 for p in params], dtype=np.uint64), np.array(requests), np.array(steps))
        numbers[4].view(np.int32)[:] = [min(p.top_k, logits.shape[1]) for p in params]
        there = device.view(-1)[:5 * rows]
        there.copy_(flat, non_blocking=True)
        event.record()
        there = there.view(5, rows)
        both = torch.empty((2, rows), dtype=torch.int32, device=self.device)
        kernels.sample_filtered(logits, there[0], there[4].view(torch.int32), there[1], there[2], there[3], both[0], both[1].view(torch.float32))
        return self._to_host(both, any(p.logprobs for p in params))

    def _to_host(self, out: torch.Tensor, with_logprobs: bool = False) -> PendingTokens:
        rows, count = out.shape[-1], out.numel()
        if not self._hosts or self._hosts[0].numel() < count:
            self._hosts = [torch.empty(max(count, 64), dtype=torch.int32, pin_memory=True) for _ in range(self._RING)]
        host = self._hosts[self._turn % self._RING]
        self._turn += 1
        host[:count].copy_(out.view(-1), non_blocking=True)
        event = torch.cuda.Event()
        event.record()
        return PendingTokens(host, event, rows, out[0] if out.dim() == 2 else out, with_logprobs)

    def launch(self, logits: torch.Tensor, params: "SamplingParams | list[SamplingParams]", requests: list[int], steps: list[int]) -> PendingTokens:
        """Start the choice and the copy of the ids to pinned host memory; the caller may do other work before
        it asks the returned object for the tokens.  ``params``: for all rows, or one for each; rows with their own are chosen by the kernel for filters
        even where they are alike, so that no row's choice depends on which others are still there."""
        rows = logits.shape[0]
        if rows != len(requests) or rows != len(steps):
            raise ValueError("one request index and one step number per logits row")
        if not isinstance(params, SamplingParams):
            params = list(params)
            if len(params) != rows:
                raise ValueError(f"{len(params)} sampling parameters for {rows} rows")
            if params:
                return self._launch_filtered(logits, params, requests, steps)
            params = SamplingParams()
        if params.min_p > 0 or params.logprobs:
            return self._launch_filtered(logits, [params] * rows, requests, steps)
        out = torch.empty(rows, dtype=torch.int32, device=self.device)
        if params.temperature == 0.0:
            kernels.argmax(logits, out)
        else:
            kernels.sample_keyed(logits, params.temperature, params.seed, self._keys_on_device(requests, steps), out,
                                 params.top_k, params.top_p)
        return self._to_host(out)

    def sample(self, logits: torch.Tensor, params: "SamplingParams | list[SamplingParams]", requests: list[int], steps: list[int]) -> list[int]:
        return self.launch(logits, params, requests, steps).tokens()
