"""Greedy and temperature / top-k sampling on the device, with the uniform
numbers made on the host by a counter-based generator: the number for
(seed, request, output position) is a pure function of the three, so a
request's tokens do not depend on which other requests share its steps, and a
plain implementation on the CPU can reproduce them."""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import ops
from .params import SamplingParams

_MASK = (1 << 64) - 1


def _splitmix64(x: int) -> int:
    x = (x + 0x9E3779B97F4A7C15) & _MASK
    z = x
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK
    return z ^ (z >> 31)


def uniform_for(seed: int, request_index: int, position: int) -> float:
    """A number in [0, 1) with 24 random bits (exact in float32)."""
    h = _splitmix64(seed & _MASK)
    h = _splitmix64(h ^ (request_index & _MASK))
    h = _splitmix64(h ^ (position & _MASK))
    return (h >> 40) / float(1 << 24)


class SampledTokens:
    """The tokens of one sampling call: on the device at once (``device``, int32 [N]), on the host
    when ``read()`` is called (their copy to pinned memory is queued right behind the sampling)."""

    def __init__(self, device_tokens: torch.Tensor):
        self.device = device_tokens
        self._host = None
        self._event = None
        if device_tokens.is_cuda:
            self._host = torch.empty(device_tokens.shape, dtype=device_tokens.dtype, pin_memory=True)
            self._host.copy_(device_tokens, non_blocking=True)
            self._event = torch.cuda.Event()
            self._event.record()

    def read(self) -> list[int]:
        if self._host is None:
            return self.device.tolist()
        self._event.synchronize()
        return self._host.tolist()


class VerifiedTokens:
    """The tokens of one verification: on the device at once (``counts`` int32 [R], how many tokens each request gained,
    and ``tokens`` int32 [N] in the rows' layout, -1 behind them), on the host when ``read()`` is called."""

    def __init__(self, counts: torch.Tensor, tokens: torch.Tensor, lengths: Sequence[int]):
        self.counts, self.tokens = counts, tokens
        self._lengths = list(lengths)
        self._both = SampledTokens(torch.cat([counts, tokens]))

    def read(self) -> list[list[int]]:
        """A list of tokens per request: its drafts that stand, and the one behind them."""
        both = self._both.read()
        R = len(self._lengths)
        out, at = [], R
        for n, count in zip(self._lengths, both[:R]):
            out.append(both[at:at + count])
            at += n
        return out


class Sampler:
    def __init__(self, device):
        self.device = torch.device(device)

    def sample(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               uniforms: Sequence[float]) -> list[int]:
        """One token per row of float32 logits [N, V]; returns host ints."""
        return self.sample_async(logits, params, uniforms).read()

    def sample_async(self, logits: torch.Tensor, params: Sequence[SamplingParams],
                     uniforms: Sequence[float]) -> SampledTokens:
        """The same without waiting for the device."""
        N = logits.shape[0]
        assert N == len(params) == len(uniforms)
        out = torch.empty(N, dtype=torch.int32, device=self.device)
        if all(p.greedy for p in params):
            ops.argmax(logits, out)
        else:
            meta = torch.tensor([[p.temperature for p in params], list(uniforms)], dtype=torch.float32)
            topk = torch.tensor([p.top_k for p in params], dtype=torch.int32)
            if self.device.type == "cuda":
                meta = meta.pin_memory().to(self.device, non_blocking=True)
                topk = topk.pin_memory().to(self.device, non_blocking=True)
            ops.sample(logits, meta[0].contiguous(), topk, meta[1].contiguous(), out)
        return SampledTokens(out)

    def verify(self, logits: torch.Tensor, params: Sequence[SamplingParams], drafts: Sequence[Sequence[int]],
               uniforms: Sequence[Sequence[float]], draft_logits: Optional[torch.Tensor] = None) -> list[list[int]]:
        """The tokens each request gains from a step that ran its newest token and its drafts: see ``verify_async``."""
        return self.verify_async(logits, params, drafts, uniforms, draft_logits).read()

    def verify_async(self, logits: torch.Tensor, params: Sequence[SamplingParams], drafts: Sequence[Sequence[int]],
                     uniforms: Sequence[Sequence[float]], draft_logits: Optional[torch.Tensor] = None) -> VerifiedTokens:
        """Hold drafted tokens against the target's logits without waiting for the device.  ``logits`` float32 [N, V]: for
        request r one row more than it has ``drafts``, in the order of the step's wanted places; ``uniforms[r]`` has a number
        for each of its rows (the last one draws the token behind the drafts that stand).  ``draft_logits`` float32 [N - R, V]:
        what the drafts were drawn from, or None for drafts that were found."""
        R = len(params)
        lengths = [len(d) + 1 for d in drafts]
        if len(drafts) != R or [len(u) for u in uniforms] != lengths or logits.shape[0] != sum(lengths):
            raise ValueError("verify: one list of drafts per request, one uniform number and one row of logits per draft and one more")
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        ints = torch.tensor(starts + [p.top_k for p in params] + [int(t) for d in drafts for t in d], dtype=torch.int32)
        floats = torch.tensor([p.temperature for p in params] + [float(u) for us in uniforms for u in us], dtype=torch.float32)
        if self.device.type == "cuda":
            ints = ints.pin_memory().to(self.device, non_blocking=True)
            floats = floats.pin_memory().to(self.device, non_blocking=True)
        tokens = torch.empty(starts[-1], dtype=torch.int32, device=self.device)
        counts = torch.empty(R, dtype=torch.int32, device=self.device)
        ops.verify_drafts(logits, ints[2 * R + 1:], draft_logits, ints[:R + 1], floats[:R], ints[R + 1:2 * R + 1], floats[R:], tokens, counts,
                          lambda shape, dtype: torch.empty(shape, dtype=dtype, device=self.device))
        return VerifiedTokens(counts, tokens, lengths)
