"""Turns logits rows into token ids on the device."""
from __future__ import annotations

import numpy as np
import torch

from .. import ops
from .params import SamplingParams


class NonFiniteLogits(RuntimeError):
    """A row of logits held NaN or infinity (reference: native/cuda-device.inc:250-257)."""


def _mix(z: np.ndarray) -> np.ndarray:
    """splitmix64's finaliser"""
    z = z + np.uint64(0x9E3779B97F4A7C15)
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def uniform_numbers(seeds: list[int], counters: list[int], lens: list[int]) -> torch.Tensor:
    """float32 in [0, 1), lens[s] of them for sequence s, that depend on its seed, its counter and their place alone."""
    seed, counter = (np.repeat(np.asarray(a, dtype=np.uint64), lens) for a in (seeds, counters))
    place = np.concatenate([np.arange(n, dtype=np.uint64) for n in lens] or [np.zeros(0, np.uint64)])
    h = _mix(_mix(_mix(seed) ^ (counter << np.uint64(32))) + place)
    return torch.from_numpy((h >> np.uint64(40)).astype(np.float32) / np.float32(1 << 24))


class Sampler:
    def __init__(self, device, vocab_size: int):
        self.device, self.vocab_size = device, vocab_size
        self._workspace = None
        self._out = None

    def _buffers(self, rows: int):
        need = ops.sample_workspace_floats(rows, self.vocab_size)
        if self._workspace is None or self._workspace.numel() < need:
            self._workspace = torch.empty(max(need, 1), dtype=torch.float32, device=self.device)
        if self._out is None or self._out.numel() < rows:
            self._out = torch.empty(max(rows, 64), dtype=torch.int32, device=self.device)
        return self._workspace, self._out[:rows]

    def sample_device(self, logits: torch.Tensor, params: list[SamplingParams], counters: list[int]) -> torch.Tensor:
        """int32 token ids on the device, one per row of `logits` (-1 marks a non-finite row)."""
        rows = logits.shape[0]
        workspace, out = self._buffers(rows)
        if any(p.temperature > 0 for p in params):
            temperature = torch.tensor([float(p.temperature) for p in params], dtype=torch.float32).to(self.device)
            seed = torch.tensor([p.seed for p in params], dtype=torch.int64).to(self.device)
            counter = torch.tensor(counters, dtype=torch.int32).to(self.device)
            ops.sample(logits, out, workspace, temperature, seed, counter)
        else:
            ops.sample(logits, out, workspace)
        return out

    def sample(self, logits: torch.Tensor, params: list[SamplingParams], counters: list[int]) -> list[int]:
        """Token ids on the host; only 4 bytes a row cross the bus."""
        if logits.shape[0] == 0:
            return []
        tokens = self.sample_device(logits, params, counters).tolist()
        if any(t < 0 or t >= self.vocab_size for t in tokens):
            raise NonFiniteLogits("Non-finite logits: the model produced NaN or infinity.")
        return tokens

    def verify(self, logits: torch.Tensor, tokens: torch.Tensor, lens: list[int], params: list[SamplingParams], counters: list[int],
               draft_logits: torch.Tensor | None = None, draft_rows: torch.Tensor | None = None) -> list[list[int]]:
        """The tokens that a step gives each sequence whose input were its last token and drafts of the next ones: the drafts that hold and
        the token after them, one to lens[s] of them, distributed as the target has them (`ops.verify_drafts`).

        logits [sum of lens, vocabulary] (float32 or bfloat16) and tokens (int32, on the device): every row of the step, sequence after
        sequence.  counters[s]: how many tokens the sequence has had so far; with its seed it settles the random numbers.  draft_logits,
        draft_rows: as for `ops.verify_drafts`."""
        n, rows = len(lens), sum(lens)
        if n == 0:
            return []
        if min(lens) < 1 or logits.shape[0] != rows or tokens.numel() != rows or len(params) != n or len(counters) != n:
            raise ValueError(f"verify: {n} sequences of {lens} rows do not fit logits {tuple(logits.shape)}, {tokens.numel()} tokens, "
                             f"{len(params)} parameters and {len(counters)} counters.")
        need = ops.verify_workspace_floats(rows, n, logits.shape[1])
        if self._workspace is None or self._workspace.numel() < need:
            self._workspace = torch.empty(need, dtype=torch.float32, device=self.device)
        starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
        ints = torch.from_numpy(np.stack([starts, np.asarray(lens), np.zeros(n), np.zeros(n)]).astype(np.int32)).to(self.device)
        temperature = uniform = None
        if any(p.temperature > 0 for p in params):
            temperature = torch.tensor([float(p.temperature) for p in params], dtype=torch.float32).to(self.device)
            uniform = uniform_numbers([p.seed for p in params], counters, lens).to(self.device)
        ops.verify_drafts(logits, tokens, ints[0], ints[1], uniform, ints[2], ints[3], self._workspace, temperature, draft_logits, draft_rows)
        both = torch.cat([tokens.reshape(-1), ints[2:].reshape(-1)]).tolist()      # 4 bytes a row cross the bus
        given, accepted, following = both[:rows], both[rows:rows + n], both[rows + n:]
        answers = [given[start + 1:start + 1 + held] + [token] for start, held, token in zip(starts.tolist(), accepted, following)]
        if any(t < 0 or t >= self.vocab_size for answer in answers for t in answer):      # (as `sample`: a padded head's rows are longer than the vocabulary)
            raise NonFiniteLogits("Non-finite logits: the model produced NaN or infinity.")
        return answers
