"""Chooses the next token of each row of logits on the device."""
from __future__ import annotations

import numpy as np
import torch

from ..kernels import ops as _ops
from ..kernels import staging as _staging
from .params import SamplingConfig

_M = (1 << 64) - 1


def uniform_at(seed: int, index: int) -> float:
    """A number in [0, 1) that depends only on (seed, index): a counter run
    through the splitmix64 finaliser, top 24 bits.  The reference seeds a
    thread-local mt19937 from the random device (src/core/runtime/InferRuntime.cu:240),
    which cannot be reproduced; this can, in any batch."""
    x = (seed * 0x9E3779B97F4A7C15 + (index + 1) * 0xD1B54A32D192ED03) & _M
    x ^= x >> 30
    x = (x * 0xBF58476D1CE4E5B9) & _M
    x ^= x >> 27
    x = (x * 0x94D049BB133111EB) & _M
    x ^= x >> 31
    return (x >> 40) / float(1 << 24)


class SeenTokens:
    """The distinct tokens of a sequence that only grows (a request's prompt and output), kept up
    to date token by token: a repetition penalty needs them at every step, and to make a set of a
    few thousand tokens anew for every request and step costs more than the step itself."""

    def __init__(self):
        self._set: set = set()
        self._buf = np.empty(256, dtype=np.int32)
        self._n = 0
        self._consumed = 0

    def update(self, tokens) -> np.ndarray:
        """``tokens``: the sequence so far, longer than (or as long as) at the last call.
        Returns its distinct tokens, int32, in the order of their first appearance."""
        for t in tokens[self._consumed:]:
            t = int(t)
            if t not in self._set:
                self._set.add(t)
                if self._n == self._buf.size:
                    self._buf = np.concatenate([self._buf, np.empty(self._buf.size, dtype=np.int32)])
                self._buf[self._n] = t
                self._n += 1
        self._consumed = len(tokens)
        return self._buf[:self._n]


class TokenLog:
    """A request's prompt and output as one int32 array, kept up to date token by token."""

    def __init__(self, prompt):
        self.prompt_len = len(prompt)
        self._n = len(prompt)
        self._buf = np.empty(2 * self._n + 256, dtype=np.int32)
        self._buf[:self._n] = prompt

    def update(self, output) -> np.ndarray:
        """``output``: the output so far, longer than (or as long as) at the last call."""
        end = self.prompt_len + len(output)
        if end > self._buf.size:
            self._buf = np.concatenate([self._buf, np.empty(max(self._buf.size, end - self._buf.size), dtype=np.int32)])
        if end > self._n:
            self._buf[self._n:end] = output[self._n - self.prompt_len:]
            self._n = end
        return self._buf[:end]


def allowed_mask(config: SamplingConfig, output: np.ndarray, vocab: int) -> np.ndarray | None:
    """What the config's ``allowed`` says about the token after ``output``: int32 [ceil(vocab / 32)], or None for all.  A copy: the
    function may fill the same array again for the next request."""
    mask = config.allowed(output) if config.allowed is not None else None
    if mask is None:
        return None
    mask = np.array(mask, order="C")
    if mask.dtype not in (np.int32, np.uint32) or mask.shape != (-(-vocab // 32),):
        raise ValueError(f"allowed() returned {mask.dtype} {mask.shape}, expected int32 or uint32 {(-(-vocab // 32),)}")
    return mask.view(np.int32)


def allows_none(mask: np.ndarray, vocab: int) -> bool:
    """Whether a mask (``allowed_mask``) has no bit for any of the ``vocab`` tokens."""
    whole, rest = divmod(vocab, 32)
    return not mask[:whole].any() and not (rest and int(mask[whole]) & ((1 << rest) - 1))


class Sampler:
    def __init__(self, device, ops=_ops):
        self.device = device
        self.ops = ops

    def _send(self, columns: list) -> list[torch.Tensor]:
        # (a copy from pageable memory would make the host wait for the step in flight, and a host that
        # waits cannot launch the next step ahead)
        return _staging.send(self.device, columns)

    def sample(self, logits: torch.Tensor, configs: list[SamplingConfig], indices: list[int],
               seen: list | None = None, histories: list | None = None, masks: list | None = None) -> list[int]:
        """One token per row.  ``indices[r]`` is the number of the output token
        row r decides (the counter of its random draw); ``seen[r]`` the tokens
        of its prompt and output so far (needed only with a repetition penalty):
        a sequence, or its distinct tokens as an int32 array (``SeenTokens``).
        ``histories[r]`` is (prompt and output as an int32 array, tokens of the prompt), for rows whose config says ``adjusts``
        and ``needs_output`` (``TokenLog``); ``masks[r]`` is ``allowed_mask`` of the row (asked for here where not given).
        ``logits`` may be changed in place by the options."""
        if logits.shape[0] == 0:
            return []
        return self.sample_on_device(logits, configs, indices, seen, histories, masks).tolist()

    def _adjust(self, logits: torch.Tensor, configs: list[SamplingConfig], seen, histories, given) -> None:
        """All options on the logits in one launch, a repetition penalty among them."""
        V = logits.shape[1]
        parts, cu, prompt_lens, ids, values, cu_bias, masks, mask_rows = [], [0], [], [], [], [0], [], []
        for r, c in enumerate(configs):
            tokens, prompt_len, mask = np.zeros(0, dtype=np.int32), 0, None
            if c.adjusts and c.needs_output:
                if histories is None or histories[r] is None:
                    raise ValueError(f"row {r}: its options need the request's prompt and output")
                tokens, prompt_len = histories[r]
                mask = allowed_mask(c, tokens[prompt_len:].copy(), V) if given is None else given[r]
            elif c.repetition_penalty != 1.0 and seen is not None:      # (which tokens it saw is all that counts)
                tokens = np.asarray(seen[r], dtype=np.int32)
                prompt_len = tokens.size
            if c.repetition_penalty == 1.0 and not (c.presence_penalty or c.frequency_penalty):
                tokens = tokens[:0]                                      # (nothing to send)
            parts.append(tokens)
            cu.append(cu[-1] + tokens.size)
            prompt_lens.append(min(prompt_len, tokens.size))
            if c.logit_bias:
                ids.extend(c.logit_bias)
                values.extend(c.logit_bias.values())
            cu_bias.append(len(ids))
            if mask is None:
                mask_rows.append(-1)
            else:
                mask_rows.append(len(masks))
                masks.append(mask)
        columns = [np.concatenate(parts) if cu[-1] else np.zeros(0, dtype=np.int32), np.asarray(cu, dtype=np.int32),
                   np.asarray(prompt_lens, dtype=np.int32), np.asarray([c.repetition_penalty for c in configs], dtype=np.float32),
                   np.asarray([c.presence_penalty for c in configs], dtype=np.float32),
                   np.asarray([c.frequency_penalty for c in configs], dtype=np.float32)]
        if ids:
            columns += [np.asarray(ids, dtype=np.int32), np.asarray(values, dtype=np.float32), np.asarray(cu_bias, dtype=np.int32)]
        if masks:
            columns += [np.stack(masks), np.asarray(mask_rows, dtype=np.int32)]
        sent = self._send(columns)
        self.ops.adjust_logits(logits, *sent[:6], bias=tuple(sent[6:9]) if ids else None, masks=tuple(sent[-2:]) if masks else None, out=logits)

    def sample_on_device(self, logits: torch.Tensor, configs: list[SamplingConfig], indices: list[int],
                         seen: list | None = None, histories: list | None = None, masks: list | None = None) -> torch.Tensor:
        """As ``sample``, but the tokens stay on the device (int32 [rows]) and
        nothing waits for them: the caller reads them when it needs them."""
        R = logits.shape[0]
        assert len(configs) == R and len(indices) == R
        if any(c.adjusts for c in configs):
            self._adjust(logits, configs, seen, histories, masks)
        elif any(c.repetition_penalty != 1.0 for c in configs):
            parts, cu = [], [0]
            for r, c in enumerate(configs):
                if c.repetition_penalty != 1.0 and seen is not None:
                    row = seen[r]
                    if not isinstance(row, np.ndarray):      # a plain sequence: its distinct tokens
                        row = np.unique(np.asarray(row, dtype=np.int32))
                    parts.append(row)
                    cu.append(cu[-1] + row.size)
                else:
                    cu.append(cu[-1])
            flat = np.concatenate(parts) if parts and cu[-1] else np.zeros(1, dtype=np.int32)
            seen_d, cu_d, pen_d = self._send([
                flat.astype(np.int32, copy=False), np.asarray(cu, dtype=np.int32),
                np.asarray([c.repetition_penalty for c in configs], dtype=np.float32)])
            self.ops.repetition_penalty(logits, seen_d, cu_d, pen_d)
        if all(c.greedy for c in configs):
            return self.ops.argmax(logits)
        eff = [c.effective() for c in configs]
        temperature, top_k, top_p, min_p, u = self._send([
            np.asarray([e[0] for e in eff], dtype=np.float32), np.asarray([e[1] for e in eff], dtype=np.int32),
            np.asarray([e[2] for e in eff], dtype=np.float32), np.asarray([e[3] for e in eff], dtype=np.float32),
            np.asarray([uniform_at(c.seed, i) for c, i in zip(configs, indices)], dtype=np.float32)])
        limit = _ops.sample_few_limit(logits.shape[1])
        return self.ops.sample(logits, temperature, u, top_k, top_p, min_p, few=any(0 < e[1] <= limit for e in eff))
