"""Request controls on logits: penalties, biases and grammar masks, ahead of the sampler.

No counterpart in the reference, whose sampler knows temperature and top-p only
(src/helios/runtime/qwen3/decode.py:457-473). ``LogitControls`` are one row's settings,
``TokenHistory`` holds the tokens of live requests on the device, and ``control_rows`` applies
the settings of a tick's logit rows (``ops.control_logits``): from the row's history the
repetition penalty (``x / r`` where ``x > 0``, else ``x * r``) on every token it holds, the frequency
penalty times a token's occurrences past the prompt, the presence penalty where there are any;
then the row's biases; then -inf where its mask does not allow a token.
"""

from __future__ import annotations

import math
from collections.abc import Mapping, Sequence
from dataclasses import dataclass, field

import torch

from helios_b200 import ops

MAX_HISTORY = 65_535
FP32_MAX, FP32_TINY = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny


@dataclass(frozen=True)
class LogitControls:
    """One request's controls. ``slot`` is its ``TokenHistory`` slot, which the penalties need;
    ``logit_bias`` maps token ids to biases (-inf bans a token); ``allowed`` is a bool tensor ``[V]`` or a packed mask
    (``pack_mask``), None for no mask."""
    repetition_penalty: float = 1.0
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Mapping[int, float] = field(default_factory=dict)
    allowed: torch.Tensor | None = None
    slot: int | None = None

    def __post_init__(self) -> None:
        # The device holds all of these in fp32.
        if not FP32_TINY <= self.repetition_penalty <= FP32_MAX:
            raise ValueError("repetition_penalty must be positive and finite in fp32")
        if not (abs(self.frequency_penalty) <= FP32_MAX and abs(self.presence_penalty) <= FP32_MAX):
            raise ValueError("frequency_penalty and presence_penalty must be finite in fp32")
        if self.penalised and self.slot is None:
            raise ValueError("penalties need the request's TokenHistory slot")
        if any(token < 0 or not (bias == -math.inf or abs(bias) <= FP32_MAX)
               for token, bias in self.logit_bias.items()):
            raise ValueError("logit_bias maps token ids >= 0 to finite numbers or -inf")

    @property
    def penalised(self) -> bool:
        return self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0 or self.presence_penalty != 0.0


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool ``[..., V]`` to int32 words ``[..., ceil(V / 32)]``, bit i of word c for token 32c + i."""
    if allowed.dtype != torch.bool:
        raise ValueError("allowed must be a bool tensor")
    pad = -allowed.shape[-1] % 32
    bits = torch.nn.functional.pad(allowed, (0, pad)).unflatten(-1, (-1, 32)).long()
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


class TokenHistory:
    """The tokens of up to ``slots`` live requests, on the device: a request opens a slot with its
    prompt, every sampled token is appended to it, and the slot is closed with the request. Appending
    takes the sampled ids from the device, so no step waits for them. Calls run on the current
    stream."""

    def __init__(self, slots: int, capacity: int, device: torch.device | str) -> None:
        if slots < 1 or not 1 <= capacity <= MAX_HISTORY:
            raise ValueError(f"a history needs slots and a capacity of 1 to {MAX_HISTORY} tokens")
        self.device = torch.device(device)
        self.capacity = capacity
        self.tokens = torch.zeros((slots, capacity), dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device=self.device)
        self.prompt_lengths = torch.zeros(slots, dtype=torch.int32, device=self.device)
        self._lengths: list[int | None] = [None] * slots  # host mirror; None: free
        self._free = list(range(slots - 1, -1, -1))

    def _upload(self, values: list, dtype: torch.dtype) -> torch.Tensor:
        host = torch.tensor(values, dtype=dtype)
        return host.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else host

    def _open_slot(self, slot: int) -> int:
        if not 0 <= slot < len(self._lengths) or self._lengths[slot] is None:
            raise ValueError(f"history slot {slot} is not open")
        return self._lengths[slot]

    def length(self, slot: int) -> int:
        return self._open_slot(slot)

    def open(self, prompt_ids: Sequence[int]) -> int:
        """A slot holding ``prompt_ids``."""
        count = len(prompt_ids)
        if count > self.capacity:
            raise ValueError(f"the prompt has {count} tokens and the history {self.capacity} places")
        if not self._free:
            raise RuntimeError("every history slot is in use")
        slot = self._free[-1]  # taken once nothing is left that can refuse the prompt
        if count:
            self.tokens[slot, :count] = self._upload(list(prompt_ids), torch.int32)
        self.lengths[slot] = count
        self.prompt_lengths[slot] = count
        self._free.pop()
        self._lengths[slot] = count
        return slot

    def append(self, slots: Sequence[int], ids: torch.Tensor | Sequence[int]) -> None:
        """One token for each of ``slots`` (distinct): ``ids`` on the device, or a list. Ids on the device
        are not looked at here: one that is no token (the -1 of a row in which nothing was allowed)
        is flagged by the next ``control_rows`` that reads it, and counts for nothing."""
        slots = list(slots)
        if len(set(slots)) != len(slots):
            raise ValueError("a history slot takes one token at a time")
        at = [self._open_slot(slot) for slot in slots]
        if any(position >= self.capacity for position in at):
            raise ValueError("a history slot is full")
        if not isinstance(ids, torch.Tensor):
            ids = self._upload(list(ids), torch.int32)
        if ids.device != self.tokens.device or ids.numel() != len(slots):
            raise ValueError("append needs one token id per slot, on the history's device")
        if not slots:
            return
        rows, columns = self._upload([slots, at], torch.long)
        self.tokens.index_put_((rows, columns), ids.reshape(-1).to(torch.int32))
        self.lengths.index_put_((rows,), (columns + 1).to(torch.int32))
        for slot, position in zip(slots, at):
            self._lengths[slot] = position + 1

    def close(self, slot: int) -> None:
        self._open_slot(slot)
        self._lengths[slot] = None
        self._free.append(slot)


def control_rows(logits: torch.Tensor, controls: Sequence[LogitControls | None],
                 history: TokenHistory | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [rows, V]`` (bf16, on the device) with each row's controls applied (None: none), in
    ``out`` (``logits`` itself works) or a new tensor. ``history`` holds the slots that they name."""
    rows, vocab = logits.shape
    if len(controls) != rows:
        raise ValueError("Each logit row needs its controls (or None).")
    if not any(controls):
        return logits.clone() if out is None else out if out is logits else out.copy_(logits)
    none = LogitControls()
    rows_of = [none if c is None else c for c in controls]
    device = logits.device

    def upload(values: list, dtype: torch.dtype) -> torch.Tensor:
        host = torch.tensor(values, dtype=dtype)
        return host.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else host

    args: dict = {}
    if any(c.penalised for c in rows_of):
        if history is None:
            raise ValueError("penalties need the TokenHistory")
        for c in rows_of:
            if c.penalised:
                history._open_slot(c.slot)
        settings = upload([[c.repetition_penalty for c in rows_of], [c.frequency_penalty for c in rows_of],
                           [c.presence_penalty for c in rows_of]], torch.float32)
        args.update(repetition=settings[0], frequency=settings[1], presence=settings[2], history=history.tokens,
                    slots=upload([c.slot if c.penalised else -1 for c in rows_of], torch.int32),
                    lengths=history.lengths, prompt_lengths=history.prompt_lengths)
    if any(c.logit_bias for c in rows_of):
        lists = [sorted(c.logit_bias.items()) for c in rows_of]
        if any(pairs and pairs[-1][0] >= vocab for pairs in lists):
            raise ValueError(f"logit_bias names a token outside the vocabulary of {vocab}")
        offsets = [0]
        for pairs in lists:
            offsets.append(offsets[-1] + len(pairs))
        args["bias"] = (upload(offsets, torch.int32), upload([t for p in lists for t, _ in p], torch.int32),
                        upload([b for p in lists for _, b in p], torch.float32))
    if any(c.allowed is not None for c in rows_of):
        words, masks, which, seen = (vocab + 31) // 32, [], [], {}
        for c in rows_of:
            if c.allowed is None:
                which.append(-1)
                continue
            if id(c.allowed) not in seen:  # rows that share a mask object share its words
                whole = c.allowed.dtype == torch.bool and c.allowed.shape == (vocab,)
                mask = pack_mask(c.allowed) if whole else c.allowed
                if mask.dtype != torch.int32 or mask.shape != (words,):
                    raise ValueError("allowed must be bool [V] or packed int32 [ceil(V / 32)]")
                seen[id(c.allowed)] = len(masks)
                masks.append(mask.to(device, non_blocking=True))
            which.append(seen[id(c.allowed)])
        args.update(mask=torch.stack(masks), mask_rows=upload(which, torch.int32))
    return ops.control_logits(logits, **args, out=out)
