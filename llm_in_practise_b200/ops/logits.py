"""Rules on the logits of a serving batch (``csrc/logits.cu``): penalties for repeated tokens, biases, temperature and a grammar's mask.

``LogitState`` holds the rules of every sequence on the device, one row each (as the KV cache has one row a sequence): its history, its
penalties, its biases, its mask. ``process_logits`` applies them to a batch of logits in one pass, ``greedy_tokens`` takes the best token of
each row without writing the logits out, ``LogitState.append`` puts the tokens that were chosen behind the histories. With l a logit in
32 bits, c how often its token stands in the row's output and seen whether it stands in the prompt or the output::

    y = l;  seen: y * r if y < 0 else y / r;  c > 0: y - f c - p;  y + bias;  y / T;  not allowed: -inf

r, f, p are HF's ``repetition_penalty`` (Quantization/GPTQModel/inference_qwen3_4b_gptq.py:58-68) and the OpenAI API's
``frequency_penalty`` and ``presence_penalty``, the bias its ``logit_bias``; the mask is what structured output hands a vLLM server.
The bias comes behind the repetition penalty, which scales what the model says and not what the caller adds. HF and vLLM add it first and scale
the sum: for a seen token with both (and r not 1) they give another value, (l + bias) r or (l + bias) / r. All other rules commute or stand in
one place only.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Dict, Optional, Sequence

import torch

from . import _native as nv

vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_PROCESS_ARGS = [vp, i64, i32, i32, vp, vp, vp, vp, i64, i32, vp]
_GREEDY_ARGS = [vp, i64, i32, i32, vp, vp, vp, vp, i32, vp]
MAX_VOCAB = 1 << 19
MAX_BIAS = 2047          # biases of one row
MAX_HISTORY = (1 << 20) - 1      # tokens of one row's history
SCALES = (2.0 ** -126, 2.0 ** 126)       # repetition penalties and temperatures: numbers whose reciprocal has all its bits
_LOCK = threading.RLock()       # held while a state's tensors are exchanged or their addresses are taken


class _Rules(ctypes.Structure):
    """``b200_logit_rules`` (include/b200_ops.h)."""
    _fields_ = [(n, vp) for n in ("tokens", "length", "prompt_length", "repetition", "presence", "frequency", "temperature", "bias_ids",
                                  "bias_length", "bias_values", "mask", "masked")] + [(n, ctypes.c_int32) for n in ("rows", "width", "bias_width", "words")]


class LogitState:
    """Rules of ``rows`` sequences over a vocabulary of ``vocab`` tokens, histories of up to ``max_len`` tokens, up to ``max_bias`` biases each.
    The tensors may be filled directly (``set_row`` does it from Python values): ``tokens`` int32 [rows, max_len], of which ``length`` [rows] are
    the history and its first ``prompt_length`` [rows] the prompt; ``repetition``, ``presence``, ``frequency``, ``temperature`` fp32 [rows];
    (the first and the last of these four within ``SCALES``); ``bias_ids`` int32 / ``bias_values`` fp32 [rows, max_bias] with ``bias_length`` [rows]; after ``allow_masks()`` ``mask`` int32
    [rows, ceil(vocab / 32)] (bit v % 32 of word v // 32 set: token v is allowed) and ``masked`` bool [rows]. Tokens outside 0 .. vocab - 1 are
    passed over, and of biases for one token the last one counts. Sequences, and calls on several streams, may share a state as long as
    nobody writes the rows that another call reads; tensors put in place of others count from the next call on."""

    def __init__(self, rows: int, vocab: int, max_len: int, max_bias: int = 0, device=None):
        if rows < 1 or not 1 <= vocab <= MAX_VOCAB or not 1 <= max_len <= MAX_HISTORY or not 0 <= max_bias <= MAX_BIAS:
            raise ValueError(f"LogitState: rows must be positive, vocab 1 .. {MAX_VOCAB}, max_len 1 .. {MAX_HISTORY}, max_bias 0 .. {MAX_BIAS}")
        self.rows, self.vocab, self.max_len, self.max_bias = rows, vocab, max_len, max_bias
        self.words = -(-vocab // 32)

        def of(dtype, *shape, value=0):
            return torch.full(shape, value, dtype=dtype, device=device)
        self.tokens, self.length, self.prompt_length = of(torch.int32, rows, max_len), of(torch.int32, rows), of(torch.int32, rows)
        self.repetition, self.temperature = of(torch.float32, rows, value=1.0), of(torch.float32, rows, value=1.0)
        self.presence, self.frequency = of(torch.float32, rows), of(torch.float32, rows)
        self.bias_ids, self.bias_values = of(torch.int32, rows, max_bias), of(torch.float32, rows, max_bias)
        self.bias_length = of(torch.int32, rows)
        self.mask = self.masked = None
        self._work = {}                                  # bytes of a workspace and launches, by batch size and form
        self.device = self.tokens.device

    def allow_masks(self) -> "LogitState":
        """Room for a mask a row (all of them off). A graph captured before there is room applies no masks."""
        if self.mask is None:
            mask = torch.zeros(self.rows, self.words, dtype=torch.int32, device=self.device)
            masked = torch.zeros(self.rows, dtype=torch.bool, device=self.device)
            with _LOCK:                                  # both at once, and not over masks that another thread made room for meanwhile
                if self.mask is None:
                    self.__dict__.update(mask=mask, masked=masked, _struct=None)
        return self

    def set_row(self, row: int, prompt: Sequence[int] = (), output: Sequence[int] = (), repetition_penalty: float = 1.0, presence_penalty: float = 0.0,
                frequency_penalty: float = 0.0, temperature: float = 1.0, logit_bias: Optional[Dict[int, float]] = None,
                allowed: Optional[Sequence[int]] = None) -> None:
        """The rules of ``row`` from Python values; what the row held is gone. ``allowed``: the only tokens that may come next (None: all)."""
        if not 0 <= row < self.rows:
            raise ValueError(f"LogitState: no row {row} of {self.rows}")
        if not all(SCALES[0] <= v <= SCALES[1] for v in (repetition_penalty, temperature)):
            raise ValueError(f"LogitState: repetition_penalty and temperature must be from {SCALES[0]:.2g} to {SCALES[1]:.2g}, not {repetition_penalty} and "
                             f"{temperature}")
        hist, bias = list(prompt) + list(output), dict(logit_bias or {})
        if len(hist) > self.max_len or len(bias) > self.max_bias:
            raise ValueError(f"LogitState: {len(hist)} tokens and {len(bias)} biases do not fit rows of {self.max_len} and {self.max_bias}")
        bad = [t for t in [*bias, *(() if allowed is None else allowed)] if not 0 <= int(t) < self.vocab]
        if bad:
            raise ValueError(f"LogitState: token {bad[0]} is not one of the vocabulary's {self.vocab}")
        # all that may fail comes before the first write
        ids = _in_32_bits(torch.tensor(hist, dtype=torch.int64))
        bias_ids = torch.tensor([int(k) for k in bias], dtype=torch.int32)
        values = torch.tensor([float(v) for v in bias.values()], dtype=torch.float32)
        numbers = [(self.length, len(hist)), (self.prompt_length, len(prompt)), (self.repetition, float(repetition_penalty)),
                   (self.presence, float(presence_penalty)), (self.frequency, float(frequency_penalty)), (self.temperature, float(temperature)),
                   (self.bias_length, len(bias))]
        for t, v in numbers:
            t[row] = v
        if hist:
            self.tokens[row, :len(hist)] = ids.to(self.device)
        if bias:
            self.bias_ids[row, :len(bias)] = bias_ids.to(self.device)
            self.bias_values[row, :len(bias)] = values.to(self.device)
        self.set_mask(row, allowed)

    def set_mask(self, row: int, allowed: Optional[Sequence[int]]) -> None:
        """The tokens that may come next in ``row`` (None: all of them)."""
        if not 0 <= row < self.rows:
            raise ValueError(f"LogitState: no row {row} of {self.rows}")
        ids = None if allowed is None else torch.as_tensor(list(allowed), dtype=torch.long)
        if ids is not None and len(ids) and not 0 <= int(ids.min()) <= int(ids.max()) < self.vocab:
            raise ValueError(f"LogitState: a mask names tokens {int(ids.min())} .. {int(ids.max())}, and the vocabulary has {self.vocab}")
        if ids is None:
            if self.mask is not None:
                self.masked[row] = False
            return
        self.allow_masks()
        bits = torch.zeros(self.words * 32, dtype=torch.bool)
        bits[ids] = True
        word = (bits.view(-1, 32).long() << torch.arange(32)).sum(1)
        self.mask[row] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32).to(self.device)
        self.masked[row] = True

    def append(self, ids: torch.Tensor, slot: Optional[torch.Tensor] = None) -> None:
        """Put ``ids[i]`` (int64 [n]) behind the history of row ``slot[i]`` (int32 [n], all different; None: row i). A full row keeps what it has."""
        _check_slot("append", self, ids.shape[0], slot)
        if ids.dtype != torch.int64 or ids.dim() != 1 or not ids.is_contiguous() or ids.device != self.device:
            raise ValueError("append: ids must be a contiguous int64 tensor on the state's device")
        if nv.use_native(self.tokens):
            fn = nv.proto("b200_append_tokens", [vp, i32, i32, vp, vp, vp, i32, vp])
            nv.check(nv.call_on(self.device, fn, nv.ptr(self.tokens), self.rows, self.max_len, nv.ptr(self.length), nv.ptr(slot), nv.ptr(ids),
                                ids.shape[0]), "append_tokens")
            nv.count_launch()
            return
        rows = range(ids.shape[0]) if slot is None else slot.tolist()
        for s, t in zip(rows, _in_32_bits(ids).tolist()):
            at = int(self.length[s]) if 0 <= s < self.rows else -1
            if 0 <= at < self.max_len:
                self.tokens[s, at] = t
                self.length[s] = at + 1

    def __setattr__(self, name, value):
        with _LOCK:
            object.__setattr__(self, name, value)
            self.__dict__["_struct"] = None              # holds the tensors' addresses

    def _address(self) -> _Rules:
        """What a native call takes the address of. Whoever calls holds it until the call is back: it keeps the tensors that it names, and another thread
        may have put others in their place by then."""
        rules = self._struct
        if rules is None:
            with _LOCK:
                self._check_tensors()
                tensors = [getattr(self, n) for n, _ in _Rules._fields_[:12]]
                rules = _Rules(*map(nv.ptr, tensors), self.rows, self.max_len, self.max_bias, self.words)
                rules.tensors = tensors
                self.__dict__["_struct"] = rules
        return rules

    def _check_tensors(self) -> None:
        """Tensors that were put in place of the state's own are like them."""
        i, f, R = torch.int32, torch.float32, (self.rows,)
        kinds = {"tokens": (i, (self.rows, self.max_len)), "length": (i, R), "prompt_length": (i, R), "repetition": (f, R), "presence": (f, R),
                 "frequency": (f, R), "temperature": (f, R), "bias_ids": (i, (self.rows, self.max_bias)), "bias_values": (f, (self.rows, self.max_bias)),
                 "bias_length": (i, R), "mask": (i, (self.rows, self.words)), "masked": (torch.bool, R)}
        for name, (dtype, shape) in kinds.items():
            t = getattr(self, name)
            if t is None and name in ("mask", "masked") and self.mask is self.masked:
                continue
            if t is None or t.dtype is not dtype or t.shape != shape or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"LogitState: {name} must be a contiguous {dtype} {list(shape)} tensor on {self.device}")


def _in_32_bits(ids: torch.Tensor) -> torch.Tensor:
    """int64 tokens as int32; those that it does not hold are -1, which is no token either."""
    return torch.where(ids == ids.to(torch.int32), ids, -1).to(torch.int32)


def _check_slot(what, state, n, slot):
    if slot is not None and (slot.dtype is not torch.int32 or slot.shape != (n,) or not slot.is_contiguous() or slot.device != state.device):
        raise ValueError(f"{what}: slot must be a contiguous int32 [{n}] tensor on the state's device")
    if slot is None and n > state.rows:
        raise ValueError(f"{what}: {n} rows, and the state has {state.rows}: name them with slot")


def _check(what, logits, state, slot):
    if logits.dim() != 2 or logits.shape[1] != state.vocab or logits.device != state.device:
        raise ValueError(f"{what}: logits must be [rows, {state.vocab}] on {state.device}, like the state")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: logits must be fp32, bf16 or fp16, not {logits.dtype}")
    if logits.stride(1) != 1 and state.vocab > 1:
        raise ValueError(f"{what}: the logits of a row must be contiguous")
    _check_slot(what, state, logits.shape[0], slot)


def process_logits(logits: torch.Tensor, state: LogitState, slot: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [B, vocab] (fp32, bf16 or fp16; rows may be strided) after the rules of rows ``slot`` (int32 [B], None: row b for batch row b; a slot
    outside the state has no rules) as fp32 [B, vocab], in ``out`` if given (fp32 logits may be their own ``out``). A row whose mask allows
    nothing is all minus infinity."""
    _check("process_logits", logits, state, slot)
    if out is None:
        out = logits.new_empty(logits.shape, dtype=torch.float32)
    elif (out.dtype != torch.float32 or out.shape != logits.shape or out.device != logits.device or (out.stride(1) != 1 and state.vocab > 1)
          or (out.stride(0) < state.vocab and out.shape[0] > 1)):
        raise ValueError("process_logits: out must be fp32, like the logits in shape, with contiguous rows, each of its own")
    elif _overlap(out, logits) and (out.data_ptr(), out.dtype, out.stride(0)) != (logits.data_ptr(), logits.dtype, logits.stride(0) if out.shape[0] > 1 else out.stride(0)):
        raise ValueError("process_logits: out and the logits overlap without being the same")
    if not nv.use_native(logits):
        return out.copy_(_rules_torch(logits, state, slot))
    if logits.shape[0] == 0:
        return out
    work, launches = _workspace(state, logits.shape[0], 0)
    fn, rules = nv.proto("b200_process_logits", _PROCESS_ARGS), state._address()
    nv.check(nv.call_on(state.device, fn, logits.data_ptr(), logits.stride(0), logits.shape[0], state.vocab, nv.ptr(slot), ctypes.addressof(rules),
                        work.data_ptr(), out.data_ptr(), out.stride(0), nv.dtype_code(logits.dtype)), "process_logits")
    nv.count_launch(launches)
    return out


def _overlap(a, b) -> bool:
    """Whether the memory from the first to the last element of one reaches into the other's."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()) for t in (a, b))
    return a0 < b1 and b0 < a1


def _workspace(state, B, greedy):
    """The call's scratch, and how many kernels it launches."""
    known = state._work.get((B, greedy))
    if known is None:
        fn = nv.lib().b200_logits_workspace
        fn.argtypes, fn.restype = [i32] * 3, i64
        known = state._work[B, greedy] = fn(B, state.vocab, greedy), nv.proto("b200_logits_launches", [i32] * 3)(B, state.vocab, greedy)
    return state.tokens.new_empty(known[0], dtype=torch.uint8), known[1]


def greedy_tokens(logits: torch.Tensor, state: LogitState, slot: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``process_logits(...).argmax(1)`` (int64 [B]) without the logits in between: the best token of each row, the lowest of equals; a NaN is
    above all, and a row whose mask allows nothing gives 0."""
    _check("greedy_tokens", logits, state, slot)
    if not nv.use_native(logits):
        return _rules_torch(logits, state, slot).argmax(1)
    B = logits.shape[0]
    ids = logits.new_empty(B, dtype=torch.int64)
    if B == 0:
        return ids
    work, launches = _workspace(state, B, 1)
    fn, rules = nv.proto("b200_greedy_tokens", _GREEDY_ARGS), state._address()
    nv.check(nv.call_on(state.device, fn, logits.data_ptr(), logits.stride(0), B, state.vocab, nv.ptr(slot), ctypes.addressof(rules),
                        work.data_ptr(), ids.data_ptr(), nv.dtype_code(logits.dtype)), "greedy_tokens")
    nv.count_launch(launches)
    return ids


def _rules_torch(logits, st, slot):
    y = logits.float().clone()
    rows = range(y.shape[0]) if slot is None else slot.tolist()
    for b, s in enumerate(rows):
        if not 0 <= s < st.rows:
            continue
        r, f, p, T = (float(t[s]) for t in (st.repetition, st.frequency, st.presence, st.temperature))
        n, m = min(max(int(st.length[s]), 0), st.max_len), max(int(st.prompt_length[s]), 0)
        hist = st.tokens[s, :n].long()
        ok = (hist >= 0) & (hist < st.vocab)
        v = y[b]
        if n and (r != 1.0 or f != 0.0 or p != 0.0):
            seen = torch.zeros(st.vocab, dtype=torch.bool, device=y.device)
            seen[hist[ok]] = True
            said = hist[m:][ok[m:]]
            c = torch.bincount(said, minlength=st.vocab)
            v = torch.where(seen, torch.where(v < 0, v * st.repetition[s], v / st.repetition[s]), v)
            v = torch.where(c > 0, v - st.frequency[s] * c.float() - st.presence[s], v)
        for i in range(min(max(int(st.bias_length[s]), 0), st.max_bias)):
            t = int(st.bias_ids[s, i])
            later = (st.bias_ids[s, i + 1:int(st.bias_length[s])] == t).any() if st.max_bias else False
            if 0 <= t < st.vocab and not bool(later):
                v = v.clone() if v is y[b] else v
                v[t] += st.bias_values[s, i]
        if T != 1.0:
            v = v / st.temperature[s]
        if st.mask is not None and bool(st.masked[s]):
            t = torch.arange(st.vocab, device=y.device)
            v = torch.where(((st.mask[s][t // 32] >> (t % 32)) & 1) == 0, torch.full_like(v, float("-inf")), v)
        y[b] = v
    return y
