"""Attention of a decode batch whose sequences share their first keys (``csrc/prefix_attn.cu``): the keys and values of the shared part
are read once for the whole group instead of once a sequence.

The sequences of a serving batch often start alike: a system prompt, a few-shot preamble, one long document with many questions. A paged
cache holds such a part once (the engine's prefix cache lists its blocks in every sequence's row), and ``paged_attention`` reads it
once for every sequence. ``prefix_attention`` is told the groups (``make_prefix_groups``) and gives the same result but for rounding: its weights, of a
token's own keys too, are rounded to the cache's 16 bits before the product with the values, on the tensor cores, where ``paged_attention`` keeps them in
32 (off from 64 bits by 2.3e-3 relative instead of 1.7e-3 in bf16, 2.6e-4 instead of 2.1e-4 in fp16). Maxima, sums and partial results have 32.

The reference's deployments turn on vLLM's prefix caching for this kind of traffic (Deployment/Ray/serve_run_examples/deepseek.py:29-34).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _native as nv
from .paged_attention import paged_attention

vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
_PLAN_ARGS = [i32] * 8
_ARGS = [vp, i64, vp, vp, i32, vp, vp, vp, i64, i32, i32, vp, vp, i32, i32, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32, f32, i32, vp]


@dataclass
class PrefixGroups:
    """Which tokens of a step share their first keys. ``groups`` int32 [n_groups, 4] = (first token, tokens, shared keys, 0); ``of`` int32 [tokens]:
    the group of every token, -1 for none. Bounds known on the host: ``longest`` (tokens of the largest group), ``max_shared`` and ``min_shared`` (shared
    keys of the group with the most; what every token of the step shares at least). A plan that a captured graph replays may be rewritten
    on the device: tokens of a group behind the ``longest``-th read all their keys by themselves, the other two only choose how the work is cut."""
    groups: torch.Tensor
    of: torch.Tensor
    n_groups: int
    longest: int
    max_shared: int
    min_shared: int = 0


def make_prefix_groups(groups: Sequence[Sequence[int]], tokens: int, device) -> PrefixGroups:
    """The plan of a step of ``tokens`` tokens from its groups ``(first token, tokens, shared keys)``: runs of consecutive tokens, none of them in
    two groups, whose sequences hold the same keys and values at positions ``0 .. shared - 1`` (in the same pages, or in copies). They are read
    from the pages that the group's first token lists."""
    rows, of = [], [-1] * tokens
    for first, n, shared in ([int(v) for v in g] for g in groups):
        if n < 0 or shared < 0 or first < 0 or first + n > tokens:
            raise ValueError(f"make_prefix_groups: group ({first}, {n}, {shared}) is not within {tokens} tokens")
        if n == 0 or shared == 0:
            continue
        if any(j >= 0 for j in of[first:first + n]):
            raise ValueError("make_prefix_groups: a token is in two groups")
        of[first:first + n] = [len(rows)] * n
        rows.append([first, n, shared, 0])
    host = torch.tensor([v for r in rows for v in r] + of, dtype=torch.int32)
    dev = torch.device(device)
    host = host.pin_memory().to(dev, non_blocking=True) if dev.type == "cuda" else host
    return PrefixGroups(host[:4 * len(rows)].view(-1, 4), host[4 * len(rows):], len(rows), max((r[1] for r in rows), default=0),
                        max((r[2] for r in rows), default=0), min((r[2] for r in rows), default=0) if -1 not in of else 0)


def prefix_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, table: torch.Tensor, pos: torch.Tensor, slot: torch.Tensor,
                     groups: Optional[PrefixGroups], n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                     sinks: Optional[torch.Tensor] = None, max_pos: int = 0, plan: int = 0) -> torch.Tensor:
    """Context [T, H * D] of token t over keys ``0 .. pos[t]`` of cache row ``slot[t]``, as ``paged_attention`` gives it (same arguments; no
    window), with the shared keys of ``groups`` read once. Tokens of a group whose position is before its last shared key, and tokens of no
    group, read all their keys by themselves. A token with ``pos`` -1, or a slot outside the table, sees no key: zeros. A table entry that names no
    page of the pools reads nothing outside of them; what its row gets is without meaning. ``max_pos``: an upper bound of ``pos`` known on the host
    (0: unknown). ``plan``: how the shared keys are cut, as ``b200_prefix_attn`` takes it (include/b200_ops.h); 0: chosen by the sizes.

    For caches of 16 bits with head sizes that are multiples of 16 up to 128, pages of a power of two from 8 on (fewer than 2^31 - 256 rows of a
    pool, fewer than 2^31 - 4096 places in a table row) and a positive scale; others go through ``paged_attention``, as does a step without groups. Captured into a graph, each
    call keeps a workspace of its own."""
    T, H, G, D = q.shape[0], n_heads, n_kv_heads, head_dim
    BS, dt = cache_k.shape[2], q.dtype
    if not nv.use_native(q):
        return _by_paged_attention(q, cache_k, cache_v, table, pos, slot, H, G, D, scale, sinks, max_pos)
    others = (groups is None or groups.n_groups == 0 or (dt is not torch.bfloat16 and dt is not torch.float16) or D % 16 or D > 128 or BS < 8 or BS & (BS - 1)
              or cache_k.shape[0] * G * BS >= 2 ** 31 - 256 or table.shape[-1] * BS >= 2 ** 31 - 4096 or not scale > 0)
    dev, pools = q.device, cache_k.shape
    if cache_k.dtype is not dt or cache_v.dtype is not dt or cache_v.shape != pools or pools[1] != G or pools[3] != D:
        raise ValueError(f"prefix_attention: caches must be {dt} [blocks, {G}, block_size, {D}], both of one shape")
    if not cache_k.is_contiguous() or not cache_v.is_contiguous() or cache_k.device != dev or cache_v.device != dev:
        raise ValueError("prefix_attention: caches must be contiguous and on the queries' device")
    q_ptr, stride = q.data_ptr(), q.stride()
    row = stride[0] if T > 1 else H * D
    if H % G or len(stride) != 2 or q.shape[1] < H * D or (T and stride[1] != 1) or (not others and (row < H * D or row % 8 or q_ptr % 16)):
        raise ValueError(f"prefix_attention: queries must be rows of {H * D} or more contiguous values that start on 16 bytes, each of its own")
    if table.dtype is not torch.int32 or table.dim() != 2 or table.device != dev or (table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError("prefix_attention: the block table is int32 [rows, blocks] with contiguous rows on the queries' device")
    if sinks is not None and (sinks.dtype is not torch.float32 or sinks.shape != (H,) or not sinks.is_contiguous() or sinks.device != dev):
        raise ValueError(f"prefix_attention: sinks must be contiguous fp32 [{H}] on the queries' device")
    tokens = (T,)
    tables = ((pos, tokens), (slot, tokens)) if others else ((pos, tokens), (slot, tokens), (groups.of, tokens), (groups.groups, (groups.n_groups, 4)))
    for t, shape in tables:
        if t.dtype is not torch.int32 or t.shape != shape or t.device != dev or not t.is_contiguous():
            raise ValueError(f"prefix_attention: pos, slot and the groups' tables must be contiguous int32 tensors for {T} tokens on the queries' device")
    if others:
        if cache_k.data_ptr() % 16 or cache_v.data_ptr() % 16:
            raise ValueError("prefix_attention: caches must start on 16 bytes")
        with torch.cuda.device(dev):
            return _by_paged_attention(q, cache_k, cache_v, table, pos, slot, H, G, D, scale, sinks, max_pos)
    of, rows, n_groups = groups.of, groups.groups, groups.n_groups
    most_own = max(1, max_pos + 1 - groups.min_shared) if max_pos else 0
    if not plan:
        plan = nv.proto("b200_prefix_attn_plan", _PLAN_ARGS)(T, n_groups, groups.longest, groups.max_shared, most_own, H, G, D)
    out = q.new_empty((T, H * D))
    part = q.new_empty(T * H * (plan % 256) * (D + 2), dtype=torch.float32)
    fn = nv.proto("b200_prefix_attn", _ARGS)
    nv.check(nv.call_on(dev, fn, q_ptr, row, cache_k.data_ptr(), cache_v.data_ptr(), pools[0], pos.data_ptr(), slot.data_ptr(), table.data_ptr(),
                        table.stride(0), *table.shape, rows.data_ptr(), of.data_ptr(), n_groups, groups.longest, nv.ptr(sinks),
                        out.data_ptr(), part.data_ptr(), plan, most_own, T, H, G, D, BS, scale, nv.dtype_code(dt)), "prefix_attn")
    nv.count_launch(2)
    return out


def _by_paged_attention(q, cache_k, cache_v, table, pos, slot, H, G, D, scale, sinks, max_pos):
    """``paged_attention`` takes slots, positions and pages as they are: what lies outside the table or the pools is seen to here."""
    if q.shape[0] == 0:
        return q.new_empty((0, H * D))
    n, last = table.shape[0], min(table.shape[1] * cache_k.shape[2], 2 ** 31) - 1
    row = slot.clamp(0, max(n - 1, 0))
    pos = torch.where(row == slot, pos.clamp(max=last), -1) if n else torch.full_like(pos, -1)
    return paged_attention(q, cache_k, cache_v, table.clamp(0, cache_k.shape[0] - 1).contiguous(), pos, row, H, G, D, scale, sinks=sinks, max_pos=max_pos)
