"""Block tables and maps of a serving step, built on the GPU from the requests' lengths (``csrc/step_maps.cu``).

A step holds ``n`` requests: request i sits in row ``rows[i]`` of a paged cache's block table, has ``cached[i]`` tokens in the cache and
brings more. What the kernels of the step read follows from these lengths: which blocks the row lists
(``extend_block_tables``), and position, cache row and place in the pool of every token, with the attention kernels' tiles
(``step_maps``). Built on the device a step's maps cost one launch, and a decode loop that stays on the device needs no host for them.

vLLM's scheduler keeps the same tables behind the reference's ``vllm serve`` deployments
(LLM_on_Kubernetes/Inference_Platfrom/README.md:1504-1509).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as nv

vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_EXTEND_ARGS = [vp, i64, i32, i32, vp, vp, vp, vp, i32, vp, i32, i32, vp]
_MAPS_ARGS = [vp, i64, i32, i32, vp, vp, vp, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp]
MOST = 2 ** 31 - 1   # sums of lengths stop there
TILE_Q = 64          # query rows per tile of the tensor-core attention kernels


@dataclass
class StepMaps:
    """Tables of one step of ``total`` tokens. ``cu`` int32 [n + 1]: request i is tokens cu[i] .. cu[i + 1] - 1; ``pos`` / ``slot`` int32 [total]:
    position and cache row; ``place`` int64 [total]: block * block_size + offset, the token's row in a pool's [blocks * block_size] (-1 where
    its row lists no block for it); ``last`` int64 [n]: the request's last token (one before its first, if it has none). With tiles:
    ``tiles`` / ``tile_of`` int32 [n_tiles, 4] and ``runs`` / ``run_tiles`` int32 [n, 4] as in ``inference.ragged.Pieces``."""
    cu: torch.Tensor
    pos: torch.Tensor
    slot: torch.Tensor
    place: torch.Tensor
    last: torch.Tensor
    tiles: Optional[torch.Tensor] = None
    tile_of: Optional[torch.Tensor] = None
    runs: Optional[torch.Tensor] = None
    run_tiles: Optional[torch.Tensor] = None


def _ints(n, device, tensors) -> bool:
    """All of them contiguous int32 [n] on the device?"""
    for t in tensors:
        if t.dtype is not torch.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
            return False
    return True


def _check(what, table, rows, block_size, *lengths):
    if (table.dtype is not torch.int32 or table.dim() != 2 or (table.stride(1) != 1 and table.shape[1] > 1)
            or (table.stride(0) < table.shape[1] and table.shape[0] > 1)):
        raise ValueError(f"{what}: the block table is int32 [rows, blocks] with contiguous rows, each of its own")
    if block_size < 1:
        raise ValueError(f"{what}: block_size must be positive, not {block_size}")
    if rows.dim() != 1 or not _ints(rows.shape[0], table.device, (rows, *lengths)):
        raise ValueError(f"{what}: rows and lengths must be contiguous int32 tensors of one size on the table's device, {table.device}")


def extend_block_tables(table: torch.Tensor, rows: torch.Tensor, cached: torch.Tensor, lens: torch.Tensor, blocks: torch.Tensor,
                        block_size: int = 1) -> torch.Tensor:
    """Give every request the blocks it lacks: row ``rows[i]`` of ``table`` (int32 [rows, max_blocks], changed in place) lists
    ``ceil(cached[i] / block_size)`` blocks and gets the next ``ceil(lens[i] / block_size) - that`` of the list ``blocks`` (int32) behind them, in the
    order of the requests (none where a length shrinks). ``rows`` are different rows. Returns the number of blocks that the requests need, int32 [1]
    on the device (``MOST`` where it is more): where it is more than ``blocks`` holds, entries beyond the list stay as they were, and so do those beyond
    the table's width. With ``block_size`` 1 ``cached`` and ``lens`` count blocks."""
    _check("extend_block_tables", table, rows, block_size, cached, lens)
    if blocks.dim() != 1 or not _ints(blocks.shape[0], table.device, (blocks,)):
        raise ValueError(f"extend_block_tables: blocks must be a contiguous int32 tensor on the table's device, {table.device}")
    n = rows.shape[0]
    used = table.new_empty(1)
    if nv.use_native(table):
        fn = nv.proto("b200_extend_block_tables", _EXTEND_ARGS)
        nv.check(nv.call_on(table.device, fn, table.data_ptr(), table.stride(0), *table.shape, rows.data_ptr(), cached.data_ptr(), lens.data_ptr(),
                            blocks.data_ptr(), blocks.shape[0], used.data_ptr(), n, block_size), "extend_block_tables")
        nv.count_launch()
        return used
    at = 0
    free = blocks.tolist()
    for row, c, k in zip(rows.tolist(), cached.tolist(), lens.tolist()):
        have, want = -(-max(c, 0) // block_size), -(-max(k, 0) // block_size)
        if 0 <= row < table.shape[0]:
            for j in range(have, min(want, table.shape[1], have + len(free) - at)):
                table[row, j] = free[at + j - have]
        at += max(want - have, 0)
    return used.fill_(min(at, MOST))


def step_maps(table: torch.Tensor, rows: torch.Tensor, cached: torch.Tensor, new: torch.Tensor, block_size: int, total: int,
              n_tiles: int = 0) -> StepMaps:
    """Maps of a step in which request i brings ``new[i]`` tokens from position ``cached[i]`` on (``rows``, ``cached``, ``new`` int32 [n]; ``table``
    int32 [rows, max_blocks] lists their blocks already). ``total``: the step's tokens, as known to the host: rows of the result, which where
    it is larger than the sum of ``new`` are not written behind that sum. ``n_tiles`` > 0: tables of the tiles too, so many of them; where the step
    has fewer, the others are of no rows (where more, they are left out). Positions are below 2^31, and ``cu`` stops at ``MOST``."""
    _check("step_maps", table, rows, block_size, cached, new)
    n, dev = rows.shape[0], table.device
    if n < 1 or total < 0 or n_tiles < 0:
        raise ValueError("step_maps: a step has at least one request, and no negative number of tokens or tiles")
    if not nv.use_native(table):
        return _step_maps_torch(table, rows, cached, new, block_size, total, n_tiles)
    four = 4 * n if n_tiles else 0
    # one allocation for the int32 tables (those of four columns first, so that they start on 16 bytes), one for the int64 ones
    at = 8 * n_tiles + 2 * four
    words = table.new_empty(at + 2 * total + n + 1)
    longs = table.new_empty(total + n, dtype=torch.int64)
    w, g = words.data_ptr(), longs.data_ptr()
    w_pos = w + 4 * at
    fn = nv.proto("b200_step_maps", _MAPS_ARGS)
    nv.check(nv.call_on(dev, fn, table.data_ptr(), table.stride(0), *table.shape, rows.data_ptr(), cached.data_ptr(), new.data_ptr(), n, block_size, total,
                        n_tiles, w_pos + 8 * total, w_pos, w_pos + 4 * total, g, g + 8 * total, w, w + 16 * n_tiles, w + 32 * n_tiles,
                        w + 32 * n_tiles + 4 * four), "step_maps")
    nv.count_launch()
    place, last = longs.split_with_sizes((total, n))
    if not n_tiles:
        pos, slot, cu = words.split_with_sizes((total, total, n + 1))
        return StepMaps(cu, pos, slot, place, last)
    fours, pos, slot, cu = words.split_with_sizes((at, total, total, n + 1))
    return StepMaps(cu, pos, slot, place, last, *fours.view(-1, 4).split_with_sizes((n_tiles, n_tiles, n, n)))


def _step_maps_torch(table, rows, cached, new, bs, total, n_tiles) -> StepMaps:
    dev, n = table.device, rows.shape[0]
    pos, slot = (torch.zeros(total, dtype=torch.int32, device=dev) for _ in range(2))
    place = torch.zeros(total, dtype=torch.int64, device=dev)
    cu, tiles, tile_of, run_tiles, at = [0], [], [], [], 0
    new_l = [max(0, k) for k in new.tolist()]
    for i, (row, c, k) in enumerate(zip(rows.tolist(), cached.tolist(), new_l)):
        nt = -(-k // TILE_Q)
        some = range(max(0, min(nt, n_tiles - at)))
        tiles += [[min(cu[-1] + j * TILE_Q, MOST), min(TILE_Q, k - j * TILE_Q), c + j * TILE_Q, row] for j in some]
        tile_of += [[i, j, nt, at] for j in some]
        run_tiles.append([min(at, MOST), nt, 0, 0])
        at += nt
        live = max(0, min(k, total - cu[-1]))
        p = torch.arange(c, c + live, device=dev)
        pos[cu[-1]:cu[-1] + live] = p.to(torch.int32)
        slot[cu[-1]:cu[-1] + live] = row
        listed = (p >= 0) & (p <= MOST) & (p // bs < table.shape[1])
        if 0 <= row < table.shape[0] and bool(listed.any()):
            blk = table[row, (p // bs).clamp(0, table.shape[1] - 1)].long()
            place[cu[-1]:cu[-1] + live] = torch.where(listed, blk * bs + p % bs, -1)
        else:
            place[cu[-1]:cu[-1] + live] = -1
        cu.append(cu[-1] + k)
    cu_t = torch.tensor([min(c, MOST) for c in cu], dtype=torch.int32, device=dev)
    maps = StepMaps(cu_t, pos, slot, place, cu_t[1:].long() - 1)
    if n_tiles:
        def table4(x, m):
            return torch.tensor((x + [[0, 0, 0, 0]] * m)[:m], device=dev).to(torch.int32).view(-1, 4)
        maps.tiles, maps.tile_of = table4(tiles, n_tiles), table4(tile_of, n_tiles)
        maps.run_tiles = table4(run_tiles, n)
        maps.runs = torch.stack([cu_t[:-1], torch.tensor(new_l, dtype=torch.int32, device=dev), cached, rows], 1)
    return maps
