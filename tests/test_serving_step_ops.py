"""Operators of a serving step that shares work between its sequences: attention over shared keys, block tables and maps from the
requests' lengths, rules on logits. Each against a statement of its own in 64 bits (or in whole numbers), token by token; the plain PyTorch
path on the CPU, the kernels on the GPU."""
import collections
import gc
import itertools
import re
import weakref

import pytest
import torch

import test_kernel_sources_cpu as sources

from llm_in_practise_b200.ops import _native as nv
from llm_in_practise_b200.ops import logits as logits_module
from llm_in_practise_b200.ops.logits import LogitState, greedy_tokens, process_logits
from llm_in_practise_b200.ops.prefix_attention import make_prefix_groups, prefix_attention
from llm_in_practise_b200.ops.step_maps import extend_block_tables, step_maps

CPU_AND_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF, NAN = float("inf"), float("nan")


@pytest.fixture
def entries(monkeypatch):
    """Names of the entry points that took a call."""
    names, real = [], nv.proto

    def proto(name, argtypes):
        fn = real(name, argtypes)

        def call(*args):
            rc = fn(*args)
            names.append(name)
            return rc
        return call
    monkeypatch.setattr(nv, "proto", proto)
    return names


# ------------------------------------------------------------------------------------------------ block tables
def grown(table, rows, cached, lens, blocks, bs):
    table, at = [list(r) for r in table], 0
    for row, c, n in zip(rows, cached, lens):
        for j in range(-(-max(c, 0) // bs), -(-max(n, 0) // bs)):
            if 0 <= row < len(table) and j < len(table[0]) and at < len(blocks):
                table[row][j] = blocks[at]
            at += 1
    return table, at


def requests(n, cached, new, seed, rows=None):
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, cached + 1, (n,), generator=g).tolist()
    k = torch.randint(0, new + 1, (n,), generator=g).tolist()
    return c, k, torch.randperm(rows or n + 2, generator=g)[:n].tolist()


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("n,cached,new,bs,spare", [(1, 0, 1, 16, 0), (1, 17, 0, 16, 0), (31, 100, 40, 16, 3), (32, 100, 40, 1, 0), (33, 5, 3, 64, -2), (200, 0, 900, 16, 9),
                                                   (64, 4000, 1, 16, 0), (1000, 30, 70, 8, 0), (4097, 9, 9, 4, -50)])
def test_block_tables(device, n, cached, new, bs, spare):
    """Blocks in the order of the requests; a list that ends too early leaves the rest of the rows as they were, and says how many it lacks."""
    c, k, rows = requests(n, cached, new, n + new)
    lens = [a + b for a, b in zip(c, k)]
    need = sum(-(-b // bs) - -(-a // bs) for a, b in zip(c, lens))
    blocks = list(range(7, 7 + max(0, need + spare)))
    width = -(-max(lens + [1]) // bs)
    wide = i32([[-5] * (width + 3)] * (n + 2), device)
    table = wide[:, :width]                                           # rows of a wider table
    before = table.tolist()
    used = extend_block_tables(table, i32(rows, device), i32(c, device), i32(lens, device), i32(blocks, device), bs)
    want, at = grown(before, rows, c, lens, blocks, bs)
    assert table.tolist() == want and used.tolist() == [at] and at == need
    assert bool((wide[:, width:] == -5).all())


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_block_tables_keep_to_their_bounds(device):
    """Rows outside the table, rows that are too short, lengths that shrink or are negative: what does not fit is left out, nothing else is touched."""
    rows, c, lens = [-1, 0, 5, 1, 2, 3], [0, 0, 0, 40, 3, -9], [64, 200, 64, 20, 36, 32]
    table = i32([[0] * 4 for _ in range(4)], device)
    used = extend_block_tables(table, i32(rows, device), i32(c, device), i32(lens, device), i32(list(range(100, 140)), device), 16)
    want, at = grown([[0] * 4 for _ in range(4)], rows, c, lens, list(range(100, 140)), 16)
    assert table.tolist() == want and used.tolist() == [at]
    none = i32([], device)
    assert extend_block_tables(table, none, none, none, none, 16).tolist() == [0] and table.tolist() == want


def maps_of(table, rows, cached, new, bs):
    cu, pos, slot, place, tiles, tile_of, run_tiles = [0], [], [], [], [], [], []
    for i, (row, c, k) in enumerate(zip(rows, cached, new)):
        run_tiles.append([len(tiles), -(-k // 64), 0, 0])
        tile_of += [[i, j, -(-k // 64), len(tiles)] for j in range(-(-k // 64))]
        tiles += [[cu[-1] + a, min(64, k - a), c + a, row] for a in range(0, k, 64)]
        for p in range(c, c + k):
            pos.append(p)
            slot.append(row)
            place.append(table[row][p // bs] * bs + p % bs if 0 <= row < len(table) and 0 <= p // bs < len(table[0]) else -1)
        cu.append(cu[-1] + k)
    runs = [[cu[i], k, c, row] for i, (row, c, k) in enumerate(zip(rows, cached, new))]
    return dict(cu=cu, pos=pos, slot=slot, place=place, last=[x - 1 for x in cu[1:]], tiles=tiles, tile_of=tile_of, runs=runs, run_tiles=run_tiles)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("n,cached,new,bs", [(1, 0, 1, 16), (1, 3, 0, 16), (1, 9, 5000, 16), (32, 50, 1, 64), (33, 700, 130, 16), (60, 3000, 2000, 16), (300, 40, 3, 1),
                                             (2000, 100, 20, 32)])
def test_step_maps(device, n, cached, new, bs):
    c, k, rows = requests(n, cached, new, n)
    width = -(-(cached + new) // bs) + 1
    g = torch.Generator().manual_seed(1)
    table = torch.randperm((n + 2) * width, generator=g).view(n + 2, width).to(torch.int32)
    want = maps_of(table.tolist(), rows, c, k, bs)
    table = table.to(device)
    bare = step_maps(table, i32(rows, device), i32(c, device), i32(k, device), bs, sum(k))
    full = step_maps(table, i32(rows, device), i32(c, device), i32(k, device), bs, sum(k), n_tiles=len(want["tiles"]) + 2)
    assert bare.tiles is None
    for m in (bare, full):
        assert all(getattr(m, f).tolist() == want[f] for f in ("cu", "pos", "slot", "place", "last"))
    for f in ("tiles", "tile_of"):                                    # two tiles more than there are: of no rows
        assert getattr(full, f).tolist() == want[f] + [[0, 0, 0, 0]] * 2
    assert full.runs.tolist() == want["runs"] and full.run_tiles.tolist() == want["run_tiles"]


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_step_maps_keep_to_their_bounds(device):
    """A table that does not list a token's block gives no place for it; tables sized for fewer tokens or tiles than there are are not left."""
    rows, c, k = [0, 7, 1, -2, 2], [0, 0, 30, 4, -2], [70, 3, 8, 2, 5]
    table = torch.arange(1, 10, dtype=torch.int32).view(3, 3)
    want = maps_of(table.tolist(), rows, c, k, 16)
    m = step_maps(table.to(device), i32(rows, device), i32(c, device), i32(k, device), 16, 40, n_tiles=3)
    assert m.cu.tolist() == want["cu"] and m.pos.tolist() == want["pos"][:40] and m.place.tolist() == want["place"][:40]
    assert m.tiles.tolist() == want["tiles"][:3]
    more = step_maps(table.to(device), i32(rows, device), i32(c, device), i32(k, device), 16, 100)
    assert more.place[:88].tolist() == want["place"] and len(more.place) == 100
    assert -1 in want["place"][70:73] and -1 in want["place"][-7:]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("n", [4, 70])
def test_lengths_whose_sums_pass_31_bits(device, n):
    """Requests that need more blocks, or bring more tokens, than 32 bits count: those before them have theirs, those behind them nothing, never the first ones'
    again; sums stop at 2^31 - 1. The last of 70 is in another CTA than the long ones."""
    most = 2 ** 31 - 1
    lens = [5, most, most] + [3] * (n - 3)
    rows = list(range(n))
    before = [[-5] * 6 for _ in range(n)]
    zeros, blocks = [0] * n, list(range(100, 109))
    table = i32(before, device)
    used = extend_block_tables(table, i32(rows, device), i32(zeros, device), i32(lens, device), i32(blocks, device), 1)
    assert used.tolist() == [most] and table[0].tolist() == [100, 101, 102, 103, 104, -5] and table[1].tolist() == [105, 106, 107, 108, -5, -5]
    assert bool((table[2:] == -5).all())
    used = extend_block_tables(table, i32(rows, device), i32(zeros, device), i32([most, 0, 0] + lens[3:], device), i32(list(range(7)), device), 16)
    assert used.tolist() == [2 ** 27 + n - 3] and table[0].tolist() == [0, 1, 2, 3, 4, 5] and bool((table[2:] == -5).all())

    table = torch.arange(6 * n, dtype=torch.int32).view(n, 6)
    lens = [70] + lens[1:]
    cached = [2, 9, most - 64] + [0] * (n - 3)
    want = [list(range(2, 72)) + list(range(9, 39)), [0] * 70 + [1] * 30]
    m = step_maps(table.to(device), i32(rows, device), i32(cached, device), i32(lens, device), 16, 100, n_tiles=5)
    assert [m.pos.tolist(), m.slot.tolist()] == want
    assert m.place.tolist() == [int(table[s, p // 16]) * 16 + p % 16 for p, s in zip(*want)]
    assert m.cu.tolist() == [0, 70] + [most] * (n - 1) and m.last.tolist() == [69] + [most - 1] * (n - 1)
    assert m.tiles.tolist() == [[0, 64, 2, 0], [64, 6, 66, 0], [70, 64, 9, 1], [134, 64, 73, 1], [198, 64, 137, 1]]
    nt = 2 ** 25
    assert m.tile_of.tolist() == [[0, 0, 2, 0], [0, 1, 2, 0], [1, 0, nt, 2], [1, 1, nt, 2], [1, 2, nt, 2]]
    assert m.runs[:4].tolist() == [[0, 70, 2, 0], [70, most, 9, 1], [most, most, most - 64, 2], [most, 3, 0, 3]]
    assert m.run_tiles[:4].tolist() == [[0, 2, 0, 0], [2, nt, 0, 0], [2 + nt, nt, 0, 0], [2 + 2 * nt, 1, 0, 0]]
    # a position behind the last of 32 bits has no place
    m = step_maps(table.to(device), i32([0], device), i32([most - 1], device), i32([4], device), 2 ** 30, 4, n_tiles=1)
    assert m.place.tolist() == [(int(table[0, 1]) * 2 ** 30) + 2 ** 30 - 2, (int(table[0, 1]) * 2 ** 30) + 2 ** 30 - 1, -1, -1] and m.tiles.tolist() == [[0, 4, most - 1, 0]]


def test_refusals_of_tables():
    t, r = torch.zeros(4, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(table=t.long()), dict(rows=r.long()), dict(cached=r[:1]), dict(lens=r.view(1, 2)), dict(block_size=0), dict(table=t.t()), dict(table=t[:1].expand(4, 4)),
                dict(blocks=torch.zeros(8, dtype=torch.int32)[::2])):
        args = dict(table=t, rows=r, cached=r, lens=r, blocks=r, block_size=16)
        args.update(bad)
        with pytest.raises(ValueError, match="extend_block_tables"):
            extend_block_tables(**args)
    for bad in (dict(new=r.float()), dict(total=-1), dict(n_tiles=-1), dict(rows=r[:0], cached=r[:0], new=r[:0])):
        args = dict(table=t, rows=r, cached=r, new=r, block_size=16, total=0)
        args.update(bad)
        with pytest.raises(ValueError, match="step_maps"):
            step_maps(**args)


# ------------------------------------------------------------------------------------------------ rules on logits
def exact_rules(x, rows):
    """One row after another in 64 bits. rows: dicts as for LogitState.set_row, or None for a row without rules. Returns values and, for each, a
    bound: six roundings to 32 bits, each half a step of what stands there, on values that a subtraction may make small."""
    out, size = [], []
    for l, r in zip(x.double(), rows):
        y, s = l.clone(), l.abs()
        if r is not None:
            prompt, said = list(r.get("prompt", ())), list(r.get("output", ()))
            V = y.shape[0]
            for t in {t for t in prompt + said if 0 <= t < V}:
                rep = f32(r.get("repetition_penalty", 1.0))
                y[t] = y[t] * rep if y[t] < 0 else y[t] / rep
                s[t] = torch.maximum(s[t], y[t].abs())
            for t in {t for t in said if 0 <= t < V}:
                f, p = f32(r.get("frequency_penalty", 0.0)), f32(r.get("presence_penalty", 0.0))
                y[t] -= f * said.count(t) + p
                s[t] += abs(f) * said.count(t) + abs(p)
            for t, v in (r.get("logit_bias") or {}).items():
                y[t] += f32(v)
                s[t] += abs(f32(v))
            T = f32(r.get("temperature", 1.0))
            y, s = y / T, s / T
            if r.get("allowed") is not None:
                keep = torch.zeros(V, dtype=torch.bool)
                keep[torch.tensor(list(r["allowed"]), dtype=torch.long)] = True
                y[~keep] = -INF
        out.append(y)
        size.append(s)
    return torch.stack(out), torch.stack(size) * 6 * 2.0 ** -24


def f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def some_rules(V, B, seed, max_len):
    """Rows of all kinds: no rules, each rule alone, all of them, histories with the same token many times and tokens outside the vocabulary."""
    g = torch.Generator().manual_seed(seed)

    def toks(n):
        return torch.where(torch.rand(n, generator=g) < 0.5, torch.randint(0, V, (n,), generator=g), torch.randint(0, min(V, 5), (n,), generator=g)).tolist()
    rows = []
    for b in range(B):
        n = int(torch.randint(0, max_len // 2 + 1, (1,), generator=g))
        r = dict(prompt=toks(n) + [-1, V, 2 ** 31 - 1][:b % 4], output=toks(max_len // 3))
        kind = b % 7
        if kind in (1, 6):
            r["repetition_penalty"] = 1.3 if b % 2 else 0.7
        if kind in (2, 6):
            r["presence_penalty"] = 0.75
        if kind in (3, 6):
            r["frequency_penalty"] = -0.31
        if kind in (4, 6):
            ids = torch.randperm(V, generator=g)[:5].tolist()
            r["logit_bias"] = dict(zip(ids, [100.0, -100.0, 0.5, -0.25, 3.0]))
        if kind in (5, 6):
            r["allowed"] = torch.randperm(V, generator=g)[:V // 3].tolist()
            r["temperature"] = 0.6
        rows.append(r)
    return rows


def state_of(rows, V, max_len, device, max_bias=8):
    st = LogitState(len(rows), V, max_len, max_bias, device)
    for b, r in enumerate(rows):
        if r is not None:
            st.set_row(b, **r)
    return st


def both(x, st, slot=None):
    """process_logits and greedy_tokens of a batch, and of one so large (the same rows again and again) that another kernel takes it: the same."""
    y, ids = process_logits(x, st, slot), greedy_tokens(x, st, slot)
    k = 801 // (x.shape[0] * -(-x.shape[1] // 4096)) + 1
    again = (torch.arange(x.shape[0], dtype=torch.int32, device=x.device) if slot is None else slot).repeat(k)
    ys, more = process_logits(x.repeat(k, 1), st, again).view(k, *y.shape), greedy_tokens(x.repeat(k, 1), st, again).view(k, -1)
    assert torch.equal(torch.isnan(ys), torch.isnan(y).expand_as(ys)) and torch.equal(ys.nan_to_num(7.0), y.nan_to_num(7.0).expand_as(ys))
    assert torch.equal(more, ids.expand_as(more))
    return y, ids


def check_rules(got, want, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got == -INF, want == -INF) and torch.equal(got == INF, want == INF)
    fin = torch.isfinite(want)
    over = ((got - want).abs() - bound)[fin]
    assert over.numel() == 0 or over.max().item() <= 0, over.max().item()


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V,B,dtype", [(1, 3, torch.float32), (31, 8, torch.float32), (33, 7, torch.bfloat16), (4096, 14, torch.float16), (4097, 7, torch.float32),
                                       (30522, 9, torch.float32), (50257, 7, torch.bfloat16), (151936, 14, torch.float32)])
def test_rules_on_logits(device, V, B, dtype):
    """Each rule and all together, at vocabularies that end in a word of the mask, a slice, a vector; two strided batches; greedy is their argmax."""
    rows = some_rules(V, B, V + B, 60) if V >= 15 else [dict(prompt=[0], repetition_penalty=2.0), dict(output=[0, 0], frequency_penalty=1.0), dict(allowed=[])]
    B = len(rows)
    st = state_of(rows, V, 100, device)
    wide = (torch.randn(B, V + 5, generator=torch.Generator().manual_seed(V)) * 3).to(dtype)
    for x in (wide[:, :V].contiguous(), wide[:, :V], wide[:, 5:]):
        want, bound = exact_rules(x, rows)
        y = process_logits(x.to(device) if x.is_contiguous() else wide.to(device)[:, x.storage_offset():x.storage_offset() + V], st)
        check_rules(y, want, bound)
        same, ids = both(x.to(device), st)
        assert torch.equal(same, y) and torch.equal(ids.cpu(), y.argmax(1).cpu())


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_rules_go_by_slot(device):
    """Batch rows take the rules of any rows of the state, the same one twice too; a slot outside of it has none."""
    V = 5000
    rows = some_rules(V, 9, 3, 40)
    st = state_of(rows, V, 64, device)
    slot = [8, 2, 2, -1, 9, 0, 6, 2 ** 31 - 1]
    x = torch.randn(len(slot), V) * 3
    want, bound = exact_rules(x, [rows[s] if 0 <= s < 9 else None for s in slot])
    y, ids = both(x.to(device), st, i32(slot, device))
    check_rules(y, want, bound)
    assert torch.equal(y[3].cpu(), x[3]) and torch.equal(ids.cpu(), y.argmax(1).cpu())


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_and_infinity_in_logits(device, dtype):
    """What stands in a masked place is gone, whatever it was; an allowed NaN stays and is the best token, as in torch; equals give the lowest."""
    V = 9000
    x = torch.zeros(7, V, dtype=dtype)
    x[0, 100] = NAN; x[0, 8000] = INF                          # both masked
    x[1, 7000] = NAN; x[1, 50] = INF                           # both allowed
    x[2, 5000], x[2, 4000] = 3.0, 3.0                          # equals in different slices
    x[3] = -INF
    x[4, 10] = torch.finfo(dtype).min
    x[5, :] = torch.finfo(dtype).min
    x[6, 3], x[6, 2] = 0.0, -0.0
    x[6, 4:] = -1.0
    x[6, :2] = -1.0
    rows = [dict(allowed=range(200, 5000))] + [dict(repetition_penalty=1.5, prompt=[1])] + [None] * 5
    st = state_of(rows, V, 8, device)
    y, ids = both(x.to(device), st)
    y = y.cpu()
    assert not torch.isnan(y[0]).any() and (y[0] == -INF).sum() == V - 4800 and (y[0, 200:5000] == 0).all()
    assert torch.isnan(y[1]).sum() == 1 and y[1, 50] == INF and torch.equal(y[2:], x[2:].float())
    assert ids.tolist() == [200, 7000, 4000, 0, 0, 0, 2] == y.argmax(1).tolist()[:4] + [0, 0, 2]


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_masked_to_nothing_and_all_allowed(device):
    V = 12345
    st = state_of([dict(allowed=[]), dict(allowed=range(V)), dict(allowed=[V - 1]), dict(allowed=[0])], V, 4, device)
    x = torch.randn(4, V)
    y = both(x.to(device), st)[0].cpu()
    assert (y[0] == -INF).all() and torch.equal(y[1], x[1]) and greedy_tokens(x.to(device), st).tolist()[0] == 0
    assert greedy_tokens(x.to(device), st).tolist()[2:] == [V - 1, 0] and (y[2] == -INF).sum() == V - 1
    st.set_mask(0, None)
    assert torch.equal(process_logits(x.to(device), st).cpu()[0], x[0])


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_biases_that_name_a_token_twice(device):
    """The last entry for a token counts, in any order that the entries are worked on."""
    V = 600
    st = LogitState(2, V, 4, 300, device)
    st.bias_ids[0, :300] = torch.arange(300, dtype=torch.int32, device=device) % 7
    st.bias_values[0, :300] = torch.arange(300, dtype=torch.float32, device=device)
    st.bias_length[0] = 300
    st.bias_ids[1, :3], st.bias_values[1, :3], st.bias_length[1] = i32([V, -1, 5], device), torch.tensor([9.0, 9.0, 2.0], device=device), 9999
    y = both(torch.zeros(2, V, device=device), st)[0].cpu()
    assert y[0, :7].tolist() == [float(max(i for i in range(300) if i % 7 == t)) for t in range(7)] and (y[0, 7:] == 0).all()
    assert y[1, 5] == 2.0 and y[1].count_nonzero() == 1          # ids outside the vocabulary are passed over, as are entries of id 0 and value 0


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V,n", [(50257, 12000), (50257, 12300), (50257, 40000), (524288, 20000), (7, 30000)])
def test_long_histories(device, V, n):
    """More tokens than the table has room for by their hashes, all different or the same few, in the largest vocabulary too; biases among them."""
    g = torch.Generator().manual_seed(n)
    toks = torch.randint(0, V, (n,), generator=g).tolist()
    rows = [dict(prompt=toks[:n // 2], output=toks[n // 2:], repetition_penalty=1.2, frequency_penalty=0.01, presence_penalty=0.5,
                 logit_bias={toks[0]: 2.0, toks[-1]: -1.0, V - 1: 0.5}), dict(output=list(range(min(V, n))), frequency_penalty=1.0)]
    st = state_of(rows, V, n, device)
    x = torch.randn(2, V, generator=g) * 3
    said = [collections.Counter(r.get("output", ())) for r in rows]
    want, bound = exact_counts(x, rows, said)
    y, ids = both(x.to(device), st)
    check_rules(y, want, bound)
    assert torch.equal(ids.cpu(), y.argmax(1).cpu())


def exact_counts(x, rows, said):
    """As exact_rules for unmasked rows, by vectors: six roundings of numbers no larger than the sum of the sizes."""
    want, size = x.double().clone(), x.double().abs()
    for y, s, r, c in zip(want, size, rows, said):
        count = torch.zeros(y.shape[0], dtype=torch.float64)
        count[torch.tensor(list(c))] = torch.tensor([float(v) for v in c.values()], dtype=torch.float64)
        seen = count > 0
        if r.get("prompt"):
            seen[torch.tensor(r["prompt"])] = True
        rep, f, p = (f32(r.get(k, d)) for k, d in (("repetition_penalty", 1.0), ("frequency_penalty", 0.0), ("presence_penalty", 0.0)))
        y.copy_(torch.where(seen, torch.where(y < 0, y * rep, y / rep), y))
        y -= f * count + p * (count > 0)
        s.copy_(torch.maximum(s * max(rep, 1.0), s) + abs(f) * count + abs(p))
        for t, v in (r.get("logit_bias") or {}).items():
            y[t] += f32(v)
            s[t] += abs(f32(v))
    return want, size * 6 * 2.0 ** -24


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_histories_grow(device):
    """Tokens come behind their rows' histories and count from the next call on; a full row and slots outside the state keep what they have."""
    V = 200
    st = LogitState(4, V, 5, 0, device)
    st.set_row(0, prompt=[7, 7], output=[8], frequency_penalty=1.0)
    st.set_row(2, prompt=[1, 2, 3, 4], repetition_penalty=2.0)
    x = torch.ones(4, V, device=device)
    st.append(torch.tensor([9, 8, 5, 6], device=device), i32([0, 2, 77, -3], device))
    st.append(torch.tensor([9, 8], device=device), i32([0, 2], device))      # row 2 is full
    assert st.length.tolist() == [5, 0, 5, 0] and st.tokens[0].tolist() == [7, 7, 8, 9, 9] and st.tokens[2].tolist() == [1, 2, 3, 4, 8]
    y = process_logits(x, st).cpu()
    assert y[0, [7, 8, 9, 10]].tolist() == [1.0, 0.0, -1.0, 1.0] and y[2, [1, 4, 8, 9]].tolist() == [0.5, 0.5, 0.5, 1.0]
    st.append(torch.tensor([3, 3, 3, 3], device=device))
    assert st.length.tolist() == [5, 1, 5, 1]
    st.set_row(0)
    assert torch.equal(process_logits(x, st).cpu()[0], torch.ones(V))


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_logits_in_place(device):
    V = 6400
    rows = some_rules(V, 7, 5, 30)
    st = state_of(rows, V, 64, device)
    x = torch.randn(7, V)
    y = x.clone().to(device)
    assert process_logits(y, st, out=y) is y
    check_rules(y, *exact_rules(x, rows))
    slot = torch.arange(7, dtype=torch.int32, device=device).repeat(60)
    many = x.repeat(60, 1).to(device)
    process_logits(many, st, slot, out=many)
    assert torch.equal(many.view(60, 7, V), y.expand(60, 7, V))
    assert process_logits(x[:0].to(device), st).shape == (0, V) and greedy_tokens(x[:0].to(device), st).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("V,n", [(6400, 30), (40000, 20000)])
def test_in_place_and_elsewhere_are_the_same(V, n):
    """Batches of several kernels, which go over logits that stay in their place in another order; rows with histories longer than a table, too. Equal are
    numbers, and any two NaN: which of its NaN an operation gives is open (IEEE 754, 6.2.3), so a row of T 1 may pass one on or divide it by 1."""
    def same(a, b):
        return bool(((a == b) | (a.isnan() & b.isnan())).all())

    rows = some_rules(V, 7, 5, 30)
    st = state_of(rows, V, n, "cuda")
    if n > 30:
        st.tokens[2] = torch.randint(0, V, (n,), dtype=torch.int32, device="cuda")
        st.length[2], st.prompt_length[2], st.frequency[2] = n, n // 2, 0.25
    slot = torch.arange(8, dtype=torch.int32, device="cuda").repeat(60)          # row 7 has no rules
    x = torch.randn(480, V, device="cuda")
    x[::3, 5], x[1::3, 9] = NAN, -INF
    y = process_logits(x, st, slot)
    z = x.clone()
    process_logits(z, st, slot, out=z)
    assert same(y, z)
    wide = torch.empty(480, V + 3, device="cuda")                             # rows that do not start on 16 bytes
    assert same(process_logits(x, st, slot, out=wide[:, 1:V + 1]), y)
    few = process_logits(x[:8], st, slot[:8])                                 # by one kernel
    assert same(few, y[:8])
    assert torch.equal(greedy_tokens(x, st, slot), y.argmax(1))


def test_refusals_of_rules():
    st = LogitState(4, 100, 8, 2)
    x = torch.zeros(4, 100)
    for bad in (dict(logits=x[0]), dict(logits=x[:, :99]), dict(logits=torch.zeros(5, 100)), dict(slot=torch.zeros(4)), dict(slot=torch.zeros(3, dtype=torch.int32)),
                dict(logits=torch.zeros(100, 4).t()), dict(logits=x.double())):
        for fn in (process_logits, greedy_tokens):
            with pytest.raises(ValueError, match=fn.__name__):
                fn(**{**dict(logits=x, state=st), **bad})
    for out in (x.double(), x[:2], torch.zeros(100, 4).t(), x[:1].clone().expand(4, 100)):
        with pytest.raises(ValueError, match="process_logits"):
            process_logits(x, st, out=out)
    for bad in (dict(row=4), dict(row=-1), dict(row=0, prompt=range(9)), dict(row=0, logit_bias={1: 1.0, 2: 1.0, 3: 1.0}), dict(row=0, logit_bias={100: 1.0}),
                dict(row=0, allowed=[-1]), dict(row=0, repetition_penalty=0.0), dict(row=0, temperature=0.0), dict(row=0, temperature=NAN)):
        with pytest.raises(ValueError, match="LogitState"):
            st.set_row(**bad)
    for bad in (dict(rows=0), dict(vocab=0), dict(vocab=(1 << 19) + 1), dict(max_len=0), dict(max_len=1 << 20), dict(max_bias=2048), dict(max_bias=-1)):
        with pytest.raises(ValueError, match="LogitState"):
            LogitState(**{**dict(rows=2, vocab=9, max_len=4), **bad})
    for ids, slot in ((torch.zeros(2), None), (torch.zeros(5, dtype=torch.int64), None), (torch.zeros(2, dtype=torch.int64), torch.zeros(2))):
        with pytest.raises(ValueError, match="append"):
            st.append(ids, slot)


def test_outputs_that_overlap_their_logits_are_refused():
    st, buf = LogitState(4, 100, 8), torch.randn(900)
    x = buf[:400].view(4, 100)
    for out in (buf[100:500].view(4, 100), buf[4:404].view(4, 100), buf[:800].view(4, 200)[:, :100], buf[399:799].view(4, 100)):
        with pytest.raises(ValueError, match="overlap"):
            process_logits(x, st, out=out)
    with pytest.raises(ValueError, match="overlap"):
        process_logits(buf.view(torch.bfloat16)[:400].view(4, 100), st, out=x)
    for out in (x, buf[400:800].view(4, 100)):
        want = x.clone()
        assert torch.equal(process_logits(x, st, out=out), want)


def test_tensors_in_place_of_the_state_s_own():
    """They are looked at before their addresses are taken."""
    for name, bad in (("tokens", torch.zeros(4, 7, dtype=torch.int32)), ("length", torch.zeros(4, dtype=torch.int64)), ("bias_values", torch.zeros(3, 2)),
                      ("temperature", torch.ones(8)[::2]), ("mask", torch.zeros(4, 4, dtype=torch.int32)), ("rows", 5)):
        st = LogitState(4, 100, 8, 2)
        st._address()
        setattr(st, name, bad)
        with pytest.raises(ValueError, match="LogitState"):
            st._address()
    st = LogitState(4, 100, 8, 2)
    st.temperature = torch.full((4,), 2.0)
    st.mask, st.masked = torch.zeros(4, 4, dtype=torch.int32), torch.ones(4, dtype=torch.bool)
    st._address()


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_tokens_that_32_bits_do_not_hold(device):
    """They are not of the vocabulary, and passed over like others that are not: in a prompt, in an output and behind a history. A row that is refused keeps what
    it has."""
    V = 50
    st = LogitState(2, V, 8, 1, device)
    st.set_row(0, prompt=[2 ** 32 + 3, 7, -2 ** 40], output=[2 ** 32 + 5, 8], frequency_penalty=1.0, repetition_penalty=2.0)
    st.append(torch.tensor([2 ** 32 + 6, 9], device=device), i32([0, 1], device))
    y = process_logits(torch.ones(2, V, device=device), st).cpu()
    assert st.length.tolist() == [6, 1] and y[0].tolist() == [{7: 0.5, 8: -0.5}.get(v, 1.0) for v in range(V)]
    before = {n: t.clone() for n, t in vars(st).items() if isinstance(t, torch.Tensor)}
    for bad in (dict(prompt=["a"]), dict(prompt=[1], logit_bias={3: "x"}), dict(prompt=[1], presence_penalty="x")):
        with pytest.raises((ValueError, TypeError)):
            st.set_row(0, **bad)
        assert all(torch.equal(t, before[n]) for n, t in vars(st).items() if n in before)


@pytest.mark.parametrize("room", [False, True])
def test_masks_of_rows_and_tokens_that_are_not_there_are_refused(room):
    """They are not counted from the end, and a refused mask leaves the rows as they were."""
    st = LogitState(3, 64, 4)
    st.set_row(2, allowed=[5])
    if not room:
        st.mask = st.masked = None
    for row, allowed in ((-1, [1]), (3, [1]), (-1, None), (3, None), (0, [-1]), (0, [1, 64]), (0, torch.tensor([2, -3]))):
        with pytest.raises(ValueError, match="LogitState"):
            st.set_mask(row, allowed)
    if room:
        assert st.masked.tolist() == [False, False, True] and st.mask.tolist() == [[0, 0], [0, 0], [32, 0]]
        st.set_mask(0, torch.tensor([0, 63]))
        st.set_mask(1, range(0))
        assert st.masked.all() and st.mask[:2].tolist() == [[1, -2 ** 31], [0, 0]]


def test_a_call_holds_what_it_was_given(monkeypatch):
    """Another thread puts a tensor in place while a call is on its way: the struct that the call was given, and the tensors it names, live until the call
    is back."""
    st, x = LogitState(4, 100, 8), torch.zeros(4, 100)
    seen = []

    def entry(*args):
        struct = weakref.ref(st._struct)
        old = [weakref.ref(t) for t in (st.tokens, st.temperature)]
        st.tokens, st.temperature = torch.zeros(4, 8, dtype=torch.int32), torch.ones(4)
        gc.collect()
        seen.append(struct() is not None and all(t() is not None for t in old))
        return 0
    monkeypatch.setattr(logits_module, "_workspace", lambda *a: (torch.zeros(16, dtype=torch.uint8), 1))
    for name, fake in (("use_native", lambda *a: True), ("proto", lambda *a: entry), ("call_on", lambda dev, fn, *a: fn(*a, 0))):
        monkeypatch.setattr(nv, name, fake)
    process_logits(x, st)
    greedy_tokens(x, st)
    assert seen == [True, True]


def test_masks_of_a_state_that_others_use(monkeypatch):
    """Room for masks, made while other threads call with the state and set a mask of their own: a call sees both tensors or none, and no mask is lost."""
    st, real, nested = LogitState(4, 100, 8), torch.zeros, []

    def zeros(*args, **kw):
        st._address()
        if not nested:
            nested.append(1)
            st.set_mask(1, [3])
        return real(*args, **kw)
    monkeypatch.setattr(torch, "zeros", zeros)
    st.allow_masks()
    monkeypatch.undo()
    assert st.masked.tolist() == [False, True, False, False] and int(st.mask[1, 0]) == 8
    struct = st._address()
    assert (struct.mask, struct.masked) == (st.mask.data_ptr(), st.masked.data_ptr())


def test_scales_at_their_bounds():
    st = LogitState(2, 8, 4)
    for v in (2.0 ** -126, 2.0 ** 126):
        st.set_row(0, [1], repetition_penalty=v, temperature=v)
    for v in (2.0 ** -127, 2.0 ** 127, float("inf"), -1.0):
        for kw in (dict(repetition_penalty=v), dict(temperature=v)):
            with pytest.raises(ValueError, match="LogitState"):
                st.set_row(0, [1], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 300])
def test_launches_are_counted(B):
    V = 12800                                                     # four slices a row: 8 and 1200 of them
    st = LogitState(B, V, 4, device="cuda")
    x = torch.randn(B, V, device="cuda")
    for fn, many in ((process_logits, 1 if B == 2 else 2), (greedy_tokens, 1 if B == 2 else 3)):
        before = nv.launch_count
        fn(x, st)
        assert nv.launch_count - before == many


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 127, 1025, 20353, 162815, 162816, 162817])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_best_of_few_rows(V, dtype):
    """Up to eight rows are a cluster's each, up to 162816 tokens; more rows and tokens go other ways. All of them give the first of the largest."""
    rows = some_rules(V, 9, V, 30)
    st = state_of(rows, V, 64, "cuda")
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(9, V, generator=g) * 4).round().div(4).to(dtype).cuda()          # many equals
    x[1], x[2, V // 2], x[3, -1] = -INF, NAN, INF
    for n in (1, 8, 9):
        y = process_logits(x[:n], st)
        first = torch.where(y.isnan().any(1, keepdim=True), y.isnan(), y == y.nan_to_num(-INF, INF, -INF).amax(1, keepdim=True)).int().argmax(1)
        assert torch.equal(greedy_tokens(x[:n], st), first)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [3, 300])
@pytest.mark.parametrize("e", [-126, -60, 0, 60, 126])
def test_temperatures_at_their_bounds(B, e):
    """Powers of two: the quotient is exact wherever 32 bits hold it (smaller ones are off by at most their last bit), infinite behind that."""
    V = 12800
    st = LogitState(B, V, 4, device="cuda")
    st.temperature.fill_(2.0 ** e)
    x = torch.randn(B, V, device="cuda")
    got, want = process_logits(x, st).double(), x.double() / 2.0 ** e
    want = torch.where(want.abs() >= 2.0 ** 128, torch.full_like(want, float("inf")).copysign(want), want)
    off = (got - want).abs().nan_to_num(0.0)                      # infinities of one sign
    assert torch.equal(got.isinf(), want.isinf()) and bool((off <= torch.where(want.abs() < 2.0 ** -126, 2.0 ** -149, 0.0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 30, 300])
def test_rules_captured_and_replayed(B):
    """Each way through the kernels in one graph of a decode step (elsewhere, in place, the best token, which joins the history): the same as eager calls with a
    state of their own, step after step; rows whose rules change between replays have the new ones."""
    V = 30522
    rows = some_rules(V, B, B, 60)
    st, eager = (state_of(rows, V, 100, "cuda").allow_masks() for _ in range(2))
    slot = torch.arange(B, dtype=torch.int32, device="cuda").flip(0)
    x = torch.randn(B, V, device="cuda")
    place, stream, graph = x.clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        y = process_logits(x, st, slot)
        process_logits(place, st, slot, out=place)
        ids = greedy_tokens(x, st, slot)
        st.append(ids, slot)
    for i in range(6):
        x.copy_(torch.randn(B, V, device="cuda") * 3)
        place.copy_(x)
        if i == 3:
            for s in (st, eager):
                s.set_row(0, [1, 2, 3], [4, 4], frequency_penalty=2.0, temperature=0.5, allowed=range(1, V, 3))
        graph.replay()
        want, best = process_logits(x, eager, slot), greedy_tokens(x, eager, slot)
        eager.append(best, slot)
        assert torch.equal(y, want) and torch.equal(place, want) and torch.equal(ids, best) and torch.equal(best, want.argmax(1))
    assert torch.equal(st.tokens, eager.tokens) and torch.equal(st.length, eager.length)


@pytest.mark.gpu
def test_a_state_on_two_streams_at_once():
    """Calls of several sizes on two streams, each with scratch of its own, and of one state that nobody writes."""
    V = 32768
    rows = some_rules(V, 40, 7, 60)
    st = state_of(rows, V, 100, "cuda")
    xs = [torch.randn(n, V, device="cuda") for n in (2, 40, 300, 9)]
    slots = [torch.arange(x.shape[0], dtype=torch.int32, device="cuda") % 40 for x in xs]
    want = [(process_logits(x, st, s), greedy_tokens(x, st, s)) for x, s in zip(xs, slots)]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                for x, s, w in zip(xs, slots, want):
                    got.append((process_logits(x, st, s), greedy_tokens(x, st, s), w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w[0]) and torch.equal(ids, w[1]) for y, ids, w in got)


@pytest.mark.gpu
def test_tables_and_maps_captured_and_replayed():
    """A decode step's tables and maps in one graph, whose requests' lengths change on the device from replay to replay."""
    n, bs, width = 70, 16, 20
    table = torch.zeros(n + 2, width, dtype=torch.int32, device="cuda")
    rows = torch.randperm(n + 2, generator=torch.Generator().manual_seed(1))[:n].to(torch.int32).cuda()
    cached, lens, new = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    blocks = torch.zeros(n * width, dtype=torch.int32, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        used = extend_block_tables(table, rows, cached, lens, blocks, bs)
        m = step_maps(table, rows, cached, new, bs, 1000, n_tiles=80)
    want, have, free = table.tolist(), [0] * n, list(range(1, n * width + 1))
    for step in range(5):
        k = torch.randint(1, 14, (n,), generator=torch.Generator().manual_seed(step)).tolist()
        for t, v in ((cached, have), (new, k), (lens, [a + b for a, b in zip(have, k)])):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        blocks[:len(free)].copy_(torch.tensor(free, dtype=torch.int32))
        graph.replay()
        want, at = grown(want, rows.tolist(), have, lens.tolist(), free, bs)
        assert table.tolist() == want and used.tolist() == [at]
        maps, T = maps_of(want, rows.tolist(), have, k, bs), sum(k)
        assert all(getattr(m, f)[:T].tolist() == maps[f] for f in ("pos", "slot", "place")) and m.cu.tolist() == maps["cu"] and m.last.tolist() == maps["last"]
        assert m.tiles.tolist() == maps["tiles"] + [[0, 0, 0, 0]] * 10 and m.runs.tolist() == maps["runs"]
        free, have = free[at:], lens.tolist()


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("B", [3, 300])
def test_quotients_next_to_the_largest_number(device, B):
    """By temperatures and repetition penalties below 1: infinite where the quotient is, and nowhere else. Off by a rounding, and by the correction's own of a
    remainder, 2^-24 of half a step."""
    V, top = 12800, torch.finfo(torch.float32).max
    g = torch.Generator().manual_seed(B)
    d = 1 - torch.randint(1, 2 ** 23, (B,), generator=g) * 2.0 ** -24
    x = (top * d.double()[:, None] * (1 - torch.randint(0, 6, (B, V), generator=g) * 2.0 ** -24)).float()
    x[:, ::2] *= -1
    want = x.double() / d.double()[:, None]
    for name in ("temperature", "repetition"):
        if name == "repetition":
            x, want = x.abs(), want.abs()
        st = LogitState(B, V, V, device=device)
        getattr(st, name).copy_(d)
        if name == "repetition":
            st.tokens.copy_(torch.arange(V, dtype=torch.int32).expand(B, V))
            st.length.fill_(V)
            st.prompt_length.fill_(V)
        got = process_logits(x.to(device), st).double().cpu()
        assert torch.equal(got.isinf(), want.abs() >= 2.0 ** 128 * (1 - 2.0 ** -25))
        fin = got.isfinite()
        assert bool(((got - want).abs()[fin] <= want.abs()[fin] * 2.0 ** -24 * (1 + 2.0 ** -20)).all())


# ------------------------------------------------------------------------------------------------ attention over shared keys
def batch_of(groups, alone, own, H, G, D, BS, dtype, seed, copies=False):
    """A decode batch on the CPU: groups (tokens, shared keys), then sequences by themselves, ``own`` keys (cyclic) behind the shared ones. Whole pages of
    the shared part are the same page for all; the page that it ends in is each sequence's copy. All that no sequence holds is NaN."""
    g = torch.Generator().manual_seed(seed)
    members, plan, first = [], [], 0
    for n, shared in groups:
        plan.append((first, n, shared))
        members += [(first, shared)] * n
        first += n
    members += [(None, 0)] * alone
    keys = [s + k for (_, s), k in zip(members, itertools.cycle(own))]
    total = sum(-(-k // BS) for k in keys) + 3
    pages = (torch.randperm(total, generator=g) + 1).tolist()
    ck, cv = (torch.full((total + 1, G, BS, D), NAN, dtype=dtype) for _ in range(2))
    rows = []
    for i, ((first, s), n) in enumerate(zip(members, keys)):
        lead = rows[first][:s // BS] if first is not None and first != i and not copies else []
        rows.append(lead + [pages.pop() for _ in range(-(-n // BS) - len(lead))])
        own_k, own_v = (torch.randn(n, G, D, generator=g).to(dtype) for _ in range(2))
        if first is not None and first != i:
            k0, v0 = keys_of(ck, rows[first], s), keys_of(cv, rows[first], s)
            own_k[:s], own_v[:s] = k0, v0
        at = torch.arange(n)
        blk = torch.tensor(rows[-1])[at // BS]
        ck[blk, :, at % BS], cv[blk, :, at % BS] = own_k, own_v
    width = max(map(len, rows)) + 1
    table = torch.zeros(len(rows), width + 2, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    T = len(rows)
    q = torch.randn(T, (H + 2 * G) * D, generator=g).to(dtype)
    return dict(q=q, ck=ck, cv=cv, table=table, pos=torch.tensor([n - 1 for n in keys], dtype=torch.int32), slot=torch.arange(T, dtype=torch.int32), plan=plan,
                H=H, G=G, D=D, BS=BS)


def keys_of(pool, row, n):
    at = torch.arange(n)
    return pool[torch.tensor(row)[at // pool.shape[2]], :, at % pool.shape[2]]


def exact_attention(b, scale, sinks=None):
    """Token by token in 64 bits, with a bound for a result of 16 bits. The result and every weight are rounded once, each by half a step; a score is a sum of D
    products in 32 bits, off by at most D 2^-24 of the sum of their sizes, and a weight by that much twice (it and the sum); 2^-20 more for exponentials
    (2^-22 each, of the weight and of two joins) and for sums in 32 bits of a few hundred blocks. Numbers below the type's smallest normal one
    are a fixed step apart (fp16: 2^-24 below 2^-14), so a rounding there is off by half of that, ``tiny``: of the result, and of a weight, which is
    rounded as a part of the largest one of its range, so by no more than ``tiny`` of the row's largest weight."""
    H, G, D, BS = b["H"], b["G"], b["D"], b["BS"]
    half = torch.finfo(b["q"].dtype).eps / 2
    tiny = torch.finfo(b["q"].dtype).smallest_normal * half
    out, bound = [], []
    for t in range(b["q"].shape[0]):
        n, row = int(b["pos"][t]) + 1, int(b["slot"][t])
        if n <= 0 or not 0 <= row < b["table"].shape[0]:
            out.append(torch.zeros(H * D, dtype=torch.float64)); bound.append(torch.zeros(H * D, dtype=torch.float64))
            continue
        k, v = (keys_of(b[c], b["table"][row].tolist(), n).double().repeat_interleave(H // G, 1) for c in ("ck", "cv"))
        q = b["q"][t, :H * D].double().view(H, D)
        s = torch.einsum("hd,nhd->hn", q, k) * scale
        err = D * 2.0 ** -24 * scale * torch.einsum("hd,nhd->hn", q.abs(), k.abs()).amax(1)
        full = s if sinks is None else torch.cat([s, sinks.double()[:, None]], 1)
        w = full.softmax(1)[:, :n]
        o, size = torch.einsum("hn,nhd->hd", w, v), torch.einsum("hn,nhd->hd", w, v.abs())
        out.append(o.reshape(-1))
        bound.append((half * o.abs() + size * (half + 2 * err[:, None] + 2.0 ** -20) * (1 + half)
                      + tiny * (1 + w.amax(1)[:, None] * v.abs().sum(0))).reshape(-1))
    return torch.stack(out), torch.stack(bound)


def call(b, device, groups=None, scale=None, sinks=None, **kw):
    on = {k: v.to(device) for k, v in b.items() if isinstance(v, torch.Tensor)}
    plan = make_prefix_groups(b["plan"] if groups is None else groups, b["q"].shape[0], device)
    return prefix_attention(on["q"], on["ck"], on["cv"], on["table"][:, :-2], on["pos"], on["slot"], plan, b["H"], b["G"], b["D"],
                            b["D"] ** -0.5 if scale is None else scale, sinks=None if sinks is None else sinks.to(device), max_pos=int(b["pos"].max()), **kw)


def close(got, b, scale=None, sinks=None):
    want, bound = exact_attention(b, b["D"] ** -0.5 if scale is None else scale, sinks)
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, over


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,D", [(16, 4, 128), (40, 8, 128), (8, 8, 128), (16, 1, 128), (12, 2, 64), (4, 4, 64), (24, 2, 64), (8, 4, 96), (6, 2, 80), (3, 1, 16), (5, 5, 112)])
@pytest.mark.parametrize("BS", [8, 16, 64, 256])
def test_shared_keys(entries, H, G, D, BS):
    """Groups of 1 to 40 tokens whose shared part ends in and beside pages, tiles and ranges; sequences by themselves between and behind them."""
    b = batch_of([(3, 64), (1, 1), (40, 257), (2, 63), (17, 640)], 3, [1, 2, 65, 31, 200, 129], H, G, D, BS, torch.bfloat16, H + D + BS)
    close(call(b, "cuda"), b)
    assert "b200_prefix_attn" in entries and "b200_paged_attn" not in entries


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("groups,own", [([(130, 2000)], [1, 7]), ([(2, 5000)], [3000, 1]), ([(33, 128), (33, 129), (33, 127)], [64]), ([(1, 4096)], [1]), ([(300, 1)], [5])])
def test_few_and_many_rows(entries, dtype, D, groups, own):
    """Work cut into many ranges and into none, tiles that are full and all but empty; copies of the shared keys instead of the same pages."""
    b = batch_of(groups, 0, own, 8, 2, D, 16, dtype, D, copies=len(own) == 1 and groups[0][0] < 40)
    close(call(b, "cuda"), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [18, 48, 70, 120])
@pytest.mark.parametrize("unknown", [False, True])
def test_tokens_with_and_without_room_beside_the_shared_keys(dtype, tokens, unknown):
    """144, 384, 560 and 960 CTAs of own keys (as many as tokens times KV heads) beside 8 to 64 of shared ones: rooms for four, three and two warps to a CTA, and for not
    even those; two only where the number of own keys is known. A token of the group sees less than the shared part, one nothing at all."""
    b = batch_of([(tokens, 130)], 0, [1, 40, 7, 100], 16, 8, 128, 16, dtype, tokens)
    b["pos"][3], b["pos"][5] = 76, -1
    if unknown:
        plan = make_prefix_groups(b["plan"], tokens, "cuda")
        on = {k: v.cuda() for k, v in b.items() if isinstance(v, torch.Tensor)}
        close(prefix_attention(on["q"], on["ck"], on["cv"], on["table"][:, :-2], on["pos"], on["slot"], plan, 16, 8, 128, 128 ** -0.5), b)
    else:
        close(call(b, "cuda"), b)


@pytest.mark.skipif(not nv.lib_path().exists(), reason="no kernel library here")
def test_plans_by_size():
    """Which kernel has the shared keys, and in how many ranges; of any sizes, some plan that the call takes."""
    fn = nv.proto("b200_prefix_attn_plan", [nv.ctypes.c_int] * 8)
    assert fn(4, 1, 4, 512, 40, 16, 4, 128) < TC                      # up to 32 rows and 1024 keys: mma.sync
    assert fn(64, 1, 64, 4096, 600, 32, 8, 96) < TC                   # a head size that tcgen05 has not
    assert fn(64, 1, 64, 4096, 600, 32, 8, 128) == TC + 7             # 28 us; in 8 ranges 31
    assert fn(128, 1, 128, 16384, 512, 32, 8, 128) == TC + 9          # 68 us; in 4 ranges 80, in 12 82
    for T, n, longest, shared, own, H, G, D in itertools.product((1, 64, 4096), (1, 5, 300), (1, 4096), (1, 64, 2 ** 31 - 1), (0, 1, 2 ** 31 - 1), (128,), (1, 128), (16, 64, 128)):
        assert 1 <= fn(T, n, longest, shared, own, H, G, D) % TC <= min(32, -(-shared // 64))
    for bad in itertools.product((0, 1), repeat=7):
        if not all(bad):
            T, n, longest, shared, H, G, D = bad
            assert fn(T, n, longest, shared, 0, H, G, 16 * D) >= 1


TC = 256                      # plan: the tcgen05 kernel


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G,D,BS", [(8, 2, 128, 8), (5, 1, 64, 16), (40, 8, 128, 16), (24, 2, 64, 64), (16, 16, 128, 128), (128, 1, 64, 32)])
def test_every_cut_of_the_shared_keys(dtype, H, G, D, BS):
    """Both kernels of the shared keys, from one range to more than there are keys for; each result by the same bound."""
    b = batch_of([(3, 64), (1, 1), (70, 257), (9, 1030)], 2, [1, 65, 31], H, G, D, BS, dtype, H + D)
    for plan in (1, 2, 5, 32, TC + 1, TC + 2, TC + 3, TC + 7, TC + 32):
        close(call(b, "cuda", plan=plan), b)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 80])
def test_sinks_and_scales(D):
    b = batch_of([(5, 300), (9, 77)], 2, [1, 40], 8, 2, D, 16, torch.float16, 3)
    sinks = torch.tensor([-INF, -50.0, 0.0, 3.0, 40.0, -1.0, 1.0, 10.0])
    close(call(b, "cuda", sinks=sinks), b, sinks=sinks)
    for scale in (1e-3, 0.5):
        close(call(b, "cuda", scale=scale), b, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 64, 48])
def test_tokens_that_do_not_see_all_of_the_shared_part(D):
    """A token before the last shared key, one at it, one without any key, slots outside the table: each as by itself; no row of the batch touches
    another's."""
    b = batch_of([(8, 200)], 2, [10], 8, 2, D, 16, torch.bfloat16, 5)
    b["pos"][[1, 2, 3, 4, 9]] = torch.tensor([0, 198, 199, -1, -1], dtype=torch.int32)
    b["slot"][[6, 8]] = torch.tensor([-1, 10], dtype=torch.int32)
    got = call(b, "cuda")
    close(got, b)
    assert (got[[4, 6, 8, 9]] == 0).all()
    sinks = torch.zeros(8)
    got = call(b, "cuda", sinks=sinks)
    close(got, b, sinks=sinks)
    assert (got[[4, 6, 8, 9]] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 96])
def test_values_of_other_sequences_stay_theirs(D):
    """A NaN or infinity in one sequence's own keys and values reaches that sequence alone; one in the shared part all of the group."""
    b = batch_of([(6, 100), (3, 50)], 1, [30, 7], 8, 2, D, 64, torch.bfloat16, 8)
    for plan in (0, 2, TC + 2) if D == 128 else (0, 2):
        nan_and_infinity(b, plan)


def nan_and_infinity(b, plan):
    clean = call(b, "cuda", plan=plan)
    for pool, bad in (("ck", NAN), ("cv", INF), ("cv", NAN)):
        c = {**b, "ck": b["ck"].clone(), "cv": b["cv"].clone()}
        row, p = 2, 110
        c[pool][int(b["table"][row, p // 64]), :, p % 64] = bad
        got = call(c, "cuda", plan=plan)
        assert torch.equal(got[[0, 1, 3, 4, 5, 6, 7, 8, 9]], clean[[0, 1, 3, 4, 5, 6, 7, 8, 9]]) and not torch.isfinite(got[2]).all()
        c = {**b, "ck": b["ck"].clone(), "cv": b["cv"].clone()}
        c[pool][int(b["table"][0, 0]), :, 5] = bad
        got = call(c, "cuda", plan=plan)
        assert torch.equal(got[6:], clean[6:]) and not torch.isfinite(got[:6]).all(1).any()


@pytest.mark.gpu
def test_pages_outside_the_pool_are_not_read():
    """A table entry that names no page of the pool: its keys are not read, the other rows have their results."""
    b = batch_of([(6, 128)], 2, [70], 8, 2, 128, 64, torch.bfloat16, 9)
    for plan, page in itertools.product((2, TC + 2), (-1, b["ck"].shape[0], 2 ** 31 - 1, -2 ** 31)):
        clean = call(b, "cuda", plan=plan)
        c = {**b, "table": b["table"].clone()}
        c["table"][3, 2] = page
        got = call(c, "cuda", plan=plan)
        others = [0, 1, 2, 4, 5, 6, 7]
        assert torch.equal(got[others], clean[others]) and not torch.equal(got[3], clean[3])
        c["table"][0, 0] = page
        assert torch.equal(call(c, "cuda", plan=plan)[6:], clean[6:])


@pytest.mark.gpu
def test_a_pool_that_32_bits_do_not_address():
    """Pages behind 2^31 elements of a pool."""
    n_pages = 2 ** 31 // (8 * 64 * 128) + 70
    if torch.cuda.mem_get_info()[0] < 3 * n_pages * 8 * 64 * 128 * 2:
        pytest.skip("not enough memory")
    b = batch_of([(5, 200)], 1, [100], 8, 8, 128, 64, torch.bfloat16, 11)
    used = b["ck"].shape[0]
    on = {k: v.cuda() for k, v in b.items() if isinstance(v, torch.Tensor)}
    ck, cv = (torch.empty(n_pages, 8, 64, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ck[-used:], cv[-used:] = on["ck"], on["cv"]
    out = prefix_attention(on["q"], ck, cv, on["table"] + (n_pages - used), on["pos"], on["slot"], make_prefix_groups(b["plan"], 6, "cuda"), 8, 8, 128, 128 ** -0.5)
    assert torch.equal(out, call(b, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("groups,own,D", [([(64, 4096)], [300, 12], 128), ([(3, 700)], [5], 64), ([(20, 900), (9, 50)], [600, 3, 90], 96), ([(2, 4096)], [3000], 128)])
def test_calls_repeat_themselves(groups, own, D):
    """Bit for bit, on two streams at once as well: no sum depends on what is done first."""
    b = batch_of(groups, 1, own, 8, 2, D, 16, torch.bfloat16, 17)
    on = {k: v.cuda() for k, v in b.items() if isinstance(v, torch.Tensor)}
    T = b["q"].shape[0]
    plan, most = make_prefix_groups(b["plan"], T, "cuda"), int(b["pos"].max())

    def once():
        return prefix_attention(on["q"], on["ck"], on["cv"], on["table"], on["pos"], on["slot"], plan, 8, 2, D, D ** -0.5, max_pos=most)
    first, outs, streams = once(), [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(once())
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 48])
def test_captured_and_on_another_stream(D):
    """Two captured calls and an eager one between their replays, on a stream of their own; the plan rewritten on the device within its bounds, and beyond
    them."""
    b = batch_of([(20, 300)], 4, [33], 16, 4, D, 16, torch.bfloat16, 13)
    on = {k: v.cuda() for k, v in b.items() if isinstance(v, torch.Tensor)}
    plan = make_prefix_groups([(0, 20, 300)], 24, "cuda")
    args = (on["q"], on["ck"], on["cv"], on["table"], on["pos"], on["slot"], plan, 16, 4, D, D ** -0.5)
    want = prefix_attention(*args)
    close(want, b)
    stream, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = prefix_attention(*args)
        graphs.append((graph, out))
    for rewrite in ([0, 20, 300, 0], [0, 5, 17, 0], [2, 18, 300, 0], [0, 20, 10 ** 6, 0], [-3, 20, 300, 0], [0, 99, 300, 0], [0, 20, 0, 0], [0, 20, -5, 0]):
        plan.groups.copy_(torch.tensor([rewrite]))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for graph, out in graphs:
                out.fill_(NAN)
                graph.replay()
            eager = prefix_attention(*args)
        stream.synchronize()
        close(eager, b)
        assert torch.equal(graphs[0][1], eager) and torch.equal(graphs[1][1], eager)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_other_caches_go_through_paged_attention(entries, device):
    """32-bit caches, head sizes, small pages and steps without groups that the kernels are not for."""
    for dtype, D, groups, BS in ((torch.float32, 64, None, 16), (torch.bfloat16, 24, None, 16), (torch.bfloat16, 160, None, 16), (torch.bfloat16, 64, [], 16),
                                 (torch.bfloat16, 64, None, 4), (torch.bfloat16, 64, None, 1)):
        b = batch_of([(4, 40)], 1, [3, 20], 4, 2, D, BS, dtype, 1)
        close(call(b, device, groups=groups), b)
    assert "b200_prefix_attn" not in entries


FALLBACKS = [(torch.float32, 64, 16), (torch.bfloat16, 24, 16), (torch.bfloat16, 64, 4)]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("dtype,D,BS", FALLBACKS)
@pytest.mark.parametrize("grouped", [True, False])
def test_other_caches_keep_to_the_same_bounds(device, dtype, D, BS, grouped):
    """What goes through paged_attention: tokens without a key and slots outside the table are zeros there as well, a position behind the table's last one sees
    all of its row, an entry that names no page of the pool reads nothing outside of it, and no row of the batch touches another's."""
    b = batch_of([(6, 40)], 3, [10], 4, 2, D, BS, dtype, 5)
    want, bound = exact_attention(b, D ** -0.5)
    b["pos"][[1, 7]] = torch.tensor([-1, 2 ** 31 - 1], dtype=torch.int32)
    b["slot"][[3, 4, 8]] = torch.tensor([-1, 9, 2 ** 31 - 1], dtype=torch.int32)
    last = b["table"][7].clone()
    b["table"][7, 1:] = last[0]                                       # entries behind the sequence's own: its first page again
    b["table"][5, 40 // BS] = 2 ** 31 - 1
    b["table"][6, 0] = -1
    for sinks in (None, torch.zeros(4)):
        got = call(b, device, groups=None if grouped else [], sinks=sinks)
        assert (got[[1, 3, 4, 8]] == 0).all()
        if sinks is None:                                             # by the bound: max_pos, another one now, chooses how the keys are cut
            assert bool(((got.double().cpu() - want).abs() <= bound)[[0, 2]].all())
    none = torch.empty(0, dtype=torch.int32)
    empty = {**b, "q": b["q"][:0], "pos": none, "slot": none, "plan": []}
    on = {k: v.to(device) for k, v in empty.items() if isinstance(v, torch.Tensor)}
    assert prefix_attention(on["q"], on["ck"], on["cv"], on["table"], on["pos"], on["slot"], None, 4, 2, D, 0.1, max_pos=5000).shape == (0, 4 * D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,BS", FALLBACKS)
def test_refusals_of_other_caches(dtype, D, BS):
    """What goes through paged_attention is looked at as well before its addresses are taken."""
    b = batch_of([(4, 40)], 1, [3], 4, 2, D, BS, dtype, 1)
    other = torch.float16 if dtype is torch.float32 else torch.float32
    for change in (dict(ck=b["ck"].to(other)), dict(cv=b["cv"].to(other)), dict(cv=b["cv"][:, :1]), dict(q=b["q"][:, :20]), dict(table=b["table"].long()),
                   dict(pos=b["pos"].long()), dict(slot=b["slot"][:2]), dict(ck=b["ck"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError, match="prefix_attention"):
            call({**b, **change}, "cuda")
    on = {k: v.cuda() for k, v in b.items() if isinstance(v, torch.Tensor)}
    args = [on["q"], on["ck"], on["cv"], on["table"], on["pos"], on["slot"], None, 4, 2, D, 0.125]
    for i, bad in ((0, on["q"].t().contiguous().t()), (3, b["table"]), (4, b["pos"]), (5, b["slot"]), (1, b["ck"]), (7, 3)):
        with pytest.raises(ValueError, match="prefix_attention"):
            prefix_attention(*args[:i], bad, *args[i + 1:])
    with pytest.raises(ValueError, match="sinks"):
        prefix_attention(*args, sinks=torch.zeros(4))


def test_refusals_of_groups():
    for groups in ([(0, 3, 5), (2, 2, 5)], [(-1, 2, 5)], [(3, 2, 5)], [(0, -1, 5)], [(0, 1, -5)]):
        with pytest.raises(ValueError, match="make_prefix_groups"):
            make_prefix_groups(groups, 4, "cpu")
    p = make_prefix_groups([(0, 2, 7), (2, 0, 9), (2, 1, 0), (3, 1, 4)], 4, "cpu")
    assert p.of.tolist() == [0, 0, -1, 1] and p.groups.tolist() == [[0, 2, 7, 0], [3, 1, 4, 0]] and (p.n_groups, p.longest, p.max_shared) == (2, 2, 7)
    assert make_prefix_groups([], 3, "cpu").n_groups == 0


@pytest.mark.gpu
def test_refusals_of_attention():
    b = batch_of([(4, 40)], 1, [3], 4, 2, 64, 16, torch.bfloat16, 1)
    for change in (dict(ck=b["ck"].float()), dict(cv=b["cv"][:, :1]), dict(q=b["q"][:, :100]), dict(table=b["table"].long()), dict(pos=b["pos"].long()),
                   dict(slot=b["slot"][:2]), dict(ck=b["ck"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError, match="prefix_attention"):
            call({**b, **change}, "cuda")
    on = {k: v.cuda() for k, v in b.items() if isinstance(v, torch.Tensor)}
    args = [on["q"], on["ck"], on["cv"], on["table"], on["pos"], on["slot"], make_prefix_groups(b["plan"], 5, "cuda"), 4, 2, 64, 0.125]
    for i, bad in ((0, torch.empty(5, 516, dtype=torch.bfloat16, device="cuda")[:, 1:513]), (0, on["q"][:1].expand(5, 512)), (0, on["q"].flatten().unfold(0, 512, 64)[:5]), (7, 3), (6, make_prefix_groups(b["plan"], 4, "cuda")),
                   (6, make_prefix_groups(b["plan"], 5, "cpu"))):
        with pytest.raises(ValueError, match="prefix_attention"):
            prefix_attention(*args[:i], bad, *args[i + 1:])
    with pytest.raises(ValueError, match="sinks"):
        prefix_attention(*args, sinks=torch.zeros(4))


def test_lanes_meet_before_instructions_of_a_warp(monkeypatch):
    """The tcgen05 kernel's source, read as the other ones are."""
    monkeypatch.setattr(sources, "WHOLE", re.compile(r"\b(issue_qk|pt_mma_ss|pt_mma_ts|pt_commit|tmem_ld_32x32)\b\s*[(<]"))
    sources.test_lanes_meet_before_instructions_of_a_warp("prefix_attn_tc.cu")
