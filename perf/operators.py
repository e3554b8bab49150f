"""The operators of a serving step that shares work between its sequences, as cases that can be run and timed one by one:

    prefix    attention of a decode batch whose sequences start with the same keys: the shared ones are read once for the group
    extend    block tables grown from the requests' lengths, blocks taken off a list in order
    maps      positions, cache rows, places in the pool and attention tiles of a step, from the requests' lengths
    logits    repetition, presence and frequency penalties, biases, temperature and a grammar's mask on a batch of logits
    greedy    the same rules, and only the best token of each row as a result

A case is a dict of plain values. ``run`` computes a case in its plain form, or, where ``own`` is true, calls the package.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TILE = 64                     # query rows of a tile of the tensor-core attention kernels


def listed():
    return [
        # four chats over one short system prompt: the smallest call, bound by latency
        {"name": "prefix_few", "kind": "prefix", "groups": "4:512", "alone": 0, "own_keys": 40, "H": 16, "G": 4, "D": 128, "page": 64, "dtype": "bf16", "sinks": False},
        # 64 requests behind one few-shot prompt of 4096 tokens, Qwen3-8B heads
        {"name": "prefix_serving", "kind": "prefix", "groups": "64:4096", "alone": 0, "own_keys": 600, "H": 32, "G": 8, "D": 128, "page": 64, "dtype": "bf16", "sinks": False},
        # three system prompts of odd lengths and sequences that share nothing, Qwen3-14B heads, small pages
        {"name": "prefix_mixed", "kind": "prefix", "groups": "17:1000,9:77,30:2511", "alone": 7, "own_keys": 900, "H": 40, "G": 8, "D": 128, "page": 16, "dtype": "fp16", "sinks": False},
        # 128 questions about one long document
        {"name": "prefix_long", "kind": "prefix", "groups": "128:16384", "alone": 0, "own_keys": 512, "H": 32, "G": 8, "D": 128, "page": 64, "dtype": "bf16", "sinks": False},
        # a decode step in which some of 64 sequences need their next block
        {"name": "extend_decode", "kind": "extend", "n": 64, "new": 1, "cached": 4000, "page": 16},
        # 200 requests admitted together, up to 8192 tokens each
        {"name": "extend_admit", "kind": "extend", "n": 200, "new": 8192, "cached": 0, "page": 16},
        # the maps of a decode step of 64 sequences
        {"name": "maps_decode", "kind": "maps", "n": 64, "new": 1, "cached": 4000, "page": 64},
        # the maps of a step with prompt pieces of up to 2000 tokens of 60 requests, some of them continued
        {"name": "maps_prompts", "kind": "maps", "n": 60, "new": 2000, "cached": 3000, "page": 16},
        # eight chats with a repetition penalty, vocabulary of Qwen3
        {"name": "logits_few", "kind": "logits", "B": 8, "V": 151936, "history": 1500, "bias": 0, "mask": 0.0, "dtype": "fp32"},
        # a full batch: long histories, biases, half of the rows under a grammar
        {"name": "logits_batch", "kind": "logits", "B": 128, "V": 151936, "history": 6000, "bias": 300, "mask": 0.5, "dtype": "fp32"},
        # one chat, greedy: the smallest call
        {"name": "greedy_one", "kind": "greedy", "B": 1, "V": 151936, "history": 900, "bias": 0, "mask": 0.0, "dtype": "fp32"},
        # tool calls of 64 sequences decoded greedily under a grammar
        {"name": "greedy_grammar", "kind": "greedy", "B": 64, "V": 151936, "history": 3000, "bias": 40, "mask": 1.0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "extend", "maps", "logits", "greedy"])
    if kind == "prefix":
        D = rng.choice([128, 128, 64, 96])
        H, G = rng.choice([(16, 4), (32, 8), (40, 8), (8, 8), (16, 2)] if D != 64 else [(16, 8), (12, 2), (12, 12)])
        k = rng.choice([1, 1, 1, 2, 4])
        left, keys, groups = _log(rng, k, 128), 16384 * 32 // max(H, 32) // k, []
        for i in range(k):
            n = max(1, left // (k - i))
            groups.append("%d:%d" % (n, _log(rng, 40, keys)))
            left -= n
        return {"kind": kind, "groups": ",".join(groups), "alone": rng.choice([0, 0, 1, 5]), "own_keys": _log(rng, 1, 512), "H": H, "G": G, "D": D,
                "page": rng.choice([64, 64, 32, 16]), "dtype": rng.choice(["bf16", "bf16", "fp16"]), "sinks": rng.random() < 0.25}
    if kind == "extend":
        n = _log(rng, 1, 200)
        return {"kind": kind, "n": n, "new": rng.choice([1, 1, _log(rng, 2, 8192)]), "cached": rng.choice([0, _log(rng, 1, 8000)]), "page": rng.choice([16, 32, 64])}
    if kind == "maps":
        n = _log(rng, 1, 512)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, min(2000, 100000 // n))
        return {"kind": kind, "n": n, "new": new, "cached": rng.choice([0, _log(rng, 1, 8000)]), "page": rng.choice([16, 32, 64])}
    V = rng.choice([151936, 151936, 32768, 30522, 50257, 6400])
    return {"kind": kind, "B": _log(rng, 1, 120), "V": V, "history": _log(rng, 1, 6000), "bias": rng.choice([0, 1, 40, 300]),
            "mask": rng.choice([0.0, 0.5, 1.0]), "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}


# ------------------------------------------------------------------------------------------------ inputs
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))
        self.c = torch.Generator().manual_seed(int(seed) + 1)

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=self.g) * std).to(dtype)

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, device=DEV, generator=self.g) * (hi - lo) + lo

    def below(self, hi, *shape, dtype=torch.int32):
        return torch.randint(0, hi, shape, device=DEV, generator=self.g, dtype=torch.int64).to(dtype)

    def host(self, lo, hi, n):
        """n whole numbers of lo .. hi, on the host."""
        return torch.randint(lo, hi + 1, (n,), generator=self.c).tolist()

    def pages(self, n):
        """The numbers 1 .. n in any order: page 0 is never handed out."""
        return (torch.randperm(n, generator=self.c) + 1).tolist()


def _pad(rows, width):
    return [r + [0] * (width - len(r)) for r in rows]


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).to(DEV)


def _prefix_inputs(case, seed):
    """Sequences of a group list the same pages for the whole pages that they share; a page in which the shared part ends is each one's own copy."""
    r = _Random(seed)
    H, G, D, BS, dt = case["H"], case["G"], case["D"], case["page"], DTYPES[case["dtype"]]
    sizes = [tuple(int(x) for x in g.split(":")) for g in case["groups"].split(",")]
    members, groups, first = [], [], 0
    for n, shared in sizes:
        groups.append((first, n, shared))
        members += [(shared, j) for j in [len(groups) - 1] * n]
        first += n
    members += [(0, None)] * case["alone"]
    keys = [shared + k for (shared, _), k in zip(members, r.host(1, case["own_keys"], len(members)))]
    total = sum(s // BS for _, s in sizes) + sum(-(-k // BS) - s // BS for (s, _), k in zip(members, keys))
    pages = r.pages(total)
    common = [[pages.pop() for _ in range(s // BS)] for _, s in sizes]
    rows = [(common[j] if j is not None else []) + [pages.pop() for _ in range(-(-k // BS) - s // BS)] for (s, j), k in zip(members, keys)]
    ck, cv = r.normal(total + 1, G, BS, D, dtype=dt), r.normal(total + 1, G, BS, D, dtype=dt)
    for first, n, shared in groups:                                  # the copies of the page that the shared part ends in
        cut = shared % BS
        for i in range(first + 1, first + n):
            if cut:
                ck[rows[i][shared // BS], :, :cut] = ck[rows[first][shared // BS], :, :cut]
                cv[rows[i][shared // BS], :, :cut] = cv[rows[first][shared // BS], :, :cut]
    T = len(members)
    return {"qkv": r.normal(T, (H + 2 * G) * D, dtype=dt), "ck": ck, "cv": cv, "table": _ints(_pad(rows, max(map(len, rows)))), "pos": _ints([k - 1 for k in keys]),
            "slot": torch.arange(T, dtype=torch.int32, device=DEV), "groups": groups, "keys": keys, "sinks": r.normal(H) if case["sinks"] else None}


def _lengths(case, r):
    """The same new lengths for every seed, in another order: a step's tensors keep their shapes."""
    n = case["n"]
    new = torch.randint(1, case["new"] + 1, (n,), generator=torch.Generator().manual_seed(n + case["new"]))
    new = new[torch.randperm(n, generator=r.c)].tolist()
    cached = r.host(0, case["cached"], n) if case["cached"] else [0] * n
    return new, cached


def _table_inputs(case, seed):
    r = _Random(seed)
    n, BS = case["n"], case["page"]
    new, cached = _lengths(case, r)
    have = [-(-c // BS) for c in cached]
    need = [-(-(c + k) // BS) - h for c, k, h in zip(cached, new, have)]
    pages = r.pages(sum(have) + sum(need) + n)
    rows = [[pages.pop() for _ in range(h)] for h in have]
    free = list(pages)                                               # what is left is handed out from the front, with some to spare
    width = -(-(case["new"] + case["cached"]) // BS)
    slots = torch.randperm(n + 3, generator=r.c)[:n].tolist()        # requests sit in any rows of the table
    table = [[0] * width for _ in range(n + 3)]
    for s, row in zip(slots, rows):
        table[s][:len(row)] = row
    if case["kind"] == "maps":
        for s, h, k in zip(slots, have, need):
            table[s][h:h + k] = [free.pop() for _ in range(k)]
    return {"table": _ints(table), "rows": _ints(slots), "cached": _ints(cached), "new": _ints(new), "lens": _ints([c + k for c, k in zip(cached, new)]),
            "blocks": _ints(free), "total": sum(new), "n_tiles": sum(-(-k // TILE) for k in new), "need": sum(need)}


def _logit_inputs(case, seed):
    """Rules of a batch as requests set them: some rows without a penalty, some with all of them; tokens of a text come again and again."""
    r = _Random(seed)
    B, V = case["B"], case["V"]
    length = r.host(1, case["history"], B)
    prompt = [r.host(0, n, 1)[0] for n in length]
    often = torch.floor(r.uniform(0.0, 1.0, B, case["history"]) ** 4 * V).to(torch.int32).clamp_(0, V - 1)
    kind = torch.arange(B, device=DEV) % 3
    one = torch.ones(B, device=DEV)
    s = {"logits": r.normal(B, V, std=3.0).to(DTYPES[case["dtype"]]), "tokens": often, "length": _ints(length), "prompt": _ints(prompt),
         "repetition": torch.where(kind != 1, r.uniform(1.01, 1.3, B), one), "presence": torch.where(kind != 0, r.uniform(-0.5, 1.5, B), 0 * one),
         "frequency": torch.where(kind == 2, r.uniform(0.0, 1.0, B), 0 * one), "temperature": r.uniform(0.5, 1.2, B)}
    if case["bias"]:
        m = case["bias"]
        s["bias_ids"] = torch.stack([torch.randperm(V, generator=r.c)[:m] for _ in range(B)]).to(torch.int32).to(DEV)
        s["bias_values"] = r.uniform(-5.0, 5.0, B, m)
        s["bias_length"] = _ints(r.host(0, m, B))
    if case["mask"]:
        words = -(-V // 32)
        dense, thin = r.below(2 ** 32, B, words, dtype=torch.int64), r.below(2 ** 32, B, words, dtype=torch.int64)
        for _ in range(4):
            thin &= r.below(2 ** 32, B, words, dtype=torch.int64)   # a grammar allows few tokens in one state and most in another
        dense = torch.where((torch.arange(B, device=DEV) % 2 == 0)[:, None], dense, thin)
        s["mask"] = torch.where(dense >= 2 ** 31, dense - 2 ** 32, dense).to(torch.int32)
        s["masked"] = torch.arange(B, device=DEV) < round(B * case["mask"])
    return s


def _inputs(case, seed):
    return (_prefix_inputs if case["kind"] == "prefix" else _logit_inputs if case["kind"] in ("logits", "greedy") else _table_inputs)(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if own and kind == "prefix":
        from llm_in_practise_b200.ops.prefix_attention import make_prefix_groups
        s["plan"] = make_prefix_groups(s["groups"], s["qkv"].shape[0], DEV)
    if own and kind in ("logits", "greedy"):
        from llm_in_practise_b200.ops.logits import LogitState
        st = LogitState(case["B"], case["V"], case["history"], max_bias=case["bias"], device=DEV)
        st.tokens.copy_(s["tokens"]); st.length.copy_(s["length"]); st.prompt_length.copy_(s["prompt"])
        for name in ("repetition", "presence", "frequency", "temperature"):
            getattr(st, name).copy_(s[name])
        if case["bias"]:
            st.bias_ids.copy_(s["bias_ids"]); st.bias_values.copy_(s["bias_values"]); st.bias_length.copy_(s["bias_length"])
        if case["mask"]:
            st.allow_masks()
            st.mask.copy_(s["mask"]); st.masked.copy_(s["masked"])
        s["state"], s["slot"] = st, torch.arange(case["B"], dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ the package's calls
def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "prefix":
        from llm_in_practise_b200.ops.prefix_attention import prefix_attention
        return prefix_attention(s["qkv"], s["ck"], s["cv"], s["table"], s["pos"], s["slot"], s["plan"], case["H"], case["G"], case["D"],
                                case["D"] ** -0.5, sinks=s["sinks"], max_pos=max(s["keys"]) - 1)
    if kind == "extend":
        from llm_in_practise_b200.ops.step_maps import extend_block_tables
        used = extend_block_tables(s["table"], s["rows"], s["cached"], s["lens"], s["blocks"], case["page"])
        return {"table": s["table"], "used": used}
    if kind == "maps":
        from llm_in_practise_b200.ops.step_maps import step_maps
        m = step_maps(s["table"], s["rows"], s["cached"], s["new"], case["page"], s["total"], n_tiles=s["n_tiles"])
        return {"cu": m.cu, "pos": m.pos, "slot": m.slot, "place": m.place, "last": m.last, "tiles": m.tiles}
    from llm_in_practise_b200.ops.logits import greedy_tokens, process_logits
    return (process_logits if kind == "logits" else greedy_tokens)(s["logits"], s["state"], s["slot"])


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_prefix(s):
    case = s["case"]
    H, G, D, BS = case["H"], case["G"], case["D"], case["page"]
    T, rep = s["pos"].shape[0], case["H"] // case["G"]
    q = s["qkv"][:, :H * D].float().view(T, G, rep, D) * D ** -0.5

    def keys_of(pool, blocks):                                       # pages in order -> [..., G, keys, D]
        x = pool[blocks.long()].float()
        return x.movedim(-3, -4).flatten(-3, -2)

    out = torch.empty(T, G, rep, D, device=DEV)
    parts = list(s["groups"])
    at = sum(n for _, n, _ in parts)
    if at < T:
        parts.append((at, T - at, 0))
    for first, n, shared in parts:
        rows, qg = s["table"][first:first + n], q[first:first + n]
        lo = shared // BS
        hi = -(-max(s["keys"][first:first + n]) // BS)
        k, v = keys_of(s["ck"], rows[:, lo:hi]), keys_of(s["cv"], rows[:, lo:hi])
        at_key = torch.arange(lo * BS, hi * BS, device=DEV)
        sc = torch.einsum("ngrd,ngkd->ngrk", qg, k)
        hidden = (at_key[None] > s["pos"][first:first + n, None]) | (at_key[None] < shared)
        sc = sc.masked_fill(hidden[:, None, None], float("-inf"))
        m = sc.amax(-1, keepdim=True)
        if shared:
            nb = -(-shared // BS)
            pk, pv = keys_of(s["ck"], rows[0, :nb])[:, :shared], keys_of(s["cv"], rows[0, :nb])[:, :shared]
            ps = torch.einsum("ngrd,gkd->ngrk", qg, pk)
            m = torch.maximum(m, ps.amax(-1, keepdim=True))
        if s["sinks"] is not None:
            m = torch.maximum(m, s["sinks"].view(1, G, rep, 1))
        p = torch.exp(sc - m)
        total, acc = p.sum(-1, keepdim=True), torch.einsum("ngrk,ngkd->ngrd", p, v)
        if shared:
            p = torch.exp(ps - m)
            total, acc = total + p.sum(-1, keepdim=True), acc + torch.einsum("ngrk,gkd->ngrd", p, pv)
        if s["sinks"] is not None:
            total = total + torch.exp(s["sinks"].view(1, G, rep, 1) - m)
        out[first:first + n] = acc / total
    return out.view(T, H * D).to(s["qkv"].dtype)


def _plain_extend(s):
    case, BS = s["case"], s["case"]["page"]
    have, want = (s["cached"] + BS - 1) // BS, (s["lens"] + BS - 1) // BS
    need = want - have
    start = need.cumsum(0) - need
    col = torch.arange(s["table"].shape[1], device=DEV)
    take = (col[None] >= have[:, None]) & (col[None] < want[:, None])
    at = (start[:, None] + col[None] - have[:, None]).clamp(0, s["blocks"].shape[0] - 1)
    rows = s["rows"].long()
    s["table"][rows] = torch.where(take, s["blocks"][at.long()], s["table"][rows])
    return {"table": s["table"], "used": need.sum().to(torch.int32).view(1)}


def _plain_maps(s):
    case, BS, T = s["case"], s["case"]["page"], s["total"]
    new, n = s["new"], s["new"].shape[0]
    cu = torch.cat([new.new_zeros(1), new.cumsum(0).to(torch.int32)])
    owner = torch.repeat_interleave(torch.arange(n, device=DEV), new.long(), output_size=T)
    pos = torch.arange(T, device=DEV, dtype=torch.int32) - cu[owner] + s["cached"][owner]
    slot = s["rows"][owner]
    block = s["table"][slot.long(), (pos // BS).long()].long()
    nt = (new + TILE - 1) // TILE
    tile_owner = torch.repeat_interleave(torch.arange(n, device=DEV), nt.long(), output_size=s["n_tiles"])
    before = (torch.arange(s["n_tiles"], device=DEV) - (nt.cumsum(0) - nt)[tile_owner]).to(torch.int32) * TILE
    tiles = torch.stack([cu[tile_owner] + before, torch.minimum(new[tile_owner] - before, torch.full_like(before, TILE)),
                         s["cached"][tile_owner] + before, s["rows"][tile_owner]], 1)
    return {"cu": cu, "pos": pos, "slot": slot, "place": block * BS + (pos % BS).long(), "last": (cu[1:] - 1).long(), "tiles": tiles}


def _plain_logits(s):
    y = s["logits"].float()
    B, V = y.shape
    at = torch.arange(s["tokens"].shape[1], device=DEV)[None]
    rows = torch.arange(B, device=DEV)[:, None].expand_as(s["tokens"])
    known = at < s["length"][:, None]
    said = known & (at >= s["prompt"][:, None])
    seen = torch.zeros(B, V, dtype=torch.bool, device=DEV)
    seen[rows[known], s["tokens"][known].long()] = True
    count = torch.zeros(B, V, dtype=torch.int32, device=DEV)
    count.index_put_((rows[said], s["tokens"][said].long()), torch.ones((), dtype=torch.int32, device=DEV), accumulate=True)
    rep = s["repetition"][:, None]
    y = torch.where(seen, torch.where(y < 0, y * rep, y / rep), y)
    y = y - s["frequency"][:, None] * count
    y = y - s["presence"][:, None] * (count > 0)
    if "bias_ids" in s:
        used = torch.arange(s["bias_ids"].shape[1], device=DEV)[None] < s["bias_length"][:, None]
        rows = torch.arange(B, device=DEV)[:, None].expand_as(s["bias_ids"])
        bias = torch.zeros(B, V, device=DEV)
        bias[rows[used], s["bias_ids"][used].long()] = s["bias_values"][used]
        y = y + bias
    y = y / s["temperature"][:, None]
    if "mask" in s:
        token = torch.arange(V, device=DEV)
        allowed = (s["mask"][:, token // 32] >> (token % 32)) & 1
        y = torch.where((allowed == 0) & s["masked"][:, None], torch.full_like(y, float("-inf")), y)
    return y


def run(s):
    with torch.no_grad():
        if own:
            return _run_own(s)
        kind = s["case"]["kind"]
        if kind == "prefix":
            return _plain_prefix(s)
        if kind == "extend":
            return _plain_extend(s)
        if kind == "maps":
            return _plain_maps(s)
        y = _plain_logits(s)
        if kind == "logits":
            return y
        best = y.amax(1, keepdim=True)                               # the lowest of the best
        return torch.where(y == best, torch.arange(y.shape[1], device=DEV)[None], y.shape[1]).amin(1)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "prefix":
        es = 2
        sizes = [tuple(int(x) for x in g.split(":")) for g in case["groups"].split(",")]
        T = sum(n for n, _ in sizes) + case["alone"]
        own_keys = T * (case["own_keys"] + 1) / 2                    # their lengths are spread evenly
        read = sum(s for _, s in sizes) + own_keys
        pairs = sum(n * s for n, s in sizes) + own_keys
        return {"bytes": read * case["G"] * case["D"] * 2 * es + 2 * T * case["H"] * case["D"] * es, "flops": 4 * pairs * case["H"] * case["D"]}
    if kind in ("extend", "maps"):
        tokens = case["n"] * (case["new"] + 1) / 2
        blocks = tokens / case["page"] + case["n"] * 0.5
        if kind == "extend":
            return {"bytes": case["n"] * 12 + blocks * 8, "flops": 0}
        return {"bytes": case["n"] * 24 + blocks * 4 + tokens * 16 + 16 * (tokens / TILE + case["n"] * 0.5), "flops": 0}
    B, V = case["B"], case["V"]
    es = 4 if case["dtype"] == "fp32" else 2
    bytes_ = B * V * es + B * (case["history"] + 1) / 2 * 4 + B * case["bias"] / 2 * 8 + round(B * case["mask"]) * (V / 8) + B * 28
    return {"bytes": bytes_ + (B * V * 4 if kind == "logits" else B * 8), "flops": B * V * 2}


# ------------------------------------------------------------------------------------------------ 64 bits, token by token and row by row
def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "prefix":
        H, G, D, BS = case["H"], case["G"], case["D"], case["page"]
        rows = []
        for t, n in enumerate(s["keys"]):                            # every sequence by itself, over its own pages
            at = torch.arange(n, device=DEV)
            block = s["table"][t, at // BS].long()
            k, v = s["ck"][block, :, at % BS].double(), s["cv"][block, :, at % BS].double()
            q = s["qkv"][t, :H * D].double().view(G, H // G, D)
            score = torch.matmul(q, k.permute(1, 2, 0)) / D ** 0.5
            if s["sinks"] is not None:
                score = torch.cat([score, s["sinks"].double().view(G, H // G, 1)], 2)
            weight = score.softmax(2)[:, :, :n]
            rows.append(torch.matmul(weight, v.transpose(0, 1)).reshape(H * D))
        return torch.stack(rows)
    if kind == "extend":
        BS = case["page"]
        table, free, used = s["table"].tolist(), s["blocks"].tolist(), 0
        for row, c, n in zip(s["rows"].tolist(), s["cached"].tolist(), s["lens"].tolist()):
            for j in range(-(-c // BS), -(-n // BS)):
                table[row][j] = free[used]
                used += 1
        return {"table": _ints(table), "used": _ints([used])}
    if kind == "maps":
        BS, table = case["page"], s["table"].tolist()
        cu, pos, slot, place, tiles = [0], [], [], [], []
        for row, c, k in zip(s["rows"].tolist(), s["cached"].tolist(), s["new"].tolist()):
            tiles += [[cu[-1] + a, min(TILE, k - a), c + a, row] for a in range(0, k, TILE)]
            pos += range(c, c + k)
            slot += [row] * k
            place += [table[row][p // BS] * BS + p % BS for p in range(c, c + k)]
            cu.append(cu[-1] + k)
        return {"cu": _ints(cu), "pos": _ints(pos), "slot": _ints(slot), "place": _ints(place, torch.int64), "last": _ints([c - 1 for c in cu[1:]], torch.int64),
                "tiles": _ints(tiles)}
    rows = []
    V = case["V"]
    for b in range(case["B"]):
        y = s["logits"][b].double()
        n, m = int(s["length"][b]), int(s["prompt"][b])
        said = torch.bincount(s["tokens"][b, m:n].long(), minlength=V).double()
        seen = torch.bincount(s["tokens"][b, :n].long(), minlength=V) > 0
        r = float(s["repetition"][b])
        y = torch.where(seen & (y > 0), y / r, torch.where(seen, y * r, y))
        y = y - float(s["frequency"][b]) * said - float(s["presence"][b]) * (said > 0).double()
        if case["bias"]:
            k = int(s["bias_length"][b])
            y.index_add_(0, s["bias_ids"][b, :k].long(), s["bias_values"][b, :k].double())
        y = y / float(s["temperature"][b])
        if case["mask"] and bool(s["masked"][b]):
            word = s["mask"][b].long() & 0xFFFFFFFF
            bits = torch.stack([(word >> i) & 1 for i in range(32)], 1).reshape(-1)[:V]
            y[bits == 0] = float("-inf")
        rows.append(y)
    y = torch.stack(rows)
    return y if kind == "logits" else y.argmax(1)
