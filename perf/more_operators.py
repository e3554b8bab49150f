"""The operators of a training step on given tokens, and what it keeps for its backward pass, as cases that can be run and timed one by one:

    score     log probabilities of given tokens under given logits, with entropy, rank and the most probable alternatives
    grad      the same with the gradient of log probabilities and entropies
    head      the same from hidden states and the weights of an output projection, forward alone or with both gradients
    embed     embedding lookup with scaling, and the table's gradient by sorted tokens
    pack      activations in 8 bits, and back
    glu       SwiGLU that keeps its input in 8 bits for the backward pass

A case is a dict of plain values. ``run`` computes a case in its plain form, or, where ``own`` is true, calls the package.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32                    # values that share a power of two


def listed():
    return [
        # one chat whose next token is shown with twenty alternatives: the smallest call, bound by latency
        {"name": "score_chat", "kind": "score", "T": 1, "V": 151936, "top": 20, "entropy": False, "rank": True, "temperature": 1.0, "masked": 0.0, "skipped": 0.0, "dtype": "fp32"},
        # the prompt tokens of a batch, scored for a report: every row with its entropy, rank and five alternatives
        {"name": "score_prompts", "kind": "score", "T": 3000, "V": 151936, "top": 5, "entropy": True, "rank": True, "temperature": 1.0, "masked": 0.0, "skipped": 0.1, "dtype": "bf16"},
        # decoding under a grammar, an odd vocabulary, logits in fp16, a temperature
        {"name": "score_grammar", "kind": "score", "T": 64, "V": 50257, "top": 8, "entropy": True, "rank": False, "temperature": 0.7, "masked": 0.9, "skipped": 0.0, "dtype": "fp16"},
        # a step of preference or reward training on sampled answers; prompt tokens are skipped
        {"name": "grad_answers", "kind": "grad", "T": 4096, "V": 151936, "entropy": True, "temperature": 1.0, "skipped": 0.3, "dtype": "bf16"},
        # answers scored by a frozen model of 8B parameters, from its hidden states
        {"name": "head_frozen", "kind": "head", "T": 2048, "K": 4096, "V": 151936, "entropy": True, "temperature": 1.0, "skipped": 0.0, "grad": False, "dtype": "bf16"},
        # a training step of a model with 2560 channels whose head is trained too, an odd number of tokens
        {"name": "head_train", "kind": "head", "T": 1001, "K": 2560, "V": 151936, "entropy": True, "temperature": 1.0, "skipped": 0.25, "grad": True, "dtype": "bf16"},
        # the input layer of a small language model in fp32: 16 sequences of 256 tokens
        {"name": "embed_gpt", "kind": "embed", "T": 4096, "V": 30522, "D": 768, "scale": 1.0, "padding": 0.0, "dtype": "fp32"},
        # the input layer of a large one in bf16, scaled, a padded batch
        {"name": "embed_llm", "kind": "embed", "T": 16384, "V": 151936, "D": 4096, "scale": 64.0, "padding": 0.3, "dtype": "bf16"},
        # a short batch's layer inputs, odd width
        {"name": "pack_short", "kind": "pack", "T": 100, "D": 1100, "add": False, "dtype": "fp16"},
        # what a layer of 4096 channels keeps of 16384 tokens: the stream and the last branch, added
        {"name": "pack_layer", "kind": "pack", "T": 16384, "D": 4096, "add": True, "dtype": "bf16"},
        # the gated unit of a small layer in fp32, odd sizes
        {"name": "glu_small", "kind": "glu", "T": 301, "F": 1000, "dtype": "fp32"},
        # the gated unit of a layer with 12288 channels, forward and backward
        {"name": "glu_layer", "kind": "glu", "T": 8192, "F": 12288, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "score", "grad", "head", "embed", "embed", "pack", "glu"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    V = rng.choice([151936, 151936, 50257, 32768, 30522, 6400, 1001])
    if kind == "score":
        return {"kind": kind, "T": _log(rng, 1, 1200), "V": V, "top": rng.choice([0, 1, 5, 20, 32]), "entropy": rng.random() < 0.5, "rank": rng.random() < 0.5,
                "temperature": rng.choice([1.0, 0.7, 1.3]), "masked": rng.choice([0.0, 0.0, 0.9, 0.999]), "skipped": rng.choice([0.0, 0.2]), "dtype": dtype}
    if kind == "grad":
        return {"kind": kind, "T": _log(rng, 1, 1800), "V": V, "entropy": rng.random() < 0.5, "temperature": rng.choice([1.0, 0.8]), "skipped": rng.choice([0.0, 0.3]), "dtype": dtype}
    if kind == "head":
        return {"kind": kind, "T": _log(rng, 1, 1000), "K": rng.choice([768, 1024, 2560]), "V": V, "entropy": rng.random() < 0.5, "temperature": rng.choice([1.0, 0.8]),
                "skipped": rng.choice([0.0, 0.3]), "grad": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "embed":
        return {"kind": kind, "T": _log(rng, 1, 16384), "V": V, "D": rng.choice([768, 1024, 2560, 200, 64]), "scale": rng.choice([1.0, 32.0]),
                "padding": rng.choice([0.0, 0.3, 0.9]), "dtype": dtype}
    if kind == "pack":
        return {"kind": kind, "T": _log(rng, 1, 8192), "D": rng.choice([768, 2560, 4096, 1100, 77, 8]), "add": rng.random() < 0.5, "dtype": dtype}
    return {"kind": kind, "T": _log(rng, 1, 4096), "F": rng.choice([12288, 9728, 2048, 1000, 36]), "dtype": dtype}


# ------------------------------------------------------------------------------------------------ inputs
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=self.g) * std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, device=DEV, generator=self.g)


def _words(r, n, V):
    """Tokens as a text has them: some come again and again, most seldom."""
    return torch.floor(r.uniform(n) ** 4 * V).to(torch.int64).clamp_(0, V - 1)


def _activations(r, T, D, dtype):
    """Rows with channels that stand out, as the stream of a trained model has them."""
    x = torch.randn(T, D, device=DEV, generator=r.g)
    x[:, ::97] *= 30.0
    return (x * (0.1 + r.uniform(T, 1))).to(dtype)


def _inputs(case, seed):
    r = _Random(seed)
    kind, T, dt = case["kind"], case["T"], DTYPES[case["dtype"]]
    if kind == "pack":
        return {"x": _activations(r, T, case["D"], dt), "add": r.normal(T, case["D"], dtype=dt) if case["add"] else None}
    if kind == "glu":
        return {"gu": r.normal(T, 2 * case["F"], dtype=dt, std=1.5), "dy": r.normal(T, case["F"], dtype=dt, std=0.1)}
    V = case["V"]
    ids = _words(r, T, V)
    if kind == "embed":
        if case["padding"]:
            ids = torch.where(r.uniform(T) < case["padding"], torch.full_like(ids, V - 1), ids)
        return {"ids": ids, "table": r.normal(V, case["D"], dtype=dt, std=0.02), "dy": r.normal(T, case["D"], dtype=dt, std=0.1),
                "pad": V - 1 if case["padding"] else None}
    s = {"tokens": torch.where(r.uniform(T) < case["skipped"], torch.full_like(ids, -100), ids)}
    if kind == "head":
        s["x"], s["w"] = r.normal(T, case["K"], dtype=dt), r.normal(V, case["K"], dtype=dt, std=3.0 / case["K"] ** 0.5)
    else:
        s["logits"] = r.normal(T, V, dtype=dt, std=3.0)
        if case.get("masked"):
            hidden = r.uniform(T, V) < case["masked"]
            hidden.scatter_(1, ids[:, None], False)                  # a token that was chosen is one that the grammar allowed
            s["logits"].masked_fill_(hidden, float("-inf"))
    if kind == "grad" or case.get("grad"):
        s["g"] = r.normal(T) / T                                     # an advantage a token
        s["h"] = r.normal(T, std=0.1) / T if case["entropy"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    leaves = {"grad": ["logits"], "head": ["x", "w"] if case.get("grad") else [], "embed": ["table"], "glu": ["gu"]}.get(case["kind"], [])
    if own:
        for name in leaves:
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ the package's calls
def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "score":
        from llm_in_practise_b200.ops.logprobs import token_logprobs
        r = token_logprobs(s["logits"], s["tokens"], top=case["top"], entropy=case["entropy"], rank=case["rank"], temperature=case["temperature"])
        return {k: v for k, v in r._asdict().items() if v is not None}
    if kind in ("grad", "head"):
        from llm_in_practise_b200.ops.logprobs import linear_token_logprobs, token_logprobs
        if kind == "grad":
            r = token_logprobs(s["logits"], s["tokens"], entropy=case["entropy"], temperature=case["temperature"])
            leaves = {"logits": s["logits"]}
        else:
            r = linear_token_logprobs(s["x"], s["w"], s["tokens"], entropy=case["entropy"], temperature=case["temperature"])
            leaves = {"x": s["x"], "w": s["w"]} if case["grad"] else {}
        out = {"logprob": r.logprob.detach()}
        if case["entropy"]:
            out["entropy"] = r.entropy.detach()
        if leaves:
            pairs = [(r.logprob, s["g"])] + ([(r.entropy, s["h"])] if case["entropy"] else [])
            grads = torch.autograd.grad([a for a, _ in pairs], list(leaves.values()), [b for _, b in pairs])
            out.update({"d" + n: g for n, g in zip(leaves, grads)})
        return out
    if kind == "embed":
        from llm_in_practise_b200.ops.elementwise import embedding
        y = embedding(s["ids"], s["table"], scale=case["scale"], padding_idx=s["pad"])
        return {"y": y.detach(), "dtable": torch.autograd.grad(y, s["table"], s["dy"])[0]}
    if kind == "pack":
        from llm_in_practise_b200.ops.act8 import pack8, unpack8
        return unpack8(pack8(s["x"], s["add"]))
    from llm_in_practise_b200.ops.act8 import swiglu8
    y = swiglu8(s["gu"])
    return {"y": y.detach(), "dgu": torch.autograd.grad(y, s["gu"], s["dy"])[0]}


# ------------------------------------------------------------------------------------------------ plain forms
def _rows(y, tokens, entropy):
    """Log probabilities and entropies of rows y in 32 bits; rows without a token give zeros. Also what the gradient needs."""
    V = y.shape[1]
    ok = (tokens >= 0) & (tokens < V)
    at = tokens.clamp(0, V - 1)[:, None]
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    lp = torch.where(ok, (y.gather(1, at) - lse)[:, 0], 0.0)
    p = e.div_(total)
    H = None
    if entropy:
        H = torch.where(ok, -(torch.where(p > 0, y - lse, 0.0) * p).sum(1), 0.0)
    return ok, at, lse, p, lp, H


def _row_grads(y, ok, at, lse, p, g, h, H, temperature):
    d = -g[:, None] * p
    if h is not None:
        d -= h[:, None] * p * (torch.where(p > 0, y - lse, 0.0) + H[:, None])
    d.scatter_add_(1, at, g[:, None])
    d.masked_fill_(~ok[:, None], 0.0)
    return d.div_(temperature)


def _plain_score(s):
    case = s["case"]
    parts = []
    for a in range(0, case["T"], 512):                               # a few rows at a time: sorting takes room
        l, t = s["logits"][a:a + 512], s["tokens"][a:a + 512]
        y = l.float() / case["temperature"]
        ok, at, lse, _, lp, H = _rows(y, t, case["entropy"])
        r = {"logprob": lp}
        if case["entropy"]:
            r["entropy"] = H
        if case["rank"]:
            r["rank"] = torch.where(ok, 1 + (l > l.gather(1, at)).sum(1), 0)
        if case["top"]:
            v, i = l.float().sort(dim=1, descending=True, stable=True)
            v, i = v[:, :case["top"]], i[:, :case["top"]]
            r["top_ids"] = torch.where(ok[:, None], i, -1)
            r["top_logprobs"] = torch.where(ok[:, None], v / case["temperature"] - lse, 0.0)
        parts.append(r)
    return {k: torch.cat([r[k] for r in parts]) for k in parts[0]}


def _plain_grad(s):
    case = s["case"]
    y = s["logits"].float() / case["temperature"]
    ok, at, lse, p, lp, H = _rows(y, s["tokens"], case["entropy"])
    out = {"logprob": lp}
    if case["entropy"]:
        out["entropy"] = H
    out["dlogits"] = _row_grads(y, ok, at, lse, p, s["g"], s["h"], H, case["temperature"]).to(s["logits"].dtype)
    return out


def _plain_head(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    y = (x @ w.t()) / case["temperature"]
    ok, at, lse, p, lp, H = _rows(y, s["tokens"], case["entropy"])
    out = {"logprob": lp}
    if case["entropy"]:
        out["entropy"] = H
    if case["grad"]:
        d = _row_grads(y, ok, at, lse, p, s["g"], s["h"], H, case["temperature"])
        out["dx"], out["dw"] = (d @ w).to(s["x"].dtype), (d.t() @ x).to(s["w"].dtype)
    return out


def _plain_embed(s):
    case = s["case"]
    y = (s["table"][s["ids"]].float() * case["scale"]).to(s["table"].dtype)
    dy = s["dy"].float() * case["scale"]
    if s["pad"] is not None:
        dy = dy.masked_fill((s["ids"] == s["pad"])[:, None], 0.0)
    d = torch.zeros(case["V"], case["D"], device=DEV).index_add_(0, s["ids"], dy)
    return {"y": y, "dtable": d.to(s["table"].dtype)}


def _power(e):
    """2 ** e in fp32 for whole numbers -127 .. 127, exactly."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _in_8_bits(x, largest):
    """The values that x (fp32, rows) has in 8 bits: blocks of 32 share the least power of two under which all of them are below 127.5."""
    T, D = x.shape
    pad = -D % BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).view(T, -1, BLOCK)
    part, power = torch.frexp(b.abs().amax(2, keepdim=True))
    e = (power - 7 + (part * 128 >= 127.5).int()).clamp(-127, largest)
    q = torch.round(b * _power(-e)).clamp(-127, 127)
    return (q * _power(e)).view(T, -1)[:, :D]


def _largest(dtype):
    return 9 if dtype is torch.float16 else 121                      # 127 times this power of two is still a number of the type


def _plain_pack(s):
    x = s["x"].float()
    if s["add"] is not None:
        x = (x + s["add"].float()).to(s["x"].dtype).float()          # the stream is rounded where a model adds it
    return _in_8_bits(x, _largest(s["x"].dtype)).to(s["x"].dtype)


def _plain_glu(s):
    F, dt = s["case"]["F"], s["gu"].dtype
    g, u = s["gu"][:, :F].float(), s["gu"][:, F:].float()
    y = g / (1 + torch.exp(-g)) * u
    g, u = _in_8_bits(g, _largest(dt)), _in_8_bits(u, _largest(dt))
    sig, dy = 1 / (1 + torch.exp(-g)), s["dy"].float()
    return {"y": y.to(dt), "dgu": torch.cat([dy * u * sig * (1 + g * (1 - sig)), dy * g * sig], 1).to(dt)}


def run(s):
    if own:
        if s["case"]["kind"] in ("grad", "embed", "glu") or s["case"].get("grad"):
            return _run_own(s)
        with torch.no_grad():
            return _run_own(s)
    with torch.no_grad():
        return {"score": _plain_score, "grad": _plain_grad, "head": _plain_head, "embed": _plain_embed, "pack": _plain_pack, "glu": _plain_glu}[s["case"]["kind"]](s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, T = case["kind"], case["T"]
    es = 4 if case["dtype"] == "fp32" else 2
    if kind == "pack":                                               # read, kept in 8 bits, read again, written
        n, kept = T * case["D"], T * (case["D"] + -(-case["D"] // BLOCK))
        return {"bytes": n * es * (3 if case["add"] else 2) + 2 * kept, "flops": 4 * n}
    if kind == "glu":
        n, kept = T * case["F"], 2 * T * (case["F"] + -(-case["F"] // BLOCK))
        return {"bytes": n * es * (2 + 1 + 1 + 2) + 2 * kept, "flops": 20 * n}
    V = case["V"]
    if kind == "embed":
        D = case["D"]
        rows = T * (1 - case["padding"])
        return {"bytes": T * (8 + 2 * D * es) + rows * D * es + V * D * es, "flops": 2 * T * D}
    rows = T * (1 - case["skipped"])
    small = T * 8 + T * 4 * (1 + bool(case["entropy"]))
    if kind == "score":
        return {"bytes": rows * V * es + small + T * (8 * bool(case["rank"]) + 12 * case["top"]), "flops": 4 * rows * V}
    if kind == "grad":
        return {"bytes": 2 * rows * V * es + T * V * es + 2 * small, "flops": 10 * rows * V}
    K = case["K"]
    n = 3 if case["grad"] else 1
    return {"bytes": (T * K + V * K) * es * (2 if case["grad"] else 1) + small, "flops": n * 2 * rows * V * K}


# ------------------------------------------------------------------------------------------------ 64 bits, row by row
def _exact_row(y, t, entropy):
    lp = torch.log_softmax(y, 0)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum() if entropy else None
    return lp, p, H


def _exact_rows(logits_of, case, s):
    """Row by row from the definition; ``logits_of(i)`` are row i's logits in 64 bits, before the temperature."""
    T, V = case["T"], case["V"]
    out = {"logprob": torch.zeros(T, dtype=torch.float64, device=DEV)}
    if case["entropy"]:
        out["entropy"] = torch.zeros(T, dtype=torch.float64, device=DEV)
    if case.get("rank"):
        out["rank"] = torch.zeros(T, dtype=torch.int64, device=DEV)
    if case.get("top"):
        out["top_ids"] = torch.full((T, case["top"]), -1, dtype=torch.int64, device=DEV)
        out["top_logprobs"] = torch.zeros(T, case["top"], dtype=torch.float64, device=DEV)
    grads = torch.zeros(T, V, dtype=torch.float64, device=DEV) if "g" in s else None
    for i, t in enumerate(s["tokens"].tolist()):
        if not 0 <= t < V:
            continue
        l = logits_of(i)
        lp, p, H = _exact_row(l / case["temperature"], t, case["entropy"])
        out["logprob"][i] = lp[t]
        if case["entropy"]:
            out["entropy"][i] = H
        if case.get("rank"):
            out["rank"][i] = 1 + (l > l[t]).sum()
        if case.get("top"):
            order = torch.argsort(-l, stable=True)[:case["top"]]
            out["top_ids"][i], out["top_logprobs"][i] = order, lp[order]
        if grads is not None:
            row = -float(s["g"][i]) * p
            row[t] += float(s["g"][i])
            if s["h"] is not None:
                row -= float(s["h"][i]) * torch.where(p > 0, p * (lp + H), torch.zeros_like(p))
            grads[i] = row / case["temperature"]
    return out, grads


def exact(case, seed):
    s = _inputs(case, seed)
    kind, T = case["kind"], case["T"]
    if kind in ("score", "grad"):
        out, grads = _exact_rows(lambda i: s["logits"][i].double(), case, s)
        if grads is not None:
            out["dlogits"] = grads
        return out
    if kind == "head":
        x, w = s["x"].double(), s["w"].double()
        y = x @ w.t()
        out, grads = _exact_rows(lambda i: y[i], case, s)
        if grads is not None:
            out["dx"], out["dw"] = grads @ w, grads.t() @ x
        return out
    if kind == "embed":
        d = torch.zeros(case["V"], case["D"], dtype=torch.float64, device=DEV)
        rows = s["dy"].double() * case["scale"]
        keep = torch.ones_like(s["ids"], dtype=torch.bool) if s["pad"] is None else s["ids"] != s["pad"]
        d.index_put_((s["ids"][keep],), rows[keep], accumulate=True)
        return {"y": s["table"].double()[s["ids"]] * case["scale"], "dtable": d}

    def power(e):                                                    # 2 ** e, exactly
        return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)

    def kept(x, dtype):                                              # a value of x in 8 bits, block by block, by trying powers of two
        T, D = x.shape
        out = torch.empty_like(x)
        for a in range(0, D, BLOCK):
            b = x[:, a:a + BLOCK]
            m = b.abs().amax(1, keepdim=True)
            e = torch.floor(torch.log2(m.clamp_min(2.0 ** -140))) - 7
            for _ in range(3):
                e = torch.where(m * power(-e) >= 127.5, e + 1, e)
            e = e.clamp(-127, 9 if dtype is torch.float16 else 121)
            out[:, a:a + BLOCK] = torch.round(b * power(-e)).clamp(-127, 127) * power(e)
        return out

    if kind == "pack":
        x = s["x"].double()
        if s["add"] is not None:
            x = (x + s["add"].double()).float().to(s["x"].dtype).double()
        return kept(x, s["x"].dtype)
    F, dt = case["F"], s["gu"].dtype
    g, u, dy = s["gu"][:, :F].double(), s["gu"][:, F:].double(), s["dy"].double()
    y = g * torch.sigmoid(g) * u
    g, u = kept(g, dt), kept(u, dt)
    sig = torch.sigmoid(g)
    return {"y": y, "dgu": torch.cat([dy * u * (sig + g * sig * (1 - sig)), dy * g * sig], 1)}
