"""Log probabilities of given tokens, the embedding's gradient by sorted tokens, activations in 8 bits: each against a statement of its own in 64 bits; edges of
vocabularies, alignments, strides, tiles and blocks, masked and empty rows, NaN and infinities, ties, refusals, graphs, streams, and a step of all together."""
import math

import pytest
import torch

from llm_in_practise_b200.ops import _native as nv, act8, elementwise as ew, logprobs as lpm
from llm_in_practise_b200.ops.act8 import Packed8, checkpoint8, pack8, swiglu8, unpack8
from llm_in_practise_b200.ops.elementwise import embedding, embedding_grad
from llm_in_practise_b200.ops.logprobs import linear_token_logprobs, token_logprobs

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
gpu = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


def half_step(dtype):
    """Half a step of a type, relative to the value; and half of its smallest number."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


# ------------------------------------------------------------------------------------------------ log probabilities
def exact_rows(l, tokens, T, g=None, h=None):
    """lp, H, rank and the gradient, row by row, from the definition in 64 bits."""
    B, V = l.shape
    out = {"lp": torch.zeros(B), "H": torch.zeros(B), "rank": torch.zeros(B), "grad": torch.zeros(B, V), "p": torch.zeros(B, V)}
    out = {k: v.double() for k, v in out.items()}
    for i, t in enumerate(tokens.tolist()):
        if not 0 <= t < V:
            continue
        y = l[i].double() / T
        logp = torch.log_softmax(y, 0)
        p = logp.exp()
        plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
        out["lp"][i], out["H"][i], out["p"][i] = logp[t], -plogp.sum(), p
        out["rank"][i] = 1 + (l[i] > l[i, t]).sum()
        if g is not None:
            d = -float(g[i]) * p - float(h[i]) * (plogp + p * out["H"][i])
            d[t] += float(g[i])
            out["grad"][i] = d / T
    return out


def exact_top(row, k):
    """Ids in order: larger first, NaN above all, the lowest id first among equals."""
    key = [(-INF if math.isnan(v) else -v, i) for i, v in enumerate(row.double().tolist())]
    nan_first = sorted(range(len(key)), key=lambda i: (not math.isnan(float(row[i])), key[i]))
    return nan_first[:k]


def sum_error(V):
    """Relative error of a row's sum of V weights: each has 2^-22 from the exponential and, as its exponent is rounded three times, 3 (2^-24) |y - max|, where
    weights beyond |y - max| = 24 no longer count (72 steps); the sum rounds once per value that a thread adds (V / 256 at the fewest threads, of which
    a value passes at most 64 more where partial sums meet)."""
    return 2.0 ** -22 + (72 + V / 256 + 64) * 2.0 ** -24


def lp_tolerance(e, V, T, spread):
    """log s has the relative error of s (absolute in the logarithm) and half a step of itself; the difference to the maximum and its quotient by T round three
    times."""
    return sum_error(V) + 2.0 ** -24 * (4 * spread + 4 * (e["lp"].abs() + math.log(V) + 1))


def masks(l, kind):
    B, V = l.shape
    low = torch.finfo(l.dtype).min
    if kind == "inf":
        l[:, 1::3] = -INF
    elif kind == "lowest":
        l[:, 1::3] = low
    elif kind == "one":                                   # a single token is allowed
        l[:, 1:] = -INF
    elif kind == "all_lowest":                            # every logit is the type's lowest: the row is uniform
        l[:] = low
    elif kind == "nothing":
        l[:] = -INF
    elif kind == "ties":
        l.copy_((l * 2).round() / 2)
    return l


VOCABS = [1, 2, 7, 8, 31, 33, 1000, 1001, 4099, 30522, 151936]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["plain", "inf", "lowest", "one", "all_lowest", "ties"])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", VOCABS)
def test_rows_and_their_gradient(V, dtype, kind, device):
    if device == "cpu" and V > 5000:
        pytest.skip("the kernels' sizes")
    B, T = 5, 0.75
    r = torch.Generator().manual_seed(V)
    l = masks((torch.randn(B, V, generator=r) * 3).to(DT[dtype]), kind)
    tokens = torch.randint(0, V, (B,), generator=r)
    tokens[0] = 0
    tokens[1:3] = torch.tensor([-100, V])                 # passed over
    if kind in ("inf", "lowest"):
        tokens[3:] -= (tokens[3:] % 3 == 1).long()        # tokens that were allowed
    elif kind == "one":
        tokens[3:] = 0
    g, h = torch.randn(B, generator=r), torch.randn(B, generator=r)
    e = exact_rows(l, tokens, T, g, h)
    k = min(20, V)
    x = l.clone().to(device).requires_grad_(True)
    got = token_logprobs(x, tokens.to(device), top=k, entropy=True, rank=True, temperature=T)
    (grad,) = torch.autograd.grad([got.logprob, got.entropy], x, [g.to(device), h.to(device)])
    plain = token_logprobs(x.detach(), tokens.to(device), temperature=T)
    assert plain[1:] == (None,) * 4 and torch.equal(plain.logprob, got.logprob)
    spread = float((l.double().amax(1, keepdim=True) - l.double()).masked_fill(l == -INF, 0).clamp_max(1e4).max()) / T
    tol = lp_tolerance(e, V, T, min(spread, 200.0))
    assert ((got.logprob.cpu().double() - e["lp"]).abs() <= tol).all()
    # the entropy is log s - u / s, two sums with that error whose second weighs differences up to log V + 1 on the average
    assert ((got.entropy.cpu().double() - e["H"]).abs() <= tol + 2 * sum_error(V) * (math.log(V) + 2)).all()
    assert got.rank.dtype == torch.int64 and torch.equal(got.rank.cpu(), e["rank"].long())
    for i in range(B):
        if not 0 <= tokens[i] < V:
            assert (got.top_ids[i] == -1).all() and (got.top_logprobs[i] == 0).all() and (grad[i] == 0).all()
            continue
        ids = exact_top(l[i], k)
        assert got.top_ids[i].tolist() == ids
        want = torch.log_softmax(l[i].double() / T, 0)[ids].float().double()       # what 32 bits do not hold is minus infinity
        seen = got.top_logprobs[i].cpu().double()
        assert ((seen - want).abs() <= tol[i] + 2.0 ** -22 * want.abs().clamp_max(1e300))[want > -INF].all() and torch.equal(seen[want == -INF], want[want == -INF])
    # a weight has the error of its exponential (with its exponent's, 4 (2^-24) |y - max|) and of 1 / s; the bracket (|h| (|log p| + H) + |g|) that of lp and H
    half, least = half_step(DT[dtype])
    logp = (l.double() / T - torch.logsumexp(l.double() / T, 1, keepdim=True)).clamp(-1e5, 0)
    size = (e["p"] * (g.abs()[:, None] + h.abs()[:, None] * (logp.abs() + e["H"][:, None] + 1)) / T).double()
    bound = (half + 2.0 ** -24) * e["grad"].abs() + size * (4 * sum_error(V) + 2.0 ** -20) + least + 2.0 ** -23 * (g.abs() / T)[:, None] * (e["grad"] != 0)
    assert ((grad.cpu().double() - e["grad"]).abs() <= bound).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
def test_rows_without_a_number(dtype, device):
    """Nothing allowed, NaN, plus infinity: NaN, as log_softmax gives; neighbours keep their values."""
    V = 1001
    l = torch.randn(5, V).to(DT[dtype])
    l[1] = -INF
    l[2, 500] = float("nan")
    l[3, 7] = INF
    want = exact_rows(l, torch.full((5,), 3), 1.0)
    x = l.clone().to(device).requires_grad_(True)
    got = token_logprobs(x, torch.full((5,), 3, device=device), entropy=True, top=3)
    (grad,) = torch.autograd.grad(got.logprob.sum() + got.entropy.sum(), x)
    for i in (1, 2, 3):
        assert got.logprob[i].isnan() and got.entropy[i].isnan() and grad[i].isnan().any()
    for i in (0, 4):
        assert abs(float(got.logprob[i]) - float(want["lp"][i])) < 1e-4 and not grad[i].isnan().any()
    assert got.top_ids[2, 0] == 500 and got.top_ids[1].tolist() == [0, 1, 2] and got.top_ids[3, 0] == 7


@pytest.mark.parametrize("device", DEVICES)
def test_alternatives_of_equal_logits_are_the_lowest_ids(device):
    for V, k in ((40, 32), (5000, 32), (5000, 1), (70001, 32)):
        if device == "cpu" and V > 5000:
            continue
        l = torch.zeros(3, V, dtype=torch.bfloat16)
        l[1, V // 2:] = 1                                   # equal ones behind smaller ones
        l[2, -1] = -0.0
        ids = token_logprobs(l.to(device), top=k).top_ids.cpu()
        assert ids[0].tolist() == list(range(k)) and ids[2].tolist() == list(range(k))
        more = list(range(V // 2, min(V, V // 2 + k)))
        assert ids[1].tolist() == (more + list(range(k)))[:k]


@gpu
@pytest.mark.parametrize("step", [4096, 8192, 1024, 8])
def test_alternatives_that_lie_apart_evenly(step):
    """The largest logits stand a power of two apart, so that the same few threads see all of them."""
    V = 151936
    l = torch.randn(2, V)
    for j in range(8):
        l[:, j::step] += 50 + torch.rand(2, l[:, j::step].shape[1])
    for dtype in (torch.float32, torch.bfloat16):
        x = l.to(dtype)
        ids = token_logprobs(x.cuda(), top=32).top_ids.cpu()
        want = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :32]
        assert torch.equal(ids, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strided_rows_and_shapes(shift, dtype, device):
    """Rows that begin anywhere and are further apart than they are long; more dimensions than two; the same bits as from a copy."""
    wide = (torch.randn(2, 3, 531) * 3).to(DT[dtype]).to(device)
    view = wide[..., shift:shift + 509]
    tokens = torch.randint(0, 509, (2, 3), device=device)
    a, b = view.detach().requires_grad_(True), view.detach().clone().requires_grad_(True)
    got, want = (token_logprobs(x, tokens, top=4, entropy=True, rank=True) for x in (a, b))
    for x, y in zip(got, want):
        assert x.shape == y.shape and x.shape[:2] == (2, 3)
        assert torch.allclose(x.double(), y.double(), rtol=0, atol=2 * sum_error(509) + 2.0 ** -20)
    ga, gb = (torch.autograd.grad(r.logprob.sum() - r.entropy.sum(), x)[0] for r, x in ((got, a), (want, b)))
    assert ga.shape == view.shape and torch.allclose(ga.double(), gb.double(), rtol=half_step(DT[dtype])[0] * 2, atol=1e-6)
    one = token_logprobs(view[0, 0], tokens[0, 0], top=4, entropy=True)
    assert one.logprob.shape == () and one.top_ids.shape == (4,) and torch.equal(one.top_ids, got.top_ids[0, 0])
    none = token_logprobs(view[:0], tokens[:0], top=2, rank=True)
    assert none.logprob.shape == (0, 3) and none.top_ids.shape == (0, 3, 2)


def test_gradients_against_differences():
    l = torch.randn(3, 17, dtype=torch.float64)
    tokens, T = torch.tensor([3, -1, 16]), 1.3
    x = l.float().requires_grad_(True)
    r = token_logprobs(x, tokens, entropy=True, temperature=T)
    (grad,) = torch.autograd.grad((r.logprob * torch.tensor([1.0, 2.0, -0.5])).sum() + 0.3 * r.entropy.sum(), x)

    def f(l):
        e = exact_rows(l, tokens, T)
        return float((e["lp"] * torch.tensor([1.0, 2.0, -0.5])).sum() + 0.3 * e["H"].sum())
    for i in range(3):
        for j in range(17):
            d = torch.zeros_like(l)
            d[i, j] = 1e-5
            # central differences of step 1e-5 in 64 bits are good to 1e-9; the gradient to its 32 bits
            assert abs((f(l + d) - f(l - d)) / 2e-5 - float(grad[i, j])) < 2e-6


def test_only_one_gradient_and_none():
    x = torch.randn(4, 9).requires_grad_(True)
    tokens = torch.tensor([0, 1, 2, 3])
    r = token_logprobs(x, tokens, entropy=True, top=2, rank=True)
    assert r.logprob.requires_grad and r.entropy.requires_grad and not r.top_logprobs.requires_grad and not r.rank.requires_grad
    (a,) = torch.autograd.grad(r.entropy.sum(), x)
    want = exact_rows(x.detach(), tokens, 1.0, torch.zeros(4), torch.ones(4))["grad"]
    assert (a.double() - want).abs().max() < 1e-6
    assert not token_logprobs(x.detach(), tokens).logprob.requires_grad
    with torch.no_grad():
        assert not token_logprobs(x, tokens).logprob.requires_grad


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,V", [(150, 140001), (150, 131080), (3, 1100001), (150, 65544), (2, 300000)])
def test_alternatives_of_long_rows(rows, V, dtype):
    """Segments of either length, rows at odd addresses, a CTA or a cluster a row: values that are far apart, equal ones across segments and their pieces, rows with few
    values that are not the lowest, of one value alone, and with more large values than a list holds."""
    dt = DT[dtype]
    l = torch.randn(rows, V, device="cuda") * 3
    r = torch.Generator().manual_seed(V)
    for i in range(rows):
        kind = i % 6
        if kind == 1:
            l[i] = l[i].clamp_max(0) - 1
            l[i, torch.randint(0, V, (12,), generator=r).cuda()] = 5.0                       # twelve equal ones, anywhere
        elif kind == 2:
            l[i] = -INF
            l[i, torch.randint(0, V, (3,), generator=r).cuda()] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
        elif kind == 3:
            l[i] = -1.5
        elif kind == 4:
            l[i] = torch.randint(-3, 3, (V,), generator=r).float().cuda()                    # a sixth of the row is the largest
        elif kind == 5:
            at = int(torch.randint(0, V - 4000, (1,), generator=r))
            l[i, at:at + 4000] = 50 + torch.rand(4000, device="cuda")                        # close together
    l = l.to(dt)
    tokens = torch.randint(0, V, (rows,), device="cuda")
    order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1]
    lp = torch.log_softmax(l.double(), 1)
    for top in (1, 5, 8, 9, 32):
        for more in ({}, {"entropy": True, "rank": True}):
            got = token_logprobs(l, tokens, top=top, **more)
            assert torch.equal(got.top_ids, order[:, :top])
            want = lp.gather(1, got.top_ids)
            # the sum's error and that of a difference of up to |log p| (2^-22 of it, in 32 bits), as for the token itself
            bound = sum_error(V) + want.abs().clamp_max(1e4) * 2.0 ** -22 + 2.0 ** -22
            fine = (got.top_logprobs.double() - want).abs() <= bound
            assert (fine | (want == -INF) & (got.top_logprobs == -INF)).all()


def test_what_log_probabilities_refuse():
    l, t = torch.randn(2, 5), torch.tensor([0, 1])
    for bad in (lambda: token_logprobs(l.double(), t), lambda: token_logprobs(l, t.int()), lambda: token_logprobs(l, t[:1]), lambda: token_logprobs(l, t, top=6),
                lambda: token_logprobs(l, t, top=-1), lambda: token_logprobs(torch.randn(2, 50), t, top=33), lambda: token_logprobs(l, t, temperature=0.0),
                lambda: token_logprobs(l, t, temperature=float("nan")), lambda: token_logprobs(l), lambda: token_logprobs(l, rank=True, top=2),
                lambda: token_logprobs(torch.randn(2, 0), t), lambda: linear_token_logprobs(torch.randn(2, 8), torch.randn(5, 9), t),
                lambda: linear_token_logprobs(torch.randn(2, 8), torch.randn(5, 8), None), lambda: linear_token_logprobs(torch.randn(2, 8), torch.randn(5, 8), t[:1]),
                lambda: linear_token_logprobs(torch.randn(2, 8), torch.randn(5, 8).bfloat16(), t)):
        with pytest.raises((ValueError, TypeError)):
            bad()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,V,passed", [(1, 64, 37, 0), (5, 128, 1001, 0), (17, 64, 4099, 0.5), (130, 72, 20011, 0), (256, 64, 5000, 0.5), (257, 64, 5000, 0.5),
                                          (300, 128, 9000, 0), (700, 64, 3000, 0.9), (600, 64, 600, 0.572), (513, 64, 600, 1)])
def test_from_hidden_states(T, K, V, passed, dtype, device, monkeypatch):
    """Chunks of the vocabulary, odd sizes; few, many and only rows that are passed over, up to the ends of tiles (256 of 600 count), whose states and weights may be
    anything; the gradients of both operands, small ones too (weights of 1e-6)."""
    monkeypatch.setattr(lpm, "_CHUNK_BYTES", 0)                         # chunks of 4096 columns at most, the last one short
    dt, tau = DT[dtype], 0.8
    r = torch.Generator().manual_seed(T)
    x, w = torch.randn(T, K, generator=r).to(dt), (torch.randn(V, K, generator=r) * 3 / K ** 0.5).to(dt)
    tokens = torch.randint(0, V, (T,), generator=r)
    if T > 3:
        tokens[2] = -100
    tokens[torch.randperm(T, generator=r)[:round(T * passed)]] = V + 3
    if T == 600:
        counting = ((tokens >= 0) & (tokens < V)).nonzero()[:, 0]
        tokens[counting[256:]] = -1
    g, h = torch.randn(T, generator=r) * 1e-6, torch.randn(T, generator=r) * 1e-6
    bad = (tokens < 0) | (tokens >= V)
    x[bad] = float("nan")
    g[bad], h[bad] = 1e20, float("inf")
    if device == "cpu":
        x[bad] = 0
    a, b = x.clone(), w                                    # what counts; a row that is passed over has no part in anything
    a[bad] = 0
    logits = a.double() @ b.double().t()
    e = exact_rows(logits, tokens, tau, g, h)
    live, keep = a.double(), (~bad).double()
    g, h = g.clone(), h.clone()
    a, b = x.to(device).requires_grad_(True), w.to(device).requires_grad_(True)
    got = linear_token_logprobs(a, b, tokens.to(device), entropy=True, temperature=tau)
    dx, dw = torch.autograd.grad([got.logprob, got.entropy], [a, b], [g.to(device), h.to(device)])
    # a logit is a sum of K exact products in 32 bits (K + 8 roundings of the sum of magnitudes); row sums as above
    logit = (K + 8) * 2.0 ** -24 * float((live.abs() @ w.double().abs().t()).max()) / tau
    tol = lp_tolerance(e, V, tau, float((logits.amax(1, keepdim=True) - logits).max()) / tau) + 2 * logit
    assert ((got.logprob.detach().cpu().double() - e["lp"]).abs() <= tol).all()
    assert ((got.entropy.detach().cpu().double() - e["H"]).abs() <= tol + 2 * (sum_error(V) + 2 * logit) * (math.log(V) + 2)).all()
    assert not got.logprob[bad.to(device)].any() and not got.entropy[bad.to(device)].any() and not dx[bad.to(device)].any()
    # gradients of logits are rounded to 16 bits before the products (half a step of each term), the results once more; sums in 32 bits
    half, least = half_step(dt)
    rel = half + 2 * logit + 8 * sum_error(V) + 2.0 ** -19
    gs, hs = torch.where(bad, 0, g).abs(), torch.where(bad, 0, h).abs()
    size = e["p"] * (gs[:, None] + hs[:, None] * ((e["p"].clamp_min(1e-30).log()).abs() + e["H"][:, None] + 1)) / tau + e["grad"].abs()
    # fp16 brings the largest gradient to 2^13 or more, so that the smallest number, 2^-24, is 2^-37 of it
    tiny = 2.0 ** -37 * float(((gs + hs * (math.log(V) + 1)) / tau).max()) * keep[:, None] if dt == torch.float16 else 0.0
    for name, u, v, want, terms in (("dx", dx, None, e["grad"] @ w.double(), (size * rel + tiny) @ w.double().abs()),
                                    ("dw", dw, None, e["grad"].t() @ live, (size * rel + tiny).t() @ live.abs())):
        assert u.dtype == dt
        assert ((u.cpu().double() - want).abs() <= terms + half * want.abs() + least + max(T, V) * 2.0 ** -24 * terms).all(), name
    frozen = linear_token_logprobs(a, w.to(device), tokens.to(device), temperature=tau)
    assert torch.equal(frozen.logprob, got.logprob) and torch.autograd.grad(frozen.logprob.sum(), a)[0].shape == x.shape
    with torch.no_grad():
        assert torch.equal(linear_token_logprobs(a, b, tokens.to(device), temperature=tau).logprob, got.logprob)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,V", [(1001, 64, 20011), (700, 256, 9000), (1001, 640, 30522), (300, 128, 151936)])
def test_gradient_of_hidden_states_cut_along_the_vocabulary(T, K, V, dtype):
    """Few tiles, whose products are cut into parts by the rows that count, from all of them to one and none; the same bits in every call, in a captured one too that
    is replayed with other rows."""
    from llm_in_practise_b200.ops.gemm import ensure_graph_workspace
    dt, tau = DT[dtype], 0.8
    half, least = half_step(dt)
    w = (torch.randn(V, K, device="cuda") * 3 / K ** 0.5).to(dt)
    x = torch.randn(T, K, device="cuda").to(dt).requires_grad_(True)
    g = torch.randn(T, device="cuda")
    tokens = torch.randint(0, V, (T,), device="cuda")
    ensure_graph_workspace(x.device)
    torch.autograd.grad(linear_token_logprobs(x, w, tokens, temperature=tau).logprob, x, g)          # what a capture needs is there
    held, graph = tokens.clone(), torch.cuda.CUDAGraph()
    leaf = x.detach().requires_grad_(True)                 # one that no eager graph holds
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        (replayed,) = torch.autograd.grad(linear_token_logprobs(leaf, w, held, temperature=tau).logprob, leaf, g)
    logits = x.detach().double() @ w.double().t()
    logit = (K + 8) * 2.0 ** -24 * float((x.detach().double().abs() @ w.double().abs().t()).max()) / tau
    p = torch.softmax(logits / tau, 1)
    del logits
    # dl: half a step, the logit's error twice (its own and the sum's), the sum's; then V additions in 32 bits
    rel = half + 2 * logit + 8 * sum_error(V) + V * 2.0 ** -24
    for passed in (0, T // 4, T * 9 // 10, T - 257, T - 256, T - 1, T):
        t = tokens.clone()
        t[torch.randperm(T, device="cuda")[:passed]] = -1
        keep = (t >= 0).double()[:, None]
        one = torch.nn.functional.one_hot(t.clamp_min(0), V).double()
        scale = g.double()[:, None] * keep / tau
        want, terms = ((one - p) * scale) @ w.double(), ((one + p) * scale.abs()) @ w.double().abs()
        tiny = 2.0 ** -37 * float(scale.abs().max()) * (keep * w.double().abs().sum(0)) if dt == torch.float16 else 0.0
        del one
        (dx,) = torch.autograd.grad(linear_token_logprobs(x, w, t, temperature=tau).logprob, x, g)
        assert ((dx.double() - want).abs() <= terms * rel + tiny + half * want.abs() + least).all(), passed
        assert torch.equal(torch.autograd.grad(linear_token_logprobs(x, w, t, temperature=tau).logprob, x, g)[0], dx)
        held.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed, dx) or ((replayed.double() - want).abs() <= terms * rel + tiny + half * want.abs() + least).all(), passed


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,V,width", [(128, 2048, 151936, 208), (1, 2560, 151936, 208), (64, 4096, 50257, 176), (100, 8192, 6400, 48), (37, 8192, 1001, 16)])
def test_tokens_at_the_ends_of_tiles_of_odd_width(T, K, V, width, dtype):
    """Tiles of an odd number of 16 columns end inside 32 that are read at a time: the log probability of the next tile's first tokens is that tile's to give."""
    tiles = nv.proto("b200_gemm_head_tiles", [lpm.i32] * 3)(T, V, K)
    assert [n for n in range(16, 257, 16) if -(-V // n) == tiles] == [width] and width % 32 == 16
    dt, r = DT[dtype], torch.Generator().manual_seed(V)
    x, w = torch.randn(T, K, generator=r).to(dt).cuda(), (torch.randn(V, K, generator=r) * 3 / K ** 0.5).to(dt).cuda()
    logits = x.double() @ w.double().t()
    want = torch.log_softmax(logits, 1)
    # as above: the logit's sum in 32 bits (its own and those of the row's sum), the row's sum, the logarithm
    logit = (K + 8) * 2.0 ** -24 * float((x.double().abs() @ w.double().abs().t()).max())
    spread = float((logits.amax(1, keepdim=True) - logits).max())
    for at in range(4):                                     # every row has each of the places
        places = torch.randint(0, V // width, (T,), generator=r) * width + torch.tensor([0, 15, 16 % width, width - 1])[(torch.arange(T) + at) % 4]
        tokens = places.clamp_max(V - 1).cuda()
        e = want.gather(1, tokens[:, None])[:, 0]
        got = linear_token_logprobs(x, w, tokens).logprob
        assert ((got.double() - e).abs() <= lp_tolerance({"lp": e}, V, 1.0, spread) + 2 * logit).all()
        for _ in range(5):
            assert torch.equal(linear_token_logprobs(x, w, tokens).logprob, got)


# ------------------------------------------------------------------------------------------------ embedding gradients
def exact_embedding(ids, dout, rows, scale, pad):
    out = torch.zeros(rows, dout.shape[-1], dtype=torch.float64)
    size = torch.zeros_like(out)
    n = torch.zeros(rows, 1, dtype=torch.float64)
    for t, i in enumerate(ids.tolist()):
        if 0 <= i < rows and i != pad:
            out[i] += dout[t].double() * scale
            size[i] += (dout[t].double() * scale).abs()
            n[i] += 1
    return out, size, n


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 5, 8), (31, 3, 8), (32, 2, 77), (33, 1023, 64), (65, 1024, 40), (500, 1, 16), (700, 7, 200), (2000, 40000, 24), (5000, 300, 1030)])
def test_embedding_gradient(T, V, D, dtype, device):
    dt = DT[dtype]
    r = torch.Generator().manual_seed(T)
    ids = (torch.rand(T, generator=r) ** 3 * V).long().clamp(0, V - 1)
    if T > 30:
        ids[3], ids[17], ids[29] = -100, V, 2 ** 40           # no rows of the table
    pad = int(ids[0]) if T > 60 and V > 1 else None
    dout = torch.randn(T, D, generator=r).to(dt)
    want, size, n = exact_embedding(ids, dout, V, 1.5, -1 if pad is None else pad)
    for out_dtype in {dt, torch.float32}:
        got = embedding_grad(ids.to(device), dout.to(device), V, 1.5, pad, out_dtype)
        assert got.dtype == out_dtype and got.shape == (V, D)
        # n sums in 32 bits, the scale, and one rounding to the type
        half, least = half_step(out_dtype)
        assert ((got.cpu().double() - want).abs() <= (n + 2) * 2.0 ** -24 * size + half * want.abs() + least).all()
        if device == "cuda":
            assert torch.equal(got, embedding_grad(ids.to(device), dout.to(device), V, 1.5, pad, out_dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_embedding_gradient_of_strided_rows_and_shapes(device):
    ids = torch.randint(0, 50, (3, 7), device=device)
    wide = torch.randn(3, 7, 90, device=device)
    for lo in (0, 1, 4):
        a = embedding_grad(ids, wide[..., lo:lo + 64], 50)
        assert torch.equal(a, embedding_grad(ids, wide[..., lo:lo + 64].clone(), 50))
    b = embedding_grad(ids, wide[:, :1, :1].expand(3, 7, 8), 50)
    assert torch.equal(b, embedding_grad(ids, wide[:, :1, :1].expand(3, 7, 8).clone(), 50))
    assert not embedding_grad(ids[:0], wide[:0], 50).any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [1.0, 8.0])
def test_embedding_and_its_gradient(scale, device):
    table, pos = torch.randn(100, 64).to(device).requires_grad_(True), torch.randn(9, 64).to(device).requires_grad_(True)
    ids = torch.randint(0, 100, (4, 9), device=device)
    ids[0, :3] = 42
    dout = torch.randn(4, 9, 64, device=device)
    y = embedding(ids, table, pos, scale, padding_idx=42)
    assert torch.equal(y.detach(), (table.detach()[ids] * scale + pos.detach()))
    a, b = torch.autograd.grad(y, [table, pos], dout)
    want, size, n = exact_embedding(ids.flatten().cpu(), dout.flatten(0, 1).cpu(), 100, scale, 42)
    assert not a[42].any() and ((a.cpu().double() - want).abs() <= (n + 2) * 2.0 ** -23 * size).all()
    assert torch.allclose(b, dout.sum(0), rtol=0, atol=1e-5)


@gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,D", [(1, 8), (3, 64), (257, 40), (1025, 16), (300, 4096)])
def test_embedding_lookup(T, D, dtype):
    """Values are rounded to 32 bits and to the type; without a scale they are the table's. Tokens outside the table give zeros, ids of 32 bits and other shapes
    are taken."""
    dt = DT[dtype]
    table, pos = torch.randn(77, D, device="cuda").to(dt), torch.randn(T, D, device="cuda").to(dt)
    ids = torch.randint(0, 77, (T,), device="cuda")
    for scale in (1.0, 3.7):
        s32 = float(torch.tensor(scale))
        for p in (None, pos):
            want = table.double()[ids] * s32 + (0 if p is None else p.double())
            half, least = half_step(dt)
            # product and sum are one operation of 32 bits (2^-24 of the result), then the type's half step
            assert ((embedding(ids, table, p, scale).double() - want).abs() <= (half + 2.0 ** -24) * want.abs() * (1 + 2.0 ** -20) + least).all()
    assert torch.equal(embedding(ids, table), table[ids]) and torch.equal(embedding(ids, table, pos), (table.float()[ids] + pos.float()).to(dt))
    assert torch.equal(embedding(ids.int(), table), table[ids]) and torch.equal(embedding(ids.view(1, 1, T), table), table[ids].view(1, 1, T, D))
    bad = ids.clone()
    bad[0], bad[-1] = -100, 77
    y = embedding(bad, table)
    assert not y[0].any() and not y[-1].any() and torch.equal(y[1:-1], table[ids[1:-1]])
    assert embedding(ids[:0], table).shape == (0, D) and embedding(ids[0], table).shape == (D,)
    wide = torch.randn(77, 2 * D, device="cuda").to(dt)
    assert torch.equal(embedding(ids, wide[:, :D]), wide[:, :D][ids])


@gpu
@pytest.mark.parametrize("L", [1, 2, 3, 5, 7, 64, 100, 255, 256, 257, 1000, 4097, 20011])
def test_positions_of_any_period(L):
    """Each row has its own position's: a sum of two numbers of 32 bits, rounded once."""
    for dt in (torch.float32, torch.bfloat16):
        table, pos = torch.randn(50, 8, device="cuda").to(dt), torch.randn(L + 3, 8, device="cuda").to(dt)
        ids = torch.randint(0, 50, (-(-40000 // L), L), device="cuda")
        assert torch.equal(embedding(ids, table, pos), (table.float()[ids] + pos[:L].float()).to(dt))


def test_what_embedding_gradients_refuse():
    ids, d = torch.zeros(3, dtype=torch.int64), torch.randn(3, 4)
    for bad in (lambda: embedding_grad(ids.int(), d, 5), lambda: embedding_grad(ids[:2], d, 5), lambda: embedding_grad(ids, d.double(), 5), lambda: embedding_grad(ids, d, 0),
                lambda: embedding_grad(ids, d, 2 ** 31 - 1), lambda: embedding_grad(ids, d, 5, dtype=torch.bfloat16), lambda: embedding_grad(ids, torch.randn(3, 0), 5)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", DEVICES)
def test_padding_tokens_count_as_torch_counts_them(device):
    table, ids = torch.randn(20, 16, device=device, requires_grad=True), torch.tensor([3, 19, 7, 19], device=device)
    dout = torch.randn(4, 16, device=device)
    for pad in (19, -1):
        (a,) = torch.autograd.grad(embedding(ids, table, padding_idx=pad), table, dout)
        (b,) = torch.autograd.grad(torch.nn.functional.embedding(ids, table, pad), table, dout)
        assert torch.equal(a, b) and torch.equal(a, embedding_grad(ids, dout, 20, padding_idx=pad)) and not a[19].any()
    for pad in (20, -21):
        for call in (lambda: embedding(ids, table, padding_idx=pad), lambda: embedding_grad(ids, dout, 20, padding_idx=pad)):
            with pytest.raises(ValueError):
                call()


@pytest.mark.skipif(not nv.lib_path().exists(), reason="no kernel library here")
def test_sizes_of_workspaces_are_not_kept_for_ever():
    """Batches of other lengths every step; pairs of ids twice and two partial sums a tile, of 32 pairs at least, are what a workspace holds."""
    for T in range(1, 1000):
        n = ew._embedding_work(T, 40)
        assert 2 * 8 * T + 2 * 4 * 40 * -(-T // 32) <= n < 2 * (8 * T + 16) + 2 * 4 * 40 * -(-T // 32) + 1
    assert ew._embedding_work.cache_info().currsize <= 128 and ew._embedding_work(0, 40) >= 16


@gpu
@pytest.mark.parametrize("dtype", DT)
def test_embeddings_of_the_c_interface(dtype):
    """What a C caller has had: rows without the table's number of rows, sums that are added to an fp32 table."""
    dt, T, D = DT[dtype], 300, 72
    table, pos, ids = torch.randn(50, D, device="cuda").to(dt), torch.randn(100, D, device="cuda").to(dt), torch.randint(0, 50, (T,), device="cuda")
    out, vp, i64, i32, f32 = torch.empty(T, D, dtype=dt, device="cuda"), lpm.vp, lpm.i64, lpm.i32, lpm.f32
    fwd, bwd = nv.proto("b200_embedding_fwd", [vp, vp, vp, vp, i64, i32, i32, f32, i32, vp]), nv.proto("b200_embedding_bwd", [vp, vp, vp, i64, i32, f32, i32, vp])
    for p in (None, pos):
        assert fwd(ids.data_ptr(), table.data_ptr(), nv.ptr(p), out.data_ptr(), T, D, 100, 1.0, nv.dtype_code(dt), nv.stream()) == 0
        assert torch.equal(out, embedding(ids.view(3, 100), table, p).view(T, D))
    start, dout = torch.randn(50, D, device="cuda"), torch.randn(T, D, device="cuda").to(dt)
    got, (want, size, n) = start.clone(), exact_embedding(ids, dout.cpu(), 50, 1.5, -1)
    assert bwd(ids.data_ptr(), dout.data_ptr(), got.data_ptr(), T, D, 1.5, nv.dtype_code(dt), nv.stream()) == 0
    want, size = want + start.cpu().double(), size + start.cpu().double().abs()
    assert ((got.cpu().double() - want).abs() <= (n + 2) * 2.0 ** -24 * size).all()          # n products and sums in 32 bits


@gpu
def test_embedding_gradient_has_no_derivative():
    """A graph of the gradient may be asked for; what is refused is to go through it."""
    table, f = torch.randn(20, 16, device="cuda", requires_grad=True), torch.randn(4, 16, device="cuda", requires_grad=True)
    ids = torch.tensor([3, 19, 7, 19], device="cuda")
    (plain,) = torch.autograd.grad((embedding(ids, table) * f).sum(), table)
    (g,) = torch.autograd.grad((embedding(ids, table) * f).sum(), table, create_graph=True)
    assert torch.equal(g, plain)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_what_embeddings_refuse():
    table, ids = torch.randn(20, 16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        embedding(ids.to("meta"), table)
    with pytest.raises(ValueError):
        embedding(ids, table, torch.randn(4, 16, device="meta"))
    with pytest.raises(ValueError):
        embedding(ids, table, torch.randn(3, 16))
    for dt in (torch.float32, torch.bool, torch.int16):
        with pytest.raises(TypeError):
            embedding(ids.to(dt), table)


def test_sizes_that_32_bits_do_not_count_are_refused():
    """On a device without memory: nothing but the check runs."""
    row, t = torch.empty(1, 2 ** 32 + 5, dtype=torch.bfloat16, device="meta"), torch.empty(1, dtype=torch.int64, device="meta")
    for bad in (lambda: token_logprobs(row, t), lambda: pack8(row), lambda: swiglu8(row[:, 1:]),
                lambda: linear_token_logprobs(row[:, :8], torch.empty(2 ** 31, 8, dtype=torch.bfloat16, device="meta"), t),
                lambda: linear_token_logprobs(torch.empty(2 ** 31, 8, device="meta"), torch.empty(9, 8, device="meta"), t.expand(2 ** 31))):
        with pytest.raises(ValueError):
            bad()


@gpu
def test_log_probabilities_of_one_row_and_of_rows_upon_one_another():
    """A single row may have any stride, and rows may share memory."""
    w = torch.randn(100, 64, device="cuda").bfloat16()
    one = torch.randn(1, 67, device="cuda").bfloat16()[:, :64]
    same = torch.randn(64, device="cuda").bfloat16().expand(5, 64)
    over = torch.randn(200, device="cuda").bfloat16().as_strided((5, 64), (8, 1))
    aside = torch.randn(1, 80, device="cuda").bfloat16()[:, 3:67]
    for x in (one, same, over, aside):
        t = torch.arange(x.shape[0], device="cuda")
        plain = x.clone(memory_format=torch.contiguous_format)
        a, b = x.detach().requires_grad_(True), plain.detach().requires_grad_(True)
        la, lb = linear_token_logprobs(a, w, t).logprob, linear_token_logprobs(b, w, t).logprob
        assert torch.equal(la, lb) and torch.equal(linear_token_logprobs(x, w, t).logprob, lb)
        g = torch.randn_like(la)
        assert torch.equal(torch.autograd.grad(la, a, g)[0], torch.autograd.grad(lb, b, g)[0])
    with pytest.raises(ValueError):
        linear_token_logprobs(plain, w[0].expand(100, 64), t)


@gpu
@pytest.mark.parametrize("T", [100000, 70000])
def test_embedding_gradient_of_many_tokens(T):
    """Tiles of more than 32 pairs, a token in most of them, tokens of three digits."""
    V, D = 200000, 16
    ids = torch.randint(0, V, (T,), device="cuda")
    ids[torch.rand(T, device="cuda") < 0.7] = 123456
    dout = torch.randn(T, D, device="cuda")
    got = embedding_grad(ids, dout, V)
    want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, ids, dout.double())
    size = torch.zeros_like(want).index_add_(0, ids, dout.double().abs())
    n = torch.bincount(ids, minlength=V)[:, None]
    assert ((got.double() - want).abs() <= (n + 2).double().clamp_max(3000) * 2.0 ** -24 * size).all()
    assert torch.equal(got, embedding_grad(ids, dout, V))


# ------------------------------------------------------------------------------------------------ 8 bits
def exact_pack(x, top):
    """The value that each of x [rows, D] has in 8 bits, block by block in whole Python numbers and fractions."""
    from fractions import Fraction
    out = torch.empty(x.shape, dtype=torch.float64)
    for i, row in enumerate(x.double().tolist()):
        for a in range(0, len(row), 32):
            block = row[a:a + 32]
            m = max([abs(Fraction(v)) for v in block if math.isfinite(v)], default=Fraction(0))
            e = -127
            while e < top and m >= Fraction(255, 2) * Fraction(2) ** e:
                e += 1
            for j, v in enumerate(block):
                if not math.isfinite(v):
                    out[i, a + j] = float("nan")
                else:
                    out[i, a + j] = float(max(-127, min(127, round(Fraction(v) / Fraction(2) ** e))) * Fraction(2) ** e)
    return out


def edges(dtype):
    """Blocks at the edges of the rule: largest magnitudes next to 127.5 steps, ties, zeros, smallest and largest numbers, what is not finite."""
    f = torch.finfo(dtype)
    rows = []
    for m in (127.0, 127.25, 127.5, 128.0, 255.0, 1.0, 0.75):
        for e in (0, -3, -14, 5):
            rows.append(torch.tensor([m, -m] + [m * k / 127 for k in range(-15, 15)]) * 2.0 ** e)
    rows.append(torch.arange(32) + 0.5)                                                       # ties of whole numbers
    rows.append(torch.cat([torch.tensor([127.0]), torch.arange(31) + 0.5]))
    rows.append(torch.zeros(32))
    rows.append(torch.tensor([f.max, -f.max, f.max / 2, f.max / 200, 1.0, 0.0] + [f.max / 127 * 63.5] * 26))
    rows.append(torch.tensor([f.smallest_normal, -f.smallest_normal / 2, f.smallest_normal * f.eps] + [0.0] * 29))
    rows.append(torch.tensor([INF, -INF, float("nan"), 1.0, -0.3] + [0.01] * 27))
    rows.append(torch.tensor([INF] * 32))
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
def test_8_bits_at_the_edges(dtype, device):
    x = edges(DT[dtype])
    want = exact_pack(x, 9 if dtype == "fp16" else 121)
    p = pack8(x.to(device))
    got = unpack8(p).cpu()
    assert torch.equal(got.double().nan_to_num(nan=7e37), want.to(DT[dtype]).double().nan_to_num(nan=7e37))
    assert torch.equal(unpack8(p, torch.float32).cpu().nan_to_num(nan=7e37), want.float().nan_to_num(nan=7e37))
    finite = x.double().isfinite()
    assert torch.equal(got.isfinite(), finite)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (2, 31), (5, 32), (4, 33), (3, 77), (2, 100), (7, 1000), (9, 1100), (33, 2048)])
def test_8_bits_and_back(rows, D, dtype, device):
    dt = DT[dtype]
    x, a = (torch.randn(rows, D) * torch.rand(rows, 1) * 20).to(dt), torch.randn(rows, D).to(dt)
    for add in (None, a):
        s = x if add is None else x + add
        want = exact_pack(s, 9 if dtype == "fp16" else 121)
        p = pack8(x.to(device), None if add is None else add.to(device))
        assert p.shape == (rows, D) and p.nbytes() == rows * -(-D // 32) * 33
        got = unpack8(p)
        assert got.dtype == dt and torch.equal(got.cpu().double(), want)
        block = torch.nn.functional.pad(s.double().abs(), (0, -D % 32)).view(rows, -1, 32).amax(2).repeat_interleave(32, 1)[:, :D]
        assert ((got.cpu().double() - s.double()).abs() <= block / 127).all()
    wide = torch.randn(rows, D + 9).to(dt).to(device)
    for lo in (0, 1, 8):
        assert torch.equal(unpack8(pack8(wide[:, lo:lo + D])), unpack8(pack8(wide[:, lo:lo + D].clone())))
        assert torch.equal(unpack8(pack8(x.to(device), wide[:, lo:lo + D])), unpack8(pack8(x.to(device), wide[:, lo:lo + D].clone())))


@pytest.mark.parametrize("device", DEVICES)
def test_8_bits_of_other_shapes(device):
    x = torch.randn(2, 3, 50, device=device)
    assert torch.equal(unpack8(pack8(x)), unpack8(pack8(x.view(6, 50))).view(2, 3, 50))
    t = torch.randn(50, 6, device=device).t()
    assert torch.equal(unpack8(pack8(t)), unpack8(pack8(t.contiguous())))
    assert unpack8(pack8(x[:0])).shape == (0, 3, 50) and unpack8(pack8(x[0, 0])).shape == (50,)
    same = torch.randn(1, 50, device=device).expand(4, 50)
    assert torch.equal(unpack8(pack8(same)), unpack8(pack8(same.clone())))


def test_what_8_bits_refuse():
    x = torch.randn(2, 40)
    p = pack8(x)
    for bad in (lambda: pack8(x.double()), lambda: pack8(x, x[:1]), lambda: pack8(x, x.half()), lambda: pack8(torch.randn(2, 0)), lambda: unpack8(p, torch.float64),
                lambda: unpack8(p._replace(shape=(2, 70))), lambda: unpack8(p._replace(shape=(3, 40))), lambda: unpack8(p._replace(e=p.e[:1])),
                lambda: unpack8(p._replace(q=p.q.to(torch.int16))), lambda: swiglu8(torch.randn(2, 5)), lambda: swiglu8(torch.randn(2, 4).double())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,F", [(1, 1), (3, 31), (2, 32), (5, 36), (4, 100), (7, 1000), (33, 512)])
def test_gated_unit_that_keeps_8_bits(rows, F, dtype, device):
    dt = DT[dtype]
    gu, dy = (torch.randn(rows, 2 * F) * 2).to(dt), torch.randn(rows, F).to(dt)
    gu[0, 0] = -90.0                                                              # e^-g is beyond the numbers of fp32
    x = gu.to(device).requires_grad_(True)
    y = swiglu8(x)
    (got,) = torch.autograd.grad(y, x, dy.to(device))
    g, u = gu[:, :F].double(), gu[:, F:].double()
    half, least = half_step(dt)
    # the exponential of g has the error of its argument, 3 (2^-24) |g|, and 2^-22 of its own; quotient and products round four times
    slack = 2.0 ** -20 + 2.0 ** -22 * g.abs()
    want = g * torch.sigmoid(g) * u
    assert ((y.detach().cpu().double() - want).abs() <= (half + slack) * want.abs() + least + 1e-36).all()
    top = 9 if dtype == "fp16" else 121
    g, u, d = exact_pack(gu[:, :F], top), exact_pack(gu[:, F:], top), dy.double()
    s = torch.sigmoid(g)
    dg, du = d * u * s * (1 + g * (1 - s)), d * g * s
    size = torch.cat([(d * u * s).abs() * (1 + (g * (1 - s)).abs()), du.abs()], 1)
    err = (got.cpu().double() - torch.cat([dg, du], 1)).abs()
    assert (err <= half * torch.cat([dg, du], 1).abs() + torch.cat([slack, slack], 1) * size + least + 1e-36).all()
    assert torch.equal(swiglu8(gu.to(device)), y.detach())                        # without a gradient: the same result, nothing kept


@pytest.mark.parametrize("device", DEVICES)
def test_gated_unit_of_strided_rows(device):
    wide = torch.randn(6, 90, device=device)
    a, b = wide[:, 3:3 + 68].detach().requires_grad_(True), wide[:, 3:3 + 68].detach().clone().requires_grad_(True)
    ya, yb = swiglu8(a), swiglu8(b)
    assert torch.equal(ya, yb)
    d = torch.randn(6, 1, device=device).expand(6, 34)
    assert torch.equal(torch.autograd.grad(ya, a, d)[0], torch.autograd.grad(yb, b, d.clone())[0])


class Layer(torch.nn.Module):
    """(delta, residual) -> (delta, residual) of a norm, a linear layer and dropout."""

    def __init__(self, D, p=0.0):
        super().__init__()
        self.w, self.p = torch.nn.Parameter(torch.randn(D, D) / D ** 0.5), p

    def forward(self, delta, residual, times=1.0):
        x = delta if residual is None else delta + residual
        y = torch.tanh(x @ self.w.t()) * times
        return ew.dropout(y, self.p, True), x


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_checkpoints_in_8_bits(p, device):
    """The result is a plain call's; gradients are those of the layer at the kept sum, under the same dropout mask, and leave the streams of numbers as they were."""
    D = 64
    layer = Layer(D, p).to(device)
    delta, residual = (torch.randn(5, D, device=device).requires_grad_(True) for _ in range(2))
    ew.manual_seed(3)
    torch.manual_seed(3)
    a = checkpoint8(layer, delta, residual, 0.5)
    after = dict(ew._seed_state), torch.rand(1)
    ew.manual_seed(3)
    torch.manual_seed(3)
    b = layer(delta, residual, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and dict(ew._seed_state) == after[0]
    ga, gb = torch.randn(5, D, device=device), torch.randn(5, D, device=device)
    state = dict(ew._seed_state), torch.get_rng_state()
    torch.autograd.backward(a, [ga, gb])
    assert dict(ew._seed_state) == state[0] and torch.equal(torch.get_rng_state(), state[1])
    got = delta.grad.clone(), residual.grad.clone(), layer.w.grad.clone()
    kept = unpack8(pack8(delta, residual)).requires_grad_(True)
    layer.w.grad = None
    ew.manual_seed(3)
    torch.manual_seed(3)
    torch.autograd.backward(layer(kept, None, 0.5), [ga, gb])
    assert torch.equal(got[0], kept.grad) and torch.equal(got[1], kept.grad) and torch.equal(got[2], layer.w.grad)


def test_checkpoints_take_layers_that_return_tuples_and_keep_autocast():
    x = torch.randn(3, 32, requires_grad=True)
    with pytest.raises(TypeError):
        checkpoint8(lambda d, r: d * 2, x, None)
    layer, seen = Layer(32), []

    def watched(d, r):
        y = layer(d, r)
        seen.append(y[0].dtype)
        return y
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = checkpoint8(watched, x, None)
    y[0].float().sum().backward()
    assert seen == [torch.bfloat16, torch.bfloat16] and x.grad is not None


@pytest.mark.parametrize("name", ["dropout", "bernoulli", "rand_like", "attention with dropout"])
def test_checkpoints_in_a_capture_refuse_torchs_random_numbers(name, monkeypatch):
    """In the forward and, where the forward ran before the capture, in the backward pass; a layer that draws nothing, or from another device's stream, is taken."""
    F = torch.nn.functional
    draw = {"dropout": lambda x: F.dropout(x, 0.5), "bernoulli": lambda x: x * torch.bernoulli(torch.full_like(x, 0.5)), "rand_like": lambda x: x * torch.rand_like(x),
            "attention with dropout": lambda x: F.scaled_dot_product_attention(x[None], x[None], x[None], dropout_p=0.5)[0]}[name]
    x = torch.randn(4, 32, requires_grad=True)
    still = lambda d, r: (F.scaled_dot_product_attention(d[None], d[None], d[None])[0] + F.dropout(d, 0.5, training=False), d)  # noqa: E731
    y = checkpoint8(lambda d, r: (draw(d), d), x, None)[0]
    monkeypatch.setattr(act8, "_capturing", lambda t: True)
    with pytest.raises(RuntimeError, match="captured"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="captured"):
        checkpoint8(lambda d, r: (draw(d), d), x, None)
    checkpoint8(still, x, None)[0].sum().backward()
    assert torch.isfinite(x.grad).all()
    monkeypatch.setattr(act8, "_no_draws", lambda t: act8._NoDraws(torch.device("meta")))
    checkpoint8(lambda d, r: (draw(d), d), x, None)[0].sum().backward()


def test_which_operators_draw():
    ops, x = torch.ops.aten, torch.zeros(2)
    for op, args, kw, draws in ((ops.native_dropout.default, (x, 0.5, True), {}, True), (ops.uniform_.default, (x,), {}, True),
                                (ops._scaled_dot_product_flash_attention.default, (x, x, x), {}, False), (ops._scaled_dot_product_flash_attention.default, (x, x, x, 0.1), {}, True),
                                (ops._scaled_dot_product_flash_attention.default, (x, x, x), {"dropout_p": 0.1}, True),
                                (ops._cudnn_rnn.default, (x, [x], 4, None, x, None, 2, 4, 0, 1, False, 0.0, True, False, [], None), {}, False)):
        assert torch.Tag.nondeterministic_seeded in op.tags and act8._NoDraws._drew(op, args, kw) == draws


@gpu
def test_captured_checkpoints():
    """A captured step gives the gradients of an eager one, whose dropout is the package's; one that draws from torch's generator is an error, and the capture after it is
    as any other."""
    D = 64
    layer, ga = Layer(D, 0.5).cuda(), torch.randn(5, D, device="cuda")
    x = torch.randn(5, D, device="cuda")

    def step(x):
        ew.manual_seed(3)
        leaf = x.detach().requires_grad_(True)
        y = checkpoint8(layer, leaf, None)[0]
        y.backward(ga)
        return y.detach(), leaf.grad
    want = [t.clone() for t in step(x)]
    dw = layer.w.grad.clone()
    layer.w.grad = None
    y = checkpoint8(lambda d, r: (torch.nn.functional.dropout(d, 0.5), d), x.requires_grad_(True), None)[0]     # eagerly: under the same mask
    y.sum().backward()
    kept = unpack8(pack8(x.detach()))
    assert torch.equal(x.grad != 0, y.detach() != 0) and torch.equal(x.grad[x.grad != 0], torch.full_like(kept, 2.0)[x.grad != 0])
    x = x.detach()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            checkpoint8(lambda d, r: (torch.nn.functional.dropout(d, 0.5), d), x.detach().requires_grad_(True), None)
    graph = torch.cuda.CUDAGraph()
    layer.w.grad = torch.zeros_like(layer.w)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step(x)
    for _ in range(2):
        layer.w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(layer.w.grad, dw)


def test_second_derivatives_are_refused():
    x = torch.randn(3, 64, requires_grad=True)
    for f in (lambda: token_logprobs(x, torch.tensor([0, 1, 2])).logprob, lambda: linear_token_logprobs(x, torch.randn(9, 64), torch.tensor([0, 1, 2])).logprob,
              lambda: swiglu8(x), lambda: checkpoint8(Layer(64), x, None)[0]):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(f().sum(), x, create_graph=True)


def test_checkpoints_behind_a_frozen_input_and_without_gradients():
    layer = Layer(32)
    x = torch.randn(3, 32)
    y, r = checkpoint8(layer, x, None)
    assert torch.equal(y.detach(), layer(x, None)[0].detach())
    y, r = checkpoint8(Layer(32), y, r)
    y.sum().backward()                                                 # the stream gets no gradient of its own
    assert layer.w.grad is not None and torch.isfinite(layer.w.grad).all()
    with torch.no_grad():
        assert not checkpoint8(layer, x, None)[0].requires_grad


# ------------------------------------------------------------------------------------------------ how they are called
def _step(ids, tokens, table, layers, head, g, h):
    """A training step on given tokens: embedding, checkpointed layers with gated units that keep 8 bits, log probabilities and entropies."""
    delta, residual = embedding(ids, table, scale=2.0, padding_idx=0), None
    for wi, wo in layers:
        def layer(d, r, wi=wi, wo=wo):
            x = d if r is None else d + r
            return ew_linear(swiglu8(ew_linear(x, wi)), wo), x
        delta, residual = checkpoint8(layer, delta, residual)
    r = linear_token_logprobs(delta + residual, head, tokens, entropy=True)
    return (r.logprob * g).sum() + (r.entropy * h).sum()


def ew_linear(x, w):
    from llm_in_practise_b200.ops.functional import linear
    return linear(x, w)


@gpu
def test_a_step_of_all_of_them():
    """Gradients of a whole step against the same step in 64 bits without 8 bits: what they cost is seen, and small; a second run gives the same bits."""
    torch.manual_seed(5)
    V, D, F, T = 1000, 128, 256, 96
    ps = [torch.randn(V, D) * 0.5] + [t for _ in range(2) for t in (torch.randn(2 * F, D) / D ** 0.5, torch.randn(D, F) / F ** 0.5)] + [torch.randn(V, D) * 0.2]
    ps = [p.bfloat16().cuda().requires_grad_(True) for p in ps]
    ids, tokens = torch.randint(0, V, (T,), device="cuda"), torch.randint(0, V, (T,), device="cuda")
    tokens[:10] = -100
    g, h = torch.randn(T, device="cuda"), 0.1 * torch.randn(T, device="cuda")
    run = lambda: torch.autograd.grad(_step(ids, tokens, ps[0], [ps[1:3], ps[3:5]], ps[5], g, h), [ps[0], ps[5]])  # noqa: E731
    a, b = run(), run()
    assert all(torch.equal(x, y) for x, y in zip(a, b))

    def plain():
        q = [p.detach().double().requires_grad_(True) for p in ps]
        x = q[0][ids] * 2.0
        delta, res = x, None
        for i in (1, 3):
            s = delta if res is None else delta + res
            gu = s @ q[i].t()
            delta, res = (torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]) @ q[i + 1].t(), s
        lp = torch.log_softmax((delta + res) @ q[5].t(), 1)
        ok = tokens >= 0
        loss = ((lp.gather(1, tokens.clamp_min(0)[:, None])[:, 0] * g)[ok]).sum() - ((lp.exp() * lp).sum(1) * h)[ok].sum()
        return torch.autograd.grad(loss, [q[0], q[5]])
    for x, y, pad in zip(a, plain(), (True, False)):
        if pad:
            y = y.clone()
            y[0] = 0
        assert float((x.double() - y).norm() / y.norm()) < 0.05


@gpu
def test_other_streams_and_replayed_graphs():
    """Calls on a stream of their own, captured and replayed with other values in the same tensors, two captures of the same calls."""
    V, D, T = 5003, 72, 300
    l, ids = torch.randn(T, V, device="cuda").bfloat16(), torch.randint(0, V, (T,), device="cuda")
    x, w, dout = torch.randn(T, D, device="cuda").bfloat16(), torch.randn(V, D, device="cuda").bfloat16(), torch.randn(T, D, device="cuda")
    gu = torch.randn(T, 2 * D, device="cuda").bfloat16()

    def calls():
        with torch.no_grad():
            r = token_logprobs(l, ids, top=7, entropy=True, rank=True)
            s = linear_token_logprobs(x, w, ids, entropy=True)
            return [*r, s.logprob, s.entropy, embedding_grad(ids, dout, V, 2.0, 5), unpack8(pack8(gu)), swiglu8(gu)]
    calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = calls()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(on_side, calls()))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = calls()
        graphs.append((g, out))
    for i in range(3):
        l.copy_(torch.randn(T, V, device="cuda")), ids.copy_(torch.randint(0, V, (T,), device="cuda")), x.copy_(torch.randn(T, D, device="cuda"))
        dout.copy_(torch.randn(T, D, device="cuda")), gu.copy_(torch.randn(T, 2 * D, device="cuda"))
        for g, out in graphs:
            g.replay()
        want = calls()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
def test_two_calls_at_once():
    l, ids = torch.randn(200, 30000, device="cuda"), torch.randint(0, 30000, (200,), device="cuda")
    dout = torch.randn(200, 512, device="cuda")
    want = token_logprobs(l, ids, top=20, rank=True), embedding_grad(ids, dout, 30000)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((token_logprobs(l, ids, top=20, rank=True), embedding_grad(ids, dout, 30000)))
    torch.cuda.synchronize()
    for a, b in got:
        assert all(torch.equal(x, y) for x, y in zip(a[:1] + a[2:], want[0][:1] + want[0][2:])) and torch.equal(b, want[1])
