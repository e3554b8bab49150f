"""Short rows of log probabilities with alternatives, a CTA of 64 threads each: which vectors of a row its threads note and read again, and what comes out for rows of
fewer vectors than threads, with masks that leave few values or none."""
import re
from pathlib import Path

import pytest
import torch

from llm_in_practise_b200.ops.logprobs import token_logprobs

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")
SOURCE = Path(__file__).resolve().parent.parent / "csrc" / "logprobs.cu"


def noted(nvec, rising, guarded):
    """The group that each of 64 threads notes of a row of ``nvec`` vectors, by the walk of lp_rows_kernel: four vectors 64 apart while all of a warp's are inside, then what
    is left, where lanes without a vector see minus infinities. ``rising``: each group is larger than those before, else none is larger than the first."""
    out = []
    for thread in range(64):
        lane, i, group, most = thread % 32, thread, -1, -INF

        def note(i):
            nonlocal group, most
            m = float(i + 1 if rising else -i) if i < nvec else -INF
            if (i < nvec or not guarded) and (m > most or group < 0):
                group, most = i, m
        while i - lane + 31 + 3 * 64 < nvec:
            note(i)
            i += 256
        if i - lane < nvec:
            note(i)
        out.append(group)
    return out


def test_threads_note_vectors_of_their_row_alone():
    """The k threads chosen read the group that they noted again: no index may lie behind the row's last vector, whatever the row holds. The kernel's own condition is
    read from its source."""
    code = " ".join(line.split("//")[0] for line in SOURCE.read_text().splitlines())
    found = re.findall(r"if \(([^{};]*group < 0[^{};]*)\) \{ most = m; group = i; \}", code)
    assert len(found) == 1
    guarded = found[0].replace(" ", "").startswith("i<at.nvec&&(")
    for nvec in [*range(0, 600), 1023, 1024, 1025, 2047, 2048]:
        for rising in (False, True):
            groups = noted(nvec, rising, guarded)
            assert all(g < nvec for g in groups), nvec
            # every thread that has a vector notes one: as many threads as there are vectors, up to all
            assert sum(g >= 0 for g in groups) == min(nvec, 64)
            for x in range(4):                               # what is read again: the group's vectors, the first one in the place of those behind the row
                assert all((g + x * 64 if g + x * 64 < nvec else g) < nvec for g in groups if g >= 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", [9, 16, 31, 33, 40, 64, 65, 100, 128, 160, 250, 255, 256, 257, 300, 383, 511, 512, 520, 1001])
def test_alternatives_of_short_rows(V, dtype, device):
    """Rows that are whole, masked but for some, for one and for none, ties; at odd addresses; the last row ends where the tensor does."""
    r = torch.Generator().manual_seed(V)
    l = torch.randn(24, V, generator=r) * 3
    for i in range(24):
        kind = i % 6
        if kind == 1:
            l[i, torch.rand(V, generator=r) < 0.95] = -INF
        elif kind == 2:
            l[i, 1 + torch.arange(V - 1)] = -INF
        elif kind == 3:
            l[i, :V - 1] = -INF                              # the last token alone
        elif kind == 4:
            l[i] = -INF
        elif kind == 5:
            l[i] = torch.randint(-1, 2, (V,), generator=r).float()
    l = l.to(DT[dtype]).to(device)
    order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1]
    lp = torch.log_softmax(l.double(), 1)
    tokens = torch.randint(0, V, (24,), generator=r).to(device)
    for top in sorted({1, 2, 5, min(20, V), min(32, V)}):
        for more in ({}, {"entropy": True, "rank": True}):
            got = token_logprobs(l, tokens, top=top, **more)
            assert torch.equal(got.top_ids, order[:, :top])
            want = lp.gather(1, got.top_ids)
            seen = got.top_logprobs.double()
            # the sum of V weights (2^-22 and 72 steps each, one rounding a value that a thread adds and where they meet), the difference and its logarithm
            bound = 2.0 ** -22 + (72 + V / 64 + 64) * 2.0 ** -24 + want.abs().clamp_max(1e4) * 2.0 ** -22 + 2.0 ** -22
            same = (want == -INF) & (seen == -INF) | want.isnan() & seen.isnan()
            assert (((seen - want).abs() <= bound) | same).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,V", [(6, 1), (6, 5), (6, 32), (6, 33), (6, 1001), (330, 20000), (6, 50257), (2, 151936)])
def test_nan_comes_before_all_others(rows, V, dtype, device):
    """A NaN at token 0, in a few places, at the end, and a row of NaN alone, up to as many alternatives as there are tokens: in rows by 64 threads, by 256 and by clusters of
    CTAs. Every log probability is NaN."""
    if device == "cpu" and rows * V > 400000:
        pytest.skip("the kernels' sizes")
    r = torch.Generator().manual_seed(V)
    nan = float("nan")
    l = torch.randn(rows, V, generator=r)
    for i in range(rows):
        kind = (i + 4 * (rows == 2)) % 6
        if kind == 0:
            l[i, 0] = nan
        elif kind == 1:
            l[i, V - 1] = nan
        elif kind == 2:
            l[i, ::max(1, V // 3)] = nan
        elif kind == 3:
            l[i] = -INF
            l[i, 0] = nan
        elif kind == 4:
            l[i] = nan
        else:
            l[i, 0] = -nan
    l = l.to(DT[dtype]).to(device)
    x = l.float()
    order = torch.sort(torch.where(x.isnan(), torch.full_like(x, nan), x), dim=1, descending=True, stable=True)[1]        # NaN above all, the lowest id first
    for top in sorted({1, min(2, V), min(5, V), min(32, V)}):
        got = token_logprobs(l, top=top)
        assert torch.equal(got.top_ids, order[:, :top]) and got.top_logprobs.isnan().all()
