"""The operators of a shared serving step where the framework calls them: generation and the engine with rules on the logits, decode steps of
sequences that share a cached prefix, block tables and maps of the ragged step built on the device."""
import gc
import weakref

import pytest
import torch
from fastapi.testclient import TestClient

from llm_in_practise_b200.data.tokenizers import ByteTokenizer
from llm_in_practise_b200.inference import GenerationConfig, Generator
from llm_in_practise_b200.inference.generate import MAX_GROUPS, KVCache, LogitRules, PagedKVCache, group_plan, set_group_plan
from llm_in_practise_b200.inference.ragged import RaggedGenerator, make_pieces
from llm_in_practise_b200.models.qwen3 import Qwen3Config, Qwen3ForCausalLM
from llm_in_practise_b200.ops import _native as nv
from llm_in_practise_b200.serve import EngineArgs, LLMEngine
from llm_in_practise_b200.serve.engine import Request
from llm_in_practise_b200.serve.openai_server import build_app
from test_serving_step_ops import entries  # noqa: F401

gpu = pytest.mark.gpu


def qwen(device="cpu", dtype=torch.float32, D=16, H=4, Hkv=2, layers=2, vocab=300):
    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=vocab, hidden_size=64 if D == 16 else 256, intermediate_size=128, num_hidden_layers=layers, num_attention_heads=H,
                      num_key_value_heads=Hkv, head_dim=D, max_position_embeddings=1024)
    return Qwen3ForCausalLM(cfg, dtype=dtype, device=device, init_std=0.1)


@pytest.fixture(scope="module")
def model():
    return qwen()


RULED = [dict(presence_penalty=1.5, frequency_penalty=0.4), dict(logit_bias={5: 4.0, 17: -100.0}, repetition_penalty=1.3),
         dict(allowed_token_ids=list(range(40, 60)), frequency_penalty=0.7), dict(frequency_penalty=-0.5), dict()]


def by_hand(model, prompt, new, kw):
    """Greedy continuation with the rules applied in 64 bits to the logits of whole passes over the sequence."""
    g, seq = Generator(model, max_len=96), list(prompt)
    for _ in range(new):
        cache = __import__("llm_in_practise_b200.inference.generate", fromlist=["KVCache"]).KVCache(2, 1, 2, 96, 16, torch.float32, "cpu")
        y = g._prefill(torch.tensor([seq]), cache)[0].double()
        said = seq[len(prompt):]
        r = kw.get("repetition_penalty", 1.0)
        for t in set(seq):
            y[t] = y[t] * r if y[t] < 0 else y[t] / r
        for t in set(said):
            y[t] -= kw.get("frequency_penalty", 0.0) * said.count(t) + kw.get("presence_penalty", 0.0)
        for t, v in (kw.get("logit_bias") or {}).items():
            y[t] += v
        if "allowed_token_ids" in kw:
            keep = torch.zeros_like(y, dtype=torch.bool)
            keep[kw["allowed_token_ids"]] = True
            y[~keep] = float("-inf")
        seq.append(int(y.argmax()))
    return seq[len(prompt):]


def test_generation_and_engine_follow_the_rules(model):
    """Requests with different rules, and one without, in one batch: each gets what it gets alone, and what the rules give by hand."""
    torch.manual_seed(1)
    prompts = [torch.randint(0, 300, (n,)).tolist() for n in (5, 9, 3, 12, 7)]
    want = [by_hand(model, p, 8, kw) for p, kw in zip(prompts, RULED)]
    g = Generator(model, max_len=96)
    for p, kw, w in zip(prompts, RULED, want):
        assert g.generate(torch.tensor([p]), max_new_tokens=8, do_sample=False, **kw)[0, len(p):].tolist() == w
    for bs in (0, 16):
        eng = LLMEngine(model, None, EngineArgs(max_num_seqs=2, max_model_len=64, block_size=bs))          # rows are used again
        reqs = [eng.submit(p, GenerationConfig(max_new_tokens=8, **kw)) for p, kw in zip(prompts, RULED)]
        while not all(r.done.is_set() for r in reqs):
            eng.step()
        assert [r.output_ids for r in reqs] == want


def test_a_grammar_is_asked_before_every_token(model):
    """prefix_allowed_tokens_fn: called with the sequence's name and its tokens so far; with allowed_token_ids both hold."""
    calls = []

    def fn(name, toks):
        calls.append((name, len(toks)))
        return [10 + len(toks) % 3, 50, 10 ** 6]

    prompt = [1, 2, 3, 4]
    out = Generator(model, max_len=64).generate(torch.tensor([prompt]), max_new_tokens=5, prefix_allowed_tokens_fn=fn, allowed_token_ids=[10, 11, 12])
    assert out[0, 4:].tolist() == [10 + n % 3 for n in range(4, 9)] and calls == [(0, n) for n in range(4, 9)]
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=2, max_model_len=64))
    calls.clear()
    r = eng.generate([[7], prompt], GenerationConfig(max_new_tokens=3, prefix_allowed_tokens_fn=fn, do_sample=True, temperature=1.0))
    assert all(t in (10 + n % 3, 50) for x in r for n, t in enumerate(x.output_ids, len(x.prompt_ids)))
    assert {c[0] for c in calls} == {x.rid for x in r}


def test_a_grammar_that_fails_ends_its_own_request(model):
    """An exception of one request's prefix_allowed_tokens_fn is that request's error; what runs beside it gets what it gets alone."""
    def fn(name, toks):
        if len(toks) == 5:
            raise KeyError("no such state")
        return [20, 21]

    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=3, max_model_len=64))
    cfgs = [GenerationConfig(max_new_tokens=6, prefix_allowed_tokens_fn=fn), GenerationConfig(max_new_tokens=6, presence_penalty=0.5), GenerationConfig(max_new_tokens=6)]
    reqs = [eng.submit([1, 2, 3], c) for c in cfgs]
    while not all(r.done.is_set() for r in reqs):
        eng.step()
    assert reqs[0].finish_reason == "error" and "no such state" in reqs[0].error and len(reqs[0].output_ids) == 2
    for r, c in zip(reqs[1:], cfgs[1:]):
        assert r.error is None and r.output_ids == Generator(model, max_len=64).generate(torch.tensor([[1, 2, 3]]), c)[0, 3:].tolist()


def test_sampling_with_rules(model):
    """Drawn tokens keep to the rules; a row whose rules allow nothing gets token 0 and spoils nobody's draw."""
    torch.manual_seed(2)
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=3, max_model_len=64, seed=3))
    cfgs = [GenerationConfig(max_new_tokens=12, do_sample=True, temperature=5.0, allowed_token_ids=[3, 4, 5]),
            GenerationConfig(max_new_tokens=12, do_sample=True, temperature=1.0, top_k=4, logit_bias={9: 1000.0}),
            GenerationConfig(max_new_tokens=12, do_sample=True, allowed_token_ids=[])]
    reqs = [eng.submit([1, 2, 3], c) for c in cfgs]
    while not all(r.done.is_set() for r in reqs):
        eng.step()
    assert set(reqs[0].output_ids) == {3, 4, 5} and set(reqs[1].output_ids) == {9} and set(reqs[2].output_ids) == {0}


@pytest.mark.parametrize("sample", [False, True])
def test_a_grammar_that_allows_nothing_ends_its_own_request(model, sample):
    """Nothing, nothing of the vocabulary, nothing beside allowed_token_ids: an error of the request's, not a token that its grammar forbids. What runs beside
    it goes on, and generate raises."""
    how = dict(do_sample=sample, temperature=1.0, max_new_tokens=5)
    cfgs = [GenerationConfig(prefix_allowed_tokens_fn=fn, allowed_token_ids=ids, **how) for fn, ids in
            ((lambda name, toks: [20, 21] if len(toks) < 5 else [], None), (lambda name, toks: [300, -1], None), (lambda name, toks: [7], [8]))]
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=4, max_model_len=64))
    reqs = [eng.submit([1, 2, 3], c) for c in cfgs + [GenerationConfig(allowed_token_ids=[4], max_new_tokens=5)]]
    while not all(r.done.is_set() for r in reqs):
        eng.step()
    for r, n in zip(reqs, (2, 0, 0)):
        assert r.finish_reason == "error" and "no token" in r.error and len(r.output_ids) == n and set(r.output_ids) <= {20, 21}
    assert reqs[3].error is None and reqs[3].output_ids == [4] * 5
    for c in cfgs:
        with pytest.raises(ValueError, match="no token"):
            Generator(model, max_len=64).generate(torch.tensor([[1, 2, 3]]), c)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("sample", [False, True])
def test_rows_of_generate_that_are_done_are_not_asked(model, tmp_path, ragged, sample):
    """A row that has ended: its grammar is not called behind its end, and what is drawn for it and thrown away does not join its history. The other rows get what
    they get with a grammar that says the same without an end."""
    if ragged:
        import gorozen_oracle as O
        from test_gorozen import build
        cfg = O.make_config(64, 96, [O.attn_layer(4, 2, 32, 16, 100.0, None, mlp=O.dense())])
        gen = RaggedGenerator(build(tmp_path, cfg, O.random_weights(cfg, seed=15), "cpu", torch.float32), None, 64)
    else:
        gen = Generator(model, max_len=64)
    calls, states = [], []

    def fn(row, toks, strict=True):
        calls.append((row, list(toks)))
        if row == 0 and 20 in toks:
            if strict:
                raise KeyError("no state behind the end")
            return [20, 30]
        return [20] if row == 0 and len(toks) == 5 else [30, 31, 32]

    real = LogitRules.__init__

    def init(self, *a, **kw):
        real(self, *a, **kw)
        states.append(self)
    kw = dict(max_new_tokens=7, eos_token_id=20, pad_token_id=9, do_sample=sample, temperature=1.0, frequency_penalty=0.5)
    prompts = torch.tensor([[1, 2, 3], [4, 5, 6]])
    LogitRules.__init__ = init
    try:
        out = gen.generate(prompts, seed=3, prefix_allowed_tokens_fn=fn, **kw)
    finally:
        LogitRules.__init__ = real
    assert out[0, 5:].tolist() == [20, 9, 9, 9, 9] and [c[1] for c in calls if c[0] == 0] == [out[0, :n].tolist() for n in (3, 4, 5)]
    assert [c[1] for c in calls if c[0] == 1] == [out[1, :n].tolist() for n in range(3, 10)]
    st = states[0].state
    assert st.length.tolist() == [6, 10] and st.tokens[0, :6].tolist() == out[0, :6].tolist() and st.tokens[1, :10].tolist() == out[1].tolist()
    free = gen.generate(prompts, seed=3, prefix_allowed_tokens_fn=lambda row, toks: fn(row, toks, False), **kw)
    assert torch.equal(out, free)


def test_grammars_of_requests_that_ended_are_let_go(model):
    """Finished, failed and aborted requests: their functions and tokens are not kept for the row, and later steps of others do not wait for their ids."""
    class Grammar:
        def __init__(self, fail=False):
            self.fail = fail

        def __call__(self, name, toks):
            if self.fail:
                raise KeyError("failed")
            return [20, 21]

    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=4, max_model_len=64))
    grammars = [Grammar(), Grammar(fail=True), Grammar()]
    refs = [weakref.ref(g) for g in grammars]
    reqs = [eng.submit([1, 2, 3], GenerationConfig(max_new_tokens=n, prefix_allowed_tokens_fn=g)) for g, n in zip(grammars, (3, 3, 40))]
    other = eng.submit([1, 2, 3], GenerationConfig(max_new_tokens=30, presence_penalty=0.5))
    for _ in range(6):
        eng.step()
    assert [r.finish_reason for r in reqs] == ["length", "error", None]
    eng.abort(reqs[2])
    eng.step()
    assert reqs[2].finish_reason == "abort" and not other.done.is_set()
    assert not eng._rules._fn and not eng._rules._tokens
    del grammars, reqs
    gc.collect()
    assert [r() for r in refs] == [None] * 3
    eng.abort(other)
    eng.step()


def test_an_empty_list_of_allowed_tokens(model):
    """generate and the HTTP server refuse it; a request of the engine's ends with an error at its first token."""
    with pytest.raises(ValueError, match="allowed_token_ids"):
        Generator(model, max_len=64).generate(torch.tensor([[1, 2, 3]]), max_new_tokens=3, allowed_token_ids=[])
    eng = LLMEngine(model, ByteTokenizer(), EngineArgs(max_num_seqs=3, max_model_len=64))
    for how in (dict(), dict(do_sample=True, temperature=1.0)):
        r, other = (eng.submit([1, 2, 3], GenerationConfig(max_new_tokens=6, allowed_token_ids=ids, **how)) for ids in ([], [9]))
        while not (r.done.is_set() and other.done.is_set()):
            eng.step()
        assert r.finish_reason == "error" and "allowed_token_ids" in r.error and len(r.output_ids) <= 1
        assert other.error is None and other.output_ids == [9] * 6
    r = eng.submit([1, 2, 3], GenerationConfig(max_new_tokens=6, allowed_token_ids=[], eos_token_id=0))          # an end that is not allowed either
    while not r.done.is_set():
        eng.step()
    assert r.finish_reason == "error"
    c = TestClient(build_app(eng, prompt_style="deepseek"))
    assert c.post("/v1/chat/completions", json={"model": "m", "messages": [{"role": "user", "content": "hi"}], "allowed_token_ids": []}).status_code == 400
    assert c.post("/v1/completions", json={"model": "m", "prompt": "hi", "allowed_token_ids": []}).status_code == 400
    assert eng.num_waiting == 0


def test_rules_that_cannot_hold_are_refused_at_submission(model):
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=2, max_model_len=64))
    for kw in (dict(logit_bias={300: 1.0}), dict(logit_bias={-1: 1.0}), dict(allowed_token_ids=[5, 300]), dict(presence_penalty=float("nan")),
               dict(logit_bias={1: float("inf")}), dict(logit_bias={i: 1.0 for i in range(2048)}), dict(frequency_penalty=1.0, repetition_penalty=0.0)):
        with pytest.raises(ValueError):
            eng.submit([1, 2], GenerationConfig(**kw))
        with pytest.raises(ValueError):
            Generator(model, max_len=64).generate(torch.tensor([[1, 2]]), max_new_tokens=2, **kw)
    assert eng.num_waiting == 0


def test_rules_that_32_bits_or_the_tables_do_not_hold_are_refused(model):
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=2, max_model_len=64))
    for kw in (dict(logit_bias={1: 1e39}), dict(presence_penalty=-1e39), dict(frequency_penalty=1.0, do_sample=True, temperature=1e-39),
               dict(frequency_penalty=1.0, repetition_penalty=1e38), dict(frequency_penalty=1.0, do_sample=True, temperature=float("inf"))):
        with pytest.raises(ValueError):
            eng.submit([1, 2], GenerationConfig(**kw))
    ruled = GenerationConfig(presence_penalty=1.0)
    ruled.check_rules(1 << 19, (1 << 20) - 1)
    for size in ((1 << 19) + 1, 0), (300, 1 << 20):
        with pytest.raises(ValueError):
            ruled.check_rules(*size)
        GenerationConfig().check_rules(*size)


def test_server_takes_penalties_and_biases():
    tok = ByteTokenizer()
    torch.manual_seed(0)
    m = qwen(vocab=300)
    eng = LLMEngine(m, tok, EngineArgs(max_num_seqs=2, max_model_len=128)).start()
    try:
        c = TestClient(build_app(eng, prompt_style="deepseek"))
        a = ord("a")
        body = {"model": "m", "messages": [{"role": "user", "content": "hi"}], "max_tokens": 6, "temperature": 0, "ignore_eos": True}
        ids = tok.encode("a")
        text = c.post("/v1/chat/completions", json={**body, "logit_bias": {str(ids[0]): 1e4}}).json()["choices"][0]["message"]["content"]
        assert text == "a" * 6
        text = c.post("/v1/completions", json={"model": "m", "prompt": "hi", "max_tokens": 6, "temperature": 0, "ignore_eos": True, "allowed_token_ids": ids}).json()
        assert text["choices"][0]["text"] == "a" * 6 and a
        assert c.post("/v1/chat/completions", json={**body, "presence_penalty": 1.0, "frequency_penalty": -1.0}).status_code == 200
        for bad in ({"logit_bias": {"999": 1.0}}, {"logit_bias": {"x": 1.0}}, {"allowed_token_ids": [-4]}):
            assert c.post("/v1/chat/completions", json={**body, **bad}).status_code == 400
            assert c.post("/v1/completions", json={"model": "m", "prompt": "hi", **bad}).status_code == 400
        for bad in ({"presence_penalty": 3.0}, {"frequency_penalty": -2.5}):
            assert c.post("/v1/chat/completions", json={**body, **bad}).status_code == 422
    finally:
        eng.shutdown()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rows_of_a_paged_cache_grow_together(device):
    def make():
        return PagedKVCache(1, 40, 1, 16, 16, torch.float32, device, 5, 256)
    one, many = make(), make()
    updates = [(3, 0, [5, 6, 7]), (0, 2, [9]), (4, 1, []), (1, 15, [30])]
    one.table[0, :2] = many.table[0, :2] = torch.tensor([1, 2], dtype=torch.int32, device=device)
    many.extend_rows(updates)
    for slot, first, blocks in updates:
        if blocks:
            one.table[slot, first:first + len(blocks)] = torch.tensor(blocks, dtype=torch.int32, device=device)
    assert torch.equal(one.table, many.table)
    many.extend_rows([])
    many.extend_rows([(2, 0, [])])
    assert torch.equal(one.table, many.table)


class _Recorder:
    """A ragged model that keeps what its step is called with."""
    max_positions = 0

    def __init__(self, device):
        self.embed_tokens = torch.zeros(50, 8, device=device)
        self.config, self.training = None, False

    def kv_layout(self):
        return [(1, 16)]

    def eval(self):
        return self

    def forward_ragged(self, ids, pos, slot, cache, want=None, max_pos=0, pieces=None, layer_outputs=None):
        self.got = (ids, pos, slot, want, max_pos, pieces)
        return torch.zeros(len(want), 50, device=ids.device)


@gpu
def test_maps_of_a_ragged_step_on_the_device():
    """Positions, rows, tiles and runs of a step as the host would lay them out."""
    gen = RaggedGenerator(_Recorder("cuda"), None, 1024)
    cache = gen.make_cache(64, 16, 6, 160)
    entries = [(2, 0, list(range(130)), [129]), (0, 77, [5], [0]), (5, 3, [], []), (4, 64, list(range(64)), [0, 63]), (1, 0, [9, 8], [])]
    gen.step(entries, cache)
    ids, pos, slot, want, max_pos, pieces = gen.model.got
    runs, p, s = [], [], []
    for row, p0, toks, _ in entries:
        if toks:
            runs.append([len(p), len(toks), p0, row])
            p += range(p0, p0 + len(toks))
            s += [row] * len(toks)
    host = make_pieces(runs, "cpu")
    assert pos.tolist() == p and slot.tolist() == s and want.tolist() == [129, 130, 131, 194] and max_pos == 129
    assert (pieces.n_tiles, pieces.n_runs, pieces.longest) == (host.n_tiles, host.n_runs, host.longest)
    for f in ("tiles", "runs", "tile_of", "run_tiles"):
        assert getattr(pieces, f).tolist() == getattr(host, f).tolist() and getattr(pieces, f).dtype == torch.int32 and getattr(pieces, f).is_contiguous()


def test_groups_need_pages(model):
    gen = Generator(model, max_len=64)
    cache = KVCache(2, 2, 2, 64, 16, torch.float32, "cpu")
    two = torch.zeros(2, dtype=torch.long)
    with pytest.raises(ValueError, match="paged"):
        gen.decode_graphed(two, cache, two.int(), two.int(), groups=[(0, 2, 8)])


def test_plans_of_captured_steps():
    plan = group_plan(6, 512, "cpu")
    assert plan.of.tolist() == [-1] * 6 and plan.n_groups == MAX_GROUPS and (plan.groups == 0).all()
    set_group_plan(plan, [(0, 2, 64), (3, 2, 100)])
    assert plan.of.tolist() == [0, 0, -1, 1, 1, -1] and plan.groups[:2].tolist() == [[0, 2, 64, 0], [3, 2, 100, 0]] and (plan.groups[2:] == 0).all()
    set_group_plan(plan, [(1, 5, 7)])
    assert plan.of.tolist() == [-1, 0, 0, 0, 0, 0] and (plan.groups[1:] == 0).all()
    with pytest.raises(ValueError):
        set_group_plan(plan, [(i, 1, 5) for i in range(MAX_GROUPS + 1)])


def test_blocks_that_a_step_cannot_have_are_not_booked(model):
    """Where the pool runs out at one of several requests, none of them has blocks that its row of the table does not list."""
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=3, max_model_len=64, block_size=8, num_kv_blocks=7))
    reqs = [Request(i, [1], GenerationConfig()) for i in range(3)]
    for i, r in enumerate(reqs):
        r.slot = i
    eng._grow_all([(reqs[0], 1)])
    before = eng.cache.table.clone(), {k: list(v) for k, v in eng._slot_blocks.items()}, list(eng._free_blocks), list(eng._block_ref)
    with pytest.raises(RuntimeError, match="exhausted"):
        eng._grow_all([(reqs[0], 9), (reqs[1], 9), (reqs[2], 40)])
    after = eng.cache.table, {k: v for k, v in eng._slot_blocks.items() if v}, eng._free_blocks, eng._block_ref
    assert torch.equal(before[0], after[0]) and before[1:] == after[1:]
    eng._grow_all([(reqs[0], 9), (reqs[1], 9)])
    for i in (0, 1):
        blocks = eng._slot_blocks[i]
        assert eng.cache.table[i, :len(blocks)].tolist() == blocks and all(eng._block_ref[b] == 1 for b in blocks)


def test_groups_are_found_among_running_requests(model):
    """Rows that list the same first blocks, whole blocks of prompts only; few shared keys and sequences by themselves are left alone; results are those
    of an engine without groups."""
    torch.manual_seed(5)
    a, b = torch.randint(0, 300, (70,)).tolist(), torch.randint(0, 300, (33,)).tolist()
    prompts = [a + [1], b + [5], a + [2, 3], [9, 9], b + [6], a[:50] + [7]]
    outs = []
    for on in (False, True):
        eng = LLMEngine(model, None, EngineArgs(max_num_seqs=8, max_model_len=128, block_size=16, shared_prefix_attention=on, shared_prefix_min=32))
        first = [eng.submit(p, GenerationConfig(max_new_tokens=20)) for p in prompts[:2]]
        eng.step()
        reqs = first + [eng.submit(p, GenerationConfig(max_new_tokens=8)) for p in prompts[2:]]
        seen = set()
        while not all(r.done.is_set() for r in reqs):
            eng.step()
            order, groups = eng._shared_groups(eng.running)
            if groups:
                seen.add((tuple(eng.running[i].rid for i in order), groups))
        outs.append([r.output_ids for r in reqs])
        assert bool(seen) == on
    assert outs[0] == outs[1]
    whole = max(seen, key=lambda s: len(s[0]))
    assert whole[0][:5] == (0, 2, 5, 1, 4) and whole[1] == ((0, 3, 48), (3, 2, 32))
    for kw in (dict(block_size=0), dict(block_size=16, enable_prefix_caching=False)):
        with pytest.raises(ValueError, match="shared_prefix_attention"):
            LLMEngine(model, None, EngineArgs(max_num_seqs=2, max_model_len=64, shared_prefix_attention=True, **kw))


@gpu
@pytest.mark.parametrize("D,H,Hkv,bs", [(64, 8, 2, 16), (128, 4, 4, 64)])
def test_engine_with_a_shared_prompt(entries, D, H, Hkv, bs):
    """A whole step as it is used: tables grown, sequences behind one system prompt decoded as a group from a captured graph, rules on some of their
    logits. Every decode step's logits against the same model in 32 bits on the CPU: as near as those of the engine without groups."""
    m = qwen("cuda", torch.bfloat16, D, H, Hkv, layers=3)
    ref = qwen("cpu", torch.float32, D, H, Hkv, layers=3)
    ref.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    torch.manual_seed(4)
    system = torch.randint(0, 300, (130,)).tolist()
    prompts = [system + torch.randint(0, 300, (n,)).tolist() for n in (9, 21, 4, 40, 2)] + [torch.randint(0, 300, (70,)).tolist()]
    cfgs = [GenerationConfig(max_new_tokens=10, ignore_eos=True, **kw) for kw in
            (dict(), dict(frequency_penalty=0.5), dict(), dict(logit_bias={7: 1.0}, presence_penalty=0.5), dict(), dict())]
    errors = {}
    for on in (False, True):
        eng = LLMEngine(m, None, EngineArgs(max_num_seqs=8, max_model_len=256, block_size=bs, warmup=False, shared_prefix_attention=on, shared_prefix_min=64))
        steps, real = [], eng._sample

        def sample(logits, reqs, real=real, steps=steps):
            steps.extend((r.prompt_ids + r.output_ids, l.float().cpu()) for r, l in zip(reqs, logits))
            return real(logits, reqs)
        eng._sample = sample
        entries.clear()
        reqs = [eng.submit(prompts[0], cfgs[0])]
        eng.step()
        reqs += [eng.submit(p, c) for p, c in zip(prompts[1:], cfgs[1:])]
        n = 0
        while not all(r.done.is_set() for r in reqs):
            eng.step()
            n += 1
            assert n < 100
        assert ("b200_prefix_attn" in entries) == on and "b200_extend_block_tables" in entries
        assert "b200_greedy_tokens" in entries and "b200_append_tokens" in entries
        assert all(len(r.output_ids) == 10 for r in reqs) and eng._reserved == 0
        g, worst = Generator(ref, max_len=256), []
        for seq, l in steps:
            cache = PagedKVCache(3, 20, Hkv, 16, D, torch.float32, "cpu", 1, 256)
            cache.set_row(0, range(1, 17))
            want = g._prefill(torch.tensor([seq]), cache)[0]
            worst.append(float((l - want).norm() / (want - want.mean()).norm()))
        errors[on] = sorted(worst)
    # both are 16-bit computations of one model whose sums are in different orders: of one size, the group's within a half more of the other's
    assert errors[True][len(errors[True]) // 2] < 1.5 * errors[False][len(errors[False]) // 2] and errors[True][-1] < 2 * errors[False][-1], errors


@gpu
@pytest.mark.parametrize("groups", [(), ((0, 2, 16),)])
def test_a_cache_that_gets_a_dead_ones_id(groups):
    """A captured step is replayed for the cache that it was captured with, and for no other that is known by the same number: its keys go where they belong."""
    gen = Generator(qwen("cuda", torch.bfloat16, 64, 8, 2), max_len=128)
    tok, pos, slots = torch.tensor([5, 6], device="cuda"), torch.full((2,), 40, dtype=torch.int32, device="cuda"), torch.arange(2, dtype=torch.int32, device="cuda")

    def make():
        cache = PagedKVCache(2, 20, 2, 16, 64, torch.bfloat16, "cuda", 3, 128)
        for row, blocks in enumerate(([1, 2, 3], [1, 4, 5])):
            cache.set_row(row, blocks)
        return cache
    old = make()
    gen.decode_graphed(tok, old, pos, slots, groups=groups)
    new = make()
    for key in list(gen._graphs):
        gen._graphs[tuple(id(new) if k == id(old) else k for k in key)] = gen._graphs.pop(key)
    for c in (old, new):
        for pool in c.k + c.v:
            pool.zero_()
    logits = gen.decode_graphed(tok, new, pos, slots, groups=groups).clone()
    again = gen.decode_graphed(tok, new, pos, slots, groups=groups)
    assert torch.equal(logits, again) and len(gen._graphs) == 1
    assert not any(bool(pool.any()) for pool in old.k + old.v)
    assert all(bool((pool[[3, 5], :, 8] != 0).any(2).all()) and int(pool.count_nonzero()) <= 2 * 2 * 64 for pool in new.k + new.v)


@gpu
def test_no_request_pays_for_a_capture():
    """warmup captures the decode steps with groups too: requests behind one system prompt, in batches of every bucket, add none."""
    m = qwen("cuda", torch.bfloat16, 64, 8, 2)
    eng = LLMEngine(m, None, EngineArgs(max_num_seqs=6, max_model_len=256, block_size=16, shared_prefix_attention=True, shared_prefix_min=32))
    eng.warmup()
    captured = set(eng.gen._graphs)
    assert {k[0] for k in captured if k[-1] == "groups"} == {2, 4, 8}
    torch.manual_seed(4)
    system = torch.randint(0, 300, (64,)).tolist()
    first = eng.submit(system + [1], GenerationConfig(max_new_tokens=12, ignore_eos=True))
    eng.step()
    reqs = [first] + [eng.submit(system + [i], GenerationConfig(max_new_tokens=3 * i, ignore_eos=True)) for i in range(1, 6)]
    grouped = 0
    while not all(r.done.is_set() for r in reqs):
        eng.step()
        grouped += bool(eng._shared_groups(eng.running)[1])
    assert grouped > 5 and set(eng.gen._graphs) == captured


@gpu
def test_gorozen_decodes_groups(tmp_path, entries):
    """The ragged step's decode graph with groups (sinks, keys as values): logits against the oracle, as near as without groups; groups change from replay
    to replay."""
    import gorozen_oracle as O
    from test_gorozen import _tokens, build, rel_err
    cfg = O.make_config(64, 96, [O.attn_layer(4, 2, 32, 16, 100.0, None, mlp=O.dense()), O.attn_layer(4, 2, 32, 16, 100.0, None, mlp=O.dense())])
    W = O.random_weights(cfg, seed=15)
    model = build(tmp_path, cfg, W, "cuda", torch.bfloat16)
    gen = RaggedGenerator(model, None, 256)
    cache = gen.make_cache(40, 16, 6, 128)
    system = _tokens(48, cfg["vocab"], 3)
    tails = [_tokens(n, cfg["vocab"], 10 + n) for n in (5, 9, 2, 17)]
    shared = [1, 2, 3]
    for i, t in enumerate(tails):
        gen.set_block_row(cache, i, shared + [4 + 5 * i + j for j in range(5)])
    gen.step([(0, 0, system + tails[0], [])], cache)
    gen.step([(i, 48, t, []) for i, t in enumerate(tails) if i], cache)
    tok = [7, 8, 9, 10]
    pos = [48 + len(t) for t in tails]
    want = [torch.as_tensor(O.forward(cfg, W, system + t + [k])[-1]) for t, k in zip(tails, tok)]
    plain = gen.decode(tok, pos, range(4), cache)
    entries.clear()
    for groups in ([(0, 4, 48)], [(0, 2, 48), (2, 2, 32)], [(1, 3, 17)]):
        got = gen.decode(tok, pos, range(4), cache, groups=groups)
        for g, p, w in zip(got, plain, want):
            assert rel_err(g[None], w[None]) < 1.5 * rel_err(p[None], w[None]) + 2.0 ** -8, groups
    assert "b200_prefix_attn" in entries and len(cache._decode_graphs) == 2
    with pytest.raises(ValueError):
        gen.decode(tok, pos, range(4), cache, groups=[(0, 1, 5)] * (MAX_GROUPS + 1))


@gpu
def test_rules_choose_the_same_tokens_on_both_devices():
    """LogitRules on the GPU and on the CPU from the same logits: greedy rows equal, step after step, histories too."""
    torch.manual_seed(6)
    V, rows = 5000, [2, 0, 3]
    cfgs = [GenerationConfig(frequency_penalty=0.8, presence_penalty=0.2, repetition_penalty=1.2), GenerationConfig(logit_bias={3: 6.0, 4: -6.0}),
            GenerationConfig(allowed_token_ids=list(range(0, V, 7)), frequency_penalty=2.0)]
    sides = []
    for device in ("cpu", "cuda"):
        r = LogitRules(4, V, 64, device, 8)
        for row, c in zip(rows, cfgs):
            r.begin(row, c, [1, 2, 3])
        sides.append(r)
    for _ in range(20):
        x = torch.randn(3, V) * 2
        a, b = (r.next(x.to(r.state.device), rows, cfgs) for r in sides)
        assert a.tolist() == b.tolist()
    assert torch.equal(sides[0].state.tokens, sides[1].state.tokens.cpu()) and torch.equal(sides[0].state.length, sides[1].state.length.cpu())
