"""Log probabilities, embedding gradients and activations in 8 bits where the framework calls them: generation, the engine and its HTTP server, Qwen3's log_probs,
checkpoints and gated units, the trainer's arguments."""
import json
import math

import pytest
import torch
from fastapi.testclient import TestClient

from llm_in_practise_b200.data.tokenizers import ByteTokenizer
from llm_in_practise_b200.inference import GenerationConfig, Generator
from llm_in_practise_b200.models.gpt import GPTLike
from llm_in_practise_b200.models.qwen3 import Qwen3Config, Qwen3ForCausalLM
from llm_in_practise_b200.serve import EngineArgs, LLMEngine
from llm_in_practise_b200.serve.openai_server import build_app

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
CFG = Qwen3Config(vocab_size=304, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=16,
                  max_position_embeddings=256)
GPU_CFG = Qwen3Config(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                      max_position_embeddings=512)


def build(device, seed=0, init_std=0.1):
    torch.manual_seed(seed)
    if device == "cpu":
        return Qwen3ForCausalLM(CFG, dtype=torch.float32, device="cpu", init_std=init_std)
    return Qwen3ForCausalLM(GPU_CFG, dtype=torch.bfloat16, device="cuda", init_std=0.05)


@pytest.fixture(scope="module")
def model():
    return build("cpu").eval()


def table(model, ids):
    """log_softmax of the model's logits behind each token of ids, in 64 bits."""
    with torch.no_grad():
        return torch.log_softmax(model(torch.tensor([ids]))["logits"][0].double(), -1)


@pytest.mark.parametrize("paged", [0, 16])
def test_engine_gives_log_probabilities(model, paged):
    """Requests that ask for none, some and many alternatives share steps; penalties and temperature do not show in them."""
    torch.manual_seed(1)
    prompts = [torch.randint(0, 304, (n,)).tolist() for n in (5, 9, 3)]
    cfgs = [GenerationConfig(max_new_tokens=6, logprobs=5, ignore_eos=True), GenerationConfig(max_new_tokens=4, ignore_eos=True),
            GenerationConfig(max_new_tokens=5, logprobs=0, do_sample=True, temperature=0.7, presence_penalty=0.5, ignore_eos=True)]
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=3, max_model_len=64, block_size=paged, seed=3))
    reqs = [eng.submit(p, c) for p, c in zip(prompts, cfgs)]
    while not all(r.done.is_set() for r in reqs):
        eng.step()
    assert not any(r.error for r in reqs) and not reqs[1].logprobs
    for r, p in ((reqs[0], prompts[0]), (reqs[2], prompts[2])):
        want = table(model, p + r.output_ids)
        assert [e.token for e in r.logprobs] == r.output_ids
        for j, e in enumerate(r.logprobs):
            row = want[len(p) - 1 + j]
            assert abs(e.logprob - float(row[e.token])) < 1e-4 and e.rank == 1 + int((row > row[e.token]).sum()) and len(e.top) == r.cfg.logprobs
            assert [i for i, _ in e.top] == row.argsort(descending=True, stable=True)[:len(e.top)].tolist()
            assert all(abs(lp - float(row[i])) < 1e-4 for i, lp in e.top)
    assert all(e.rank == 1 for e in reqs[0].logprobs)


def test_engine_refuses_too_many_alternatives(model):
    eng = LLMEngine(model, None, EngineArgs(max_num_seqs=1, max_model_len=32))
    for bad in (-1, 33):
        with pytest.raises(ValueError):
            eng.submit([1, 2], GenerationConfig(logprobs=bad))


@pytest.fixture(scope="module")
def client(model):
    eng = LLMEngine(model, ByteTokenizer(), EngineArgs(max_num_seqs=2, max_model_len=128)).start()
    yield TestClient(build_app(eng))
    eng.shutdown()


def test_server_chat_logprobs(client):
    body = {"model": "m", "messages": [{"role": "user", "content": "hi"}], "max_tokens": 6, "temperature": 0, "ignore_eos": True}
    assert "logprobs" not in client.post("/v1/chat/completions", json=body).json()["choices"][0]
    c = client.post("/v1/chat/completions", json={**body, "logprobs": True, "top_logprobs": 3}).json()["choices"][0]
    content = c["logprobs"]["content"]
    assert len(content) == 6
    for e in content:
        assert set(e) == {"token", "logprob", "bytes", "top_logprobs"} and e["logprob"] <= 0 and len(e["top_logprobs"]) == 3
        assert e["top_logprobs"][0]["logprob"] == e["logprob"] and bytes(e["bytes"]).decode() == e["token"]
    assert client.post("/v1/chat/completions", json={**body, "logprobs": True}).json()["choices"][0]["logprobs"]["content"][0]["top_logprobs"] == []
    assert client.post("/v1/chat/completions", json={**body, "top_logprobs": 3}).status_code == 400
    assert client.post("/v1/chat/completions", json={**body, "logprobs": True, "top_logprobs": 21}).status_code == 422


def test_server_completion_logprobs(client):
    body = {"model": "m", "prompt": ["ab", "cde"], "max_tokens": 5, "temperature": 0, "ignore_eos": True}
    assert [c["logprobs"] for c in client.post("/v1/completions", json=body).json()["choices"]] == [None, None]
    for c in client.post("/v1/completions", json={**body, "logprobs": 2}).json()["choices"]:
        lp = c["logprobs"]
        assert {k: len(v) for k, v in lp.items()} == {"tokens": 5, "token_logprobs": 5, "text_offset": 5, "top_logprobs": 5}
        assert lp["text_offset"][0] == 0 and all(b - a == len(t) for a, b, t in zip(lp["text_offset"], lp["text_offset"][1:], lp["tokens"]))
        assert all(x <= 0 and math.isfinite(x) for x in lp["token_logprobs"])


def events(r):
    return [json.loads(line[6:]) for line in r.text.splitlines() if line.startswith("data: {")]


def test_server_streams_logprobs(client):
    """The chunks' entries together are those of the whole answer, each token once (the second request's prompt comes from the first one's cache: its sums are in
    another order, some steps of 2^-24 of values around 4)."""
    chat = {"model": "m", "messages": [{"role": "user", "content": "hi"}], "max_tokens": 9, "temperature": 0, "ignore_eos": True, "logprobs": True, "top_logprobs": 1}
    whole = client.post("/v1/chat/completions", json=chat).json()["choices"][0]["logprobs"]["content"]
    parts = [e["choices"][0].get("logprobs") for e in events(client.post("/v1/chat/completions", json={**chat, "stream": True}))]
    got = [t for p in parts if p for t in p["content"]]
    assert [t["token"] for t in got] == [t["token"] for t in whole] and all(abs(a["logprob"] - b["logprob"]) < 1e-5 for a, b in zip(got, whole))
    text = {"model": "m", "prompt": "ab", "max_tokens": 9, "temperature": 0, "ignore_eos": True, "logprobs": 1}
    whole = client.post("/v1/completions", json=text).json()["choices"][0]["logprobs"]
    parts = [e["choices"][0]["logprobs"] for e in events(client.post("/v1/completions", json={**text, "stream": True}))]
    got = [t for p in parts for t in p["token_logprobs"]]
    assert len(got) == 9 and all(abs(a - b) < 1e-5 for a, b in zip(got, whole["token_logprobs"]))
    assert [t for p in parts for t in p["tokens"]] == whole["tokens"]


class Counting(ByteTokenizer):
    """How often it was asked for text."""

    def decode(self, *args, **kw):
        self.decoded = getattr(self, "decoded", 0) + 1
        return super().decode(*args, **kw)


@pytest.fixture(scope="module")
def counting(model):
    eng = LLMEngine(model, Counting(), EngineArgs(max_num_seqs=2, max_model_len=128)).start()
    yield TestClient(build_app(eng)), eng.tokenizer, eng
    eng.shutdown()


def test_streams_without_logprobs_decode_a_token_once(counting):
    """The text behind each token, and the whole once more at the end, in both forms of a stream."""
    client, tok, _ = counting
    for path, body in (("/v1/completions", {"prompt": "ab"}), ("/v1/chat/completions", {"messages": [{"role": "user", "content": "hi"}]})):
        tok.decoded = 0
        r = client.post(path, json={"model": "m", "max_tokens": 40, "temperature": 0, "ignore_eos": True, "stream": True, **body})
        assert r.status_code == 200 and tok.decoded == 41


def test_server_logprobs_end_at_a_stop_string(client):
    body = {"model": "m", "prompt": "ab", "max_tokens": 9, "temperature": 0, "ignore_eos": True, "logprobs": 0}
    free = client.post("/v1/completions", json=body).json()["choices"][0]
    at = next((i for i, t in enumerate(free["logprobs"]["tokens"]) if t and "�" not in t and i), None)
    if at is None:
        pytest.skip("no token of this model is text by itself")
    c = client.post("/v1/completions", json={**body, "stop": free["logprobs"]["tokens"][at]}).json()["choices"][0]
    assert c["finish_reason"] == "stop" and len(c["logprobs"]["tokens"]) <= at + 1


def test_the_token_of_a_stop_string_is_found_by_halves(counting, monkeypatch):
    """As many tokens as a walk from the first one on takes, wherever the stop string is, with some ten decodes beside those of the tokens' own texts."""
    client, tok, eng = counting
    submit, reqs = eng.submit, []
    monkeypatch.setattr(eng, "submit", lambda *a, **k: reqs.append(submit(*a, **k)) or reqs[-1])
    body = {"model": "m", "prompt": "ab", "max_tokens": 100, "temperature": 0, "ignore_eos": True, "logprobs": 0}
    free = client.post("/v1/completions", json=body).json()["choices"][0]
    text, tokens = free["text"], free["logprobs"]["tokens"]
    assert len(tokens) == 100
    places = [at for at in range(0, len(text), 7) if "\ufffd" not in text[at:at + 2]] + [None]
    assert len(places) > 3
    for at in places:
        stop = "not in it" if at is None else text[at:at + 2]
        tok.decoded = 0
        c = client.post("/v1/completions", json={**body, "stop": stop}).json()["choices"][0]
        n = len(c["logprobs"]["tokens"])
        assert c["text"] == text[:text.index(stop) if at is not None else None] and c["finish_reason"] == ("length" if at is None else "stop")
        assert tok.decoded <= 2 + 7 + n                      # 100 places are halved 7 times
        assert n == next((i for i in range(1, 101) if stop in ByteTokenizer().decode(reqs[-1].output_ids[:i], skip_special_tokens=True)), 100)


def test_generate_returns_log_probabilities(model):
    ids = torch.randint(0, 304, (1, 7))
    out, lp = Generator(model, max_len=64).generate(ids, max_new_tokens=5, do_sample=False, return_logprobs=True)
    want = table(model, out[0].tolist())
    assert lp.shape == (1, 5) and all(abs(float(lp[0, j]) - float(want[6 + j, out[0, 7 + j]])) < 1e-4 for j in range(5))


@pytest.mark.parametrize("device", DEVICES)
def test_qwen3_log_probs(device):
    """Their mean is the loss of forward(); labels of -100 are passed over; gradients of a weighted sum reach the embedding and the head."""
    m = build(device)
    ids = torch.randint(0, 300, (2, 33), device=device)
    labels = ids.clone()
    labels[0, :20] = -100
    r = m.log_probs(ids, labels, entropy=True)
    assert r.logprob.shape == r.entropy.shape == (2, 32) and not r.logprob[0, :19].any() and not r.entropy[0, :19].any()
    loss = float(m(ids, labels=labels)["loss"].detach())
    # forward() rounds its logits to the model's type (bf16: a step of 2^-8 of logits up to 8)
    assert abs(-float(r.logprob.detach().sum()) / int((labels[:, 1:] != -100).sum()) - loss) < (1e-4 if device == "cpu" else 0.02)
    adv = torch.randn(2, 32, device=device)
    ((r.logprob * adv).sum() + 0.1 * r.entropy.sum()).backward()
    got = [p.grad.clone() for p in (m.embed_tokens, m.lm_head)]
    m.zero_grad()
    with torch.enable_grad():
        lp = torch.log_softmax(m.hidden_states(ids).view(2, 33, -1)[:, :-1].float() @ m.lm_head.float().t(), -1)
        t = labels[:, 1:]
        w = (t != -100).float()
        picked = lp.gather(2, t.clamp_min(0).unsqueeze(2)).squeeze(2)
        ((picked * adv * w).sum() - 0.1 * ((lp.exp() * lp).sum(-1) * w).sum()).backward()
    for a, b in zip(got, (m.embed_tokens.grad, m.lm_head.grad)):
        assert float((a.double() - b.double()).norm() / b.double().norm()) < (1e-4 if device == "cpu" else 0.03)


def gradients(m, ids):
    m.zero_grad()
    m.train()
    loss = m(ids, labels=ids)["loss"]
    loss.backward()
    return float(loss.detach()), {n: p.grad.double().clone() for n, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("how", ["checkpoints", "gated", "both"])
def test_qwen3_trains_with_activations_in_8_bits(device, how):
    """Losses are those of 16 bits (the gated unit rounds once instead of twice); gradients are within what 1 / 127 of a block's largest value costs."""
    m = build(device)
    ids = torch.randint(0, 300, (2, 32), device=device)
    loss, want = gradients(m, ids)
    if how in ("gated", "both"):
        m.set_activation_bits(8)
    if how in ("checkpoints", "both"):
        m.gradient_checkpointing_enable(activation_bits=8, use_reentrant=False)
    l8, got = gradients(m, ids)
    again = gradients(m, ids)[1]
    assert abs(l8 - loss) < (1e-5 if device == "cpu" else 0.01) and got.keys() == want.keys()
    for n, g in got.items():
        assert torch.equal(g, again[n]) and float((g - want[n]).norm() / want[n].norm()) < 0.06, n
    m.set_activation_bits(16)
    m.gradient_checkpointing_disable()
    for n, g in gradients(m, ids)[1].items():
        assert torch.equal(g, want[n]) or device == "cuda" and torch.allclose(g, want[n], rtol=0.02, atol=1e-4), n
    for bad in (4, 32):
        with pytest.raises(ValueError):
            m.set_activation_bits(bad)
        with pytest.raises(ValueError):
            m.gradient_checkpointing_enable(activation_bits=bad)


def test_trainer_arguments_reach_the_model():
    from llm_in_practise_b200.trainer import Trainer, TrainingArguments
    m = build("cpu")
    Trainer(model=m, args=TrainingArguments(output_dir="out", gradient_checkpointing=True, gradient_checkpointing_kwargs={"use_reentrant": False, "activation_bits": 8},
                                            report_to="none"))
    assert m.gradient_checkpointing and m.checkpoint_bits == 8


def test_checkpoints_keep_the_bits_that_were_set():
    from llm_in_practise_b200.trainer import Trainer, TrainingArguments
    m = build("cpu")
    m.gradient_checkpointing_enable()
    assert m.checkpoint_bits == 16
    m.gradient_checkpointing_enable(gradient_checkpointing_kwargs={"use_reentrant": False, "activation_bits": 8})
    assert m.checkpoint_bits == 8
    Trainer(model=m, args=TrainingArguments(output_dir="out", gradient_checkpointing=True, report_to="none"))
    assert m.checkpoint_bits == 8
    m.gradient_checkpointing_enable(16)
    assert m.checkpoint_bits == 16


def test_lora_behind_8_bit_checkpoints():
    """A frozen base: nothing in front of the first layer needs a gradient, and the adapters still get theirs."""
    from llm_in_practise_b200.peft import LoraConfig, get_peft_model
    m = build("cpu")
    get_peft_model(m, LoraConfig(r=4, lora_alpha=8, lora_dropout=0.0, target_modules=["q_proj", "v_proj"]))
    m.gradient_checkpointing_enable(activation_bits=8)
    m.train()
    ids = torch.randint(0, 300, (2, 16))
    m(ids, labels=ids)["loss"].backward()
    trained = [p for p in m.parameters() if p.requires_grad]
    assert trained and any(p.grad is not None and p.grad.abs().sum() > 0 for p in trained)


@pytest.mark.gpu
def test_gpt_embedding_gradient_is_the_same_every_time():
    torch.manual_seed(0)
    m = GPTLike(vocab_size=500, block_size=32, n_layer=1, n_head=2, d_model=64, dropout=0.0, tie_weights=False).cuda()
    ids = torch.randint(0, 500, (4, 32), device="cuda")

    weights = torch.randn(64, device="cuda")

    def run():
        m.zero_grad()
        (m.hidden(ids).view(-1, 64).float() * weights).sum().backward()
        return m.tok_emb.grad.clone()
    a = run()
    assert torch.equal(a, run()) and a.abs().sum() > 0
