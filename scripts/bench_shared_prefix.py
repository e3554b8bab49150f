"""Decode steps whose sequences share a cached prefix (ops/prefix_attention.py), random weights and keys, CUDA events.

    python scripts/bench_shared_prefix.py model       # a captured step of 36 layers (Qwen3-8B sizes) without groups and with them
    python scripts/bench_shared_prefix.py attention   # the attention alone: the plan of an exact call, that of a captured step, given numbers of ranges
    python scripts/bench_shared_prefix.py once        # two calls of 128 tokens over 16384 shared keys, for a profiler

``attention`` times graphs of thirty calls on three sets of inputs in turn (device time; together they exceed L2 but for the smallest); the best of eight."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(1, os.path.join(sys.path[0], "perf"))
import torch

import operators
from llm_in_practise_b200.inference.generate import Generator, PagedKVCache, group_plan, set_group_plan
from llm_in_practise_b200.models.qwen3 import QWEN3_PRESETS, Qwen3ForCausalLM
from llm_in_practise_b200.ops import _native as nv
from llm_in_practise_b200.ops.prefix_attention import prefix_attention

# name: (groups, own keys at most, heads, KV heads, head size, ranges to try)
SIZES = {"4 x 512 + 40": ("4:512", 40, 16, 4, 128, ()), "64 x 4096 + 600": ("64:4096", 600, 32, 8, 128, (4, 6, 7, 8, 9)), "40 x 4096 + 600": ("40:4096", 600, 32, 8, 128, ()),
         "40 x 3000 + 512, 16 / 2": ("40:3000", 512, 16, 2, 128, (4, 8, 11, 24)), "128 x 16384 + 512": ("128:16384", 512, 32, 8, 128, (4, 8, 9, 12)),
         "100 x 8000 + 512, 12 / 2 of 64": ("100:8000", 512, 12, 2, 64, (4, 9, 12, 14, 18)), "64 x 2000 + 300, 16 / 8 of 64": ("64:2000", 300, 16, 8, 64, ()),
         "64 x 4096 + 600, 32 / 8 of 96": ("64:4096", 600, 32, 8, 96, ()), "64 x 2000 + 300, 16 / 4 of 80": ("64:2000", 300, 16, 4, 80, ())}


def inputs(size, n):
    groups, own, H, G, D, _ = SIZES[size]
    operators.own = True
    return [operators.prepare({"kind": "prefix", "groups": groups, "alone": 0, "own_keys": own, "H": H, "G": G, "D": D, "page": 64, "dtype": "bf16", "sinks": False}, i)
            for i in range(n)]


def call(s, plan=0, groups=None):
    c = s["case"]
    return prefix_attention(s["qkv"], s["ck"], s["cv"], s["table"], s["pos"], s["slot"], groups or s["plan"], c["H"], c["G"], c["D"], c["D"] ** -0.5,
                            max_pos=0 if groups else max(s["keys"]) - 1, plan=plan)


def device_us(fns, rounds=10):
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        for fn in fns:
            fn()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(rounds):
            for fn in fns:
                fn()
    times = []
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1000 / rounds / len(fns))
    return min(times)


def attention():
    plan_of = nv.proto("b200_prefix_attn_plan", [nv.ctypes.c_int] * 8)

    def text(plan):
        return f"{plan % 256} ranges on {'tcgen05' if plan >= 256 else 'mma.sync'}"
    for size, (_, _, H, G, D, ranges) in SIZES.items():
        ss = inputs(size, 3)
        T, p = ss[0]["qkv"].shape[0], ss[0]["plan"]
        plan = plan_of(T, p.n_groups, p.longest, p.max_shared, max(1, max(ss[0]["keys"]) - p.min_shared), H, G, D)
        cols = [f"exact plan ({text(plan)}) {device_us([lambda s=s: call(s) for s in ss]):.1f}"]
        for max_len in (8192, 32768):
            if max_len >= max(ss[0]["keys"]):
                captured = group_plan(T, max_len, "cuda")
                set_group_plan(captured, ss[0]["groups"])
                cols.append(f"captured step, max_len {max_len} ({text(plan_of(T, captured.n_groups, captured.longest, captured.max_shared, 0, H, G, D))}) "
                            f"{device_us([lambda s=s: call(s, groups=captured) for s in ss]):.1f}")
        cols += [f"{n} ranges {device_us([lambda s=s: call(s, plan=plan // 256 * 256 + n) for s in ss]):.1f}" for n in ranges]
        print(f"{size}: us: " + ", ".join(cols), flush=True)


def model():
    torch.manual_seed(0)
    cfg = QWEN3_PRESETS["qwen3-8b"]
    gen = Generator(Qwen3ForCausalLM(cfg, dtype=torch.bfloat16, device="cuda", init_std=0.02), max_len=20480)
    for B, shared, own in ((64, 4096, 300), (8, 1024, 100), (32, 16384, 300), (64, 256, 300)):
        bs, n0 = 64, shared // 64
        per = -(-(own + 1) // bs) + 1
        cache = PagedKVCache(cfg.num_hidden_layers, n0 + B * per + 1, cfg.num_key_value_heads, bs, cfg.head_dim, torch.bfloat16, "cuda", B + 1, 20480)
        for pool in cache.k + cache.v:
            pool.normal_(std=0.5)
        for i in range(B):
            cache.set_row(i, list(range(n0)) + list(range(n0 + i * per, n0 + (i + 1) * per)))
        tok = torch.randint(0, 150000, (B,), device="cuda")
        pos, slots = torch.full((B,), shared + own, dtype=torch.int32, device="cuda"), torch.arange(B, dtype=torch.int32, device="cuda")

        def timed(groups):
            for _ in range(5):
                gen.decode_graphed(tok, cache, pos, slots, groups=groups)
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            for _ in range(20):
                y = gen.decode_graphed(tok, cache, pos, slots, groups=groups)
            b.record()
            b.synchronize()
            return a.elapsed_time(b) / 20, y.clone()
        plain, y0 = timed(())
        grouped, y1 = timed([(0, B, shared)])
        print(f"{B} sequences, {shared} shared and {own} own keys: {plain:.2f} ms without groups, {grouped:.2f} with them; logits differ by "
              f"{float((y0 - y1).norm() / y0.norm()):.1e}", flush=True)
        gen._graphs.clear()
        del cache


def once():
    s, = inputs("128 x 16384 + 512", 1)
    for _ in range(2):
        call(s)
    torch.cuda.synchronize()


{"model": model, "attention": attention, "once": once}[sys.argv[1] if len(sys.argv) > 1 else "attention"]()
