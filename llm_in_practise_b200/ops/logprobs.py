"""Log probabilities of given tokens (``csrc/logprobs.cu``): what scoring, an API's ``logprobs`` and training on answers need of a model's logits.

``token_logprobs(logits, tokens)``            from logits: log probabilities, and where asked entropies, ranks and the most probable alternatives.
``linear_token_logprobs(x, w, tokens)``       from hidden states and the output projection, without a [tokens, vocab] tensor.

With y = logits / temperature and p = softmax(y): ``logprob = log p[token]``, ``entropy = -sum p log p``, ``rank = 1 +`` the number of larger logits.
Log probabilities and entropies have gradients, formed where autograd delivers the weights of the rows (a policy gradient, a preference loss, a
distillation): a mean cross entropy whose gradient is known in the forward is ``ops.loss``. A row whose token is not one of the vocabulary (-100,
say) is passed over: zeros, rank 0, alternatives -1, no gradient.

Reference: perplexities and answers scored in Quantization/LLM-Compressor/AWQ/eval_qwen3_4b_awq.py through vLLM, whose server gives ``logprobs``.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple, Optional

import torch

from . import _native as nv
from .gemm import _stream_k_workspace, gemm

vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
MAX_TOP = 32             # alternatives of a row
_HERE = contextlib.nullcontext()
_ROWS_ARGS = [vp, i64, i64, i32, vp, f32, i32, vp, vp, vp, vp, vp, vp, i32, vp]
_GRAD_ARGS = [vp, i64, i64, i32, vp, f32, vp, vp, vp, vp, i64, i32, vp]


class TokenLogprobs(NamedTuple):
    """What was not asked for is None. Shapes are the tokens' (``top_ids`` and ``top_logprobs`` have one dimension more)."""
    logprob: Optional[torch.Tensor]           # fp32
    entropy: Optional[torch.Tensor] = None    # fp32
    rank: Optional[torch.Tensor] = None       # int64: 1 = no logit is larger
    top_ids: Optional[torch.Tensor] = None    # int64, the most probable first, the lowest id first among equals
    top_logprobs: Optional[torch.Tensor] = None


_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_MOST = 2 ** 30          # columns, and tokens from hidden states, are counted in 32 bits


def _check(what, tokens, shape, device):
    if tokens.dtype is not torch.int64 or tokens.shape != shape or tokens.device != device:
        raise ValueError(f"{what}: tokens must be int64 {list(shape)} on {device}")


def _check_temperature(what, temperature):
    if not 2.0 ** -60 <= temperature <= 2.0 ** 60:
        raise ValueError(f"{what}: temperature must be from 2^-60 to 2^60, not {temperature}")


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """[rows, last] with contiguous rows; a view where there is one."""
    x = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _rows(logits, tokens, temperature, top, entropy, rank, save, shape=None):
    """(lp, H, rank, ids, lps, stats) of logits [B, V], with leading dimensions ``shape`` (None: [B]); ``stats`` fp32 [B, 4] is what the gradient needs."""
    if not nv.use_native(logits):
        got = _rows_torch(logits, tokens, temperature, top, entropy, rank)
        if shape is None:
            return got
        return (*(t if t is None else t.view(shape) for t in got[:3]), *(t if t is None else t.view(*shape, top) for t in got[3:5]), got[5])
    B, V = logits.shape
    new, one = logits.new_empty, (B,) if shape is None else shape
    lp = H = r = ids = lps = stats = None
    if tokens is not None:
        lp = new(one, dtype=torch.float32)
    if entropy:
        H = new(one, dtype=torch.float32)
    if rank:
        r = new(one, dtype=torch.int64)
    if top:
        ids, lps = new((*one, top), dtype=torch.int64), new((*one, top), dtype=torch.float32)
    if save:
        stats = new((B, 4), dtype=torch.float32)
    if B:
        ptr = nv.ptr
        rc = nv.call_on(logits.device, nv.proto("b200_token_logprobs", _ROWS_ARGS), logits.data_ptr(), logits.stride(0) if B > 1 else V, B, V, ptr(tokens),
                        1.0 / temperature, top, ptr(lp), ptr(H), ptr(r), ptr(ids), ptr(lps), ptr(stats), nv.dtype_code(logits.dtype))
        if rc:
            nv.check(rc, "token_logprobs")
        nv.count_launch()
    return lp, H, r, ids, lps, stats


def _rows_torch(logits, tokens, temperature, top, entropy, rank):
    B, V = logits.shape
    ok = torch.ones(B, dtype=torch.bool, device=logits.device) if tokens is None else (tokens >= 0) & (tokens < V)
    m = logits.float().amax(1, keepdim=True)
    d = (logits.float() - m) / temperature
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    ls = torch.log(s)
    zero = torch.zeros(B, device=logits.device)
    lp = H = r = ids = lps = None
    if tokens is not None:
        at = tokens.clamp(0, V - 1)[:, None]
        lp = torch.where(ok, (d.gather(1, at) - ls)[:, 0], zero)
    if entropy:
        H = torch.where(ok, (ls - (e * d.clamp_min(-150.0)).sum(1, keepdim=True) / s)[:, 0], zero)
    if rank:
        r = torch.where(ok, 1 + (logits > logits.gather(1, at)).sum(1), 0)
    if top:
        ids = _order(logits)[:, :top]
        lps = torch.where(ok[:, None], d.gather(1, ids) - ls, zero[:, None])
        ids = torch.where(ok[:, None], ids, -1)
    stats = torch.cat([m, 1 / s, ls, torch.zeros_like(ls) if H is None else H[:, None]], 1)
    return lp, H, r, ids, lps, stats


def _order(logits):
    """Ids by logit, the largest first, the lowest id first among equals; NaN above all."""
    x = logits.float()
    return torch.sort(torch.where(x.isnan(), torch.full_like(x, float("nan")), x), dim=1, descending=True, stable=True)[1]


def _rows_grad(logits, tokens, temperature, stats, g, h):
    B, V = logits.shape
    if not nv.use_native(logits):
        return _grad_torch(logits.float(), tokens, temperature, stats, g, h, 0, V).to(logits.dtype)
    out = torch.empty(B, V, dtype=logits.dtype, device=logits.device)
    if B:
        fn = nv.proto("b200_token_logprobs_grad", _GRAD_ARGS)
        nv.check(nv.call_on(logits.device, fn, logits.data_ptr(), logits.stride(0) if B > 1 else V, B, V, nv.ptr(tokens), 1.0 / temperature, nv.ptr(stats),
                            nv.ptr(g), nv.ptr(h), nv.ptr(out), V, nv.dtype_code(logits.dtype)), "token_logprobs_grad")
        nv.count_launch()
    return out


def _grad_torch(l, tokens, temperature, stats, g, h, c0, vocab):
    """fp32 gradient of columns c0 .. of the logits, whose fp32 values are l."""
    m, inv_s, ls, H = stats.unsqueeze(2).unbind(1)
    zero = torch.zeros_like(m)
    g, h = (zero if x is None else x.reshape(-1, 1).float() for x in (g, h))
    d = ((l - m) / temperature)
    p = torch.exp(d) * inv_s                         # zero below -150, where d would be no factor beside it
    out = -p * (g + h * (d.clamp_min(-150.0) - ls + H))
    if tokens is not None:
        t = tokens[:, None] - c0
        here = (t >= 0) & (t < l.shape[1])
        out = out + torch.zeros_like(out).scatter_(1, t.clamp(0, l.shape[1] - 1), torch.where(here, g, zero))
        out = torch.where((tokens >= 0)[:, None] & (tokens < vocab)[:, None], out, torch.zeros_like(out))
    return out / temperature


def _first_order_only(what):
    """In a backward pass: gradients are being recorded for a second one only where it was asked for."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no second derivative (create_graph)")


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top, entropy, rank):
        shape = logits.shape[:-1]
        rows = _as_rows(logits)
        lp, H, r, ids, lps, stats = _rows(rows, tokens, temperature, top, entropy, rank, True, None if len(shape) == 1 else shape)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if rank or top:
            ctx.mark_non_differentiable(*(t for t in (r, ids, lps) if t is not None))
        return lp, H, r, ids, lps

    @staticmethod
    def backward(ctx, g, h, *_):
        _first_order_only("token_logprobs")
        if g is None and h is None:
            return (None,) * 6
        logits, tokens, stats = ctx.saved_tensors
        g, h = (None if x is None else x.to(torch.float32).reshape(-1).contiguous() for x in (g, h))
        d = _rows_grad(_as_rows(logits), tokens, ctx.temperature, stats, g, h)
        return (d if logits.dim() == 2 else d.view(logits.shape)), None, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top: int = 0, entropy: bool = False, rank: bool = False,
                   temperature: float = 1.0) -> TokenLogprobs:
    """``logits`` [..., vocab] (fp32, bf16 or fp16; rows an equal distance apart are read where they are, others, as of ``logits[:, :-1]`` of several sequences, are copied
    first, in the backward pass too), ``tokens`` int64 [...] (None: no tokens are given, for entropies and
    alternatives alone). ``top``: how many alternatives, up to ``MAX_TOP``. Sums in 32 bits. A row of minus infinities alone, or with a NaN or plus infinity,
    gives NaN, as log_softmax does. Ranks and alternatives are those of the logits as they are given."""
    shape = logits.shape
    if not shape or shape[-1] < 1 or logits.dtype not in _TYPES:
        raise ValueError("token_logprobs: logits must be [..., vocab] in fp32, bf16 or fp16")
    if tokens is not None:
        _check("token_logprobs", tokens, shape[:-1], logits.device)
        tokens = tokens if len(shape) == 2 and tokens.is_contiguous() else tokens.reshape(-1).contiguous()
    elif rank or not (entropy or top):
        raise ValueError("token_logprobs: without tokens there are entropies and alternatives only")
    _check_temperature("token_logprobs", temperature)
    if shape[-1] >= _MOST:
        raise ValueError(f"token_logprobs: a row of {shape[-1]} logits; there is room for {_MOST - 1}")
    if not 0 <= top <= min(MAX_TOP, shape[-1]):
        raise ValueError(f"token_logprobs: top must be from 0 to {min(MAX_TOP, shape[-1])}, not {top}")
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, temperature, top, entropy, rank))
    return TokenLogprobs(*_rows(_as_rows(logits), tokens, temperature, top, entropy, rank, False, None if len(shape) == 2 else shape[:-1])[:5])


# ------------------------------------------------------------------------------------------------
# from hidden states
# ------------------------------------------------------------------------------------------------
_CHUNK_BYTES = 128 << 20         # 16-bit gradients of logits that exist at a time in the backward pass
_COMPACT_ROWS = 256              # more rows than one tile of the products has: those that are passed over leave them
_HEAD = [vp, i64, vp, i64, i32, i32, i32, i32, vp]
_HEAD_SUMS = _HEAD + [vp, f32, i32, vp, vp, vp]
_HEAD_GRADS = _HEAD + [vp, vp, i32, i32, f32, vp, vp, vp, vp, vp, i64, vp]
_ACTIVE_GEMM = [vp, i64, i32, vp, i64, i32, i32, i32, i32, i32, vp, i32, vp, i64, i32, f32, vp, i64, vp]
_FINISH = [vp, i32, i64, i32, vp, vp, vp, vp, f32, vp, vp, vp, vp]
_ACTIVE = [vp, vp, i64, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp]


class _Active:
    """Rows whose tokens are not passed over, side by side in ``x`` [T, K]; their number stays on the device. ``maps`` int32 [2 T + 1]: which row each is, where each
    row went, how many; ``tokens`` int64 [T]: theirs."""

    def __init__(self, x, tokens, V, maps, mine, lp=None, H=None):
        T, K = x.shape
        self.x, self.maps, self.mine = torch.empty(T, K, dtype=x.dtype, device=x.device), maps, mine
        self.rows, self.place, self.count = maps.data_ptr(), maps.data_ptr() + 4 * T, maps.data_ptr() + 8 * T
        rc = nv.proto("b200_logprob_active", _ACTIVE)(nv.ptr(tokens), x.data_ptr(), x.stride(0), T, K, V, self.rows, self.place, nv.ptr(mine), self.count, nv.ptr(lp),
                                                      nv.ptr(H), self.x.data_ptr(), nv.stream())
        if rc:
            nv.check(rc, "logprob_active")
        nv.count_launch(1 + (tokens is not None))


def _on(x: torch.Tensor):
    """x's device as the current one; nothing to enter where it is."""
    return _HERE if not x.is_cuda or x.device.index == torch._C._cuda_getDevice() else torch.cuda.device(x.device)


def _chunks(T: int, V: int):
    """Columns of the vocabulary whose gradients exist at a time: chunks of about the same size."""
    n = -(-V // min(max(_CHUNK_BYTES // (2 * max(T, 1)), 4096), V))
    C = (-(-V // n) + 255) // 256 * 256
    return [(a, min(V, a + C)) for a in range(0, V, C)], min(C, V)


def _linear_forward(x, w, tokens, temperature, entropy, save):
    T, K = x.shape
    V = w.shape[0]
    if not nv.use_native(x):
        lp, H, _, _, _, stats = _rows_torch(x.float() @ w.float().t(), tokens, temperature, 0, entropy, False)
        return lp, H, (stats, None, None)
    new, dt = x.new_empty, torch.float32
    lp, H, stats = new((T,), dtype=dt) if tokens is not None else None, new((T,), dtype=dt) if entropy else None, new((T, 4), dtype=dt) if save else None
    if T == 0:
        return lp, H, (stats, None, None)
    maps = mine = None
    rows = count = 0
    if tokens is not None and T > _COMPACT_ROWS:
        maps, mine = new((2 * T + 1,), dtype=torch.int32), new((T,), dtype=torch.int64)
        act = _Active(x, tokens, V, maps, mine, lp, H)
        x, rows, count, tokens = act.x, act.rows, act.count, mine
    tiles = nv.proto("b200_gemm_head_tiles", [i32] * 3)(T, V, K)
    if tiles < 0:
        nv.check(-tiles, "gemm_head_tiles")
    work = new((tiles * T * 4 + T,), dtype=dt)                           # sums of tiles, then the tokens' logits
    part, inv_t, st, tok = work.data_ptr(), 1.0 / temperature, nv.stream(), nv.ptr(tokens)
    lt = part + tiles * T * 16
    rc = nv.proto("b200_gemm_head_sums", _HEAD_SUMS)(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), T, V, K, nv.dtype_code(x.dtype), count, tok, inv_t,
                                                     int(entropy), part, lt, st)
    if rc:
        nv.check(rc, "gemm_head_sums")
    rc = nv.proto("b200_logprob_finish", _FINISH)(part, tiles, T, V, count, rows, tok, lt, inv_t, nv.ptr(lp), nv.ptr(H), nv.ptr(stats), st)
    if rc:
        nv.check(rc, "logprob_finish")
    nv.count_launch(2)
    return lp, H, (stats, maps, mine)


def _linear_backward(x, w, tokens, temperature, saved, g, h, need_dx, need_dw):
    T, K = x.shape
    V = w.shape[0]
    stats, maps, mine = saved
    if not nv.use_native(x):
        d = _grad_torch(x.float() @ w.float().t(), tokens, temperature, stats, g, h, 0, V)
        return (d @ w.float()).to(x.dtype) if need_dx else None, (d.t() @ x.float()).to(w.dtype) if need_dw else None
    dev, dt, inv_t, f32_ = x.device, nv.dtype_code(x.dtype), 1.0 / temperature, torch.float32
    dw = torch.empty(V, K, dtype=w.dtype, device=dev) if need_dw else None
    if T == 0:
        return (torch.empty_like(x) if need_dx else None), (None if dw is None else dw.zero_())
    chunks, C = _chunks(T, V)
    ld = (C + 7) // 8 * 8
    dl = torch.empty(T, ld, dtype=x.dtype, device=dev)
    half = x.dtype == torch.float16
    scale = part = None
    if half:             # gradients of single logits lie below fp16's numbers: they are brought up by a power of two, the results back down
        scale = torch.empty(2, dtype=f32_, device=dev)
        fs = nv.proto("b200_logprob_scale", [vp, vp, vp, i64, f32, i32, vp, vp])
        nv.check(fs(nv.ptr(g), nv.ptr(h), nv.ptr(tokens), T, inv_t, V, nv.ptr(scale), nv.stream()), "logprob_scale")
        part = torch.empty(C, K, dtype=f32_, device=dev) if need_dw else None
    act, rows, count = None, 0, 0
    if maps is not None:
        act = _Active(x, None, V, maps, mine)
    elif tokens is not None and need_dw:                  # zeros times what stands in a row that is passed over would not do: it may be no number
        mine = x.new_empty((T,), dtype=torch.int64)
        act = _Active(x, tokens, V, x.new_empty((2 * T + 1,), dtype=torch.int32), mine)
    if act is not None:
        x, rows, count, tokens = act.x, act.rows, act.count, mine
    direct = len(chunks) == 1 and not half                # one product gives dx: no sums in 32 bits between chunks
    dx = torch.empty(T, K, dtype=x.dtype, device=dev) if need_dx else None
    acc = None
    if need_dx:
        acc = dx if direct and act is None else torch.empty(T, K, dtype=x.dtype if direct else f32_, device=dev)
    fg = nv.proto("b200_gemm_head_grads", _HEAD_GRADS)
    fc = nv.proto("b200_logprob_cast", [vp, vp, i64, vp, i32, vp])
    fa = nv.proto("b200_gemm_active", _ACTIVE_GEMM)
    st = nv.stream()
    ws = _stream_k_workspace(dev) if act is not None else None      # dx has few tiles where tokens are few: it is cut along the vocabulary
    ws = (0, 0) if ws is None else (ws.data_ptr(), ws.numel())

    def product(n, depth, c0, out, beta):
        """dl w of the chunk (rows), or dl^T x (depth)."""
        d, wc = dl[:, :n], w[c0:c0 + n]
        if act is None:
            gemm(d, x, a_mn=True, b_mn=True, out=out) if depth else gemm(d, wc, b_mn=True, out=out, beta=beta)
            return
        o = (x.data_ptr(), x.stride(0)) if depth else (wc.data_ptr(), w.stride(0))
        rc = fa(dl.data_ptr(), ld, int(depth), *o, 1, n if depth else T, K, T if depth else n, dt, count, int(depth), out.data_ptr(), out.stride(0),
                nv.dtype_code(out.dtype), beta, *ws, st)
        if rc:
            nv.check(rc, "gemm_active")
        nv.count_launch()
    for c0, c1 in chunks:
        n = c1 - c0
        nv.check(fg(nv.ptr(x), x.stride(0), nv.ptr(w[c0:c1]), w.stride(0), T, n, K, dt, count, rows, nv.ptr(tokens), V, c0, inv_t, nv.ptr(stats), nv.ptr(g), nv.ptr(h),
                    nv.ptr(scale), nv.ptr(dl), ld, st), "gemm_head_grads")
        if need_dx:
            product(n, False, c0, acc, 1.0 if c0 else 0.0)
        if need_dw and not half:
            product(n, True, c0, dw[c0:c1], 0.0)
        elif need_dw:
            product(n, True, c0, part[:n], 0.0)
            nv.check(fc(nv.ptr(part), nv.ptr(dw[c0:c1]), n * K, nv.ptr(scale), dt, st), "logprob_cast")
    if need_dx and act is not None:
        fr = nv.proto("b200_logprob_return", [vp, i32, vp, i32, i32, vp, vp, i32, vp])
        nv.check(fr(nv.ptr(acc), nv.dtype_code(acc.dtype), nv.ptr(dx), T, K, act.place, nv.ptr(scale), dt, st), "logprob_return")
    elif need_dx and not direct:
        nv.check(fc(nv.ptr(acc), nv.ptr(dx), T * K, nv.ptr(scale), dt, st), "logprob_cast")
    nv.count_launch(len(chunks) * (2 if half and need_dw else 1) + bool(need_dx and acc is not dx) + half)
    return dx, dw


class _LinearLogprobsFn(torch.autograd.Function):
    """Saves nothing of the size of the logits: the backward pass computes them again, a chunk at a time."""

    @staticmethod
    def forward(ctx, x, w, tokens, temperature, entropy):
        with _on(x):
            lp, H, saved = _linear_forward(x, w, tokens, temperature, entropy, True)
        if w.requires_grad:
            from ..utils.arena import note_use
            note_use(w, False)                   # its gradient arrives through autograd
        ctx.save_for_backward(x, w, tokens, *saved)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return lp, H

    @staticmethod
    def backward(ctx, g, h):
        _first_order_only("linear_token_logprobs")
        if g is None and h is None:
            return (None,) * 5
        x, w, tokens, *saved = ctx.saved_tensors
        g, h = (None if t is None else t.to(torch.float32).contiguous() for t in (g, h))
        with _on(x):
            dx, dw = _linear_backward(x, w, tokens, ctx.temperature, saved, g, h, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dw, None, None, None


def linear_token_logprobs(x: torch.Tensor, w: torch.Tensor, tokens: Optional[torch.Tensor], *, entropy: bool = False, temperature: float = 1.0) -> TokenLogprobs:
    """``token_logprobs(x @ w.T, tokens)`` for hidden states ``x`` [..., K] and an output projection ``w`` [vocab, K] (bf16 or fp16, K a multiple of 8),
    without the logits: their sums are taken from the product's accumulators (fp32), and in the backward pass, where the product is computed again, their
    gradients, which exist in 16 bits a chunk of the vocabulary at a time. Rows whose tokens are passed over leave the products before they begin (how many stays
    on the device) and may hold anything. Gradients for ``x`` and ``w``. Tensor cores add up a logit's K products with an error of about K * 2^-30 of it (4.6e-6 of a log
    probability at K = 4096, where ``token_logprobs`` has 6e-8 of the logits it is given)."""
    shape, native = x.shape, nv.use_native(x)
    if w.dim() != 2 or w.shape[0] < 1 or not shape or shape[-1] != w.shape[1] or x.dtype != w.dtype or x.device != w.device:
        raise ValueError("linear_token_logprobs: x [..., K] and w [vocab, K] must agree in K, type and device")
    if x.dtype not in (_TYPES[1:] if native else _TYPES):
        raise TypeError(f"linear_token_logprobs: x and w must be bf16 or fp16, not {x.dtype}; token_logprobs takes logits of 32 bits")
    if native and (shape[-1] % 8 or w.stride(1) != 1 or w.stride(0) % 8 or w.stride(0) < shape[-1] or w.data_ptr() % 16):
        raise ValueError("linear_token_logprobs: rows of w must be contiguous, start at multiples of 16 bytes and have a multiple of 8 values")
    shape = shape[:-1]
    if tokens is not None:
        _check("linear_token_logprobs", tokens, shape, x.device)
    _check_temperature("linear_token_logprobs", temperature)
    if tokens is None and not entropy:
        raise ValueError("linear_token_logprobs: without tokens there are entropies only")
    rows = _as_rows(x)
    if max(rows.shape[0], *w.shape) >= _MOST:
        raise ValueError(f"linear_token_logprobs: {rows.shape[0]} tokens, a vocabulary of {w.shape[0]}; there is room for {_MOST - 1}")
    if native:
        K = rows.shape[1]
        if rows.data_ptr() % 16 or rows.stride(0) % 8 or rows.stride(0) < K:     # a row to a multiple of 16 bytes, none upon another
            rows = rows.clone(memory_format=torch.contiguous_format)
        if rows.shape[0] == 1 and rows.stride(0) != K:                           # one row is contiguous, whatever its stride says
            rows = rows.view(K).unsqueeze(0)
    flat = None if tokens is None else tokens.reshape(-1).contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        lp, H = _LinearLogprobsFn.apply(rows, w, flat, temperature, entropy)
    else:
        with _on(rows):
            lp, H, _ = _linear_forward(rows, w, flat, temperature, entropy, False)
    if len(shape) == 1:
        return TokenLogprobs(lp, H)
    return TokenLogprobs(None if lp is None else lp.view(shape), None if H is None else H.view(shape))
