"""Operators over packed sequences of tokens: what a relation-transformer layer (`lib/transformer.py:20-30, 49-58`) is made of,
as single calls -- for training it (gradients, dropout), for longer clips (rotary positions, order and prefix masks, distance
bias, capped scores) and for clips that grow token by token.

    q, k = rotary_qk(q, k, positions, rotary_frequencies(64, device=q.device), q_weight, k_weight)
    out = packed_attention(q, k, v, seq_off, causal=True)            # differentiable in q, k, v
    x = dropout_add(proj(out.flatten(1)), x, p=0.1, rng_state=state) # x + dropout(...), no mask stored
    out = attention_step(q1, k_cache, v_cache, lengths)              # one new token a sequence

float32 or bfloat16 throughout a call (statistics and sums in float32); tensors on one MI355X, no CPU path.  Work is enqueued
on the current stream of the tensors' device and may be captured into a graph; nothing is read back.  (As with every torch
operator: to capture a backward pass, let the results of eager calls on the same leaves go first.)  Bad arguments raise
ValueError before anything is launched.  Derivatives are reverse-mode and of first order: tensors with a forward-mode tangent are
refused, and so are calls under a tracer that would record the result's allocation without the kernel.  The last dimension of
q / k / v must be contiguous (others are copied), other strides are free."""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _native as nat

_DTYPES = {torch.float32: nat.DTYPE_F32, torch.bfloat16: nat.DTYPE_BF16}
_ATT_SIZE, _STEP_SIZE, _ROT_SIZE = (C.sizeof(t) for t in (nat.SttranAttention, nat.SttranAttentionStep, nat.SttranRotary))
_MAX_ROW_BYTES, _MAX_CACHE_ROW_BYTES, _MAX_HEAD_ROWS = 1 << 24, 1 << 22, (1 << 29) - 1024


def _launch(fn, args, dev):
    """`fn(args..., stream)` on the device's current stream; the entry points have no handle and so no device of their own.  (The
    stream's raw handle: building a torch.cuda.Stream costs 2 us of the 11 that a small call takes.)"""
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc != nat.STTRAN_OK:
        raise nat.SttranError(rc, f"{fn.__name__} failed")


_tracing, _dispatch_modes, _dispatch_mode, _PROXY = (torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode,
                                                     torch._C._TorchDispatchModeKey.PROXY)


def _no_tangents(name, *tensors):
    """A kernel gives its result no tangent, which reads as a derivative of zero.  (Called at a forward-mode level alone: by
    themselves these checks would take 0.7 us of the 8 that a small call takes.)"""
    if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError(f"{name} has no forward-mode derivative, and one of its tensors has a tangent")


def _checked(name, *tensors):
    """The library, if `tensors` share a served dtype and device and the call may run as it is."""
    t = tensors[0]
    if forward_ad._current_level >= 0:
        _no_tangents(name, *tensors)
    if _tracing() or (_dispatch_modes() and _dispatch_mode(_PROXY)):
        raise RuntimeError(f"{name} cannot be traced: its kernels are launched beside torch's operators")
    if not t.is_cuda:
        raise RuntimeError(f"{name} runs on an MI355X only (no CPU path)")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: float32 or bfloat16 tensors, not {t.dtype}")
    for x in tensors[1:]:
        if x.dtype != t.dtype or x.device != t.device:
            raise ValueError(f"{name}: tensors must share dtype and device, got {x.dtype} on {x.device} next to {t.dtype} on {t.device}")
    return nat.load()


def _rows(x, limit=True):
    """x as the kernels take it: innermost dimension contiguous, no overlapping row stride above the limit."""
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        return x.contiguous()
    if limit and x.shape[-3] > 1 and x.stride(-3) * x.element_size() > _MAX_ROW_BYTES:
        return x.contiguous()
    return x


def _small(name, what, x, dtype, shape, dev):
    """An index / parameter vector: exact dtype, shape and device, contiguous."""
    if forward_ad._current_level >= 0:
        _no_tangents(name, x)
    if x.dtype != dtype or tuple(x.shape) != shape or x.device != dev:
        raise ValueError(f"{name}: {what} must be {dtype} {list(shape)} on {dev}, got {x.dtype} {list(x.shape)} on {x.device}")
    return x.contiguous()


def _like(x):
    """An uninitialised contiguous tensor of x's shape (half the time of torch.empty with its shape, dtype and device)."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _heads(name, q, k, v):
    if not (1 <= q.shape[-1] <= 256) or k.shape[-1] != q.shape[-1] or v.shape != k.shape:
        raise ValueError(f"{name}: head dims 1..256 alike in q, k, v and k, v of one shape; got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    hq, hk = q.shape[-2], k.shape[-2]
    if hq < 1 or hk < 1 or hq % hk or hq > 4096:
        raise ValueError(f"{name}: {hq} query heads cannot share {hk} key heads")
    return hq, hk


def _number(name, what, x):
    """A plain number; of a tensor its value, unless a gradient would get lost with it."""
    if isinstance(x, torch.Tensor):
        if forward_ad._current_level >= 0:
            _no_tangents(name, x)
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name}: {what} is a number, it gets no gradient")
    return float(x)


def _score(name, scale, cap, d):
    scale = d ** -0.5 if scale is None else _number(name, "scale", scale)
    cap = 0.0 if cap is None else _number(name, "score_cap", cap)
    if not math.isfinite(scale) or not math.isfinite(cap) or cap < 0:
        raise ValueError(f"{name}: scale must be finite and score_cap finite and >= 0 (0: none)")
    if not max(abs(scale), cap, abs(scale) / cap if cap else 0.0) < 1e38 or (cap and cap < 1e-37):
        raise ValueError(f"{name}: scale, score_cap and their quotient must fit float32")
    return scale, cap


# ---- attention over packed sequences -----------------------------------------------------------------------------------


def _attention_struct(q, k, v, seq_off, key_off, prefix, slope, causal, cap, scale):
    a = nat.SttranAttention(_ATT_SIZE, _DTYPES[q.dtype], seq_off.shape[0] - 1, q.shape[1], k.shape[1], q.shape[2], q.shape[0], k.shape[0],
                            q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                            v.stride(1), seq_off.data_ptr(), key_off.data_ptr(), _ptr(prefix), _ptr(slope), int(causal), cap, scale)
    for n, rows in (("q", q.shape[0]), ("k", k.shape[0]), ("v", k.shape[0])):      # a single row's stride says nothing
        if rows <= 1:
            setattr(a, n + "_row_stride", 0)
    return a


def _attention_forward(q, k, v, seq_off, key_off, prefix, slope, causal, cap, scale, train):
    lib = nat.load()
    out = _like(q)
    a = _attention_struct(q, k, v, seq_off, key_off, prefix, slope, causal, cap, scale)
    a.out = out.data_ptr()
    low = lse = None
    if train:
        lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
        low = torch.empty_like(out) if q.dtype == torch.bfloat16 else None
        a.lse, a.out_residual = lse.data_ptr(), _ptr(low)
    need = lib.sttran_attention_workspace_bytes(C.byref(a), 0)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _launch(lib.sttran_attention_forward, (C.byref(a),), q.device)
    return out, low, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seq_off, key_off, prefix, slope, causal, cap, scale):
        out, low, lse = _attention_forward(q, k, v, seq_off, key_off, prefix, slope, causal, cap, scale, True)
        ctx.save_for_backward(q, k, v, seq_off, key_off, prefix, slope, out, low, lse)
        ctx.plain = (causal, cap, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, seq_off, key_off, prefix, slope, out, low, lse = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _no_tangents("packed_attention", dout)
        lib = nat.load()
        dout = _rows(dout)
        a = _attention_struct(q, k, v, seq_off, key_off, prefix, slope, *ctx.plain)
        grads = [_like(x) for x in (q, k, v)]
        a.out, a.out_residual, a.lse = out.data_ptr(), _ptr(low), lse.data_ptr()
        a.dout, a.dout_row_stride, a.dout_head_stride = dout.data_ptr(), dout.stride(0) if dout.shape[0] > 1 else 0, dout.stride(1)
        a.dq, a.dk, a.dv = (g.data_ptr() for g in grads)
        need = lib.sttran_attention_workspace_bytes(C.byref(a), 1)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _launch(lib.sttran_attention_backward, (C.byref(a),), q.device)
        return (*grads, None, None, None, None, None, None, None)


def packed_attention(q, k, v, seq_off, key_off=None, *, causal=False, prefix_len=None, distance_slope=None, score_cap=0.0, scale=None):
    """Softmax attention inside each of many sequences packed behind one another; differentiable in q, k and v.

    q [rows, query heads, head dim], k / v [key rows, key heads, head dim]; head dims 1..256, query heads a multiple of the key heads
    (query head h reads key head h // (query heads // key heads)).  `seq_off` (int32 [sequences + 1]) bounds each sequence's query
    rows, `key_off` its key rows (None: the same rows).  The newest query stands at the newest key: row i of lq queries over lk keys
    has place i + lk - lq.

    causal          a row sees keys up to its place only; of `prefix_len` (int32 [sequences]) the first keys stay visible to all rows
    distance_slope  float32 [query heads]: z -= slope * |place - key|; a constant, it gets no gradient
    score_cap       z = cap * tanh(z / cap) before the distance is taken off; 0: none
    scale           of q.k, head_dim ** -0.5 if None

    Rows that see no key, and rows outside every sequence, come out as zeros (and get zero gradients).  Offsets must ascend within
    the tensors' rows; they live on the device and are not checked (wrong ones give wrong rows, never an access out of bounds).
    Values under a mask do not reach a result, infinities and NaN included (a call that meets them is slow).  Gradients are the
    same in every run.  In bfloat16, probabilities and their derivatives are rounded to 8 bits on their way into the products
    where sequences are long, and carry 16 where they are short (below 64 rows in the forward pass, 512 in the backward), by the
    average over the call: a short sequence answers a little less exactly beside long ones (up to 1.5 times its result's own
    rounding) than by itself."""
    name = "packed_attention"
    _checked(name, q, k, v)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{name}: q, k, v are [rows, heads, head dim]")
    hq, _ = _heads(name, q, k, v)
    dev = q.device
    if seq_off.dim() != 1 or seq_off.shape[0] < 1:
        raise ValueError(f"{name}: seq_off is a vector of sequences + 1 offsets")
    n = seq_off.shape[0]
    if n - 1 > 1 << 30:
        raise ValueError(f"{name}: at most 2^30 sequences a call")
    seq_off = _small(name, "seq_off", seq_off, torch.int32, (n,), dev)
    if key_off is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"{name}: {q.shape[0]} query rows over {k.shape[0]} key rows need key_off")
        key_off = seq_off
    else:
        key_off = _small(name, "key_off", key_off, torch.int32, (n,), dev)
    if prefix_len is not None:
        if not causal:
            raise ValueError(f"{name}: prefix_len is part of the causal mask")
        prefix_len = _small(name, "prefix_len", prefix_len, torch.int32, (n - 1,), dev)
    if distance_slope is not None:
        if distance_slope.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name}: distance_slope is a constant, it gets no gradient")
        distance_slope = _small(name, "distance_slope", distance_slope, torch.float32, (hq,), dev)
    if max(q.shape[0] * hq, k.shape[0] * k.shape[1]) >= _MAX_HEAD_ROWS:
        raise ValueError(f"{name}: rows times heads must be below 2^29 - 1024 a call")
    scale, cap = _score(name, scale, score_cap, q.shape[2])
    q, k, v = _rows(q), _rows(k), _rows(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, seq_off, key_off, prefix_len, distance_slope, bool(causal), cap, scale)
    return _attention_forward(q, k, v, seq_off, key_off, prefix_len, distance_slope, bool(causal), cap, scale, False)[0]


def attention_step(q, k_cache, v_cache, lengths, *, distance_slope=None, score_cap=0.0, scale=None, out=None):
    """Attention of one new token a sequence over its cache.

    q [sequences, query heads, head dim], caches [sequences, capacity, key heads, head dim], `lengths` int32 [sequences]: live rows of
    each cache, the new token's own key (already written) being the last of them; rows behind are not read, length 0 gives zeros,
    a length above the capacity counts as the capacity.  Scores as in packed_attention.  `out`: a contiguous tensor like q to write
    into (q itself, too).  No gradient."""
    name = "attention_step"
    lib = _checked(name, q, k_cache, v_cache)
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.dim() != 4 or k_cache.shape[0] != q.shape[0]:
        raise ValueError(f"{name}: q [sequences, heads, head dim] and caches [sequences, capacity, heads, head dim]")
    hq, hk = _heads(name, q, k_cache, v_cache)
    n, dev, d = q.shape[0], q.device, q.shape[2]
    if n > 65535:
        raise ValueError(f"{name}: at most 65535 sequences a call")
    if k_cache.shape[1] > 1 << 30:
        raise ValueError(f"{name}: at most 2^30 rows a cache")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")
    lengths = _small(name, "lengths", lengths, torch.int32, (n,), dev)
    if distance_slope is not None:
        distance_slope = _small(name, "distance_slope", distance_slope, torch.float32, (hq,), dev)
    scale, cap = _score(name, scale, score_cap, d)
    q = _rows(q, limit=False)
    if out is None:
        out = _like(q)
    else:
        if forward_ad._current_level >= 0:
            _no_tangents(name, out)
        if out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
            raise ValueError(f"{name}: out must be contiguous and like q")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} has no gradient: out must not require one")
        torch.autograd.graph.increment_version(out)        # an earlier call's backward pass that saved it must not use what is written now
    for what, x in (("k_cache", k_cache), ("v_cache", v_cache)):
        if d > 1 and x.stride(3) != 1 or x.shape[1] > 1 and x.stride(1) * x.element_size() > _MAX_CACHE_ROW_BYTES:
            raise ValueError(f"{name}: {what}'s head dim must be contiguous and its rows at most {_MAX_CACHE_ROW_BYTES} bytes apart (a cache is never copied)")
    cap_rows = k_cache.shape[1]
    a = nat.SttranAttentionStep(_STEP_SIZE, _DTYPES[q.dtype], n, hq, hk, d, cap_rows, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                q.stride(0), q.stride(1), k_cache.stride(0), k_cache.stride(1) if cap_rows > 1 else 0, k_cache.stride(2),
                                v_cache.stride(0), v_cache.stride(1) if cap_rows > 1 else 0, v_cache.stride(2), lengths.data_ptr(),
                                _ptr(distance_slope), cap, scale, out.data_ptr())
    need = lib.sttran_attention_step_workspace_bytes(C.byref(a))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _launch(lib.sttran_attention_step, (C.byref(a),), dev)
    return out


# ---- per-head norm and rotary positions --------------------------------------------------------------------------------


def rotary_frequencies(rotary_dim, *, base=10000.0, factor=1.0, method="linear", original_length=None, low_turns=1.0, high_turns=32.0,
                       device=None):
    """Angles a position step of the rotary_dim / 2 pairs, float32: base ** (-2 i / rotary_dim), stretched for contexts `factor`
    times as long.

    "linear"    every frequency / factor (positions are squeezed into the old range)
    "base"      base * factor ** (rotary_dim / (rotary_dim - 2)): the slowest pair is stretched by factor, the fastest not at all
    "by_parts"  pairs that turn more than high_turns times over `original_length` keep their frequency, those below low_turns are
                divided by factor, linearly in between"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_frequencies: rotary_dim is a positive even number")
    if not (factor >= 1.0 and base > 1.0):
        raise ValueError("rotary_frequencies: factor >= 1 and base > 1")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if method == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-2.0 * i / rotary_dim)
    if method == "linear" or (method == "base" and rotary_dim == 2):
        freq = freq / factor
    elif method == "by_parts":
        if not original_length or not high_turns > low_turns:
            raise ValueError("rotary_frequencies: by_parts needs original_length and low_turns < high_turns")
        turns = original_length * freq / (2 * math.pi)
        keep = ((turns - low_turns) / (high_turns - low_turns)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    elif method != "base":
        raise ValueError(f"rotary_frequencies: method {method!r} is not one of linear, base, by_parts")
    return freq.to(device=device, dtype=torch.float32)


def _rotary_struct(q, k, positions, freq, q_weight, k_weight, eps, interleaved):
    return nat.SttranRotary(_ROT_SIZE, _DTYPES[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2], 2 * freq.shape[0], q.data_ptr(),
                            k.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1), positions.data_ptr(), freq.data_ptr(),
                            _ptr(q_weight), _ptr(k_weight), eps, int(interleaved))


def _rotary_forward(q, k, positions, freq, q_weight, k_weight, eps, interleaved):
    a = _rotary_struct(q, k, positions, freq, q_weight, k_weight, eps, interleaved)
    yq, yk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=q.device)
    a.q_out, a.k_out = yq.data_ptr(), yk.data_ptr()
    _launch(nat.load().sttran_rotary_forward, (C.byref(a),), q.device)
    return yq, yk


class _RotaryQK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freq, q_weight, k_weight, eps, interleaved):
        ctx.save_for_backward(q, k, positions, freq, q_weight, k_weight)
        ctx.plain = (eps, interleaved)
        return _rotary_forward(q, k, positions, freq, q_weight, k_weight, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, positions, freq, wq, wk = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _no_tangents("rotary_qk", dyq, dyk)
        lib, dev = nat.load(), q.device
        dyq, dyk = _rows(dyq, limit=False), _rows(dyk, limit=False)
        a = _rotary_struct(q, k, positions, freq, wq, wk, *ctx.plain)
        dq, dk = _like(q), _like(k)
        a.dq_out, a.dk_out, a.dq, a.dk = dyq.data_ptr(), dyk.data_ptr(), dq.data_ptr(), dk.data_ptr()
        a.dq_row_stride, a.dq_head_stride, a.dk_row_stride, a.dk_head_stride = dyq.stride(0), dyq.stride(1), dyk.stride(0), dyk.stride(1)
        dwq = dwk = None
        if wq is not None:
            dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
            need = lib.sttran_rotary_workspace_bytes(C.byref(a))
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            a.dq_weight, a.dk_weight, a.workspace, a.workspace_bytes = dwq.data_ptr(), dwk.data_ptr(), ws.data_ptr(), need
        _launch(lib.sttran_rotary_backward, (C.byref(a),), dev)
        return dq, dk, None, None, dwq, dwk, None, None


def rotary_qk(q, k, positions, frequencies, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False):
    """Rotary positions of queries and keys, behind a norm of every head's row where the weights are given; differentiable.

    q [tokens, query heads, head dim], k [tokens, key heads, head dim] (views of one projection are fine), `positions` int64 [tokens],
    `frequencies` float32 [pairs] on the device (rotary_frequencies): the first 2 * pairs columns are turned by position * frequency
    (angles in 64 bits, however far the position), the others pass.  Pairs are neighbours (2i, 2i + 1) with `interleaved`, else column i
    and i + pairs.  q_weight / k_weight (float32 [head dim], both or neither): y = weight * x / sqrt(mean(x^2) + eps) first.
    Returns contiguous (q, k)."""
    name = "rotary_qk"
    _checked(name, q, k)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{name}: q and k are [tokens, heads, head dim] of the same tokens and head dim")
    d, dev = q.shape[2], q.device
    if not 1 <= d <= 256 or not 1 <= q.shape[1] <= 4096 or not 1 <= k.shape[1] <= 4096:
        raise ValueError(f"{name}: head dims 1..256, 1..4096 heads")
    positions = _small(name, "positions", positions, torch.int64, (q.shape[0],), dev)
    if frequencies.dim() != 1 or 2 * frequencies.shape[0] > d:
        raise ValueError(f"{name}: frequencies of at most {d // 2} pairs")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: frequencies are constants, they get no gradient")
    frequencies = _small(name, "frequencies", frequencies, torch.float32, (frequencies.shape[0],), dev)
    if (q_weight is None) != (k_weight is None):
        raise ValueError(f"{name}: q_weight and k_weight are given both or neither")
    if q_weight is not None:
        q_weight = _small(name, "q_weight", q_weight, torch.float32, (d,), dev)
        k_weight = _small(name, "k_weight", k_weight, torch.float32, (d,), dev)
    eps = _number(name, "eps", eps)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"{name}: eps is finite and >= 0")
    q, k = _rows(q, limit=False), _rows(k, limit=False)
    args = (q, k, positions, frequencies, q_weight, k_weight, eps, bool(interleaved))
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, q_weight, k_weight)):
        return _RotaryQK.apply(*args)
    return _rotary_forward(*args)


# ---- dropout -----------------------------------------------------------------------------------------------------------


def _dropout(x, residual, p, rng_state, key, offset, used):
    y = _like(x)
    _launch(nat.load().sttran_dropout_add, (x.data_ptr(), _ptr(residual), y.data_ptr(), x.numel(), _DTYPES[x.dtype], p, _ptr(rng_state), key,
                                            offset, _ptr(used)), x.device)
    return y


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng_state, key, offset):
        # the state may move on (or be replayed from a graph with other contents) before the backward pass: keep what was drawn from
        used = None if rng_state is None else torch.empty(2, dtype=torch.int64, device=x.device)
        y = _dropout(x, residual, p, rng_state, key, offset, used)
        ctx.save_for_backward(used)
        ctx.plain = (p, key, offset, residual is not None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        used, = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _no_tangents("dropout_add", dy)
        p, key, offset, added = ctx.plain
        dx = _dropout(dy.contiguous(), None, p, used, key, offset, None) if ctx.needs_input_grad[0] else None
        return dx, dy if added and ctx.needs_input_grad[1] else None, None, None, None, None


def dropout_add(x, residual=None, *, p, rng_state=None, seed=None, offset=0):
    """residual + dropout(x): each element of x is dropped with probability p, kept ones are divided by 1 - p; differentiable in x and
    residual.  The mask is not stored: it is a function of (seed, offset, element), recomputed by the backward pass.

    Give `seed` and `offset` (integers; another offset, another mask: count the calls of a training run in it), or `rng_state`, an
    int64 [2] tensor (seed, offset) on the device, which a captured graph reads anew at every replay (`rng_state[1] += 1` between
    calls).  Element i is dropped where word i of the stream is below round(p * 2^32); word i is word i % 4 of the Philox 4x32-10
    block with counter (i // 4, offset) and key seed."""
    name = "dropout_add"
    _checked(name, x, *([residual] if residual is not None else []))
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{name}: residual {list(residual.shape)} is not x's shape {list(x.shape)}")
    p = _number(name, "p", p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"{name}: p is in [0, 1)")
    if (rng_state is None) == (seed is None):
        raise ValueError(f"{name}: give rng_state or seed")
    key = off = 0
    if rng_state is not None:
        rng_state = _small(name, "rng_state", rng_state, torch.int64, (2,), x.device)
    else:
        key, off = int(seed), int(offset)
        if not (-2 ** 63 <= key < 2 ** 63 and -2 ** 63 <= off < 2 ** 63):
            raise ValueError(f"{name}: seed and offset are 64-bit integers")
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutAdd.apply(x, residual, p, rng_state, key, off)
    return _dropout(x, residual, p, rng_state, key, off, None)
