"""Sequence operators on the paths that a size or an address chooses: bfloat16 heads of 65 .. 128 columns whose probabilities enter the
products with 8 bits (64 rows a sequence and more; 512 and more for the gradients), rows at odd multiples of two bytes, rows at the largest
distance and beyond it.  Tolerances against the definition in float64 as test_sequence_long_gpu.py derives them; forms of the same call
that only load in another way answer with the same bits."""
import pytest
import test_sequence_long_gpu as long_sequences
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from nl_vsgg_amd.lib import sequence_ops
    return sequence_ops


_i32, _normal, _run = long_sequences._i32, long_sequences._normal, long_sequences._run


# ---- the kernels of long bfloat16 sequences --------------------------------------------------------------------------------


@pytest.mark.parametrize("mask", long_sequences.MASKS)
@pytest.mark.parametrize("d", [66, 96, 128])
def test_long_bfloat16_masks(ops, mask, d):
    """two query heads share a key head; a key tile's work falls to several workgroups and is joined"""
    lens = [1100, 999]
    long_sequences._check(ops, lens, lens, 2, 1, d, torch.bfloat16, seed=61, tail=(5, 5), **long_sequences.MASKS[mask])


@pytest.mark.parametrize("d", [68, 100, 126, 128])
@pytest.mark.parametrize("hq,hk", [(8, 8), (8, 1)])
def test_long_bfloat16_heads(ops, d, hq, hk):
    """as many key tiles as leave each its own workgroup (8 key heads), and few of many query heads"""
    lens = [600, 513, 700, 650, 599, 530, 610, 577]
    long_sequences._check(ops, lens, lens, hq, hk, d, torch.bfloat16, seed=63, causal=True)


@pytest.mark.parametrize("d", [80, 128])
def test_long_bfloat16_queries_and_keys_of_other_lengths(ops, d):
    """rows that see nothing, more keys than queries and fewer, tails of tiles"""
    x, (out, dq, dk, dv) = long_sequences._check(ops, [700, 1, 900, 641], [650, 40, 1100, 641], 4, 2, d, torch.bfloat16, seed=65, tail=(9, 17), causal=True)
    assert not out[:50].any() and not dq[:50].any() and not out[2242:].any() and not dk[2431:].any() and not dv[2431:].any()


@pytest.mark.parametrize("d", [96, 128])
@pytest.mark.parametrize("rows", [64, 65, 127, 128, 129, 511, 512])
def test_bfloat16_where_the_kernels_change(ops, d, rows):
    """64 rows a sequence and one more or fewer, 512 likewise"""
    for n in (rows, rows + 1, rows - 1):
        long_sequences._check(ops, [n, n], [n, n], 2, 2, d, torch.bfloat16, seed=67, score_cap=5.0)


# ---- addresses and strides -------------------------------------------------------------------------------------------------


def _shifted(x, by=1, pad=3):
    """the same numbers in rows that begin `by` elements behind an aligned address and lie an odd number of elements apart"""
    return torch.full((*x.shape[:-1], x.shape[-1] + pad), 7.0, dtype=x.dtype, device="cuda")[..., by:by + x.shape[-1]].copy_(x)


@pytest.mark.parametrize("d", [2, 64, 96, 128, 242])
@pytest.mark.parametrize("lens", [[37, 90], [600, 530]])
def test_attention_rows_at_odd_addresses(ops, d, lens):
    """bfloat16, an even head dim: all of q, k, v and dout, and each alone, against the definition"""
    x = long_sequences._inputs(lens, lens, 2, 1, d, torch.bfloat16, 71)
    ref = long_sequences._ref(*x, causal=True)
    for odd in ((0, 1, 2, 3), (0,), (1,), (2,), (3,)):
        y = [_shifted(t) if i in odd else t for i, t in enumerate(x[:4])]
        for n, g, (r, tol) in zip(("out", "dq", "dk", "dv"), _run(ops, *y, *x[4:], causal=True), ref):
            assert (g.double().cpu() - r).norm() <= tol, (n, odd)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [64, 128, 242])
def test_step_over_rows_at_odd_addresses(ops, dtype, d):
    q, kc, vc, lens = _normal(1, 3, 4, d, dtype=DT[dtype]), _normal(2, 3, 500, 2, d, dtype=DT[dtype]), _normal(3, 3, 500, 2, d, dtype=DT[dtype]), [500, 1, 77]
    k, v = (torch.cat([c[i, :n] for i, n in enumerate(lens)]) for c in (kc, vc))
    (out, tol), *_ = long_sequences._ref(q, k, v, q, [0, 1, 2, 3], [0, 500, 501, 578])
    for odd in ((0, 1, 2), (0,), (1,), (2,)):
        args = [_shifted(t) if i in odd else t for i, t in enumerate((q, kc, vc))]
        assert (ops.attention_step(*args, _i32(lens)).double().cpu() - out).norm() <= tol, odd


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (242, 242), (128, 96)])
def test_rotary_rows_at_odd_addresses(ops, dtype, inter, d, rot):
    """any alignment of two bytes or more loads the same numbers: the same bits, forward and backward"""
    q, k, pos, freq = _normal(1, 21, 3, d, dtype=DT[dtype]), _normal(2, 21, 2, d, dtype=DT[dtype]), torch.arange(21, device="cuda"), ops.rotary_frequencies(rot, device="cuda")
    w, dy = (1 + 0.1 * _normal(3, d)).requires_grad_(), [_normal(4, 21, 3, d, dtype=DT[dtype]), _normal(5, 21, 2, d, dtype=DT[dtype])]

    def both(form):
        leaves = [form(q).requires_grad_(), form(k).requires_grad_()]
        y = ops.rotary_qk(*leaves, pos, freq, w, w, interleaved=inter)
        return [*y, *torch.autograd.grad(y, [*leaves, w], [form(g) for g in dy])]
    for a, b in zip(both(lambda x: _shifted(x).detach()), both(lambda x: x.clone())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,rows", [("bf16", 130), ("bf16", 300), ("f32", 70), ("f32", 300)])
@pytest.mark.parametrize("over", [0, 64])
def test_attention_rows_far_apart(ops, dtype, rows, over):
    """2^24 bytes a row, the most that the kernels step over, and a little more, which is copied; all of a call's rows in one buffer that
    passes 2^31 bytes"""
    dt, d = DT[dtype], 64
    step = (1 << 24) // torch.finfo(dt).bits * 8 + over
    room = torch.zeros(rows * step, dtype=dt, device="cuda")
    near = [_normal(81 + i, rows, h, d, dtype=dt) for i, h in enumerate((4, 2, 2, 4))]
    far, at = [], 128
    for x in near:
        far.append(torch.as_strided(room, x.shape, (step, d, 1), at).copy_(x))
        at += x[0].numel() + 32
    off = [0, rows // 3, rows]
    for a, b in zip(_run(ops, *far, off, off, causal=True), _run(ops, *near, off, off, causal=True)):
        assert torch.equal(a, b)


def test_step_rows_far_apart(ops):
    """2^22 bytes a row of the cache and no more: a cache is never copied"""
    n, cap, d = 2, 300, 64
    step = (1 << 22) // 2
    room = torch.zeros(cap * step + 4096, dtype=torch.bfloat16, device="cuda")
    near = [_normal(91 + i, n, cap, 2, d, dtype=torch.bfloat16) for i in range(2)]
    far = [torch.as_strided(room, x.shape, (4 * d, step, d, 1), 128 + 1024 * i).copy_(x) for i, x in enumerate(near)]
    q, lens = _normal(93, n, 4, d, dtype=torch.bfloat16), _i32([300, 201])
    assert torch.equal(ops.attention_step(q, *far, lens), ops.attention_step(q, *near, lens))
    wide = torch.as_strided(room, (n, 4, 2, d), (4 * d, step + 64, d, 1))
    with pytest.raises(ValueError, match="bytes apart"):
        ops.attention_step(q, wide, wide, lens)


def test_rotary_rows_far_apart(ops):
    rows, d, step = 140, 64, (1 << 24) + 32
    room = torch.zeros(rows * step, dtype=torch.bfloat16, device="cuda")
    q, k, pos, freq = _normal(1, rows, 2, d, dtype=torch.bfloat16), _normal(2, rows, 1, d, dtype=torch.bfloat16), torch.arange(rows, device="cuda"), ops.rotary_frequencies(d, device="cuda")
    far = [torch.as_strided(room, x.shape, (step, d, 1), at).copy_(x) for x, at in ((q, 0), (k, 1024))]
    for a, b in zip(ops.rotary_qk(*far, pos, freq), ops.rotary_qk(q, k, pos, freq)):
        assert torch.equal(a, b)
