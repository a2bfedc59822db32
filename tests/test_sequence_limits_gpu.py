"""The sequence operators at the limits of their arguments: what lies beside a buffer, the largest and smallest numbers, the largest calls.

Tolerances of attention are those that test_sequence_long_gpu.py derives (half a step, 2^-8, of the 2-norm in bfloat16, 4e-6 of it in
float32 and what dp - delta loses), against the definition in float64.  A cap adds to them: tanh is taken to 3 * 2^-24 of itself, with the
roundings of its argument and of the product with the cap 5 * 2^-24 of a score, and a probability is off by that times the score, below 6
here: 2e-6 of itself, within float32's 4e-6 as it is spread over the keys; in bfloat16, up to a cap of 1024, 1024 * 2^-22 = 2.5e-4 of
itself at most, a sixteenth of 2^-8, where the roundings that are counted in 2^-8 add up to sqrt(2 / 3) of it."""
import math

import pytest
import test_sequence_long_gpu as long_sequences
import test_sequence_ops_gpu as short_sequences
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from nl_vsgg_amd.lib import sequence_ops
    return sequence_ops


@pytest.fixture(scope="module")
def native(ops):
    from nl_vsgg_amd import _native
    return _native


def _normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float32).to(dtype).cuda()


# ---- dropout -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [1, 2, 3, 5, 7, 8, 9, 15, 17, 2047, 2049])
def test_dropout_leaves_what_lies_behind_its_elements(ops, native, dtype, n):
    """the C entry on a part of a larger buffer, at an address of 16 bytes' alignment: only its n elements are written"""
    dt, stream = DT[dtype], torch.cuda.current_stream().cuda_stream
    x, r = _normal(1, n + 24, dtype=dt), _normal(2, n + 24, dtype=dt)
    y = torch.full_like(x, 7.0)
    for at in (8, 0):
        y.fill_(7.0)
        rc = native.load().sttran_dropout_add(x[at:].data_ptr(), r[at:].data_ptr(), y[at:].data_ptr(), n, native.DTYPE_BF16 if dtype == "bf16" else native.DTYPE_F32,
                                              0.25, None, 5, 6, None, stream)
        assert rc == 0
        assert bool((y[:at] == 7).all()) and bool((y[at + n:] == 7).all())
        assert torch.equal(y[at:at + n], ops.dropout_add(x[at:at + n].clone(), r[at:at + n].clone(), p=0.25, seed=5, offset=6))


@pytest.mark.parametrize("dtype", DT)
def test_dropout_of_everything(ops, dtype):
    """where p * 2^32 rounds to 2^32 no word is as large: nothing is kept, infinities neither.  Word 2 is 2^32 - 1 at this key and offset,
    the largest there is (the first offset under key 0 that a search over the generator's definition finds)"""
    key, offset, at = 0, 389732782, 2
    assert short_sequences._philox(0, offset, key)[at] == 2 ** 32 - 1
    x = torch.full((8,), math.inf, dtype=DT[dtype], device="cuda")
    for p in (1 - 2.0 ** -34, 1 - 2.0 ** -53):
        assert not ops.dropout_add(x, p=p, seed=key, offset=offset).any()
    kept = ops.dropout_add(x, p=1 - 2.0 ** -32, seed=key, offset=offset)            # round(p * 2^32) = 2^32 - 1: that word alone is kept
    assert kept[at] == math.inf and kept.isinf().sum() == 1


# ---- attention ---------------------------------------------------------------------------------------------------------


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _run(ops, q, k, v, do, off_q, off_k, **kw):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*leaves, _i32(off_q), _i32(off_k), **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, do)]


@pytest.mark.parametrize("dtype,d,rows", [("f32", 129, (1 << 26) + 3), ("bf16", 66, (1 << 28) + 5)])
def test_attention_gradients_of_the_most_rows(ops, dtype, d, rows):
    """a row for each of more lanes than a launch has threads: queries and gradient broadcast over the rows, the last 50 see 40 keys and
    answer as by themselves (their tiles begin elsewhere: sums in another order, 2^-6 of the largest in bfloat16, 1e-5 in float32)"""
    n, nk, dt = 50, 40, DT[dtype]
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GB of device memory")
    q, do, k, v = (_normal(i, m, 1, d, dtype=dt) for i, m in enumerate((1, 1, nk, nk)))
    small = _run(ops, q.expand(n, 1, d), k, v, do.expand(n, 1, d), [0, n], [0, nk], causal=True)
    got = _run(ops, q.expand(rows, 1, d), k, v, do.expand(rows, 1, d), [0, rows - n, rows], [0, 0, nk], causal=True)
    rel = 2.0 ** -6 if dtype == "bf16" else 1e-5
    for g, w in zip((got[0][-n:], got[1][-n:], got[2], got[3]), small):
        torch.testing.assert_close(g.float(), w.float(), rtol=rel, atol=rel * w.float().abs().max().item())
    for g in got[:2]:
        assert not g[:rows - n].any()
    del got, g
    torch.cuda.empty_cache()                         # tests in processes of their own come behind this one


CAPS = [30.0, 1024.0, 1025.0, 1e4, 1e6, 1e9, 1e37]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("d,lens", [(64, [33, 20]), (64, [600, 700]), (128, [40, 50]), (128, [600, 700]), (242, [50, 30]), (33, [90, 70])])
def test_attention_under_large_caps(ops, dtype, cap, d, lens):
    """the larger the cap, the nearer to no cap at all: results and gradients, short and long sequences, odd rows"""
    long_sequences._check(ops, lens, lens, 2, 1, d, DT[dtype], seed=29, causal=True, score_cap=cap)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cap", CAPS)
def test_attention_under_large_caps_and_distances(ops, dtype, cap):
    long_sequences._check(ops, [90, 60], [90, 75], 2, 2, 64, DT[dtype], seed=31, causal=True, score_cap=cap, distance_slope=[0.2, 0.03], scale=-0.2)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("d", [64, 242])
def test_step_under_large_caps(ops, dtype, cap, d):
    dt, lens = DT[dtype], [700, 1, 64]
    q, kc, vc = _normal(1, 3, 4, d, dtype=dt), _normal(2, 3, 700, 2, d, dtype=dt), _normal(3, 3, 700, 2, d, dtype=dt)
    k, v = (torch.cat([c[i, :n] for i, n in enumerate(lens)]) for c in (kc, vc))
    (out, tol), *_ = long_sequences._ref(q, k, v, q, [0, 1, 2, 3], [0, 700, 701, 765], score_cap=cap)
    assert (ops.attention_step(q, kc, vc, _i32(lens), score_cap=cap).double().cpu() - out).norm() <= tol


@pytest.mark.parametrize("d", [64, 128])
def test_large_caps_with_what_is_not_finite(ops, d):
    """a NaN key under a large cap reaches the rows that see it and no others"""
    n, at = 150, 100
    q, k, v, do = (_normal(50 + i, n, 2, d, dtype=torch.bfloat16) for i in range(4))
    base = _run(ops, q, k, v, do, [0, n], [0, n], causal=True, score_cap=1e6)
    k[at] = math.nan
    got = _run(ops, q, k, v, do, [0, n], [0, n], causal=True, score_cap=1e6)
    for g, b in zip(got[:2], base[:2]):
        assert torch.isnan(g[at:]).all()
        torch.testing.assert_close(g[:at].float(), b[:at].float(), rtol=2.0 ** -6, atol=2.0 ** -6 * b.float().abs().max().item())


def test_tangents_are_refused_wherever_they_come_in(ops):
    """constants, the buffer to write into, and the gradient that a backward pass is given"""
    import torch.autograd.forward_ad as fw
    q, k, freq, w, off = _normal(1, 6, 4, 16), _normal(2, 6, 2, 16), ops.rotary_frequencies(16, device="cuda"), torch.ones(16, device="cuda"), _i32([0, 6])
    pos, slope, lens, cache = torch.arange(6, device="cuda"), torch.ones(4, device="cuda"), _i32([3] * 6), _normal(3, 6, 5, 2, 16)
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call in (lambda: ops.packed_attention(q, k, k, off, distance_slope=dual(slope)), lambda: ops.attention_step(q, cache, cache, lens, distance_slope=dual(slope)),
                     lambda: ops.attention_step(q, cache, cache, lens, out=dual(torch.empty_like(q))), lambda: ops.rotary_qk(q, k, pos, dual(freq)),
                     lambda: ops.rotary_qk(q, k, pos, freq, dual(w), w), lambda: ops.rotary_qk(q, k, pos, freq, w, dual(w))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        ql = q.clone().requires_grad_()
        for y in (ops.packed_attention(ql, k, k, off), ops.rotary_qk(ql, k, pos, freq)[0], ops.dropout_add(ql, p=0.5, seed=1)):
            with pytest.raises(ValueError, match="forward-mode"):
                torch.autograd.grad(y, ql, dual(torch.ones_like(y)))
        ops.packed_attention(q, k, k, off), ops.attention_step(q, cache, cache, lens), ops.rotary_qk(q, k, pos, freq), ops.dropout_add(q, p=0.5, seed=1)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: ops.packed_attention(x, k, k, off))(q[None])


def test_attention_refuses_more_sequences_than_it_counts(ops):
    q = _normal(1, 4, 1, 8)
    off = torch.zeros(1, dtype=torch.int32, device="cuda").expand((1 << 30) + 2)
    with pytest.raises(ValueError, match="sequences"):
        ops.packed_attention(q, q, q, off)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("cap", [100, 3000])
def test_step_writes_into_a_tensor_as_torch_does(ops, dtype, cap):
    """q itself; a tensor that autograd saved is marked as written; one that requires a gradient is refused"""
    q, kc, vc, lens = _normal(1, 2, 4, 64, dtype=DT[dtype]), _normal(2, 2, cap, 2, 64, dtype=DT[dtype]), _normal(3, 2, cap, 2, 64, dtype=DT[dtype]), _i32([cap, 7])
    want = ops.attention_step(q, kc, vc, lens)
    same = q.clone()
    assert ops.attention_step(same, kc, vc, lens, out=same) is same and torch.equal(same, want)
    x = torch.ones_like(q).requires_grad_()
    saved = q.clone()
    y = x * saved
    ops.attention_step(q, kc, vc, lens, out=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(ValueError, match="no gradient"):
        ops.attention_step(q, kc, vc, lens, out=x)
    with torch.no_grad():
        assert torch.equal(ops.attention_step(q, kc, vc, lens, out=x), want)
    with torch.inference_mode():
        assert torch.equal(ops.attention_step(q, kc, vc, lens, out=torch.empty_like(q)), want)


def test_numbers_that_want_a_gradient_are_refused(ops):
    """a learned scale, cap, eps or probability would get none, without a word; without a gradient a tensor is its value"""
    import torch.autograd.forward_ad as fw
    q, pos, off, lens, cache = _normal(1, 6, 2, 16), torch.arange(6, device="cuda"), _i32([0, 6]), _i32([3] * 6), _normal(2, 6, 5, 2, 16)
    freq, w = ops.rotary_frequencies(16, device="cuda"), torch.ones(16, device="cuda")
    calls = (lambda x: ops.packed_attention(q, q, q, off, scale=x), lambda x: ops.packed_attention(q, q, q, off, score_cap=x), lambda x: ops.attention_step(q, cache, cache, lens, scale=x),
             lambda x: ops.attention_step(q, cache, cache, lens, score_cap=x), lambda x: ops.rotary_qk(q, q, pos, freq, w, w, eps=x)[0], lambda x: ops.dropout_add(q, p=x, seed=3))
    for call in calls:
        for x in (torch.tensor(0.5, requires_grad=True), torch.tensor([0.5], device="cuda", requires_grad=True)):
            with pytest.raises(ValueError, match="no gradient"):
                call(x)
            with torch.no_grad():
                assert torch.equal(call(x), call(0.5))
        with fw.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            call(fw.make_dual(torch.tensor(0.5), torch.tensor(1.0)))
        assert torch.equal(call(torch.tensor(0.5)), call(0.5))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d,n", [(64, 300), (64, 1100), (128, 1100), (242, 60), (242, 1100), (33, 90)])
@pytest.mark.parametrize("kw", [{}, dict(causal=True, score_cap=4.0)])
def test_a_sequence_of_nan_beside_another(ops, dtype, d, n, kw):
    """a diverged sequence: all of its results and gradients are NaN (each row is known after the first key that it sees), the one beside it
    answers as ever -- tiles that both share are done again pair by pair, sums in another order: 2^-6 of the largest in bfloat16, 1e-5"""
    q, k, v, do = (_normal(60 + i, 2 * n + 40, 2, d, dtype=DT[dtype]) for i in range(4))
    off = [0, n, 2 * n + 40]
    base = _run(ops, q, k, v, do, off, off, **kw)
    rel = 2.0 ** -6 if dtype == "bf16" else 1e-5
    for bad in ((q, k, v), (k,)):
        args = [x.clone() for x in (q, k, v)]
        for x, y in zip((q, k, v), args):
            if any(x is z for z in bad):
                y[:n] = math.nan
        got = _run(ops, *args, do, off, off, **kw)
        for g, b in zip(got, base):
            assert torch.isnan(g[:n]).all()
            torch.testing.assert_close(g[n:].float(), b[n:].float(), rtol=rel, atol=rel * b.float().abs().max().item())
