"""Attention over long packed sequences: float32 tensors on bfloat16 planes, shares of the keys joined, in 64 bits' sight.

Tolerances.  Beside those of short sequences (4e-6 of the 2-norm in float32, 2^-8 in bfloat16): a sum over n keys takes n roundings of
its running value, about sqrt(n) * 2^-24 of its terms, so what was derived for 256 of them grows by sqrt(n / 256).  Three planes hold a
number to 2^-26 of itself, and the three products of planes that are left out are below 2^-27 of the whole each: less than one rounding
of the sum.  dq and dk further carry what dp - delta loses (4e-6 of the terms' 2-norms, weighted as ds is) and in bfloat16 the rounding
of the probabilities in delta: at most 2^-8 sum_j p_j |dp_j|, and 2^-16 sum |dout out|."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from nl_vsgg_amd.lib import sequence_ops
    return sequence_ops


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _offsets(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


def _normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float32).to(dtype).cuda()


def _ref(q, k, v, do, off_q, off_k, causal=False, prefix_len=None, distance_slope=None, score_cap=0.0, scale=None):
    """The definition in float64, finite inputs; (result, allowed error in its 2-norm) of out, dq, dk, dv."""
    f32 = 4e-6 * max(1.0, math.sqrt(max(b - a for a, b in zip(off_k, off_k[1:])) / 256))
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    q, k, v, do = (x.detach().double().cpu() for x in (q, k, v, do))
    grp, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5 if scale is None else scale
    out, dq, dk, dv, xq, xk = (torch.zeros_like(x) for x in (q, q, k, v, q, k))
    for s in range(len(off_q) - 1):
        a, b, c, d = off_q[s], off_q[s + 1], off_k[s], off_k[s + 1]
        place, key = torch.arange(b - a)[:, None] + (d - c) - (b - a), torch.arange(d - c)[None]
        see = torch.ones(b - a, d - c, dtype=torch.bool)
        if causal:
            see = (key <= place) | (key < (0 if prefix_len is None else prefix_len[s]))
        for h in range(q.shape[1]):
            Q, K, V, G = q[a:b, h], k[c:d, h // grp], v[c:d, h // grp], do[a:b, h]
            z, bend = scale * Q @ K.T, 1.0
            if score_cap:
                t = torch.tanh(z / score_cap)
                z, bend = score_cap * t, 1 - t * t
            if distance_slope is not None:
                z = z - distance_slope[h] * (place - key).abs()
            z = z.masked_fill(~see, -math.inf)
            p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
            O = p @ V
            out[a:b, h] = O
            dp, delta = G @ V.T, (G * O).sum(1, keepdim=True)
            ds = p * (dp - delta) * bend
            off = f32 * (((G * G) @ (V * V).T).sqrt() + (G * O).norm(dim=1, keepdim=True))
            off = p * bend * (off + half * (p * dp.abs()).sum(1, keepdim=True) + half * half * (G * O).abs().sum(1, keepdim=True))
            dq[a:b, h], xq[a:b, h] = scale * ds @ K, scale * off @ K.abs()
            dk[c:d, h // grp] += scale * ds.T @ Q
            xk[c:d, h // grp] += scale * off.T @ Q.abs()
            dv[c:d, h // grp] += p.T @ G
    rel = half or f32
    return [(x, rel * x.norm() + e) for x, e in ((out, 0.0), (dq, xq.norm()), (dk, xk.norm()), (dv, 0.0))]


def _run(ops, q, k, v, do, off_q, off_k, prefix_len=None, distance_slope=None, **kw):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*leaves, _i32(off_q), _i32(off_k), prefix_len=None if prefix_len is None else _i32(prefix_len),
                               distance_slope=None if distance_slope is None else torch.tensor(distance_slope, device="cuda"), **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, do)]


def _inputs(lq, lk, hq, hk, d, dtype, seed=0, tail=(0, 0)):
    off_q, off_k = _offsets(lq), _offsets(lk)
    tq, tk = off_q[-1] + tail[0], off_k[-1] + tail[1]
    return [_normal(seed + i, n, h, d, dtype=dtype) for i, (n, h) in enumerate(((tq, hq), (tk, hk), (tk, hk), (tq, hq)))] + [off_q, off_k]


def _check(ops, lq, lk, hq, hk, d, dtype, seed=0, tail=(0, 0), **kw):
    x = _inputs(lq, lk, hq, hk, d, dtype, seed, tail)
    got = _run(ops, *x, **kw)
    for n, g, (r, tol) in zip(("out", "dq", "dk", "dv"), got, _ref(*x, **kw)):
        assert bool(torch.isfinite(g).all()), n
        off = (g.double().cpu() - r).norm()
        assert off <= tol, f"{n}: off by {off / r.norm():.2e} of its norm, {tol / r.norm():.2e} allowed"
    plain = ops.packed_attention(x[0], x[1], x[2], _i32(x[4]), _i32(x[5]), **{
        n: (_i32(v) if n == "prefix_len" else torch.tensor(v, device="cuda") if n == "distance_slope" else v) for n, v in kw.items()})
    assert torch.equal(plain, got[0]), "the training forward answers like the other"
    return x, got


def _on_planes(ops, q, k, v, off):
    """whether a call takes the planes: its workspace holds 6 bytes an element of q, k and v"""
    from nl_vsgg_amd import _native
    a = ops._attention_struct(q, k, v, _i32(off), _i32(off), None, None, False, 0.0, 1.0)
    return _native.load().sttran_attention_workspace_bytes(ctypes.byref(a), 0) >= 6 * (q.numel() + k.numel() + v.numel())


MASKS = {
    "all": {},
    "causal": dict(causal=True),
    "prefix": dict(causal=True, prefix_len=[700, 90]),
    "distance": dict(distance_slope=[0.3, 0.01]),
    "cap": dict(score_cap=1.5),
    "everything": dict(causal=True, prefix_len=[9, 2000], distance_slope=[0.05, 0.002], score_cap=2.0, scale=0.3),
    "falling": dict(causal=True, scale=-0.1),
}


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("d", [64, 128, 242])
def test_planes_masks(ops, mask, d):
    lens = [1100, 999]
    x, _ = _check(ops, lens, lens, 2, 1, d, torch.float32, tail=(5, 5), **MASKS[mask])
    assert _on_planes(ops, *x[:3], x[4])


@pytest.mark.parametrize("d", [40, 57, 63, 65, 99, 127, 129, 143, 200, 255, 256])
def test_planes_head_dims(ops, d):
    lens = [1033, 1, 2100]
    x, _ = _check(ops, lens, lens, 2, 2, d, torch.float32, seed=3, causal=True)
    assert _on_planes(ops, *x[:3], x[4])


@pytest.mark.parametrize("d", [64, 100, 242])
def test_planes_few_queries_over_many_keys(ops, d):
    """rows that see nothing, sequences of no rows, keys shared out: lengths of queries and keys that differ"""
    x, got = _check(ops, [90, 0, 40, 700], [30, 50, 5000, 3000], 4, 2, d, torch.float32, seed=5, tail=(9, 17), causal=True)
    out, dq, dk, dv = got
    assert not out[:60].any() and not dq[:60].any() and not out[830:].any() and not dk[30:80].any() and not dv[8080:].any()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [64, 128, 242])
@pytest.mark.parametrize("mask", ["all", "causal", "everything"])
def test_shares_of_the_keys(ops, dtype, d, mask):
    """few rows over many keys: each share's sums are joined, in the forward pass and in dk and dv; one of 2 rows over 3"""
    _check(ops, [17, 2], [2500, 3], 2, 1, d, DT[dtype], seed=7, **MASKS[mask])


@pytest.mark.parametrize("dtype", DT)
def test_shares_of_a_key_tile(ops, dtype):
    """many query heads on few key heads: dk and dv summed by several workgroups; again and again the same bits"""
    x, got = _check(ops, [800], [800], 16, 1, 64, DT[dtype], seed=9, causal=True)
    for _ in range(3):
        for a, b in zip(got, _run(ops, *x, causal=True)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d,lens", [(64, [700, 900]), (128, [700, 900]), (242, [1100, 1300])])
def test_masked_infinities_stay_out(ops, dtype, d, lens):
    """NaN and infinities in later tokens and behind the last sequence: rows that do not see them answer as without them"""
    x = _inputs(lens, lens, 2, 1, d, DT[dtype], 11, (9, 9))
    q, k, v, do, off, _ = x
    at, rel = off[1] + 333, 2.0 ** -6 if dtype == "bf16" else 1e-5
    base = _run(ops, *x, causal=True)
    for bad in (math.nan, math.inf, -math.inf):
        q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
        k2[at], v2[at] = bad, bad
        for t in (q2, k2, v2, do2):
            t[off[-1]:] = bad
        got = _run(ops, q2, k2, v2, do2, off, off, causal=True)
        for g, b in zip(got[:2], base[:2]):
            assert bool(torch.isfinite(g[:at]).all())
            torch.testing.assert_close(g[:at].float(), b[:at].float(), rtol=rel, atol=rel * b.float().abs().max().item())
            assert not g[off[-1]:].any()
        for g, b in zip(got[2:], base[2:]):
            torch.testing.assert_close(g[:off[1]].float(), b[:off[1]].float(), rtol=rel, atol=rel * b.float().abs().max().item())
            assert not g[off[-1]:].any()
        if math.isnan(bad):
            assert bool(torch.isnan(got[0][at:off[-1]]).all()) and bool(torch.isnan(got[1][at:off[-1]]).all())


@pytest.mark.parametrize("d,n", [(64, 900), (242, 1200)])
def test_planes_hold_the_largest_numbers(ops, d, n):
    """values whose upper 8 bits round to infinity: a first token that is seen alone passes its value, the others weigh it"""
    big = torch.finfo(torch.float32).max
    q, k, v, do, off, _ = _inputs([n], [n], 2, 2, d, torch.float32, 13)
    v[0] = big
    assert _on_planes(ops, q, k, v, off)
    out = ops.packed_attention(q, k, v, _i32(off), causal=True).double().cpu()
    assert bool(torch.isfinite(out).all()) and bool((out[0] >= big * (1 - 2.0 ** -21)).all())
    z = torch.einsum("qhd,hd->qh", q.double().cpu(), k[0].double().cpu()) * d ** -0.5
    s = torch.einsum("qhd,khd->hqk", q.double().cpu(), k.double().cpu()) * d ** -0.5
    s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf)
    p = torch.exp(z - torch.logsumexp(s, 2).T)                  # of the first token, whose value outweighs all others
    torch.testing.assert_close(out, (p[..., None] * big).expand_as(out), rtol=1e-5, atol=0)


def test_planes_strides(ops):
    n, d = 1000, 64
    off = [0, 400, n]
    qkv, do = _normal(15, n, 8, d), _normal(16, n, 4, d)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    assert _on_planes(ops, q, k, v, off)
    want = _run(ops, q.contiguous(), k.contiguous(), v.contiguous(), do, off, off, causal=True)
    for form in (lambda x: x, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)):
        for g, w in zip(_run(ops, form(q), form(k), form(v), form(do), off, off, causal=True), want):
            assert torch.equal(g, w)
    odd = [torch.empty(x.shape[0], x.shape[1], d + 3, device="cuda")[..., 1:d + 1].copy_(x) for x in (q, k, v, do)]      # rows at any 4 bytes
    for g, w in zip(_run(ops, *odd, off, off, causal=True), want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", DT)
def test_graphs_with_their_own_workspaces(ops, dtype):
    """planes and shares of the keys in two captured graphs, replayed side by side with eager calls between"""
    lens, d = ([600, 500], 64)
    dt = DT[dtype]
    offs, offd = _i32(_offsets(lens)), _i32([0, 5, 9])

    def step(q, k, v, do, few):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = ops.packed_attention(*leaves, offs, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, do), ops.packed_attention(few, k, v, offd, offs)]

    def fresh(seed):
        return [_normal(seed + i, n, h, d, dtype=dt) for i, (n, h) in enumerate(((1100, 4), (1100, 2), (1100, 2), (1100, 4), (9, 4)))]
    side, graphs = torch.cuda.Stream(), []
    for j in range(2):
        static = fresh(j)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*static)
        graphs.append((g, static, res))
    for seed in (100, 200, 300):
        sets = [fresh(seed + 10 * j) for j in range(2)]
        for (g, static, _), x in zip(graphs, sets):
            for s, y in zip(static, x):
                s.copy_(y)
            g.replay()
        want = [step(*x) for x in sets]
        torch.cuda.synchronize()
        for (_, _, res), w in zip(graphs, want):
            for a, b in zip(res, w):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
def test_one_token_steps_over_a_long_cache(ops, dtype):
    """the step over a cache and the packed form of the same call: 1 row over all the keys"""
    dt, lens, hq, hk, d = DT[dtype], [3000, 1, 700], 16, 1, 96
    cap = 3100
    q, kc, vc = _normal(1, 3, hq, d, dtype=dt), _normal(2, 3, cap, hk, d, dtype=dt), _normal(3, 3, cap, hk, d, dtype=dt)
    k, v = (torch.cat([c[i, :n] for i, n in enumerate(lens)]) for c in (kc, vc))
    (out, tol), *_ = _ref(q, k, v, q, [0, 1, 2, 3], _offsets(lens))
    for got in (ops.attention_step(q, kc, vc, _i32(lens)), ops.packed_attention(q, k, v, _i32([0, 1, 2, 3]), _i32(_offsets(lens)))):
        assert (got.double().cpu() - out).norm() <= tol


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d,lens", [(64, [20, 50]), (64, [700, 650]), (242, [60, 9]), (128, [600, 800])])
def test_rows_before_the_first_sequence(ops, dtype, d, lens):
    """sequences that begin at row 7 answer as they do from row 0, the rows around them are zeros with zero gradients"""
    n = sum(lens)
    q, k, v, do = _inputs([n], [n], 2, 2, d, DT[dtype], 17, (19, 19))[:4]
    off = [7, 7 + lens[0], 7 + n]
    got = _run(ops, q, k, v, do, off, off, causal=True)
    want = _run(ops, q[7:7 + n], k[7:7 + n], v[7:7 + n], do[7:7 + n], _offsets(lens), _offsets(lens), causal=True)
    rel = 2.0 ** -6 if dtype == "bf16" else 1e-5                # tiles begin at other rows: sums in another order
    for g, w in zip(got, want):
        assert not g[:7].any() and not g[7 + n:].any()
        torch.testing.assert_close(g[7:7 + n].float(), w.float(), rtol=rel, atol=rel * w.float().abs().max().item())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_columns_that_pass_keep_infinities(ops, dtype, interleaved):
    """a column behind the turned ones passes as it is, next to an infinite one too, forward and backward"""
    n, d, rot = 6, 64, 48
    q, k = _normal(1, n, 2, d, dtype=DT[dtype]), _normal(2, n, 1, d, dtype=DT[dtype])
    q[1, 0, 50], q[2, 1, 63], k[3, 0, 49] = math.inf, -math.inf, math.nan
    freq, pos = ops.rotary_frequencies(rot, device="cuda"), torch.arange(n, device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k)]
    out = ops.rotary_qk(*leaves, pos, freq, interleaved=interleaved)
    back = torch.autograd.grad(out, leaves, [q, k])
    for x, y, g in zip((q, k), out, back):
        assert torch.equal(y[..., rot:].nan_to_num(7.0, 8.0, 9.0), x[..., rot:].nan_to_num(7.0, 8.0, 9.0))
        assert torch.equal(g[..., rot:].nan_to_num(7.0, 8.0, 9.0), x[..., rot:].nan_to_num(7.0, 8.0, 9.0))
        assert bool(torch.isfinite(y[..., :rot]).all()) and bool(torch.isfinite(g[..., :rot]).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d,lens", [(64, [50, 90]), (128, [70, 60]), (242, [50, 90]), (64, [700, 650]), (128, [600, 800]), (242, [1100, 1300])])
def test_gradients_that_are_not_finite_reach_what_they_saw(ops, dtype, d, lens):
    """an infinite or NaN gradient row reaches the keys its row saw and its own query, nothing else"""
    x = _inputs(lens, lens, 4, 2, d, DT[dtype], 19)
    q, k, v, do, off, _ = x
    at, rel = off[1] + 21, 2.0 ** -6 if dtype == "bf16" else 1e-5
    base = _run(ops, *x, causal=True)
    for bad in (math.inf, math.nan):
        do2 = do.clone()
        do2[at, 1] = bad                              # query head 1 reads key head 0
        out, dq, dk, dv = _run(ops, q, k, v, do2, off, off, causal=True)
        assert torch.equal(out, base[0])
        rows = [i for i in range(off[-1]) if i != at]
        for g, b, keep in ((dq, base[1], rows), (dk, base[2], [*range(off[1]), *range(at + 1, off[-1])]), (dv, base[3], [*range(off[1]), *range(at + 1, off[-1])])):
            torch.testing.assert_close(g[keep].float(), b[keep].float(), rtol=rel, atol=rel * b.float().abs().max().item())
        assert torch.equal(dk[:, 1], base[2][:, 1]) and torch.equal(dv[:, 1], base[3][:, 1])
        assert not torch.isfinite(dq[at, 1]).any() and not torch.isfinite(dv[off[1]:at + 1, 0]).any()
        assert bool(torch.isfinite(dq[at, [0, 2, 3]]).all())


@pytest.mark.parametrize("dtype", DT)
def test_two_threads_on_two_streams(ops, dtype):
    """calls from two host threads at once, each on its own stream, answer as calls in turn"""
    import threading
    sets = [_inputs([300, 333], [300, 333], 4, 2, 64, DT[dtype], 30 + 10 * i) for i in range(2)]
    want = [_run(ops, *x, causal=True) for x in sets]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = _run(ops, *sets[i], causal=True)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                        # shown by the assertion below
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("d", [64, 96, 128, 131, 242])
def test_short_bfloat16_sequences_round_once(ops, d):
    """below 64 rows probabilities and their derivatives enter the products with 16 bits: each is off by 2^-17 of itself, as delta is, a
    hundredth of the result's own rounding (2^-8 / sqrt(6) of it in its 2-norm); terms that cancel to a tenth bring that to a tenth, and
    what is off in quadrature to it adds under 1%.  A quarter more than the rounding of the exact result is allowed, rounding each product
    to 8 bits would take 1.4 times."""
    lens = [20, 41, 9, 63, 33]
    x = _inputs(lens, lens, 4, 2, d, torch.bfloat16, 23)
    for n, g, (r, _) in zip(("out", "dq", "dk", "dv"), _run(ops, *x), _ref(*x)):
        own = (r.to(torch.bfloat16).double() - r).norm()
        assert (g.double().cpu() - r).norm() <= 1.25 * own, n


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,most", [(64, 3), (65, 3), (700, 1), (4097, 2), (300, 40)])
def test_many_short_sequences(ops, dtype, n, most):
    """hundreds of sequences of 0 .. `most` rows: more than 64 of them may end within a wave's 32 rows, empty ones among them"""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, most + 1, (n,), generator=g).tolist()
    lens[n // 2:n // 2 + 80] = [0] * len(lens[n // 2:n // 2 + 80])
    off = _offsets(lens)
    q, k, v, do = (_normal(40 + i, off[-1] + 3, 2, 64, dtype=DT[dtype]) for i in range(4))
    out, dq, dk, dv = _run(ops, q, k, v, do, off, off, causal=True)
    # the same rows by their definition: one softmax over all rows, other sequences' masked
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(lens))
    see = (seq[:, None] == seq[None]).tril()
    Q, K, V, G = (x[:off[-1]].double().cpu().transpose(0, 1) for x in (q, k, v, do))
    p = torch.softmax((Q @ K.transpose(1, 2) / 8).masked_fill(~see, -math.inf), -1)
    dp = G @ V.transpose(1, 2)
    ds = p * (dp - (G * (p @ V)).sum(-1, keepdim=True)) / 8
    rel = 2.0 ** -8 if dtype == "bf16" else 4e-6
    for name, got, want, terms in (("out", out, p @ V, 0.0), ("dv", dv, p.transpose(1, 2) @ G, 0.0),
                                   ("dq", dq, ds @ K, (p * dp.abs()).norm()), ("dk", dk, ds.transpose(1, 2) @ Q, (p * dp.abs()).norm())):
        # dq, dk: dp - delta cancels, to zero for a first row, so its terms' rounding counts: 2^-16 of them in bfloat16 (delta's two parts)
        more = (2.0 ** -16 if dtype == "bf16" else 4e-6) * terms * 8
        assert (got[:off[-1]].double().cpu().transpose(0, 1) - want).norm() <= rel * want.norm() + more, name
        assert not got[off[-1]:].any()
