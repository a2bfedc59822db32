"""The sequence operators against plain implementations in 64 bits, through their public calls.

Tolerances.  A float32 result is a chain of sums of at most 256 products (relative error about sqrt(256) * 2^-24 of the terms), an
exponential (2^-23 and the error of its argument, some units times 2^-23) and a sum over the keys: F32 = 4e-6 of the result's 2-norm
leaves a factor of about 3.  A bfloat16 result is rounded once at the end and its probabilities (or their derivatives) once on the
way: two errors of at most half a step, 2^-8, spread evenly, so sqrt(2/3) * 2^-8 = 3.2e-3 of the 2-norm; BF16 = 2^-8.  Each element
is bounded too, by 2^-8 of what it sums in absolute value and 2^-8 of itself.  dq and dk have a third source: ds = p (dp - delta) with
delta = dout.out, where out carries the rounding of its probabilities, at most 2^-8 sum_j p_j |dp_j| in delta, and is kept to
2^-8 * 2^-8 of itself (the value and the residual of its rounding), 2^-16 sum |dout out|.  In float32 dp - delta cancels (to zero for
a row with one key), so their own errors count by their terms: F32 of the terms' 2-norms, weighted as ds is."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = 4e-6, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from nl_vsgg_amd.lib import sequence_ops
    return sequence_ops


def _offsets(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float32).to(dtype).cuda()


def _attention_ref(q, k, v, off_q, off_k, causal=False, prefix=None, slope=None, cap=0.0, scale=None, do=None):
    """Textbook attention in float64 on the CPU, a sequence and a head at a time; also each output's sum of absolute terms."""
    rounds = q.dtype == torch.bfloat16
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    do = None if do is None else do.detach().cpu().double()
    grp, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5 if scale is None else scale
    out, outa = torch.zeros_like(q), torch.zeros_like(q)
    g = [torch.zeros_like(x) for x in (q, k, v)]
    ga = [torch.zeros_like(x) for x in (q, k, v)]
    gx = [torch.zeros_like(x) for x in (q, k, v)]
    for s in range(len(off_q) - 1):
        a, b, c, d = off_q[s], off_q[s + 1], off_k[s], off_k[s + 1]
        lq, lk = b - a, d - c
        if lq == 0 or lk == 0:
            continue
        place = torch.arange(lq)[:, None] + lk - lq
        key = torch.arange(lk)[None]
        see = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            see = (key <= place) | (key < (0 if prefix is None else prefix[s]))
        for h in range(q.shape[1]):
            raw = scale * torch.where(see[..., None], (q[a:b, h][:, None] * k[c:d, h // grp][None]), 0.0).sum(-1)
            bend = torch.ones_like(raw)
            z = raw
            if cap:
                t = torch.tanh(raw / cap)
                z, bend = cap * t, 1 - t * t
            if slope is not None:
                z = z - float(slope[h]) * (place - key).abs()
            z = z.masked_fill(~see, -math.inf)
            top = z.max(1, keepdim=True).values
            p = torch.where(see, torch.exp(z - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)

            def weigh(w, x):                                  # sums over what the mask shows alone: 0 * inf must not appear
                return torch.where(see[..., None], w[..., None] * x[None], 0.0).sum(1)

            def weigh_t(w, x):
                return torch.where(see[..., None], w[..., None] * x[:, None], 0.0).sum(0)
            out[a:b, h] = weigh(p, v[c:d, h // grp])
            outa[a:b, h] = weigh(p, v[c:d, h // grp].abs())
            if do is None:
                continue
            dp = torch.where(see[..., None], do[a:b, h][:, None] * v[c:d, h // grp][None], 0.0).sum(-1)
            ds = torch.where(see, p * (dp - (do[a:b, h] * out[a:b, h]).sum(1, keepdim=True)) * bend, 0.0)
            dpn = torch.where(see[..., None], do[a:b, h][:, None] * v[c:d, h // grp][None], 0.0).norm(dim=-1)
            dn = (do[a:b, h] * out[a:b, h]).norm(dim=1, keepdim=True)
            off = F32 * (dpn + dn)
            if rounds:
                off = off + 2.0 ** -8 * (p * dp.abs()).sum(1, keepdim=True) + 2.0 ** -16 * (do[a:b, h] * out[a:b, h]).abs().sum(1, keepdim=True)
            off = p * bend * off
            gx[0][a:b, h] = scale * weigh(off, k[c:d, h // grp].abs())
            gx[1][c:d, h // grp] += scale * weigh_t(off, q[a:b, h].abs())
            g[0][a:b, h] = scale * weigh(ds, k[c:d, h // grp])
            g[1][c:d, h // grp] += scale * weigh_t(ds, q[a:b, h])
            g[2][c:d, h // grp] += weigh_t(p, do[a:b, h])
            ga[0][a:b, h] = scale * weigh(ds.abs(), k[c:d, h // grp].abs())
            ga[1][c:d, h // grp] += scale * weigh_t(ds.abs(), q[a:b, h].abs())
            ga[2][c:d, h // grp] += weigh_t(p, do[a:b, h].abs())
    return (out, outa) if do is None else (out, outa, g, ga, gx)


def _close(got, ref, terms, dtype, what, more=0.0):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, what
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(got)), f"{what}: infinities or NaN in other places"
    d, r, t = (got - ref)[fine], ref[fine], terms[fine]
    if d.numel() == 0:
        return
    more = more[fine] if torch.is_tensor(more) else torch.zeros(1)
    tol = (F32 if dtype == torch.float32 else BF16) * r.norm() + more.norm()
    assert d.norm() <= tol, f"{what}: off by {d.norm() / r.norm():.2e} of its norm, {tol / r.norm():.2e} allowed"
    if dtype == torch.bfloat16:
        assert bool((d.abs() <= (2.0 ** -8 * (t + r.abs()) + more) * (1 + 2.0 ** -7) + F32 * t).all()), f"{what}: an element off by more than its roundings"


def _run(ops, q, k, v, off_q, off_k, do=None, **kw):
    args = dict(kw)
    for n in ("prefix_len",):
        if args.get(n) is not None:
            args[n] = _i32(args[n])
    if args.get("distance_slope") is not None:
        args["distance_slope"] = torch.tensor(args["distance_slope"], dtype=torch.float32, device="cuda")
    oq, ok = _i32(off_q), _i32(off_k)
    if do is None:
        return ops.packed_attention(q, k, v, oq, ok, **args)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*leaves, oq, ok, **args)
    return (out.detach(),) + torch.autograd.grad(out, leaves, do)


def _check(ops, dtype, lq, lk, hq, hk, d, seed=0, tail=(0, 0), **kw):
    off_q, off_k = _offsets(lq), _offsets(lk)
    tq, tk = off_q[-1] + tail[0], off_k[-1] + tail[1]
    q, k, v, do = (_normal(seed + i, n, h, d, dtype=dtype) for i, (n, h) in enumerate(((tq, hq), (tk, hk), (tk, hk), (tq, hq))))
    ref = _attention_ref(q, k, v, off_q, off_k, kw.get("causal", False), kw.get("prefix_len"), kw.get("distance_slope"), kw.get("score_cap", 0.0),
                         kw.get("scale"), do)
    out = _run(ops, q, k, v, off_q, off_k, **kw)
    _close(out, ref[0], ref[1], dtype, "out")
    got = _run(ops, q, k, v, off_q, off_k, do=do, **kw)
    assert torch.equal(got[0], out), "the training forward answers like the other"
    for i, n in enumerate(("dq", "dk", "dv")):
        _close(got[1 + i], ref[2][i], ref[3][i], dtype, n, ref[4][i])
    return q, k, v, do, got


# ---- attention over packed sequences -----------------------------------------------------------------------------------

MASKS = {
    "all": {},
    "causal": dict(causal=True),
    "prefix": dict(causal=True, prefix_len=True),
    "distance": dict(distance_slope=True),
    "cap": dict(score_cap=1.5),
    "everything": dict(causal=True, prefix_len=True, distance_slope=True, score_cap=2.0, scale=0.3),
}


def _mask(name, hq, lk):
    kw = dict(MASKS[name])
    if kw.get("prefix_len"):
        kw["prefix_len"] = [(5 * i) % (n + 3) for i, n in enumerate(lk)]
    if kw.get("distance_slope"):
        kw["distance_slope"] = [0.5 / (i + 1) for i in range(hq)]
    return kw


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("d", [64, 128, 242])
def test_attention_masks(ops, dtype, mask, d):
    lq = [1, 33, 0, 70, 128, 7]
    lk = [1, 50, 4, 70, 131, 7]
    _check(ops, DT[dtype], lq, lk, 4, 2, d, **_mask(mask, 4, lk))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [1, 2, 7, 8, 17, 31, 33, 66, 99, 127, 129, 143, 255, 256])
def test_attention_head_dims(ops, dtype, d):
    """every alignment of a row: odd dims of 2-byte elements, tails of 4, 8 and 12 bytes, rows under 16 bytes"""
    _check(ops, DT[dtype], [37, 90], [37, 90], 2, 1, d, causal=True)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lens", [[1], [31], [32], [33], [64], [65], [128], [129], [257], [1] * 40, [5, 0, 0, 0, 300, 0, 1]])
def test_attention_lengths(ops, dtype, lens):
    _check(ops, DT[dtype], lens, lens, 3, 3, 64, distance_slope=[0.1, 0.01, 0.3])


@pytest.mark.parametrize("dtype", DT)
def test_attention_rows_that_see_nothing(ops, dtype):
    """fewer keys than queries in order: the first rows are before every key; sequences without keys; rows in no sequence"""
    q, k, v, do, (out, dq, dk, dv) = _check(ops, DT[dtype], [40, 9, 70], [13, 0, 70], 2, 2, 64, tail=(21, 35), causal=True)
    assert not out[:27].any() and not dq[:27].any() and not out[40:49].any() and not dq[40:49].any()
    assert not out[119:].any() and not dq[119:].any() and not dk[83:].any() and not dv[83:].any()
    assert out[27:40].any() and out[49:119].any()


@pytest.mark.parametrize("dtype", DT)
def test_attention_without_keys_queries_or_sequences(ops, dtype):
    dt = DT[dtype]
    q, k = _normal(1, 5, 2, 64, dtype=dt), _normal(2, 0, 2, 64, dtype=dt)
    out, dq, dk, dv = _run(ops, q, k, k, [0, 5], [0, 0], do=q)
    assert not out.any() and not dq.any() and dk.shape == k.shape
    out, dq, dk, dv = _run(ops, k, q, q, [0, 0], [0, 5], do=k)
    assert out.shape == k.shape and not dk.any() and not dv.any() and dk.shape == q.shape
    out, dq, dk, dv = _run(ops, q, q, q, [0], [0], do=q)
    assert not out.any() and not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [64, 242])
def test_attention_masked_infinities_stay_out(ops, dtype, d):
    """NaN and infinities in a later token (causal), in a neighbour sequence and behind the last one: rows that do not see them
    answer as without them, forward and backward; rows that do see them answer with NaN where the definition does"""
    dt = DT[dtype]
    lens = [20, 45, 1, 60]
    off = _offsets(lens)
    q, k, v, do = (_normal(10 + i, off[-1] + 9, 2, d, dtype=dt) for i in range(4))
    base = _run(ops, q, k, v, off, off, do=do, causal=True)
    for bad in (float("nan"), float("inf"), -float("inf")):
        k2, v2, q2, do2 = k.clone(), v.clone(), q.clone(), do.clone()
        k2[50] = bad; v2[50] = bad                    # token 30 of sequence 1: rows 50 .. 64 see it
        k2[off[-1]:] = bad; v2[off[-1]:] = bad; q2[off[-1]:] = bad; do2[off[-1]:] = bad
        got = _run(ops, q2, k2, v2, off, off, do=do2, causal=True)
        for g, b in zip(got[:2], base[:2]):
            assert torch.equal(torch.isfinite(g[:50]).all(), torch.tensor(True, device="cuda"))
            torch.testing.assert_close(g[:50].float(), b[:50].float(), rtol=2 ** -6 if dtype == "bf16" else 1e-5, atol=2e-2 if dtype == "bf16" else 1e-5)
            torch.testing.assert_close(g[65:].float(), b[65:].float(), rtol=2 ** -6 if dtype == "bf16" else 1e-5, atol=2e-2 if dtype == "bf16" else 1e-5)
        for g, b in zip(got[2:], base[2:]):           # keys of the other sequences get their old gradients
            for a, e in ((0, 20), (65, off[-1])):
                torch.testing.assert_close(g[a:e].float(), b[a:e].float(), rtol=2 ** -6 if dtype == "bf16" else 1e-5, atol=4e-2 if dtype == "bf16" else 1e-5)
            assert not g[off[-1]:].any()
        if math.isnan(bad):
            assert torch.isnan(got[0][50:65]).all() and torch.isnan(got[1][50:65]).all()


@pytest.mark.parametrize("dtype", DT)
def test_attention_queries_that_are_not_finite(ops, dtype):
    """a NaN query row spoils its own output and the gradients of the keys that it sees, nothing else"""
    dt = DT[dtype]
    off = [0, 40, 100]
    q, k, v, do = (_normal(20 + i, 100, 2, 64, dtype=dt) for i in range(4))
    base = _run(ops, q, k, v, off, off, do=do, causal=True)
    q2 = q.clone(); q2[60] = float("nan")             # token 20 of sequence 1 sees keys 40 .. 60
    got = _run(ops, q2, k, v, off, off, do=do, causal=True)
    keep = [i for i in range(100) if i != 60]
    for g, b in zip(got[:2], base[:2]):
        assert torch.isnan(g[60]).all()
        assert torch.equal(g[keep], b[keep])
    for g, b in zip(got[2:], base[2:]):
        assert torch.isnan(g[40:61]).all() and torch.isfinite(g[:40]).all() and torch.isfinite(g[61:]).all()
        torch.testing.assert_close(g[61:].float(), b[61:].float(), rtol=2 ** -6 if dtype == "bf16" else 1e-5, atol=4e-2 if dtype == "bf16" else 1e-5)


@pytest.mark.parametrize("dtype", DT)
def test_attention_strides(ops, dtype):
    """views of one fused projection, heads in front of rows, a broadcast key head, a gradient that is an expanded scalar"""
    dt, t, hq, hk, d = DT[dtype], 77, 4, 2, 48
    off = [0, 30, 77]
    qkv = _normal(3, t, hq + 2 * hk, d, dtype=dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    do = _normal(4, t, hq, d, dtype=dt)
    want = _run(ops, q.contiguous(), k.contiguous(), v.contiguous(), off, off, do=do)
    for g, w in zip(_run(ops, q, k, v, off, off, do=do), want):
        assert torch.equal(g, w)
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, do)]
    for g, w in zip(_run(ops, *hm[:3], off, off, do=hm[3]), want):
        assert torch.equal(g, w)
    inner = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, do)]      # head dim strided: copied
    for g, w in zip(_run(ops, *inner[:3], off, off, do=inner[3]), want):
        assert torch.equal(g, w)
    one = k[:, :1]
    a = _run(ops, q, one.expand(-1, 2, -1), one.expand(-1, 2, -1), off, off)
    assert torch.equal(a, _run(ops, q, one.repeat(1, 2, 1), one.repeat(1, 2, 1), off, off))
    qg = q.detach().clone().requires_grad_()
    ops.packed_attention(qg, k, v, _i32(off)).sum().backward()
    full = _run(ops, q, k, v, off, off, do=torch.ones_like(do))
    assert torch.equal(qg.grad, full[1])


def test_attention_gradient_against_differences(ops):
    """central differences of the float32 kernel along random directions: steps of 2^-7 leave a truncation of about h^2 = 6e-5 and a
    rounding of 2^-24 / 2^-7 = 8e-6 of the loss's terms; 2e-3 of the derivative's scale"""
    lq, lk = [9, 40], [12, 40]
    off_q, off_k = _offsets(lq), _offsets(lk)
    kw = dict(causal=True, prefix_len=[3, 5], distance_slope=[0.2, 0.05], score_cap=3.0)
    q, k, v, w = (_normal(30 + i, n, 2, 24) for i, n in enumerate((49, 52, 52, 49)))
    grads = _run(ops, q, k, v, off_q, off_k, do=w, **kw)[1:]
    h = 2.0 ** -7
    for i, x in enumerate((q, k, v)):
        u = _normal(40 + i, *x.shape)
        ends = []
        for sgn in (1, -1):
            args = [q, k, v]
            args[i] = x + sgn * h * u
            ends.append((_run(ops, *args, off_q, off_k, **kw).double() * w.double()).sum().item())
        slope, want = (ends[0] - ends[1]) / (2 * h), (grads[i].double() * u.double()).sum().item()
        scale = (grads[i].double().norm() * u.double().norm() / math.sqrt(u.numel())).item()
        assert abs(slope - want) <= 2e-3 * max(abs(want), scale), (i, slope, want)


@pytest.mark.parametrize("dtype", DT)
def test_attention_repeats_bit_for_bit(ops, dtype):
    lens = [200, 3, 77]
    off = _offsets(lens)
    q, k, v, do = (_normal(50 + i, off[-1], h, 96, dtype=DT[dtype]) for i, h in enumerate((8, 2, 2, 8)))
    a = _run(ops, q, k, v, off, off, do=do, causal=True)
    for _ in range(3):
        for x, y in zip(a, _run(ops, q, k, v, off, off, do=do, causal=True)):
            assert torch.equal(x, y)


def test_attention_large_offsets(ops):
    """rows beyond 2^31 elements of q, k and v: the last sequence answers as by itself"""
    t, h, d = 560000, 16, 256
    q = torch.zeros(t, h, d, dtype=torch.bfloat16, device="cuda")
    k, v = torch.zeros_like(q), torch.zeros_like(q)
    n = 50
    tails = [_normal(60 + i, n, h, d, dtype=torch.bfloat16) for i in range(4)]
    for x, y in zip((q, k, v), tails):
        x[-n:] = y
    off = list(range(0, t - n, 10007)) + [t - n, t]
    out = _run(ops, q, k, v, off, off)
    small = _run(ops, *tails[:3], [0, n], [0, n], do=tails[3])
    torch.testing.assert_close(out[-n:].float(), small[0].float(), rtol=2 ** -6, atol=2e-2)
    assert not out[:t - n].any()
    # gradients: a few rows of the last sequence carry all of dout
    do = torch.zeros_like(q)
    do[-n:] = tails[3]
    off = [0, t - n, t]
    off_k = [0, 0, n]                                   # the long first sequence sees no keys
    got = _run(ops, q, tails[1], tails[2], off, off_k, do=do)
    assert not got[0][:t - n].any() and not got[1][:t - n].any()
    for g, s in zip((got[1][-n:], got[2], got[3]), small[1:]):
        torch.testing.assert_close(g.float(), s.float(), rtol=2 ** -6, atol=4e-2)


def test_attention_offsets_are_clamped(ops):
    """offsets beyond the tensors, falling or negative: some answer, no access out of bounds, and the next call is right"""
    q, k, v, do = (_normal(70 + i, 64, 2, 64) for i in range(4))
    for off_q, off_k in (([0, 500], [0, 500]), ([0, 64], [-40, 900]), ([50, 10, 64], [64, 3, 20]), ([-5, 64], [-5, 64]), ([2 ** 31 - 1, 5], [5, -2 ** 31])):
        _run(ops, q, k, v, off_q, off_k, do=do, causal=True)
        torch.cuda.synchronize()
    _check(ops, torch.float32, [64], [64], 2, 2, 64)


def test_attention_on_another_stream_and_in_graphs(ops):
    """a side stream; forward and backward captured, two graphs with workspaces of their own, replayed with other inputs and eager
    work between"""
    off = _i32([0, 60, 100])
    q, k, v, do = (_normal(80 + i, 100, h, 64, dtype=torch.bfloat16) for i, h in enumerate((4, 2, 2, 4)))

    def step(q, k, v, do):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = ops.packed_attention(*leaves, off, causal=True)
        return (out.detach(),) + torch.autograd.grad(out, leaves, do)
    eager = step(q, k, v, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(q, k, v, do)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        static = [x.clone() for x in (q, k, v, do)]
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*static)
        graphs.append((g, static, res))
    for seed in range(3):
        fresh = [[_normal(100 * seed + 10 * j + i, 100, h, 64, dtype=torch.bfloat16) for i, h in enumerate((4, 2, 2, 4))] for j in range(2)]
        for (g, static, _), x in zip(graphs, fresh):
            for s, y in zip(static, x):
                s.copy_(y)
            g.replay()
        want = [step(*x) for x in fresh]
        torch.cuda.synchronize()
        for (_, _, res), w in zip(graphs, want):
            for a, b in zip(res, w):
                assert torch.equal(a, b)


def test_attention_refusals(ops):
    q, k = _normal(1, 6, 4, 16), _normal(2, 6, 2, 16)
    off = _i32([0, 6])
    ok = dict(q=q, k=k, v=k, seq_off=off)
    ops.packed_attention(**ok)
    for bad in (dict(k=k.half()), dict(k=k.bfloat16()), dict(q=q.double(), k=k.double(), v=k.double()), dict(k=k.cpu()), dict(v=k[:5]), dict(q=q[:, :3]),
                dict(q=q[0]), dict(k=_normal(1, 6, 2, 17)), dict(seq_off=off.long()), dict(seq_off=off.cpu()), dict(seq_off=off[None]),
                dict(q=q[:5]), dict(key_off=_i32([0, 3, 6])), dict(prefix_len=_i32([2])), dict(causal=True, prefix_len=_i32([1, 2])),
                dict(distance_slope=torch.ones(2, device="cuda")), dict(distance_slope=torch.ones(4, device="cuda", requires_grad=True)),
                dict(score_cap=-1.0), dict(score_cap=math.nan), dict(scale=math.inf), dict(q=_normal(1, 6, 4, 300), k=_normal(1, 6, 2, 300), v=_normal(1, 6, 2, 300))):
        with pytest.raises(ValueError):
            ops.packed_attention(**{**ok, **bad})


# ---- one new token over its cache ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (6, 3), (8, 2), (8, 1), (15, 1)])
@pytest.mark.parametrize("d", [64, 242, 33])
def test_step_equals_the_definition(ops, dtype, hq, hk, d):
    dt, cap = DT[dtype], 300
    lens = [0, 1, 2, 63, 64, 65, 299, 300, 517]
    n = len(lens)
    q, kc, vc = _normal(1, n, hq, d, dtype=dt), _normal(2, n, cap, hk, d, dtype=dt), _normal(3, n, cap, hk, d, dtype=dt)
    for i, x in enumerate(lens):                       # rows behind a sequence's length must not be read into anything
        kc[i, min(x, cap):] = float("nan")
        vc[i, min(x, cap):] = float("inf")
    for kw in ({}, dict(score_cap=2.0), dict(distance_slope=[0.3 / (i + 1) for i in range(hq)], scale=0.2)):
        args = dict(kw)
        if "distance_slope" in args:
            args["distance_slope"] = torch.tensor(args["distance_slope"], device="cuda")
        out = ops.attention_step(q, kc, vc, _i32(lens), **args)
        for i, x in enumerate(lens):
            x = min(x, cap)
            # the token as a sequence of one query over its x keys
            ref = _attention_ref(q[i:i + 1], kc[i, :x], vc[i, :x], [0, 1], [0, x], False, None, kw.get("distance_slope"), kw.get("score_cap", 0.0), kw.get("scale"))
            _close(out[i:i + 1], *ref, dt, f"length {x}")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("length", [5000, 20000])
def test_step_over_a_long_cache(ops, dtype, length):
    dt = DT[dtype]
    q, kc, vc = _normal(1, 1, 4, 64, dtype=dt), _normal(2, 1, length + 7, 2, 64, dtype=dt), _normal(3, 1, length + 7, 2, 64, dtype=dt)
    out = ops.attention_step(q, kc, vc, _i32([length]))
    ref = _attention_ref(q, kc[0, :length], vc[0, :length], [0, 1], [0, length])
    _close(out, *ref, dt, "long")


def test_step_cache_layouts_and_out(ops):
    """caches as [sequence, head, row, dim], every second row, one allocation for both; `out` given; the same sequence twice"""
    n, cap, hk, d = 3, 90, 2, 64
    q = _normal(1, n, 4, d)
    kc, vc = _normal(2, n, cap, hk, d), _normal(3, n, cap, hk, d)
    lens = _i32([90, 7, 33])
    want = ops.attention_step(q, kc, vc, lens)
    hm = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc)]
    assert torch.equal(ops.attention_step(q, *hm, lens), want)
    both = torch.stack((kc, vc), 2)
    assert torch.equal(ops.attention_step(q, both[:, :, 0], both[:, :, 1], lens), want)
    wide = torch.zeros(n, 2 * cap, hk, d, device="cuda")
    wide[:, ::2] = kc
    assert torch.equal(ops.attention_step(q, wide[:, ::2], vc, lens), want)
    out = torch.full_like(q, 7.0)
    assert ops.attention_step(q, kc, vc, lens, out=out) is out and torch.equal(out, want)
    one = ops.attention_step(q[:1].expand(3, -1, -1), kc[:1].expand(3, -1, -1, -1), vc[:1].expand(3, -1, -1, -1), lens[:1].repeat(3))
    assert torch.equal(one[0], one[1]) and torch.equal(one[0], one[2])
    assert ops.attention_step(q[:0], kc[:0], vc[:0], lens[:0]).shape == (0, 4, d)
    assert not ops.attention_step(q, kc[:, :0], vc[:, :0], lens).any()


def test_step_large_offsets(ops):
    """a cache of more than 2^31 elements, its last sequence's last rows"""
    n, cap, hk, d = 5, 1 << 17, 16, 256
    kc = torch.zeros(n, cap, hk, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    q = _normal(1, n, hk, d, dtype=torch.bfloat16)
    kt, vt = _normal(2, 40, hk, d, dtype=torch.bfloat16), _normal(3, 40, hk, d, dtype=torch.bfloat16)
    kc[-1, -40:] = kt * 8; vc[-1, -40:] = vt
    out = ops.attention_step(q, kc, vc, _i32([0, 1, 0, 5, cap]))
    s = (q[-1].double()[:, None] * (kt * 8).double().transpose(0, 1)).sum(-1) * d ** -0.5          # [heads, 40], on the GPU
    e = torch.exp(s)
    ref = (e[..., None] * vt.double().transpose(0, 1)).sum(1) / (e.sum(1, keepdim=True) + cap - 40)
    assert ((out[-1].double() - ref).norm() / ref.norm()).item() <= BF16
    assert not out[:4].any()


def test_step_in_a_graph_with_growing_lengths(ops):
    n, cap = 2, 4096
    q, kc, vc, lens = _normal(1, n, 4, 64), _normal(2, n, cap, 2, 64), _normal(3, n, cap, 2, 64), _i32([5, 9])
    ops.attention_step(q, kc, vc, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.attention_step(q, kc, vc, lens)
        lens.add_(700)
    for at in range(4):
        lens.copy_(_i32([5 + 1000 * at, 9 + 3 * at]))
        want = ops.attention_step(q, kc, vc, lens)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_step_refusals(ops):
    q, kc = _normal(1, 2, 4, 16), _normal(2, 2, 10, 2, 16)
    ok = dict(q=q, k_cache=kc, v_cache=kc, lengths=_i32([3, 4]))
    ops.attention_step(**ok)
    for bad in (dict(q=q[0]), dict(k_cache=kc[0]), dict(q=q[:1]), dict(lengths=_i32([3])), dict(lengths=_i32([3, 4]).long()), dict(v_cache=kc[:, :5]),
                dict(q=q[:, :3]), dict(q=q.bfloat16()), dict(out=q[:1]), dict(out=q.bfloat16()), dict(q=q.clone().requires_grad_()), dict(score_cap=-1.0),
                dict(k_cache=kc.transpose(2, 3).contiguous().transpose(2, 3)), dict(distance_slope=torch.ones(3, device="cuda"))):
        with pytest.raises(ValueError):
            ops.attention_step(**{**ok, **bad})


# ---- norm and rotary positions ------------------------------------------------------------------------------------------


def _rotary_ref(x, pos, freq, w, eps, inter, dy=None):
    """In float64: output, and with dy the gradients of x and w, by complex multiplication and autograd."""
    x = x.detach().cpu().double().requires_grad_(dy is not None)
    w = None if w is None else w.detach().cpu().double().requires_grad_(dy is not None)
    rot = 2 * freq.numel()
    y = x if w is None else x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    ang = (pos.cpu().double()[:, None] * freq.cpu().double())[:, None]
    turn = torch.complex(torch.cos(ang), torch.sin(ang))
    if inter:
        z = torch.complex(y[..., 0:rot:2], y[..., 1:rot:2]) * turn
        front = torch.stack((z.real, z.imag), -1).flatten(-2)
    else:
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * turn
        front = torch.cat((z.real, z.imag), -1)
    y = torch.cat((front, y[..., rot:]), -1)
    if dy is None:
        return y
    g = torch.autograd.grad(y, (x,) if w is None else (x, w), dy.detach().cpu().double())
    return (y.detach(),) + g


def _near(got, ref, dtype, what, f32=2e-6, terms=0.0):
    """float32: a few roundings (2^-24 each) and the angle's fraction (2^-25 of a turn: 2e-7); bfloat16: one rounding, at most 2^-8.
    `terms`: the 2-norm of what a difference is taken of (the norm's gradient: w g - xh mean(w g xh), nothing left of it at
    head dim 1), whose float32 share counts by itself"""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, what
    if not ref.numel():
        return
    off, tol = (got - ref).norm().item(), (f32 if dtype == torch.float32 else BF16 / math.sqrt(3) * 1.1 + f32) * ref.norm().item() + f32 * terms
    assert off <= tol, f"{what}: {off:.2e} of {ref.norm().item():.2e}, {tol:.2e} allowed"


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("d,rot,hq,hk", [(64, 64, 4, 2), (242, 242, 8, 8), (128, 96, 3, 1), (17, 6, 2, 2), (33, 32, 1, 1), (256, 250, 2, 1), (2, 2, 1, 1), (5, 0, 2, 2),
                                         (1, 0, 1, 1), (40, 20, 5, 5)])
def test_rotary(ops, dtype, inter, norm, d, rot, hq, hk):
    dt, t = DT[dtype], 37
    qkv = _normal(1, t, hq + 2 * hk, d, dtype=dt)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    pos = torch.randint(0, 5000, (t,), generator=torch.Generator().manual_seed(5)).cuda()
    freq = ops.rotary_frequencies(rot, device="cuda") if rot else torch.empty(0, device="cuda")
    w = [1.0 + 0.2 * _normal(7 + i, d) if norm else None for i in range(2)]
    dy = [_normal(9, t, hq, d, dtype=dt), _normal(10, t, hk, d, dtype=dt)]
    plain = ops.rotary_qk(q, k, pos, freq, *w, interleaved=inter)
    leaves = [x.detach().requires_grad_() for x in (q, k)] + [x.detach().requires_grad_() for x in w if x is not None]
    y = ops.rotary_qk(leaves[0], leaves[1], pos, freq, *leaves[2:], interleaved=inter)
    grads = torch.autograd.grad(y, leaves, dy)
    for i, (x, n) in enumerate(((q, "q"), (k, "k"))):
        ref = _rotary_ref(x, pos, freq, w[i], 1e-6, inter, dy[i])
        assert torch.equal(y[i], plain[i]) and y[i].is_contiguous()
        _near(y[i], ref[0], dt, n)
        terms = 0.0
        if norm:
            inv = 1 / torch.sqrt(x.cpu().double().pow(2).mean(-1, keepdim=True) + 1e-6)
            terms = (inv * dy[i].cpu().double().norm(dim=-1, keepdim=True)).norm().item() * w[i].abs().max().item()
        _near(grads[i], ref[1], dt, "d" + n, 2e-6, terms)
        if norm:
            _near(grads[2 + i], ref[2], torch.float32, "dw" + n, 4e-6)


@pytest.mark.parametrize("tokens", [0, 1, 3, 4095, 4097, 20000])
def test_rotary_tokens(ops, tokens):
    q, k = _normal(1, tokens, 2, 16), _normal(2, tokens, 1, 16)
    pos, freq = torch.arange(tokens, device="cuda"), ops.rotary_frequencies(16, device="cuda")
    w = (1 + 0.1 * _normal(3, 16)).requires_grad_()
    ql = q.clone().requires_grad_()
    y = ops.rotary_qk(ql, k, pos, freq, w, w)
    dy = (_normal(4, tokens, 2, 16), _normal(5, tokens, 1, 16))
    dq, dw = torch.autograd.grad(y, (ql, w), dy)
    rq, rk = _rotary_ref(q, pos, freq, w, 1e-6, False, dy[0]), _rotary_ref(k, pos, freq, w, 1e-6, False, dy[1])
    _near(y[0], rq[0], torch.float32, "q"); _near(y[1], rk[0], torch.float32, "k"); _near(dq, rq[1], torch.float32, "dq")
    _near(dw, rq[2] + rk[2], torch.float32, "dw", 4e-6)                  # the same weight for both: its gradients add
    again = torch.autograd.grad(ops.rotary_qk(ql, k, pos, freq, w, w), (ql, w), dy)
    assert torch.equal(again[0], dq) and torch.equal(again[1], dw)


@pytest.mark.parametrize("start", [10 ** 6, 2 ** 31 + 5, 10 ** 12, -10 ** 6])
def test_rotary_far_positions(ops, start):
    """the angle's fraction of a turn is taken in 64 bits: at 1e12 a position times a frequency is rounded by 2^-53 * 1e12 = 1.1e-4 radians, twice here (by the kernel and the reference)"""
    q = _normal(1, 9, 2, 64)
    pos, freq = start + torch.arange(9, device="cuda"), ops.rotary_frequencies(64, factor=4.0, method="base", device="cuda")
    y, _ = ops.rotary_qk(q, q, pos, freq)
    _near(y, _rotary_ref(q, pos, freq, None, 0, False), torch.float32, "far", 2e-6 if abs(start) < 2 ** 39 else 5e-4)


def test_rotary_in_a_graph_and_rows_that_are_not_finite(ops):
    q, k, pos, freq = _normal(1, 50, 4, 32), _normal(2, 50, 2, 32), torch.arange(50, device="cuda"), ops.rotary_frequencies(32, device="cuda")
    w = torch.ones(32, device="cuda")
    ops.rotary_qk(q, k, pos, freq, w, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.rotary_qk(q, k, pos, freq, w, w)
    for s in range(3):
        q.copy_(_normal(20 + s, 50, 4, 32)); pos.add_(1000)
        want = ops.rotary_qk(q, k, pos, freq, w, w)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])
    base = ops.rotary_qk(q, k, pos, freq, w, w)
    q2 = q.clone(); q2[7, 1] = float("nan"); q2[8, 0, 3] = float("inf")
    got = ops.rotary_qk(q2, k, pos, freq, w, w)[0]
    mask = torch.ones(50, 4, dtype=torch.bool, device="cuda"); mask[7, 1] = mask[8, 0] = False
    assert torch.equal(got[mask], base[0][mask]) and torch.isnan(got[7, 1]).all()


def test_rotary_refusals(ops):
    q, k, pos, freq, w = _normal(1, 6, 4, 16), _normal(2, 6, 2, 16), torch.arange(6, device="cuda"), ops.rotary_frequencies(16, device="cuda"), torch.ones(16, device="cuda")
    ok = dict(q=q, k=k, positions=pos, frequencies=freq)
    ops.rotary_qk(**ok)
    for bad in (dict(k=k[:5]), dict(k=k.bfloat16()), dict(k=_normal(2, 6, 2, 18)), dict(positions=pos.int()), dict(positions=pos[:5]), dict(positions=pos.cpu()),
                dict(frequencies=torch.ones(9, device="cuda")), dict(frequencies=freq.double()), dict(frequencies=freq.clone().requires_grad_()), dict(q_weight=w),
                dict(k_weight=w), dict(q_weight=w[:8], k_weight=w), dict(q_weight=w.bfloat16(), k_weight=w), dict(eps=-1.0), dict(eps=math.nan), dict(q=q[0])):
        with pytest.raises(ValueError):
            ops.rotary_qk(**{**ok, **bad})


# ---- dropout ------------------------------------------------------------------------------------------------------------


def _philox(block, offset, key):
    """Philox 4x32-10 in Python integers."""
    c, k, m = [block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, (offset >> 32) & 0xFFFFFFFF], [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF], 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def _kept(n, p, key, offset):
    words = [w for b in range((n + 3) // 4) for w in _philox(b, offset % 2 ** 64, key % 2 ** 64)][:n]
    return torch.tensor([w >= round(p * 2 ** 32) for w in words], dtype=torch.bool)


def test_generator_known_answers():
    """the published test vectors of philox4x32-10: all zeros, all ones"""
    assert _philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox(2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [0, 1, 3, 4, 5, 8, 1023, 4099])
@pytest.mark.parametrize("key,offset", [(0, 0), (-1, -1), (0x123456789ABCDEF, 77), (5, -2 ** 63)])
def test_dropout_mask_and_values(ops, dtype, n, key, offset):
    """the mask is the generator's, kept values are x / (1 - p) (+ residual) rounded once, dropped ones the residual"""
    dt, p = DT[dtype], 0.3
    x, r, dy = (_normal(i, n, dtype=dt) for i in range(3))
    keep = _kept(n, p, key, offset).cuda()
    scaled = torch.where(keep, x.double() / (1 - p), 0.0)
    half = torch.finfo(dt).eps / 2
    state = torch.tensor([key, offset], dtype=torch.int64, device="cuda")
    for how in (dict(rng_state=state), dict(seed=key, offset=offset)):
        y = ops.dropout_add(x, p=p, **how)
        # one product (its factor off by 2^-24) and, with a residual, one sum in float32, then the rounding
        assert bool(((y.double() - scaled).abs() <= scaled.abs() * (half + 2.0 ** -22)).all()) and torch.equal(y != 0, keep & (x != 0))
        full = scaled + r.double()
        z = ops.dropout_add(x, r, p=p, **how)
        assert bool(((z.double() - full).abs() <= full.abs() * half * 1.01 + (scaled.abs() + r.double().abs()) * 2.0 ** -22).all())
        xl, rl = x.clone().requires_grad_(), r.clone().requires_grad_()
        gx, gr = torch.autograd.grad(ops.dropout_add(xl, rl, p=p, **how), (xl, rl), dy)
        want = torch.where(keep, dy.double() / (1 - p), 0.0)
        assert bool(((gx.double() - want).abs() <= want.abs() * (half + 2.0 ** -22)).all()) and torch.equal(gr, dy)


def test_dropout_rate_and_independence(ops):
    """2^22 elements: the kept share within 5 standard deviations; masks of two offsets or seeds agree as independent ones do"""
    n, p = 1 << 22, 0.1
    x = torch.ones(n, device="cuda")
    a, b, c = (ops.dropout_add(x, p=p, seed=s, offset=o) != 0 for s, o in ((1, 0), (1, 1), (2, 0)))
    for m in (a, b, c):
        assert abs(m.double().mean().item() - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n)
    both = (1 - p) ** 2 + p ** 2
    for m in (b, c):
        assert abs((a == m).double().mean().item() - both) < 5 * math.sqrt(both * (1 - both) / n)
    assert torch.equal(ops.dropout_add(x, p=0.0, seed=3), x)


def test_dropout_backward_after_the_state_moved(ops):
    state = torch.tensor([9, 0], dtype=torch.int64, device="cuda")
    x = _normal(1, 1000).requires_grad_()
    y = ops.dropout_add(x, p=0.5, rng_state=state)
    state[1] += 1
    y2 = ops.dropout_add(x, p=0.5, rng_state=state)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    g2, = torch.autograd.grad(y2, x, torch.ones_like(y))
    assert torch.equal(g != 0, y != 0) and torch.equal(g2 != 0, y2 != 0) and not torch.equal(g, g2)


def test_dropout_in_a_graph(ops):
    """each replay reads the state anew, forward and backward of one replay agree"""
    state = torch.tensor([9, 0], dtype=torch.int64, device="cuda")
    x, dy = _normal(1, 333, 7), _normal(2, 333, 7)

    def step():
        xl = x.detach().requires_grad_()
        y = ops.dropout_add(xl, x, p=0.25, rng_state=state)
        return y.detach(), torch.autograd.grad(y, xl, dy)[0]
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, dx = step()
        state[1] += 1
    for i in (0, 1, 5):
        state.copy_(torch.tensor([9, i], device="cuda"))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1]) and state[1].item() == i + 1


def test_dropout_layouts_and_refusals(ops):
    x = _normal(1, 8, 6)
    t = x.t()
    assert torch.equal(ops.dropout_add(t, t, p=0.2, seed=1), ops.dropout_add(t.contiguous(), t.contiguous(), p=0.2, seed=1))
    half = _normal(2, 9, dtype=torch.bfloat16)[1:]                     # an address of 2 bytes' alignment
    assert torch.equal(ops.dropout_add(half, p=0.2, seed=1), ops.dropout_add(half.clone(), p=0.2, seed=1))
    for bad in (dict(p=1.0), dict(p=-0.1), dict(p=math.nan), dict(seed=None), dict(rng_state=torch.zeros(2, dtype=torch.int64, device="cuda")),
                dict(residual=x[:4]), dict(residual=x.bfloat16()), dict(x=x.half()), dict(seed=2 ** 63), dict(seed=None, rng_state=torch.zeros(2, dtype=torch.int64)),
                dict(seed=None, rng_state=torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            ops.dropout_add(**{**dict(x=x, p=0.1, seed=1), **bad})


# ---- together -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DT)
def test_attention_half_of_a_layer(ops, dtype):
    """norm and positions -> attention -> output projection -> dropout with the residual, on one fused projection: the output and
    every gradient against float64 by autograd.  bfloat16: q, k, out, the projection and the sum are each rounded (and again in the
    backward pass), at most 8 roundings of 2^-8 / sqrt(3) of the 2-norm in a chain: sqrt(8 / 3) * 2^-8 = 6.4e-3, taken as 2^-6"""
    dt, h, d, lens, p = DT[dtype], 4, 32, [19, 40, 1, 66], 0.1
    off, t = _offsets(lens), sum(lens)
    x, wqkv, wo = _normal(1, t, h * d, dtype=dt), (_normal(2, h * d, 3 * h * d) * (h * d) ** -0.5).to(dt), (_normal(3, h * d, h * d) * (h * d) ** -0.5).to(dt)
    nq, nk = 1 + 0.1 * _normal(4, d), 1 + 0.1 * _normal(5, d)
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    freq, state, dy = ops.rotary_frequencies(d, device="cuda"), torch.tensor([3, 8], dtype=torch.int64, device="cuda"), _normal(6, t, h * d, dtype=dt)
    leaves = [y.clone().requires_grad_() for y in (x, wqkv, wo, nq, nk)]
    qkv = (leaves[0] @ leaves[1]).view(t, 3 * h, d)
    q, k = ops.rotary_qk(qkv[:, :h], qkv[:, h:2 * h], pos, freq, leaves[3], leaves[4])
    att = ops.packed_attention(q, k, qkv[:, 2 * h:], _i32(off), causal=True, score_cap=20.0)
    y = ops.dropout_add(att.flatten(1) @ leaves[2], leaves[0], p=p, rng_state=state)
    grads = torch.autograd.grad(y, leaves, dy)

    ref = [z.detach().cpu().double().requires_grad_() for z in (x, wqkv, wo, nq, nk)]
    rqkv = (ref[0] @ ref[1]).view(t, 3 * h, d)
    ang = (pos.cpu().double()[:, None] * freq.cpu().double())[:, None]

    def turned(z, w):
        z = z / torch.sqrt(z.pow(2).mean(-1, keepdim=True) + 1e-6) * w
        a, b = z[..., :d // 2], z[..., d // 2:]
        return torch.cat((a * torch.cos(ang) - b * torch.sin(ang), b * torch.cos(ang) + a * torch.sin(ang)), -1)
    rq, rk, outs = turned(rqkv[:, :h], ref[3]), turned(rqkv[:, h:2 * h], ref[4]), []
    for a, b in zip(off, off[1:]):
        s = torch.tanh(rq[a:b].transpose(0, 1) @ rk[a:b].permute(1, 2, 0) * d ** -0.5 / 20.0) * 20.0
        s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), -math.inf)
        outs.append((torch.softmax(s, -1) @ rqkv[a:b, 2 * h:].transpose(0, 1)).transpose(0, 1))
    keep = _kept(t * h * d, p, 3, 8).view(t, h * d)
    ry = ref[0] + torch.where(keep, torch.cat(outs).flatten(1) @ ref[2] / (1 - p), 0.0)
    rg = torch.autograd.grad(ry, ref, dy.cpu().double())
    tol = 2e-5 if dtype == "f32" else 2.0 ** -6                         # float32: the library's products at their own 1e-6 each
    for got, want, n in zip((y,) + grads, (ry,) + rg, ("y", "dx", "dwqkv", "dwo", "dnq", "dnk")):
        rel = ((got.detach().cpu().double() - want.detach()).norm() / want.norm()).item()
        assert rel <= tol, (n, rel)


@pytest.mark.parametrize("dtype", DT)
def test_growing_clips_equal_the_whole(ops, dtype):
    """token by token through positions, cache and step, against the packed causal call over the whole clips"""
    dt, h, hk, d, lens = DT[dtype], 4, 2, 64, [7, 12, 3]
    n, cap, slope = len(lens), 16, torch.tensor([0.3, 0.1, 0.05, 0.01], device="cuda")
    freq = ops.rotary_frequencies(d, device="cuda")
    q, k, v = (_normal(i, n, cap, x, d, dtype=dt) for i, x in enumerate((h, hk, hk)))
    kc, vc = torch.full((n, cap, hk, d), float("nan"), dtype=dt, device="cuda"), torch.full((n, cap, hk, d), float("nan"), dtype=dt, device="cuda")
    steps = []
    for t in range(max(lens)):
        pos = torch.full((n,), t, dtype=torch.int64, device="cuda")
        q1, k1 = ops.rotary_qk(q[:, t], k[:, t], pos, freq, interleaved=True)
        kc[:, t], vc[:, t] = k1, v[:, t]
        steps.append(ops.attention_step(q1, kc, vc, _i32([t + 1] * n), distance_slope=slope))
    off = _offsets(lens)
    rows = [(i, t) for i, x in enumerate(lens) for t in range(x)]
    pick = lambda y: torch.stack([y[i, t] for i, t in rows])  # noqa: E731
    pos = torch.tensor([t for _, t in rows], device="cuda")
    pq, pk = ops.rotary_qk(pick(q), pick(k), pos, freq, interleaved=True)
    whole = ops.packed_attention(pq, pk, pick(v), _i32(off), causal=True, distance_slope=slope)
    got = torch.stack([steps[t][i] for i, t in rows])
    rel = ((got.double() - whole.double()).norm() / whole.double().norm()).item()
    assert rel <= (F32 if dtype == "f32" else BF16)
