"""The sequence operators at the limits of their arguments: what lies beside a buffer, the largest and smallest numbers, the largest calls."""
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
