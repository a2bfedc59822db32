"""The sequence operators' refusals and host-side parts: everything here runs without a GPU (arguments are checked before anything
is launched)."""
import ctypes as C
import math
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def native():
    import __graft_entry__ as ge
    from nl_vsgg_amd import _native
    if not os.path.exists(_native.LIB_PATH):
        ge.build()
    return _native


def _attention(nat, **over):
    a = nat.SttranAttention(struct_size=C.sizeof(nat.SttranAttention), dtype=0, num_seq=1, num_q_heads=4, num_kv_heads=2, head_dim=64,
                            q_rows=8, kv_rows=8, q=4096, k=4096, v=4096, q_row_stride=256, q_head_stride=64, k_row_stride=128,
                            k_head_stride=64, v_row_stride=128, v_head_stride=64, seq_off=4096, key_off=4096, scale=0.125, out=4096,
                            lse=4096, dout=4096, dout_row_stride=256, dout_head_stride=64, dq=4096, dk=4096, dv=4096, workspace=4096,
                            workspace_bytes=1 << 20)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over", [dict(struct_size=8), dict(dtype=1), dict(num_kv_heads=3), dict(num_q_heads=0), dict(head_dim=0), dict(head_dim=257),
                                  dict(num_seq=-1), dict(q_rows=-1), dict(q_rows=2 ** 31), dict(kv_rows=2 ** 31), dict(q=None), dict(v=None),
                                  dict(seq_off=None), dict(key_off=None), dict(score_cap=-1.0), dict(score_cap=float("nan")),
                                  dict(scale=float("inf")), dict(k_row_stride=-1), dict(k_row_stride=(1 << 22) + 1), dict(q_head_stride=-64),
                                  dict(k=4097), dict(out=4098)])
def test_attention_refusals(native, over):
    lib = native.load()
    assert lib.sttran_attention_backward(C.byref(_attention(native, **over)), None) == 1
    assert lib.sttran_attention_forward(C.byref(_attention(native, **over)), None) == 1


@pytest.mark.parametrize("over", [dict(dout=None), dict(lse=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(workspace=None),
                                  dict(workspace_bytes=16), dict(workspace=4104), dict(dout_row_stride=-1), dict(dq=4097)])
def test_attention_backward_refusals(native, over):
    assert native.load().sttran_attention_backward(C.byref(_attention(native, **over)), None) == 1


def test_attention_without_rows_launches_nothing(native):
    lib = native.load()
    assert lib.sttran_attention_forward(C.byref(_attention(native, q_rows=0, q=None, out=None)), None) == 0
    assert lib.sttran_attention_backward(C.byref(_attention(native, q_rows=0, kv_rows=0)), None) == 0
    assert lib.sttran_attention_forward(None, None) == 1
    assert lib.sttran_attention_workspace_bytes(C.byref(_attention(native)), 1) >= 8 * 4 * 4 + 8 * 16


@pytest.mark.parametrize("over", [dict(struct_size=8), dict(dtype=2), dict(num_seq=65536), dict(num_seq=-1), dict(capacity=-1), dict(head_dim=300),
                                  dict(num_q_heads=5), dict(q=None), dict(k=None), dict(out=None), dict(lengths=None), dict(score_cap=-0.5),
                                  dict(k_seq_stride=-1), dict(v_row_stride=1 << 23), dict(v=4098), dict(workspace=None)])
def test_attention_step_refusals(native, over):
    lib = native.load()
    a = native.SttranAttentionStep(struct_size=C.sizeof(native.SttranAttentionStep), dtype=0, num_seq=2, num_q_heads=4, num_kv_heads=2, head_dim=64,
                                   capacity=1024, q=4096, k=4096, v=4096, q_seq_stride=256, q_head_stride=64, k_seq_stride=131072,
                                   k_row_stride=128, k_head_stride=64, v_seq_stride=131072, v_row_stride=128, v_head_stride=64, lengths=4096,
                                   scale=0.125, out=4096, workspace=4096, workspace_bytes=1 << 24)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.sttran_attention_step(C.byref(a), None) == 1


@pytest.mark.parametrize("over", [dict(struct_size=8), dict(dtype=1), dict(tokens=-1), dict(head_dim=257), dict(rotary_dim=3), dict(rotary_dim=66),
                                  dict(rotary_dim=-2), dict(num_q_heads=0, num_kv_heads=0), dict(q=None), dict(k_out=None), dict(positions=None),
                                  dict(freq=None), dict(q_weight=4096), dict(eps=-1.0), dict(eps=float("nan")), dict(q_row_stride=-1), dict(q=4098)])
def test_rotary_refusals(native, over):
    lib = native.load()
    a = native.SttranRotary(struct_size=C.sizeof(native.SttranRotary), dtype=0, tokens=4, num_q_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=64,
                            q=4096, k=4096, q_row_stride=256, q_head_stride=64, k_row_stride=128, k_head_stride=64, positions=4096, freq=4096,
                            eps=1e-6, q_out=4096, k_out=4096)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.sttran_rotary_forward(C.byref(a), None) == 1
    assert lib.sttran_rotary_backward(C.byref(a), None) == 1                  # no gradients given at all


def test_rotary_backward_wants_workspace_for_weights(native):
    lib = native.load()
    a = native.SttranRotary(struct_size=C.sizeof(native.SttranRotary), dtype=0, tokens=4, num_q_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=64,
                            q=4096, k=4096, positions=4096, freq=4096, q_weight=4096, k_weight=4096, dq_out=4096, dk_out=4096, dq=4096, dk=4096,
                            dq_weight=4096, dk_weight=4096)
    need = lib.sttran_rotary_workspace_bytes(C.byref(a))
    assert need >= 4 * 2 * 64 * 4                                             # a share of both weights' gradients a token
    for ws, n in ((None, need), (4096, need - 1), (4104, need)):
        a.workspace, a.workspace_bytes = ws, n
        assert lib.sttran_rotary_backward(C.byref(a), None) == 1


@pytest.mark.parametrize("args", [(None, None, 4096, 8, 0, 0.1), (4096, None, None, 8, 0, 0.1), (4096, None, 4096, -1, 0, 0.1), (4096, None, 4096, 8, 1, 0.1),
                                  (4096, None, 4096, 8, 0, 1.0), (4096, None, 4096, 8, 0, -0.1), (4096, None, 4096, 8, 0, float("nan")),
                                  (4097, None, 4096, 8, 3, 0.1), (4096, 4097, 4096, 8, 3, 0.1)])
def test_dropout_refusals(native, args):
    assert native.load().sttran_dropout_add(*args, None, 0, 0, None, None) == 1


@pytest.mark.parametrize("over", [dict(q_rows=1 << 27), dict(kv_rows=1 << 28), dict(scale=3e38), dict(score_cap=2e38), dict(score_cap=1e-39),
                                  dict(scale=1e20, score_cap=1e-20)])
def test_attention_refuses_what_it_cannot_count(native, over):
    """more threads than a launch has, scores whose base-2 factors are infinite"""
    lib = native.load()
    a = _attention(native, **over)
    assert lib.sttran_attention_forward(C.byref(a), None) == 1 and lib.sttran_attention_backward(C.byref(a), None) == 1
    assert lib.sttran_attention_workspace_bytes(C.byref(a), 0) == 0


def test_attention_step_refuses_rows_it_cannot_count(native):
    lib = native.load()
    a = native.SttranAttentionStep(struct_size=C.sizeof(native.SttranAttentionStep), dtype=3, num_seq=1, num_q_heads=1, num_kv_heads=1, head_dim=2,
                                   capacity=(1 << 30) + 1, q=4096, k=4096, v=4096, q_seq_stride=2, q_head_stride=2, k_row_stride=2, v_row_stride=2,
                                   lengths=4096, scale=1.0, out=4096, workspace=4096, workspace_bytes=1 << 40)
    assert lib.sttran_attention_step(C.byref(a), None) == 1 and lib.sttran_attention_step_workspace_bytes(C.byref(a)) == 0


def test_struct_layouts_match_the_c_header(native, tmp_path):
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    src = tmp_path / "sizes.c"
    src.write_text("""
#include <stddef.h>
#include <stdio.h>
#include "sttran_hip.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu %d\\n", sizeof(SttranAttention), sizeof(SttranAttentionStep), sizeof(SttranRotary),
         offsetof(SttranAttention, dout), offsetof(SttranAttention, workspace_bytes), offsetof(SttranAttentionStep, workspace_bytes),
         offsetof(SttranRotary, workspace_bytes), STTRAN_DTYPE_BF16);
  return 0;
}
""")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    n = native
    assert got == [C.sizeof(n.SttranAttention), C.sizeof(n.SttranAttentionStep), C.sizeof(n.SttranRotary), n.SttranAttention.dout.offset,
                   n.SttranAttention.workspace_bytes.offset, n.SttranAttentionStep.workspace_bytes.offset, n.SttranRotary.workspace_bytes.offset,
                   n.DTYPE_BF16]


def test_no_cpu_path(native):
    from nl_vsgg_amd.lib import sequence_ops as ops
    x = torch.zeros(2, 1, 8)
    off = torch.tensor([0, 2], dtype=torch.int32)
    for call in (lambda: ops.packed_attention(x, x, x, off), lambda: ops.attention_step(x, x[None], x[None], off[1:]),
                 lambda: ops.rotary_qk(x, x, torch.arange(2), torch.ones(4)), lambda: ops.dropout_add(x, p=0.1, seed=1)):
        with pytest.raises(RuntimeError, match="MI355X only"):
            call()


def test_rotary_frequencies():
    """the stretches against their definitions in 64 bits; float32 results: half a step, 2^-24"""
    from nl_vsgg_amd.lib.sequence_ops import rotary_frequencies as f
    dim, base, s = 64, 10000.0, 8.0
    want = [base ** (-2.0 * i / dim) for i in range(dim // 2)]

    def near(got, ref):
        assert got.dtype == torch.float32 and got.shape == (len(ref),)
        for g, r in zip(got.double().tolist(), ref):
            assert abs(g - r) <= 2.0 ** -24 * r * 1.01
    near(f(dim), want)
    near(f(dim, factor=s), [w / s for w in want])
    b2 = base * s ** (dim / (dim - 2))
    stretched = [b2 ** (-2.0 * i / dim) for i in range(dim // 2)]
    near(f(dim, factor=s, method="base"), stretched)
    assert abs(stretched[-1] * s / want[-1] - 1) < 1e-12 and stretched[0] == 1.0
    parts = f(dim, factor=s, method="by_parts", original_length=2048).double().tolist()
    for w, g in zip(want, parts):
        turns = 2048 * w / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        assert abs(g - (w * keep + w / s * (1 - keep))) <= 2.0 ** -24 * g * 1.01
    assert parts[0] == 1.0 and abs(parts[-1] * s / want[-1] - 1) < 1e-6
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, method="other"),
                dict(rotary_dim=8, method="by_parts"), dict(rotary_dim=8, method="by_parts", original_length=64, low_turns=4, high_turns=4)):
        with pytest.raises(ValueError):
            f(**bad)
