"""The sequence operators at the limits of their arguments, as far as the host decides them: everything here runs without a GPU."""
import ctypes as C
import os

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    import __graft_entry__ as ge
    from nl_vsgg_amd import _native
    if not os.path.exists(_native.LIB_PATH):
        ge.build()
    return _native


def _step(nat, n, heads, capacity, d=1):
    """a cache that all sequences share (sequence stride 0)"""
    return nat.SttranAttentionStep(struct_size=C.sizeof(nat.SttranAttentionStep), dtype=nat.DTYPE_BF16, num_seq=n, num_q_heads=heads, num_kv_heads=heads, head_dim=d,
                                   capacity=capacity, q=4096, k=4096, v=4096, q_seq_stride=heads * d, q_head_stride=d, k_row_stride=heads * d, k_head_stride=d,
                                   v_row_stride=heads * d, v_head_stride=d, lengths=4096, scale=1.0, out=4096)


@pytest.mark.parametrize("n,heads,capacity", [(16384, 1, 1 << 30), (24576, 1, 1 << 30), (65535, 1, 1 << 30), (65535, 64, 1 << 21), (65535, 4096, 1 << 30), (4096, 1, 1000)])
def test_step_of_many_sequences_over_one_cache_takes_it_whole(native, n, heads, capacity):
    """rows a workgroup are counted in 64 bits until they are known to be the cache's at most: one share, nothing to join"""
    assert native.load().sttran_attention_step_workspace_bytes(C.byref(_step(native, n, heads, capacity))) == 0


@pytest.mark.parametrize("n,heads,capacity", [(1, 1, 1 << 30), (1, 1, 193), (4095, 1, 1 << 20), (3, 2, 5000)])
def test_step_shares_cover_the_cache(native, n, heads, capacity):
    need = native.load().sttran_attention_step_workspace_bytes(C.byref(_step(native, n, heads, capacity)))
    shares, rest = divmod(need, heads * n * (1 + 2) * 4)
    assert rest == 0 and 2 <= shares <= 4096 + 1 and -(-capacity // shares) >= 97           # 192 rows a share, or what is left of them


def _calls(ops):
    """each operator, its tensors by name (float32 unless counted or placed by them) and which of them are numbers"""
    f = lambda *s: torch.randn(*s)  # noqa: E731
    off, pos = torch.tensor([0, 4], dtype=torch.int32), torch.arange(4)
    return [
        (lambda **t: ops.packed_attention(t["q"], t["k"], t["v"], off), dict(q=f(4, 2, 8), k=f(4, 2, 8), v=f(4, 2, 8))),
        (lambda **t: ops.attention_step(t["q"], t["k"], t["v"], off[:1]), dict(q=f(1, 2, 8), k=f(1, 5, 2, 8), v=f(1, 5, 2, 8))),
        (lambda **t: ops.rotary_qk(t["q"], t["k"], pos, torch.ones(4)), dict(q=f(4, 2, 8), k=f(4, 2, 8))),
        (lambda **t: ops.dropout_add(t["x"], t["residual"], p=0.1, seed=1), dict(x=f(6), residual=f(6))),
    ]


def test_forward_mode_is_refused():
    """a tangent would be lost without a word: each operator refuses one in each of its tensors, by dual numbers and by torch.func.jvp"""
    import torch.autograd.forward_ad as fw
    from nl_vsgg_amd.lib import sequence_ops as ops
    for call, tensors in _calls(ops):
        for name, x in tensors.items():
            with fw.dual_level():
                with pytest.raises(ValueError, match="forward-mode"):
                    call(**{**tensors, name: fw.make_dual(x, torch.ones_like(x))})
            with pytest.raises(ValueError, match="forward-mode"):
                torch.func.jvp(lambda y: call(**{**tensors, name: y}), (x,), (torch.ones_like(x),))
        with fw.dual_level(), pytest.raises(RuntimeError, match="MI355X only"):
            call(**tensors)                          # without a tangent: the next check's answer


def test_tracers_are_refused():
    """a trace would hold the result's allocation and not the kernel"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from nl_vsgg_amd.lib import sequence_ops as ops
    for call, tensors in _calls(ops):
        names = list(tensors)
        flat = lambda *a: call(**dict(zip(names, a)))  # noqa: E731
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(flat, tuple(tensors.values()), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(flat)(*tensors.values())


@pytest.mark.parametrize("n,want", [(1 << 30, 0), ((1 << 30) + 1, 1), (2 ** 31 - 1, 1)])
def test_attention_counts_its_sequences(native, n, want):
    """a row's sequence is found by halving: two numbers of sequences, added, stay within 32 bits.  (No rows: nothing is launched)"""
    lib = native.load()
    a = native.SttranAttention(struct_size=C.sizeof(native.SttranAttention), dtype=0, num_seq=n, num_q_heads=1, num_kv_heads=1, head_dim=64, seq_off=4096, key_off=4096,
                               scale=1.0)
    assert lib.sttran_attention_forward(C.byref(a), None) == want and lib.sttran_attention_backward(C.byref(a), None) == want


def test_one_set_of_compiler_flags():
    """a change of the flags makes every object anew, and the tools that compile single sources take the flags from the same place"""
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc = os.path.join(root, "nl-vsgg_amd", "csrc")
    run = lambda *a: subprocess.run(["make", "-C", csrc, "--no-print-directory", *a], capture_output=True, text=True, check=True).stdout  # noqa: E731
    flags = run("-s", "print-flags").split()
    assert flags[:4] == ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"] and "--offload-arch=gfx950" in flags
    anew = run("-n", "-W", "Makefile")
    sources = [f for f in os.listdir(csrc) if f.endswith(".hip")]
    assert len(sources) > 20 and all(f"-c {f} " in anew for f in sources)
    for tool in ("kernel_resources.py", "experiments/build_variant.sh", "experiments/build_mc_trace.sh"):
        text = open(os.path.join(root, "tools", tool)).read()
        assert "print-flags" in text and "-O3" not in text, tool


def test_a_number_that_wants_a_gradient_is_refused():
    from nl_vsgg_amd.lib import sequence_ops as ops
    x = torch.tensor(0.5, requires_grad=True)
    for args in ((x, 0.0), (None, x)):
        with pytest.raises(ValueError, match="no gradient"):
            ops._score("packed_attention", *args, 64)
        with torch.no_grad():
            ops._score("packed_attention", *args, 64)
    assert ops._score("packed_attention", torch.tensor(0.5), None, 64) == (0.5, 0.0)
