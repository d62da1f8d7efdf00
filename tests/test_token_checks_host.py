"""Refusals of the token and AdamW entry points at the borders of their arguments' types; no GPU."""
import ctypes as C
import glob
import os
import re
import subprocess
import sys

import pytest

from illumina import _lib
from tests.conftest import PKG_DIR
from tests.test_tokens_host import attention_args, refused


def rotary_args(**over):
    a = _lib.RotaryArgs(precision=0, batch=1, tokens=4, head_dim=16, pairs=8, axes=2, positions=0x1000, turns=0x1000, axis=0x1000)
    a.first.x = a.first.y = 0x1000
    a.first.heads = 2
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("pairs", [2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, -1, -2 ** 31])
def test_rotary_pairs_whose_double_leaves_the_type(pairs):
    # in a process of its own: a count that passed the check would divide by zero in the launch's sizes
    code = f"""
import ctypes as C, sys
sys.path[:0] = [{PKG_DIR!r}]
from illumina import _lib
a = _lib.RotaryArgs(precision=0, batch=1, tokens=4, head_dim=16, pairs={pairs}, axes=2, positions=0x1000, turns=0x1000, axis=0x1000)
a.first.x = a.first.y = 0x1000
a.first.heads = 2
print(_lib.lib().illumina_op_rotary(C.byref(a), None), _lib.lib().illumina_last_error().decode())
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.startswith(f"{_lib.INVALID_ARG} ") and "pairs" in run.stdout


def test_vectors_between_the_places_of_their_type():
    lib = _lib.lib()
    at, off = 0x1000, 0x1002
    for n in range(4):  # w, b, mean, rstd
        w, b, mean, rstd = (off if i == n else at for i in range(4))
        refused(lib.illumina_op_layer_norm(0, at, 8, 4, 8, w, b, 1e-6, at, 8, mean, rstd, None), "misaligned")
    for n in range(5):  # w, mean, rstd, dw, db
        w, mean, rstd, dw, db = (off if i == n else at for i in range(5))
        refused(lib.illumina_op_layer_norm_backward(0, at, 8, at, 8, 4, 8, w, mean, rstd, at, 8, dw, db, at, 1 << 20, None), "misaligned")
    for over in (dict(positions=off), dict(turns=0x1004), dict(axis=off)):
        refused(lib.illumina_op_rotary(C.byref(rotary_args(**over)), None), "misaligned")
    for over in (dict(q_lens=off), dict(k_lens=off), dict(lse=off)):
        refused(lib.illumina_op_attention(C.byref(attention_args(**over)), None), "misaligned")
        a = attention_args(workspace=at, workspace_bytes=1 << 40, **over)
        refused(lib.illumina_op_attention_backward(C.byref(a), None), "misaligned")
    for name in ("m_scale", "v_scale"):
        o = _lib.AdamwOptions(device=0, tensors=1, params=(C.c_void_p * 1)(at), counts=(C.c_longlong * 1)(5), moment_bits=8,
                              m=at, v=at, m_scale=at, v_scale=at)
        setattr(o, name, off)
        refused(lib.illumina_adamw_create(C.byref(o), C.byref(C.c_void_p())), "misaligned")


def test_kernels_that_start_early_promise_nothing_about_memory():
    """A kernel launched to start while the one before it still writes must not declare what that one writes read-only for
    its own life (const __restrict__ lets the compiler load it early, or through a cache that is not kept coherent)."""
    sources = {f: open(f).read() for f in glob.glob(os.path.join(PKG_DIR, "csrc", "*.cu"))}
    started = {(f, name) for f, text in sources.items() for name in re.findall(r"launch_next\((k_\w+)", text)}
    assert {name for _, name in started} >= {"k_norm_reduce", "k_attn_join", "k_attn_dkv", "k_attn_dkv_join", "k_attn_dkv_tc"}
    for f, name in started:
        head, body = re.search(r"__global__[^;{]*?\b" + name + r"\((.*?)\)\s*\{(.*?)\n\}", sources[f], re.S).groups()
        assert "__restrict__" not in head, name
        assert "cudaGridDependencySynchronize();" in body, name


def test_gradients_are_not_lost_in_silence():
    torch = pytest.importorskip("torch")
    import illumina
    from illumina import ops
    x, q, w = torch.zeros(4, 8), torch.zeros(1, 4, 2, 8), torch.zeros(8, requires_grad=True)
    g, qg = x.clone().requires_grad_(), q.clone().requires_grad_()
    lse, stats, positions = torch.zeros(1, 2, 4), torch.zeros(4), torch.zeros(1, 4, dtype=torch.int32)
    plan = illumina.createRotary(8, [4], device="cpu")
    calls = [lambda: ops.layerNorm(g), lambda: ops.layerNorm(x, w), lambda: ops.layerNorm(x, None, w), lambda: ops.layerNorm(x, out=g),
             lambda: ops.layerNormBackward(g, x, stats, stats), lambda: ops.layerNormBackward(x, g, stats, stats),
             lambda: ops.layerNormBackward(x, x, stats, stats, w), lambda: ops.rotary(qg, positions, plan),
             lambda: ops.rotary(q, positions, plan, k=qg), lambda: ops.rotary(q, positions, plan, outQ=qg),
             lambda: ops.attention(qg, q, q), lambda: ops.attention(q, qg, q), lambda: ops.attention(q, q, qg),
             lambda: ops.attentionBackward(qg, q, q, q, q, lse), lambda: ops.attentionBackward(q, q, q, q, qg, lse)]
    for i, call in enumerate(calls):
        with pytest.raises(illumina.IlluminaError, match="requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(illumina.IlluminaError, match="CUDA tensor"):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(illumina.IlluminaError, match="tangent"):
            ops.layerNorm(dual)


def test_attention_wait_limit_refusal():
    refused(_lib.lib().illumina_op_attention_set_wait_limit(-1), "negative")
    assert _lib.lib().illumina_op_attention_set_wait_limit(0) == _lib.OK


def shares(backward, **over):
    """Shares that the workspace has room for: of the keys (forward), of the query tiles (backward)."""
    a, n = attention_args(precision=0, **over), C.c_size_t(0)
    assert _lib.lib().illumina_op_attention_workspace(C.byref(a), backward, C.byref(n)) == _lib.OK
    rows = a.batch * a.heads * a.q_tokens
    if not backward:
        return n.value // (4 * rows * (a.head_dim + 1)) or 1
    return (n.value - 4 * ((rows + 3) // 4 * 4)) // (8 * a.batch * a.kv_heads * a.k_tokens * a.head_dim) or 1


@pytest.mark.parametrize("tokens", [25000, 3000, 513, 512, 511, 200, 64, 1])
@pytest.mark.parametrize("heads", [(1, 1), (4, 1), (12, 4)])
@pytest.mark.parametrize("d", [32, 104])
def test_no_share_of_the_cuda_core_kernels_is_planned_empty(tokens, heads, d):
    wide = 64 if d <= 64 else 32
    h, hk = heads
    for backward in (0, 1):
        n = shares(backward, batch=1, heads=h, kv_heads=hk, head_dim=d, q_tokens=tokens if backward else 30,
                   k_tokens=30 if backward else tokens)
        tiles = -(-tokens // wide) * (h // hk if backward else 1)
        per = -(-tiles // n)
        assert n == 1 or (n - 1) * per < tiles, (backward, n, tiles)


def test_streams_of_another_device_are_refused():
    torch = pytest.importorskip("torch")
    import illumina
    from illumina import ops

    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 0

    with pytest.raises(illumina.IlluminaError, match="stream of cuda:0") as e:
        ops._On(torch.device("cuda", 0), Stream())
    assert e.value.status == _lib.INVALID_ARG
    x = torch.zeros(4, 8)
    for stream in (0, Stream()):
        with pytest.raises(illumina.IlluminaError, match="CUDA tensor"):
            ops.layerNorm(x, stream=stream)
