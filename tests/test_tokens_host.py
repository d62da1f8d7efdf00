"""Refusals of the token and AdamW entry points that need no GPU: bad arguments are answered before any CUDA call."""
import ctypes as C

import pytest

from illumina import _lib


def refused(status, word):
    assert status == _lib.INVALID_ARG
    assert word in _lib.lib().illumina_last_error().decode()


def attention_args(**over):
    a = _lib.AttentionArgs(precision=1, batch=2, heads=4, kv_heads=2, head_dim=64, q_tokens=10, k_tokens=12, scale=1.0)
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        getattr(a, name).data = 0x1000
    a.lse = 0x1000
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,word", [
    (dict(precision=2), "precision"), (dict(kv_heads=3), "multiple"), (dict(kv_heads=0), "multiple"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=129), "head_dim"), (dict(batch=-1), "negative"),
    (dict(q_tokens=-1), "negative"), (dict(causal_block=-2), "causal_block"), (dict(lse=None), "lse"),
    (dict(q=_lib.AttentionTensor()), "null pointer"), (dict(k=_lib.AttentionTensor()), "null pointer"),
    (dict(v=_lib.AttentionTensor(data=0x1001)), "misaligned"), (dict(batch=2 ** 30, heads=2 ** 30, kv_heads=1), "too many"),
])
def test_attention_refusals(over, word):
    lib = _lib.lib()
    refused(lib.illumina_op_attention(C.byref(attention_args(**over)), None), word)
    refused(lib.illumina_op_attention_backward(C.byref(attention_args(workspace=0x1000, workspace_bytes=1 << 40, **over)), None), word)


def test_attention_workspace_refusals():
    lib = _lib.lib()
    n = C.c_size_t(0)
    assert lib.illumina_op_attention_workspace(C.byref(attention_args()), 1, C.byref(n)) == _lib.OK
    assert n.value >= 2 * 4 * 10 * 4
    a = attention_args(workspace=0x1000, workspace_bytes=n.value - 1)
    refused(lib.illumina_op_attention_backward(C.byref(a), None), "workspace")
    a = attention_args(workspace=0x1004, workspace_bytes=n.value)
    refused(lib.illumina_op_attention_backward(C.byref(a), None), "workspace")
    a = attention_args(dk=_lib.AttentionTensor(), workspace=0x1000, workspace_bytes=n.value)
    refused(lib.illumina_op_attention_backward(C.byref(a), None), "null pointer")
    refused(lib.illumina_op_attention_workspace(None, 0, C.byref(n)), "null")
    refused(lib.illumina_op_attention(None, None), "null")


def test_norm_refusals():
    lib = _lib.lib()
    fwd = lambda p=0, x=0x1000, rows=4, c=8, eps=1e-6, y=0x1000: lib.illumina_op_layer_norm(  # noqa: E731
        p, x, c, rows, c, None, None, eps, y, c, None, None, None)
    refused(fwd(p=7), "precision")
    refused(fwd(x=None), "null")
    refused(fwd(x=0x1002), "misaligned")
    refused(fwd(rows=-1), "rows")
    refused(fwd(c=0), "width")
    refused(fwd(eps=-1.0), "eps")
    n = C.c_size_t(0)
    assert lib.illumina_op_layer_norm_workspace(1000, 96, C.byref(n)) == _lib.OK and n.value > 0
    bwd = lambda ws, size: lib.illumina_op_layer_norm_backward(  # noqa: E731
        0, 0x1000, 96, 0x1000, 96, 1000, 96, None, 0x1000, 0x1000, 0x1000, 96, 0x1000, 0x1000, ws, size, None)
    refused(bwd(None, n.value), "workspace")
    refused(bwd(0x1000, n.value - 1), "workspace")


def test_rotary_refusals():
    lib = _lib.lib()

    def args(**over):
        a = _lib.RotaryArgs(precision=0, batch=1, tokens=4, head_dim=16, pairs=8, axes=2, positions=0x1000, turns=0x1000, axis=0x1000)
        a.first.x = a.first.y = 0x1000
        a.first.heads = 2
        for k, v in over.items():
            setattr(a, k, v)
        return a

    for over, word in ((dict(precision=3), "precision"), (dict(pairs=9), "pairs"), (dict(pairs=0), "pairs"), (dict(axes=0), "axes"),
                       (dict(head_dim=2000), "head_dim"), (dict(turns=None), "null"), (dict(tokens=-1), "negative"),
                       (dict(tokens=2 ** 40), "tokens"), (dict(first=_lib.RotaryTensor(heads=2)), "null"),
                       (dict(second=_lib.RotaryTensor(heads=-1)), "head count")):
        refused(lib.illumina_op_rotary(C.byref(args(**over)), None), word)
    refused(lib.illumina_op_rotary(None, None), "null")


def test_adamw_blocks_and_refusals():
    lib = _lib.lib()
    n = C.c_longlong(0)
    counts = (C.c_longlong * 5)(1, 256, 257, 0, 1000)
    assert lib.illumina_adamw_blocks(counts, 5, C.byref(n)) == _lib.OK
    assert n.value == 1 + 1 + 2 + 0 + 4
    refused(lib.illumina_adamw_blocks((C.c_longlong * 1)(-1), 1, C.byref(n)), "size")
    out = C.c_void_p()
    params = (C.c_void_p * 5)(*[0x1000] * 5)

    def options(**over):
        o = _lib.AdamwOptions(device=0, tensors=5, params=params, counts=counts, moment_bits=32, m=0x1000, v=0x1000)
        for k, v in over.items():
            setattr(o, k, v)
        return o

    for over, word in ((dict(tensors=0), "no tensors"), (dict(moment_bits=16), "moment_bits"), (dict(m=None), "moments"),
                       (dict(v=0x1004), "moments"), (dict(moment_bits=8), "scales"), (dict(grad_precision=5), "precision"),
                       (dict(params=(C.c_void_p * 5)()), "parameter"), (dict(counts=(C.c_longlong * 5)()), "empty")):
        refused(lib.illumina_adamw_create(C.byref(options(**over)), C.byref(out)), word)
    refused(lib.illumina_adamw_step(None, None, None, None), "null")
    refused(lib.illumina_adamw_moments(None, None, None, None), "moments")
    assert lib.illumina_adamw_destroy(None) == _lib.OK


def test_tensors_off_the_gpu_are_refused():
    torch = pytest.importorskip("torch")
    import illumina
    from illumina import ops
    x, q = torch.zeros(4, 8), torch.zeros(1, 4, 2, 8)
    positions = torch.zeros(1, 4, dtype=torch.int32)
    plan = illumina.createRotary(8, [4], device="cpu")
    calls = [lambda: ops.layerNorm(x), lambda: ops.layerNormBackward(x, x, x[:, 0], x[:, 0]),
             lambda: ops.rotary(q, positions, plan), lambda: ops.attention(q, q, q),
             lambda: ops.attentionBackward(q, q, q, q, q, None), lambda: illumina.createOptimizer([x])]
    for call in calls:
        with pytest.raises(illumina.IlluminaError) as e:
            call()
        assert e.value.status == _lib.INVALID_ARG and "CUDA tensor" in str(e.value)
