"""The token operators on the GPU against 64-bit implementations, with tolerances derived from the roundings
(token_reference.py): types, odd sizes, strides, masks that leave rows empty, padding that holds NaN, other streams,
captured graphs, and a transformer block's training step built from them."""
import pytest

from tests import token_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.fixture(scope="module")
def ops():
    from illumina import ops
    return ops


TYPES = ["float32", "bfloat16"]


def randn(torch, *shape, dtype="float32", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g, device="cuda").to(getattr(torch, dtype))


# ---- layer norm ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 8), (7, 33), (5, 96), (2, 128), (9, 176), (300, 257), (1000, 704), (64, 1023),
                                    (64, 1024), (33, 1025), (40, 2048), (17, 4095), (9, 4096), (5, 5000), (3, 8200)])
def test_norm(torch, ops, dtype, rows, c):
    x = randn(torch, rows, c, dtype=dtype) * 3 + randn(torch, c).to(getattr(torch, dtype))
    w, b, dy = 1 + randn(torch, c, seed=1) * 0.3, randn(torch, c, seed=2), randn(torch, rows, c, dtype=dtype, seed=3)
    y, mean, rstd = ops.layerNorm(x, w, b, eps=1e-5)
    want, _, _, tol = R.norm(x, w, b, 1e-5)
    R.close(y, want, tol, "y")
    assert y.dtype == x.dtype and mean.dtype == rstd.dtype == torch.float32
    got = ops.layerNormBackward(dy, x, mean, rstd, w)
    for name, g, wt, t in zip(("dx", "dw", "db"), got, *R.norm_backward(dy, x, w, 1e-5)):
        R.close(g, wt, t, name)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_without_weights_strided_and_in_place(torch, ops, dtype):
    wide = randn(torch, 50, 3, 208, dtype=dtype)
    x = wide[:, 1, 8:184]  # rows 624 elements apart
    want, _, _, tol = R.norm(x, None, None, 1e-6)
    y, mean, rstd = ops.layerNorm(x)
    R.close(y, want, tol, "y")
    dy = randn(torch, 50, 400, dtype=dtype, seed=4)[:, 3:179]  # not 16-byte aligned
    dx, dw, db = ops.layerNormBackward(dy, x, mean, rstd, needWeight=False)
    assert dw is None and db is None
    ref, tols = R.norm_backward(dy, x, None, 1e-6)
    R.close(dx, ref[0], tols[0], "dx")
    other = wide.clone()
    ops.layerNorm(x, out=x)
    assert torch.equal(x, y)
    assert torch.equal(wide[:, 0], other[:, 0]) and torch.equal(wide[:, 1, :8], other[:, 1, :8])
    assert torch.equal(wide[:, 1, 184:], other[:, 1, 184:])


def test_norm_shapes_and_empty(torch, ops):
    x = randn(torch, 2, 5, 7, 24)
    y, mean, _ = ops.layerNorm(x)
    assert y.shape == x.shape and mean.numel() == 70
    y, mean, rstd = ops.layerNorm(x[:0])
    assert y.shape == (0, 5, 7, 24)
    dx, dw, db = ops.layerNormBackward(x[:0], x[:0], mean, rstd)
    assert dx.shape == (0, 5, 7, 24) and not dw.any() and not db.any()
    row = randn(torch, 24).expand(6, 24)  # one row seen six times
    assert torch.equal(ops.layerNorm(row)[0], ops.layerNorm(row.contiguous())[0])
    constant = torch.full((4, 96), 3.0, device="cuda")
    y, _, rstd = ops.layerNorm(constant, eps=1e-4)
    assert not y.any() and torch.allclose(rstd, torch.full_like(rstd, 100.0))


def test_norm_same_bits_again(torch, ops):
    x, dy = randn(torch, 5000, 320), randn(torch, 5000, 320, seed=1)
    _, mean, rstd = ops.layerNorm(x)
    first = ops.layerNormBackward(dy, x, mean, rstd)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.layerNormBackward(dy, x, mean, rstd)))


# ---- rotary positions -----------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,h,hk,d,sections,interleaved", [
    (1, 1, 1, 1, 2, [1], False), (2, 5, 3, 1, 32, [8, 8], False), (1, 196, 6, 2, 64, [10, 11, 11], True),
    (2, 33, 4, 4, 48, [5, 7], False), (1, 7, 2, 1, 50, [3, 4, 5], True), (3, 17, 8, 8, 128, [64], False),
    (1, 9, 5, 1, 200, [40, 0, 30], True), (2, 300, 12, 4, 64, [16, 8, 8], False)])
def test_rotary(torch, ops, dtype, b, t, h, hk, d, sections, interleaved):
    import illumina
    packed = randn(torch, b, t, h + 2 * hk, d, dtype=dtype)
    q, k = packed[:, :, :h], packed[:, :, h:h + hk]
    plan = illumina.createRotary(d, sections, interleaved=interleaved)
    g = torch.Generator(device="cuda").manual_seed(5)
    positions = torch.randint(-1000, 1000000, (len(sections), b, t), generator=g, device="cuda", dtype=torch.int32)
    for inverse in (False, True):
        got = ops.rotary(q, positions, plan, k=k, inverse=inverse)
        for name, x, y in zip("qk", (q, k), got):
            want, tol = R.rotate(x, positions, plan.turns, plan.axis, interleaved, inverse)
            R.close(y, want, tol, name)
    alone = ops.rotary(q, positions, plan)
    assert torch.equal(alone, ops.rotary(q, positions, plan, k=k)[0])


def test_rotary_plans(torch):
    import math

    import illumina
    p = illumina.createRotary(32, [4, 6], base=100.0)
    want = [100.0 ** (-j / 4) for j in range(4)] + [100.0 ** (-j / 6) for j in range(6)]
    assert torch.allclose(p.turns.cpu() * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-14)
    assert p.axis.tolist() == [0] * 4 + [1] * 6
    p = illumina.createRotary(32, [4, 6], base=100.0, spectrum="shared")
    assert torch.allclose(p.turns.cpu() * 2 * math.pi, torch.tensor([100.0 ** (-j / 10) for j in range(10)], dtype=torch.float64), rtol=1e-14)


def test_rotary_in_place_shared_and_fractional_positions(torch, ops):
    import illumina
    plan = illumina.createRotary(40, [8, 8])
    q = randn(torch, 3, 11, 4, 40)
    positions = torch.rand(2, 11, device="cuda") * 30
    want, tol = R.rotate(q, positions[:, None].expand(2, 3, 11), plan.turns, plan.axis, False, False)
    y = ops.rotary(q, positions, plan)
    R.close(y, want, tol, "fractional")
    x = q.clone()
    ops.rotary(x, positions, plan, outQ=x)
    assert torch.equal(x, y)
    assert ops.rotary(q[:0], positions, plan).shape == (0, 11, 4, 40)
    assert ops.rotary(q[:, :0], positions[:, :0], plan).shape == (3, 0, 4, 40)


# ---- attention --------------------------------------------------------------------

# b, tq, tk, heads, key heads, head size, causal block, query lengths, key lengths
ATTENTION = [
    (1, 1, 1, 1, 1, 64, 0, None, None),
    (2, 1, 300, 4, 1, 64, 0, None, [300, 7]),
    (1, 3, 5, 2, 1, 8, 1, None, None),
    (2, 17, 17, 3, 3, 32, 0, None, None),
    (1, 64, 64, 2, 2, 64, 1, None, None),
    (1, 128, 128, 1, 1, 128, 0, None, None),
    (2, 129, 129, 4, 2, 64, 1, None, None),
    (1, 196, 588, 6, 2, 64, 196, None, None),
    (1, 130, 260, 2, 1, 96, 49, None, None),
    (3, 100, 100, 4, 4, 40, 0, [100, 37, 1], [100, 50, 3]),
    (3, 150, 140, 8, 2, 128, 1, [150, 0, 90], [140, 100, 0]),
    (2, 90, 40, 2, 2, 64, 1, None, None),        # more queries than keys: the first 50 rows see nothing
    (2, 70, 130, 2, 2, 64, 7, [70, 64], [65, 130]),
    (1, 257, 513, 2, 1, 72, 1000, None, None),   # one causal block over all
    (1, 300, 300, 5, 1, 16, 3, None, None),
    (2, 40, 40, 2, 1, 33, 1, None, [40, 20]),    # an odd head size
    (1, 20, 50, 1, 1, 1, 0, None, None),
    (1, 400, 400, 2, 1, 64, 64, [399], [400]),
    (1, 700, 700, 1, 1, 64, 1, None, None),
    (1, 2, 3000, 3, 1, 128, 0, None, [2999]),
]


def attention_inputs(torch, case, dtype, poison=True):
    b, tq, tk, h, hk, d, block, qlens, klens = case
    q, dout = randn(torch, b, tq, h, d, dtype=dtype), randn(torch, b, tq, h, d, dtype=dtype, seed=1)
    k, v = randn(torch, b, tk, hk, d, dtype=dtype, seed=2), randn(torch, b, tk, hk, d, dtype=dtype, seed=3)
    if poison:  # padding holds anything
        for n in range(b):
            if qlens:
                q[n, qlens[n]:], dout[n, qlens[n]:] = float("nan"), float("inf")
            if klens:
                k[n, klens[n]:], v[n, klens[n]:] = float("-inf"), float("nan")
    lens = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, k, v, dout, {"causalBlock": block, "qLens": lens(qlens), "kLens": lens(klens)}


def check_attention(torch, ops, q, k, v, dout, masks, scale=None):
    out, lse = ops.attention(q, k, v, scale=scale, **masks)
    grads = ops.attentionBackward(dout, q, k, v, out, lse, scale=scale, **masks)
    res, tol = R.attention(q, k, v, q.shape[-1] ** -0.5 if scale is None else scale, masks["causalBlock"], masks["qLens"],
                           masks["kLens"], dout)
    got = {"out": out, "lse": lse, "dq": grads[0], "dk": grads[1], "dv": grads[2]}
    for name in got:
        R.close(got[name], res[name], tol[name], name)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(map(str, c[:7])))
def test_attention(torch, ops, dtype, case):
    check_attention(torch, ops, *attention_inputs(torch, case, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_packed_projection_and_scale(torch, ops, dtype, d):
    packed = randn(torch, 2, 150, 6 + 2 * 2, d, dtype=dtype)
    q, k, v = packed[:, :, :6], packed[:, :, 6:8], packed[:, :, 8:]
    dout = randn(torch, 2, 6, 150, d, dtype=dtype, seed=1).transpose(1, 2)  # heads before tokens
    check_attention(torch, ops, q, k, v, dout, {"causalBlock": 10, "qLens": None, "kLens": None}, scale=0.3)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_broadcast_and_misaligned(torch, ops, dtype):
    q, dout = randn(torch, 3, 70, 2, 64, dtype=dtype), randn(torch, 3, 70, 2, 64, dtype=dtype, seed=1)
    k = randn(torch, 1, 80, 1, 64, dtype=dtype, seed=2).expand(3, 80, 2, 64)  # one cache for all sequences and heads
    v = randn(torch, 80 * 64 + 1, dtype=dtype, seed=3)[1:].view(1, 80, 1, 64).expand(3, 80, 2, 64)  # an odd address
    check_attention(torch, ops, q, k, v, dout, {"causalBlock": 0, "qLens": None, "kLens": None})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 4.0])
def test_attention_scales(torch, ops, dtype, scale):
    q, k, v, dout, masks = attention_inputs(torch, (1, 140, 150, 2, 1, 64, 1, None, None), dtype)
    check_attention(torch, ops, q, k, v, dout, masks, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_empty_sizes(torch, ops, dtype):
    for b, tq, tk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0)):
        q, k, v = (randn(torch, b, n, 2, 64, dtype=dtype) for n in (tq, tk, tk))
        out, lse = ops.attention(q, k, v)
        assert out.shape == q.shape and not out.any() and bool((lse == float("-inf")).all())
        dq, dk, dv = ops.attentionBackward(q, q, k, v, out, lse)
        assert not dq.any() and not dk.any() and not dv.any() and dk.shape == k.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_logits_and_infinite_logit_rows(torch, ops, dtype):
    # logits of hundreds: one key takes all; a key of -inf logit takes nothing
    q, k, v, dout, masks = attention_inputs(torch, (1, 140, 260, 1, 1, 64, 0, None, None), dtype)
    out, lse = ops.attention(q * 30, k, v)
    res, tol = R.attention(q * 30, k, v, 64 ** -0.5, 0, None, None)
    R.close(out, res["out"], tol["out"], "out")
    R.close(lse, res["lse"], tol["lse"], "lse")
    q = q.abs()
    k[:, 1::2] = float("-inf")  # every second key's logit is -inf
    out, lse = ops.attention(q, k, v)
    few, _ = ops.attention(q, k[:, ::2].contiguous(), v[:, ::2].contiguous())
    # the same sums in another order: both are within the tolerance of the exact result
    res, tol = R.attention(q, k[:, ::2], v[:, ::2], 64 ** -0.5, 0, None, None)
    R.close(out, res["out"], tol["out"], "out")
    R.close(few, res["out"], tol["out"], "few")
    k[:] = float("-inf")  # no key has any weight
    out, lse = ops.attention(q, k, v)
    assert not out.any() and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_offsets_past_32_bits(torch, ops, dtype):
    size = 2 if dtype == "bfloat16" else 4
    far = 2 ** 31 + 64  # elements between the two sequences of a cache
    if torch.cuda.mem_get_info()[0] < 3 * far * size:
        pytest.skip("not enough device memory")
    buf = torch.empty(far + 200 * 2 * 64, dtype=getattr(torch, dtype), device="cuda")
    k = buf.as_strided((2, 200, 2, 64), (far, 2 * 64, 64, 1))
    k.copy_(randn(torch, 2, 200, 2, 64, dtype=dtype))
    q, dout = randn(torch, 2, 100, 4, 64, dtype=dtype, seed=1), randn(torch, 2, 100, 4, 64, dtype=dtype, seed=2)
    got = check_attention(torch, ops, q, k, k, dout, {"causalBlock": 1, "qLens": None, "kLens": None})
    near = k.contiguous()
    out, _ = ops.attention(q, near, near, causalBlock=1)
    assert torch.equal(out, got["out"])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_padding_rows_and_guards(torch, ops, dtype):
    """Nothing outside the tensors is written: outputs are views between guards."""
    import ctypes as C

    from illumina import _lib
    q, k, v, dout, masks = attention_inputs(torch, (2, 130, 140, 4, 2, 64, 1, [130, 60], [140, 33]), dtype)
    want_out, want_lse = ops.attention(q, k, v, **masks)
    want = ops.attentionBackward(dout, q, k, v, want_out, want_lse, **masks)
    assert not want_out[1, 60:].any() and not want[0][1, 60:].any() and not want[1][1, 33:].any() and not want[2][1, 33:].any()

    def guarded(like):
        big = torch.full((like.shape[0], like.shape[1] + 2, like.shape[2] + 1, 72), 7.0, dtype=like.dtype, device="cuda")
        return big, big[:, 1:-1, :-1, :64]

    def field(x):
        return _lib.AttentionTensor(x.data_ptr(), (C.c_longlong * 3)(*x.stride()[:3]))

    outs = {n: guarded(x) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    args = _lib.AttentionArgs(precision=q.dtype == torch.bfloat16, batch=2, heads=4, kv_heads=2, head_dim=64, q_tokens=130,
                              k_tokens=140, causal_block=1, scale=64 ** -0.5, q=field(q), k=field(k), v=field(v),
                              q_lens=masks["qLens"].data_ptr(), k_lens=masks["kLens"].data_ptr(), lse=want_lse.data_ptr(),
                              dout=field(dout), workspace=work.data_ptr(), workspace_bytes=work.numel(),
                              **{n: field(x) for n, (_, x) in outs.items()})
    _lib.check(_lib.lib().illumina_op_attention(C.byref(args), torch.cuda.current_stream().cuda_stream))
    _lib.check(_lib.lib().illumina_op_attention_backward(C.byref(args), torch.cuda.current_stream().cuda_stream))
    for (n, (big, x)), w in zip(outs.items(), (want_out, *want)):
        assert torch.equal(x, w), n
        x.fill_(7.0)
        assert bool((big == 7.0).all()), n


def test_attention_gradient_against_differences(torch, ops):
    q, k, v, dout, masks = attention_inputs(torch, (2, 9, 13, 4, 2, 24, 4, [9, 5], [13, 11]), "float32", poison=False)
    out, lse = ops.attention(q, k, v, **masks)
    grads = ops.attentionBackward(dout, q, k, v, out, lse, **masks)

    def loss(*qkv):
        res, _ = R.attention(*qkv, 24 ** -0.5, 4, masks["qLens"], masks["kLens"])
        valid = R.seen(2, 9, 13, 4, masks["qLens"], masks["kLens"], "cuda").any(2)
        return (res["out"] * torch.where(valid[:, :, None, None], dout.double(), 0.0)).sum()

    step = 1e-5
    for n, (x, g) in enumerate(zip((q, k, v), grads)):
        for seed in range(3):
            way = randn(torch, *x.shape, seed=40 + seed).double()
            ends = [[t.double() + (sign * step * way if i == n else 0) for i, t in enumerate((q, k, v))] for sign in (1, -1)]
            slope = (loss(*ends[0]) - loss(*ends[1])) / (2 * step)
            # central differences in 64 bits are off by step^2 of the third derivative; the gradient by 32-bit sums
            assert abs(float(slope - (g.double() * way).sum())) <= 2e-5 * float((g.double() * way).abs().sum() + 1)


def test_same_bits_again(torch, ops):
    for dtype in TYPES:
        q, k, v, dout, masks = attention_inputs(torch, (2, 500, 500, 8, 2, 64, 1, [500, 320], [500, 320]), dtype)
        out, lse = ops.attention(q, k, v, **masks)
        first = ops.attentionBackward(dout, q, k, v, out, lse, **masks)
        for _ in range(3):
            out2, lse2 = ops.attention(q, k, v, **masks)
            assert torch.equal(out, out2) and torch.equal(lse, lse2)
            again = ops.attentionBackward(dout, q, k, v, out, lse, **masks)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- together ----------------------------------------------------------------------

def block_step(torch, ops, plan, x, dy, w, positions, masks, stream=None):
    """A pre-norm attention block's forward and backward pass; projections are torch products."""
    b, t, c = x.shape
    h, hk, d = 4, 2, 32
    y, mean, rstd = ops.layerNorm(x, w["g"], w["b"], stream=stream)
    qkv = (y @ w["qkv"]).view(b, t, h + 2 * hk, d)
    q, k = ops.rotary(qkv[:, :, :h], positions, plan, k=qkv[:, :, h:h + hk], stream=stream)
    v = qkv[:, :, h + hk:]
    a, lse = ops.attention(q, k, v, stream=stream, **masks)
    out = a.reshape(b, t, h * d) @ w["o"]
    grads = {"o": a.reshape(-1, h * d).t() @ dy.reshape(-1, c)}
    da = (dy @ w["o"].t()).view(b, t, h, d)
    dq, dk, dv = ops.attentionBackward(da, q, k, v, a, lse, stream=stream, **masks)
    dq, dk = ops.rotary(dq, positions, plan, k=dk, inverse=True, stream=stream)
    dqkv = torch.cat((dq, dk, dv), 2).view(b, t, -1)
    grads["qkv"] = y.reshape(-1, c).t() @ dqkv.reshape(b * t, -1)
    dx, grads["g"], grads["b"] = ops.layerNormBackward(dqkv @ w["qkv"].t(), x, mean, rstd, w["g"], stream=stream)
    return x + out, dy + dx, grads


def block_inputs(torch):
    import illumina
    c, h, hk, d = 96, 4, 2, 32
    x, dy = randn(torch, 2, 98, c), randn(torch, 2, 98, c, seed=1)
    w = {"g": 1 + 0.1 * randn(torch, c), "b": 0.1 * randn(torch, c, seed=1),
         "qkv": randn(torch, c, (h + 2 * hk) * d) / c ** 0.5, "o": randn(torch, h * d, c) / (h * d) ** 0.5}
    i = torch.arange(98, device="cuda")
    positions = torch.stack((i // 49, i // 7 % 7, i % 7)).to(torch.int32)
    masks = {"causalBlock": 49, "qLens": None, "kLens": None}
    return illumina.createRotary(d, [4, 6, 6]), x, dy, w, positions, masks


def test_block_step_matches_autograd_in_64_bits(torch, ops):
    plan, x, dy, w, positions, masks = block_inputs(torch)
    out, dx, grads = block_step(torch, ops, plan, x, dy, w, positions, masks)
    x64, w64 = x.double().requires_grad_(), {k: v.double().requires_grad_() for k, v in w.items()}
    mean = x64.mean(-1, keepdim=True)
    y = (x64 - mean) / ((x64 - mean).square().mean(-1, keepdim=True) + 1e-6).sqrt() * w64["g"] + w64["b"]
    qkv = (y @ w64["qkv"]).view(2, 98, 8, 32)
    angle = positions.double()[plan.axis.long()].t() * plan.turns * 2 * torch.pi
    c, s = angle.cos()[None, :, None], angle.sin()[None, :, None]

    def turn(z):
        a, b = z.chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    q, k, v = turn(qkv[:, :, :4]), turn(qkv[:, :, 4:6]).repeat_interleave(2, 2), qkv[:, :, 6:].repeat_interleave(2, 2)
    logits = torch.einsum("bihd,bjhd->bhij", q, k) * 32 ** -0.5
    mask = R.seen(2, 98, 98, 49, None, None, "cuda")[:, None]
    p = torch.softmax(logits.masked_fill(~mask, float("-inf")), -1)
    want = x64 + torch.einsum("bhij,bjhd->bihd", p, v).reshape(2, 98, 128) @ w64["o"]
    want.backward(dy.double())
    # every stage keeps a relative error of a few hundred 2^-24 (sums of up to 196 terms); five stages in a row
    limit = 5 * 400 * 2.0 ** -24
    for name, a, b in [("out", out, want), ("dx", dx, x64.grad)] + [(n, grads[n], w64[n].grad) for n in grads]:
        b = b.detach()
        assert float((a.double() - b).norm() / b.norm()) <= limit, name


def test_block_step_captured_and_on_another_stream(torch, ops):
    plan, x, dy, w, positions, masks = block_inputs(torch)
    want = block_step(torch, ops, plan, x, dy, w, positions, masks)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block_step(torch, ops, plan, x, dy, w, positions, masks)
    side.synchronize()
    same = lambda a, b: torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(a[2][n], b[2][n]) for n in a[2])  # noqa: E731
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    x_in = x.clone()
    with torch.cuda.graph(graph):
        held = block_step(torch, ops, plan, x_in, dy, w, positions, masks)
    for seed in range(2):
        x_in.copy_(randn(torch, *x.shape, seed=50 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert same(held, block_step(torch, ops, plan, x_in.clone(), dy, w, positions, masks))


def test_stream_argument(torch, ops):
    q, k, v, dout, masks = attention_inputs(torch, (1, 200, 200, 2, 2, 64, 0, None, None), "bfloat16")
    want, _ = ops.attention(q, k, v)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        out, lse = ops.attention(q, k, v, stream=stream)
        grads = ops.attentionBackward(dout, q, k, v, out, lse, stream=stream)
        side.synchronize()
        assert torch.equal(out, want) and grads[0].shape == q.shape


def test_refusals(torch, ops):
    import illumina
    x = randn(torch, 4, 64)
    q = randn(torch, 1, 10, 4, 64)
    plan = illumina.createRotary(64, [32])
    pos = torch.zeros(1, 10, dtype=torch.int32, device="cuda")
    out, lse = ops.attention(q, q, q)
    mean = torch.zeros(4, device="cuda")
    bad = [
        lambda: ops.layerNorm(x.cpu()), lambda: ops.layerNorm(x.half()), lambda: ops.layerNorm(x.t()),
        lambda: ops.layerNorm(x, weight=mean), lambda: ops.layerNorm(x, eps=-1.0), lambda: ops.layerNorm(x, out=x[:2]),
        lambda: ops.layerNorm(torch.zeros(3, 0, device="cuda")),
        lambda: ops.layerNormBackward(x[:2], x, mean, mean), lambda: ops.layerNormBackward(x.bfloat16(), x, mean, mean),
        lambda: ops.layerNormBackward(x, x, mean[:3], mean), lambda: ops.layerNormBackward(x, x, None, mean),
        lambda: ops.layerNorm(randn(torch, 6, 5, 8).transpose(0, 1)),
        lambda: ops.rotary(q[..., :32], pos, plan), lambda: ops.rotary(q, pos[:, :5], plan),
        lambda: ops.rotary(q, pos.long(), plan), lambda: ops.rotary(q[0], pos, plan),
        lambda: ops.rotary(q, pos, plan, k=q[:, :5]), lambda: ops.rotary(q, pos.cpu(), plan),
        lambda: illumina.createRotary(64, [40]), lambda: illumina.createRotary(64, []),
        lambda: illumina.createRotary(64, [4], spectrum="none"),
        lambda: ops.attention(q, q[:, :, :3], q[:, :, :3]), lambda: ops.attention(q, q, q[:, :5]),
        lambda: ops.attention(q, q.bfloat16(), q), lambda: ops.attention(q[..., ::2], q, q),
        lambda: ops.attention(q, q, q, causalBlock=-1), lambda: ops.attention(q, q, q, qLens=pos[0, :1].long()),
        lambda: ops.attention(q, q, q, kLens=pos[0, :2]), lambda: ops.attention(q.half(), q.half(), q.half()),
        lambda: ops.attention(*[randn(torch, 1, 4, 1, 136)] * 3),
        lambda: ops.attentionBackward(q[:, :5], q, q, q, out, lse), lambda: ops.attentionBackward(q, q, q, q, out, None),
        lambda: ops.attentionBackward(q, q, q, q, out, lse[..., :5]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(illumina.IlluminaError) as e:
            call()
        assert e.value.status == 1, i
