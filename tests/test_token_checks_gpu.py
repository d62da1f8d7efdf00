"""Refusals of calls on torch tensors that the operators could not answer rightly, and what they keep of their arguments."""
import pytest

from tests.test_tokens_gpu import TYPES, attention_inputs, ops, randn, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def refused(call, word):
    import illumina
    from illumina import _lib
    with pytest.raises(illumina.IlluminaError, match=word) as e:
        call()
    assert e.value.status == _lib.INVALID_ARG


def test_rotary_plans_made_by_hand(torch, ops):  # noqa: F811
    """A plan's fields are vectors of one length on the device of q, as createRotary makes them."""
    from dataclasses import replace

    import illumina
    plan = illumina.createRotary(64, [16, 16])
    q, pos = randn(torch, 1, 10, 4, 64), torch.ones(2, 10, dtype=torch.int32, device="cuda")
    for over, word in ((dict(axis=plan.axis.cpu()), "axis"), (dict(axis=plan.axis[:8]), "axis"), (dict(axis=plan.axis.long()), "axis"),
                       (dict(axis=plan.axis.repeat(2)[::2]), "axis"), (dict(turns=plan.turns.repeat(2)[::2]), "turns"),
                       (dict(turns=plan.turns[::2], axis=plan.axis[::2]), "turns"), (dict(turns=plan.turns.float()), "turns"),
                       (dict(turns=plan.turns.cpu()), "turns"), (dict(turns=plan.turns.repeat(2), axis=plan.axis.repeat(2)), "pairs"),
                       (dict(turns=plan.turns[:0], axis=plan.axis[:0]), "pairs")):
        refused(lambda: ops.rotary(q, pos, replace(plan, **over)), word)
    few = replace(plan, turns=plan.turns[:8].clone(), axis=plan.axis[:8].clone())
    assert torch.equal(ops.rotary(q, pos, few)[..., 16:], q[..., 16:])


@pytest.mark.parametrize("dtype", TYPES)
def test_outputs_that_share_memory_in_views_with_gaps(torch, ops, dtype):  # noqa: F811
    import illumina
    plan = illumina.createRotary(32, [16])
    pos = torch.arange(10, dtype=torch.int32, device="cuda")[None]
    packed = randn(torch, 2, 10, 8, 32, dtype=dtype)
    kept = packed.clone()
    q, k = packed[:, :, :4], packed[:, :, 4:6]
    wide = randn(torch, 20, 3, 208, dtype=dtype)
    x = wide[:, 1, 8:184]
    heads_first = randn(torch, 2, 8, 10, 32, dtype=dtype).transpose(1, 2)
    rows = randn(torch, 40, 64, dtype=dtype)
    flat = randn(torch, 4000, dtype=dtype)
    for call in (lambda: ops.rotary(q, pos, plan, outQ=packed[:, :, 1:5]), lambda: ops.rotary(q, pos, plan, k=k, outK=packed[:, :, 3:5]),
                 lambda: ops.rotary(q, pos, plan, k=k, outQ=packed[:, :, 2:6]), lambda: ops.rotary(q[:, :9], pos[:, :9], plan, outQ=q[:, 1:]),
                 lambda: ops.rotary(q, pos, plan, k=k, outQ=packed[:, :, 4:8]),
                 lambda: ops.rotary(q, pos, plan, outQ=packed.view(-1)[1:].as_strided(q.shape, q.stride())),
                 lambda: ops.rotary(heads_first[:, :, :4], pos, plan, outQ=heads_first[:, :, 1:5]),
                 lambda: ops.layerNorm(x, out=wide[:, 1, 9:185]), lambda: ops.layerNorm(x[:19], out=x[1:]),
                 lambda: ops.layerNorm(x[:10], out=wide.view(-1)[624 + 208 + 8:].as_strided((10, 176), (312, 1))),
                 lambda: ops.layerNorm(rows[:20], out=rows.view(-1).as_strided((20, 64), (128, 1)))):
        refused(call, "overlap an input")
    # results that lie under themselves
    refused(lambda: ops.layerNorm(randn(torch, 20, 64, dtype=dtype), out=flat.as_strided((20, 64), (32, 1))), "under itself")
    refused(lambda: ops.rotary(q, pos, plan, outQ=flat.as_strided(q.shape, (640, 64, 16, 1))), "under itself")
    assert torch.equal(packed, kept)
    # parts of the same rows that do not meet, and results in place
    want = ops.rotary(q, pos, plan, k=k)
    got = ops.rotary(q, pos, plan, k=k, outK=packed[:, :, 6:])
    assert torch.equal(got[1], want[1]) and torch.equal(packed[:, :, :6], kept[:, :, :6])
    got = ops.rotary(q, pos, plan, k=k, outQ=q, outK=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    half = ops.rotary(heads_first[:, :, :4], pos, plan)
    ops.rotary(heads_first[:, :, :4], pos, plan, outQ=heads_first[:, :, 4:])
    assert torch.equal(half, heads_first[:, :, 4:])
    y = ops.layerNorm(x)[0]
    ops.layerNorm(x, out=wide[:, 0, 8:184])
    assert torch.equal(y, wide[:, 0, 8:184])
    y = ops.layerNorm(rows[::2])[0]
    ops.layerNorm(rows[::2], out=rows[1::2])
    assert torch.equal(y, rows[1::2])
    one = randn(torch, 1, 64, dtype=dtype)  # the stride of a single row says nothing
    y = ops.layerNorm(one)[0]
    ops.layerNorm(one, out=one.as_strided((1, 64), (7, 1)))
    assert torch.equal(y, one)


def test_outputs_that_share_memory_with_weights_or_positions(torch, ops):  # noqa: F811
    import illumina
    w, x = randn(torch, 64), randn(torch, 1, 64)
    refused(lambda: ops.layerNorm(x, w, out=w[None]), "overlap an input")
    refused(lambda: ops.layerNorm(x, None, w, out=w[None]), "overlap an input")
    plan = illumina.createRotary(32, [16])
    place = torch.zeros(1, 10, 4, 32, device="cuda")
    refused(lambda: ops.rotary(randn(torch, 1, 10, 4, 32), place.view(-1)[100:110][None], plan, outQ=place), "overlap an input")


def test_autograd_sees_what_the_calls_overwrite(torch, ops):  # noqa: F811
    import illumina
    plan, pos = illumina.createRotary(32, [16]), torch.arange(10, dtype=torch.int32, device="cuda")[None]
    leaf = torch.ones(1, 10, 4, 32, device="cuda", requires_grad=True)
    flat = torch.ones(40, 32, device="cuda", requires_grad=True)
    for call in (lambda x: ops.rotary(x, pos, plan, outQ=x), lambda x: ops.rotary(x.clone(), pos, plan, k=x, outK=x)):
        x = randn(torch, 1, 10, 4, 32)
        loss = (leaf * x).sum()  # saves x
        call(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    x = randn(torch, 40, 32)
    loss = (flat * x).sum()
    ops.layerNorm(x, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    p = [torch.nn.Parameter(torch.ones(8, 8, device="cuda")), torch.nn.Parameter(torch.ones(0, device="cuda"))]
    opt = illumina.createOptimizer(p)
    a = torch.ones(8, 8, device="cuda", requires_grad=True)
    loss = (a @ p[0]).sum()  # saves p[0]
    opt.step([torch.ones(8, 8, device="cuda"), torch.ones(0, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        x = randn(torch, 40, 32)
        want = ops.layerNorm(x)[0]
        ops.layerNorm(x, out=x)
        assert torch.equal(x, want)


def test_parameters_are_taken_without_a_graph(torch, ops):  # noqa: F811
    x, w = randn(torch, 40, 32), torch.nn.Parameter(torch.ones(32, device="cuda"))
    refused(lambda: ops.layerNorm(x, w), "requires a gradient")
    want = ops.layerNorm(x, w.detach())[0]
    with torch.no_grad():
        assert torch.equal(ops.layerNorm(x, w)[0], want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", [(500, 96), (700, 264), (301, 257), (40, 2048), (20, 1033), (5, 5000)])
def test_norm_entry_points_without_some_results(torch, ops, dtype, rows, c):  # noqa: F811
    """Through the C entry points: statistics not kept, dx not wanted or in dy's place, one of dw and db alone."""
    import ctypes as C

    from illumina import _lib
    lib, precision, stream = _lib.lib(), dtype == "bfloat16", torch.cuda.current_stream().cuda_stream
    x, dy = randn(torch, rows, c, dtype=dtype), randn(torch, rows, c, dtype=dtype, seed=1)
    w, b = 1 + randn(torch, c, seed=2) * 0.3, randn(torch, c, seed=3)
    y, mean, rstd = ops.layerNorm(x, w, b)
    dx, dw, db = ops.layerNormBackward(dy, x, mean, rstd, w)
    got = torch.empty_like(x)
    _lib.check(lib.illumina_op_layer_norm(precision, x.data_ptr(), c, rows, c, w.data_ptr(), b.data_ptr(), 1e-6, got.data_ptr(), c,
                                          None, None, stream))
    assert torch.equal(got, y)
    size = C.c_size_t(0)
    _lib.check(lib.illumina_op_layer_norm_workspace(rows, c, C.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device="cuda")

    def backward(dy, dx, dw, db):
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        space = (work.data_ptr(), size.value) if dw is not None or db is not None else (None, 0)
        _lib.check(lib.illumina_op_layer_norm_backward(precision, dy.data_ptr(), c, x.data_ptr(), c, rows, c, w.data_ptr(),
                                                       mean.data_ptr(), rstd.data_ptr(), at(dx), c, at(dw), at(db), *space, stream))

    new = lambda: (torch.empty_like(x), torch.empty_like(w), torch.empty_like(w))  # noqa: E731
    x1, w1, b1 = new()
    backward(dy, None, w1, b1)
    assert torch.equal(w1, dw) and torch.equal(b1, db)
    x1, w1, b1 = new()
    backward(dy, x1, w1, None)
    assert torch.equal(x1, dx) and torch.equal(w1, dw)
    x1, w1, b1 = new()
    backward(dy, x1, None, b1)
    assert torch.equal(x1, dx) and torch.equal(b1, db)
    x1 = dy.clone()
    backward(x1, x1, w1, b1)
    assert torch.equal(x1, dx) and torch.equal(w1, dw) and torch.equal(b1, db)
    x1, _, _ = new()
    backward(dy, x1, None, None)
    assert torch.equal(x1, dx)


def test_views_with_a_lazy_negation(torch, ops):  # noqa: F811
    import illumina
    z = torch.view_as_complex(randn(torch, 10, 1, 2)).conj()
    column = z.imag  # [10, 1]: rows of one element, whose values are not those in memory
    assert column.is_neg()
    refused(lambda: ops.layerNorm(column), "lazy negation")
    assert ops.layerNorm(column.resolve_neg())[0].shape == (10, 1)
    plan, q = illumina.createRotary(32, [16]), randn(torch, 1, 10, 4, 32)
    refused(lambda: ops.rotary(q, column.t(), plan), "lazy negation")
    one = z[:1, 0].imag
    refused(lambda: ops.layerNorm(randn(torch, 4, 1), one), "lazy negation")
    opt = illumina.createOptimizer([torch.ones(1, device="cuda")])
    refused(lambda: opt.step([one]), "lazy negation")
    opt.lr = one
    refused(lambda: opt.step([torch.ones(1, device="cuda")]), "lazy negation")
    refused(lambda: illumina.createOptimizer([one]), "contiguous float32")
