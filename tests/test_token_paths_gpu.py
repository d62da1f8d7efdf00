"""The token operators' variants (chosen by sizes, types and alignment) and uses that stress their launches: every width
class of the norm, shares of the key pass, results overwritten straight after a call, two streams at once, graphs."""
import pytest

from tests import token_reference as R
from tests.test_tokens_gpu import TYPES, attention_inputs, check_attention, ops, randn, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", [(5000, 136), (3000, 256), (2500, 264), (2400, 512), (2400, 516), (2500, 768), (2400, 776),
                                    (1300, 1024), (700, 1032), (300, 2056), (5000, 124), (2, 4096)])
def test_norm_width_classes(torch, ops, dtype, rows, c):  # noqa: F811
    """More rows than the backward's CTAs take at once, and widths on both sides of every class."""
    x, w = randn(torch, rows, c, dtype=dtype), 1 + randn(torch, c, seed=1) * 0.3
    b, dy = randn(torch, c, seed=2), randn(torch, rows, c, dtype=dtype, seed=3)
    y, mean, rstd = ops.layerNorm(x, w, b)
    want, _, _, tol = R.norm(x, w, b, 1e-6)
    R.close(y, want, tol, "y")
    got = ops.layerNormBackward(dy, x, mean, rstd, w)
    for name, g, wt, t in zip(("dx", "dw", "db"), got, *R.norm_backward(dy, x, w, 1e-6)):
        R.close(g, wt, t, name)
    alone = ops.layerNormBackward(dy, x, mean, rstd, w, needWeight=False)
    assert torch.equal(alone[0], got[0]) and alone[1] is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 4, 8])
def test_norm_backward_of_rows_apart(torch, ops, dtype, shift):  # noqa: F811
    """Rows with gaps, at 16-byte boundaries and between them; without weights."""
    wide = randn(torch, 900, 2, 280, dtype=dtype)
    x, dy = wide[:, 0, shift:shift + 264], randn(torch, 900, 264, dtype=dtype, seed=1)
    _, mean, rstd = ops.layerNorm(x)
    got = ops.layerNormBackward(dy, x, mean, rstd)
    for name, g, wt, t in zip(("dx", "dw", "db"), got, *R.norm_backward(dy, x, None, 1e-6)):
        R.close(g, wt, t, name)


# few key tiles with many query tiles each: the CUDA-core key pass shares them out (odd head sizes for bf16)
SHARES = [(1, 324, 324, 24, 6, 104, 0, None, None), (2, 150, 260, 8, 1, 40, 49, [150, 77], [260, 131]),
          (1, 1000, 70, 2, 1, 64, 0, None, None), (1, 900, 900, 1, 1, 128, 1, None, None),
          (2, 500, 64, 4, 2, 32, 1, [500, 0], [64, 9])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SHARES, ids=lambda c: "-".join(map(str, c[:7])))
def test_attention_shares_of_the_key_pass(torch, ops, dtype, case):  # noqa: F811
    if dtype == "bfloat16":
        case = (*case[:5], case[5] - 1, *case[6:])
    check_attention(torch, ops, *attention_inputs(torch, case, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(2, 520, 520, 4, 2, 64, 1, [520, 300], [520, 300]), (1, 300, 5000, 2, 1, 64, 0, None, None),
                                  (1, 700, 700, 2, 2, 128, 0, None, None)], ids=lambda c: "-".join(map(str, c[:7])))
def test_inputs_overwritten_straight_after_the_calls(torch, ops, dtype, case):  # noqa: F811
    """A call's kernels start while the one before finishes; what follows the call on its stream finds all of them done."""
    q, k, v, dout, masks = attention_inputs(torch, case, dtype, poison=False)
    out, lse = ops.attention(q, k, v, **masks)
    want = (out, lse, *ops.attentionBackward(dout, q, k, v, out, lse, **masks))
    torch.cuda.synchronize()
    for _ in range(10):
        q2, k2, v2, dout2 = q.clone(), k.clone(), v.clone(), dout.clone()
        out2, lse2 = ops.attention(q2, k2, v2, **masks)
        held = out2.clone(), lse2.clone()
        grads = ops.attentionBackward(dout2, q2, k2, v2, out2, lse2, **masks)
        for t in (q2, k2, v2, dout2, out2, lse2):
            t.fill_(float("nan"))
        assert all(torch.equal(a, b) for a, b in zip(want, (*held, *grads)))


def test_norm_gradients_read_straight_after_the_call(torch, ops):  # noqa: F811
    x, dy = randn(torch, 20000, 704, dtype="bfloat16"), randn(torch, 20000, 704, dtype="bfloat16", seed=1)
    _, mean, rstd = ops.layerNorm(x)
    want = ops.layerNormBackward(dy, x, mean, rstd)
    torch.cuda.synchronize()
    for _ in range(10):
        x2, dy2, m2, r2 = x.clone(), dy.clone(), mean.clone(), rstd.clone()
        got = ops.layerNormBackward(dy2, x2, m2, r2)
        for t in (x2, dy2, m2, r2):
            t.fill_(float("nan"))
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_streams_at_once(torch, ops):  # noqa: F811
    cases = [attention_inputs(torch, c, "bfloat16") for c in ((1, 196, 6000, 8, 2, 64, 0, None, None),
                                                             (2, 600, 600, 4, 4, 128, 1, None, None))]
    run = lambda c: (lambda out, lse: (out, lse, *ops.attentionBackward(c[3], *c[:3], out, lse, **c[4])))(*ops.attention(*c[:3], **c[4]))  # noqa: E731
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


def test_two_graphs_of_bf16_attention(torch, ops):  # noqa: F811
    graphs = []
    for seed in range(2):
        q, k, v, dout, masks = attention_inputs(torch, (1, 100 + seed, 4000, 4, 2, 64, 0, None, None), "bfloat16")
        ops.attention(q, k, v)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = ops.attention(q, k, v)
            grads = ops.attentionBackward(dout, q, k, v, out, lse)
        graphs.append((graph, q, k, v, dout, (out, lse, *grads)))
    for round in range(2):
        for n, (graph, q, k, v, dout, _) in enumerate(graphs):
            for t in (q, k, v, dout):
                t.copy_(randn(torch, *t.shape, dtype="bfloat16", seed=10 * round + n))
        for graph, *_ in graphs:
            graph.replay()
        for _, q, k, v, dout, held in graphs:
            out, lse = ops.attention(q, k, v)
            want = (out, lse, *ops.attentionBackward(dout, q, k, v, out, lse))
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_refuses_overlapping_outputs(torch, ops):  # noqa: F811
    import illumina
    buf = randn(torch, 101, 64)
    qk = randn(torch, 2, 2, 10, 4, 32)
    q, k = qk[0], qk[1]
    plan = illumina.createRotary(32, [16])
    pos = torch.zeros(1, 10, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.layerNorm(buf[:-1], out=buf[1:]), lambda: ops.rotary(q, pos, plan, k=k, outQ=k),
                 lambda: ops.rotary(q, pos, plan, k=k, outK=q), lambda: ops.rotary(q, pos, plan, k=k, outQ=q, outK=q),
                 lambda: ops.layerNorm(buf, out=buf[:1].expand(101, 64))):
        with pytest.raises(illumina.IlluminaError):
            call()
    y = ops.rotary(q, pos, plan, k=k, outQ=q, outK=k)  # both in place
    assert y[0].data_ptr() == q.data_ptr() and y[1].data_ptr() == k.data_ptr()


def test_refuses_a_parameter_listed_twice(torch):  # noqa: F811
    import illumina
    p = torch.zeros(1000, device="cuda")
    for params in ([p, p], [p[:600], p[500:]], [p, torch.zeros(3, device="cuda"), p[10:20]]):
        with pytest.raises(illumina.IlluminaError, match="overlap"):
            illumina.createOptimizer(params)
    illumina.createOptimizer([p[:500], p[500:], p[:0]]).destroy()


def test_two_optimizers_on_two_streams(torch):  # noqa: F811
    import illumina
    g = torch.Generator(device="cuda").manual_seed(3)
    start = torch.randn(300000, generator=g, device="cuda")
    grad = torch.randn(300000, generator=g, device="cuda")

    def steps(bits, stream):
        p = start.clone()
        torch.cuda.synchronize()
        opt = illumina.createOptimizer([p], momentBits=bits)
        return p, opt, lambda: opt.step([grad], stream=stream)

    alone = [steps(bits, None) for bits in (32, 8)]
    for _, _, step in alone:
        for _ in range(20):
            step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [steps(bits, s) for bits, s in zip((32, 8), streams)]
    for _ in range(20):
        for _, _, step in both:
            step()
    torch.cuda.synchronize()
    for (a, _, _), (b, opt, _) in zip(alone, both):
        assert torch.equal(a, b) and opt.steps == 20
