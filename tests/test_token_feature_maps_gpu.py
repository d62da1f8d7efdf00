"""The token operators on a feature map of the depth network: a frame's bottleneck pixels as tokens, normed, rotated by their
row and column, attended to, and back; against the 64-bit formulas stage by stage, in both types."""
import pytest

from tests import token_reference as R
from tests.test_tokens_gpu import TYPES, ops, randn, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def feature_map(torch):  # noqa: F811
    import illumina
    model = illumina.createDepthModel(illumina.buildArchitecture(224), synthSeed=5, keepIntermediates=True)
    frames = torch.rand(1, 3, 224, 224, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    model.forward(frames)
    model.sync()
    name = max(model.arch.tensors, key=lambda n: model.arch.tensors[n].c)  # the widest map
    data, _ = model.debugTensor(name)
    model.destroy()
    return torch.from_numpy(data).cuda()


@pytest.mark.parametrize("dtype", TYPES)
def test_stage_over_a_feature_map(torch, ops, feature_map, dtype):  # noqa: F811
    import illumina
    h, w, c = feature_map.shape
    x = feature_map.to(getattr(torch, dtype)).reshape(1, h * w, c)
    assert bool(torch.isfinite(x).all()) and float(x.float().std()) > 0
    heads, d = 4, 32
    weight, bias = 1 + randn(torch, c) * 0.1, randn(torch, c, seed=1) * 0.1
    y, mean, rstd = ops.layerNorm(x, weight, bias)
    want, _, _, tol = R.norm(x, weight, bias, 1e-6)
    R.close(y, want, tol, "y")
    at = torch.arange(h * w, device="cuda")
    positions = torch.stack((at // w, at % w)).to(torch.int32)
    plan = illumina.createRotary(d, [d // 4, d // 4])
    q = y[:, :, :heads * d].reshape(1, h * w, heads, d)  # tokens' columns as heads, without a projection
    k, v = q[:, :, :1], q[:, :, 1:2]
    rq, rk = ops.rotary(q, positions, plan, k=k)
    for got, given in ((rq, q), (rk, k)):
        want, tol = R.rotate(given, positions[:, None], plan.turns, plan.axis, False, False)
        R.close(got, want, tol, "rotated")
    out, lse = ops.attention(rq, rk, v)
    dout = randn(torch, *out.shape, dtype=dtype, seed=2)
    grads = ops.attentionBackward(dout, rq, rk, v, out, lse)
    want, tol = R.attention(rq, rk, v, d ** -0.5, 0, None, None, dout)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        R.close(got, want[name], tol[name], name)
    dq, dk = ops.rotary(grads[0], positions, plan, k=grads[1], inverse=True)
    dy = torch.zeros_like(y)
    dy[:, :, :heads * d] = dq.reshape(1, h * w, heads * d)
    dy[:, :, :d] += dk[:, :, 0]
    dy[:, :, d:2 * d] += grads[2][:, :, 0]
    got = ops.layerNormBackward(dy, x, mean, rstd, weight)
    for name, g, wt, t in zip(("dx", "dw", "db"), got, *R.norm_backward(dy, x, weight, 1e-6)):
        R.close(g, wt, t, name)
