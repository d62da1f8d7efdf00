"""AdamW on the GPU: against 64 bits, the 8-bit codes bit for bit, captured steps, checkpoints, and a depth model's
weights through a step and back into a model."""
import math

import numpy as np
import pytest

from tests import token_reference as R

pytestmark = pytest.mark.gpu
BLOCK = 256


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


COUNTS = [1, 255, 256, 257, 4, 0, 5000, 2048, 33, 70001]


def tensors(torch, counts, seed=0, grad="float32", gap=0):
    """Parameters and gradients as views of flat buffers, `gap` elements apart (odd addresses)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    size = sum(counts) + gap * (len(counts) + 1)
    flat, grads = torch.randn(size, generator=g, device="cuda"), torch.randn(size, generator=g, device="cuda") * 0.01
    grads = grads.to(getattr(torch, grad))
    at, p, d = gap, [], []
    for n in counts:
        p.append(flat[at:at + n])
        d.append(grads[at:at + n])
        at += n + gap
    return flat, p, d


def places(counts):
    """Element ranges of the flat moments."""
    at, out = 0, []
    for n in counts:
        out.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return out


HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weightDecay=0.1)


@pytest.mark.parametrize("grad", ["float32", "bfloat16"])
@pytest.mark.parametrize("gap", [0, 1, 8])
def test_32_bit_moments(torch, grad, gap):
    import illumina
    flat, p, d = tensors(torch, COUNTS, grad=grad, gap=gap)
    guard = torch.ones_like(flat, dtype=torch.bool)
    for x in p:
        guard[x.storage_offset():x.storage_offset() + x.numel()] = False
    kept = flat[guard].clone()
    decay = [i % 2 == 0 for i in range(len(COUNTS))]
    opt = illumina.createOptimizer(p, decay=decay, gradDtype=d[0].dtype, **HYPER)
    want = [(x.double(), torch.zeros_like(x).double(), torch.zeros_like(x).double()) for x in p]
    steps = 4
    for t in range(1, steps + 1):
        grads = [x * (1 + t) for x in d]
        opt.step(grads)
        want = [R.adamw(a, g, m, v, t, 2e-3, 0.9, 0.99, 1e-8, 0.1 if k else 0.0) for (a, m, v), g, k in zip(want, grads, decay)]
    assert opt.steps == steps
    m, v = opt.moments()
    for x, (a, b, c), (at, n) in zip(p, want, places(COUNTS)):
        # a step rounds each moment's two products and their sum, the parameter's few operations on up to lr each
        R.close(m[at:at + n], b, steps * 4 * R.E32 * (b.abs() + 0.05), "m")
        R.close(v[at:at + n], c, steps * 6 * R.E32 * (c + 0.0025), "v")
        R.close(x, a, steps * (4 * R.E32 * a.abs() + 2e-3 * 64 * R.E32 * 10), "p")
    assert torch.equal(flat[guard], kept)


def plain_8_bit(torch, p, g, m, v, ms, vs, step, lr, b1, b2, eps, wd):
    """One step of one tensor with 8-bit moments on the CPU in 32-bit operations, as documented; (p in 64 bits, codes...)."""
    f = np.float32
    n = p.size
    size = -(-n // BLOCK) * BLOCK
    gp = np.zeros(size, f)
    gp[:n] = g
    at = np.arange(size, dtype=np.uint64)
    mm = (m.astype(f) * np.repeat(ms, BLOCK)).astype(f)
    vv = (v.astype(f) * np.repeat(vs, BLOCK)).astype(f)
    vv = (vv * vv).astype(f)
    mm = ((mm * f(b1)).astype(f) + (gp * f(1 - b1)).astype(f)).astype(f)
    vv = ((vv * f(b2)).astype(f) + ((gp * gp).astype(f) * f(1 - b2)).astype(f)).astype(f)
    new = p.astype(np.float64) * (1 - lr * wd) - lr * (mm[:n].astype(np.float64) / (1 - b1 ** step)) / (
        np.sqrt(vv[:n].astype(np.float64) / (1 - b2 ** step)) + eps)
    return new, mm, np.sqrt(vv).astype(f), at


def codes(x, first, step, levels, signed):
    f = np.float32
    blocks = x.reshape(-1, BLOCK)
    top = np.abs(blocks).max(1)
    scale = np.where(top < f(2.0 ** -100), f(0), (top * f(1 / levels)).astype(f)).astype(f)
    inv = np.zeros_like(scale)
    inv[scale > 0] = (f(1) / scale[scale > 0]).astype(f)
    place = np.arange(x.size, dtype=np.uint64) + np.uint64(first)
    u = ((place * np.uint64(0x85EBCA6B) + np.uint64(step) * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)) >> np.uint64(8)
    u = (u.astype(f) * f(2.0 ** -24)).astype(f).reshape(-1, BLOCK)
    c = np.floor(((blocks * inv[:, None]).astype(f) + u).astype(f))
    c = np.clip(c, -levels if signed else 0, levels)
    if not signed:
        c = np.where((blocks > 0) & (scale[:, None] > 0), np.maximum(c, 1), c)
    return c.reshape(-1), scale


@pytest.mark.parametrize("grad", ["float32", "bfloat16"])
def test_8_bit_moments_bit_for_bit(torch, grad):
    import illumina
    flat, p, d = tensors(torch, COUNTS, grad=grad, seed=3)
    d[8].zero_()  # a tensor without gradient keeps zero moments
    opt = illumina.createOptimizer(p, momentBits=8, gradDtype=d[0].dtype, **HYPER)
    held = [(x.cpu().numpy().copy(),) for x in p]
    m = [np.zeros(-(-n // BLOCK) * BLOCK, np.int8) for n in COUNTS]
    v = [np.zeros(-(-n // BLOCK) * BLOCK, np.uint8) for n in COUNTS]
    s = [(np.zeros(x.size // BLOCK, np.float32), np.zeros(x.size // BLOCK, np.float32)) for x in m]
    for step in (1, 2, 3):
        grads = [x * step for x in d]
        opt.step(grads)
        for i, (at, n) in enumerate(places(COUNTS)):
            if not n:
                continue
            new, mm, root, _ = plain_8_bit(torch, held[i][0], grads[i].float().cpu().numpy(), m[i], v[i], *s[i], step, 2e-3,
                                           0.9, 0.99, 1e-8, 0.1)
            mc, msc = codes(mm, at, step, 127, True)
            vc, vsc = codes(root, at, step, 255, False)
            size = m[i].size
            assert np.array_equal(opt.m[at:at + size].cpu().numpy(), mc), (step, i)
            assert np.array_equal(opt.v[at:at + size].cpu().numpy(), vc), (step, i)
            assert np.array_equal(opt.mScale[at // BLOCK:(at + size) // BLOCK].cpu().numpy(), msc)
            assert np.array_equal(opt.vScale[at // BLOCK:(at + size) // BLOCK].cpu().numpy(), vsc)
            m[i], v[i], s[i] = mc.astype(np.int8), vc.astype(np.uint8), (msc, vsc)
            got = p[i].cpu().numpy()
            assert np.abs(got - new).max() <= 2 ** -24 * 4 * np.abs(new).max() + 2e-3 * 64 * 2 ** -24 * 10
            held[i] = (got.copy(),)
    mv, vv = opt.moments()
    size = sum(x.size for x in m)
    assert mv.numel() == vv.numel() == size
    want = np.concatenate([c.astype(np.float32) * np.repeat(sc[0], BLOCK) for c, sc in zip(m, s)])
    assert np.array_equal(mv.cpu().numpy(), want)


def test_8_bit_second_moment_follows_a_change_of_scale(torch):
    """Rounding to the nearest code would hold the second moment where it is: a step moves it by less than a code."""
    import illumina
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.zeros(4096, device="cuda")
    opt = illumina.createOptimizer([p], lr=0.0, betas=(0.9, 0.999), momentBits=8)
    big = torch.ones(4096, device="cuda")
    big[::2] = 0.25
    opt.step([big])
    for _ in range(1500):
        opt.step([torch.full((4096,), 0.5, device="cuda") * torch.sign(torch.randn(4096, generator=g, device="cuda"))])
    _, v = opt.moments()
    # exactly: v = b^1500 (1 - b) g0^2 + (1 - b^1500) / 4; the codes' noise is a few hundredths of a root
    want = 0.25 * (1 - 0.999 ** 1500)
    for half in (v[::2], v[1::2]):
        assert abs(float(half.mean()) / want - 1) < 0.1


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_count_on(torch, bits):
    import illumina
    runs = []
    for captured in (False, True):
        _, p, d = tensors(torch, COUNTS, seed=7)
        lr = torch.tensor([1e-2], device="cuda")
        opt = illumina.createOptimizer(p, lr=lr, momentBits=bits)
        opt.step(d)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step(d)
        for k in range(5):
            lr.fill_(1e-2 / (k + 1))
            if captured:
                graph.replay()
            else:
                opt.step(d)
        assert opt.steps == 6
        runs.append((p, opt.state()))
        torch.cuda.synchronize()
    (a, sa), (b, sb) = runs
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(sa["m"], sb["m"]) and torch.equal(sa["v"], sb["v"])


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_resumes_bit_for_bit(torch, bits):
    import illumina
    _, p, d = tensors(torch, COUNTS, seed=9)
    opt = illumina.createOptimizer(p, momentBits=bits)
    for _ in range(3):
        opt.step(d)
    state, params = opt.state(), [x.clone() for x in p]
    opt.step(d)
    again = illumina.createOptimizer(params, momentBits=bits)
    again.loadState(state)
    again.step(d)
    assert again.steps == 4 and all(torch.equal(x, y) for x, y in zip(p, params))
    assert torch.equal(opt.m, again.m) and torch.equal(opt.v, again.v)
    opt.destroy()
    with pytest.raises(illumina.IlluminaError):
        opt.step(d)


def test_more_tensors_than_one_launch_carries(torch):
    import illumina
    counts = [(7 * i) % 600 for i in range(1000)]  # some empty
    _, p, d = tensors(torch, counts, seed=11)
    before = [x.clone() for x in p]
    opt = illumina.createOptimizer(p, lr=1e-2, weightDecay=0.0)
    opt.step(d)
    assert opt.steps == 1
    for x, y, g in zip(p, before, d):
        # the first step moves every element by lr * sign(g), up to eps / |g|
        want = y.double() - 1e-2 * g.double() / (g.double().abs() + 1e-8)
        R.close(x, want, 4 * R.E32 * want.abs() + 1e-2 * 64 * R.E32, "p")


def test_special_gradients(torch):
    import illumina
    for bits in (32, 8):
        p = torch.ones(1024, device="cuda")
        g = torch.full((1024,), 0.1, device="cuda")
        g[300] = math.nan
        opt = illumina.createOptimizer([p], momentBits=bits)
        opt.step([g])
        m, _ = opt.moments()
        spoiled = torch.isnan(m)
        assert bool(spoiled[300]) and not spoiled[:256].any() and not spoiled[512:].any()
        assert int(torch.isnan(p).sum()) == 1
        p = torch.ones(512, device="cuda")
        opt = illumina.createOptimizer([p], momentBits=bits, weightDecay=0.0)
        opt.step([torch.zeros(512, device="cuda")])
        assert bool((p == 1).all())
        opt.step([torch.full((512,), 1e-36, device="cuda")])
        assert bool(torch.isfinite(p).all()) and bool(torch.isfinite(opt.moments()[0]).all())


def test_depth_model_weights_through_a_step(torch):
    import illumina
    arch = illumina.buildArchitecture(64)
    weights = illumina.synthesizeWeights(arch, 3)
    specs = illumina.weightSpecs(arch)
    params = [torch.from_numpy(weights[n]).cuda() for n, _ in specs]
    grads = [torch.ones_like(p) for p in params]
    opt = illumina.createOptimizer(params, lr=1e-3, weightDecay=0.0, decay=[len(s) > 1 for _, s in specs])
    opt.step(grads)
    stepped = {n: p.cpu().numpy() for (n, _), p in zip(specs, params)}
    for n, _ in specs:
        assert np.abs(stepped[n] - (weights[n] - np.float32(1e-3))).max() <= 1e-6
    back = illumina.parseWeights(illumina.serializeWeights(arch, stepped), arch)
    assert all(np.array_equal(back[n], stepped[n]) for n in stepped)
    frames = torch.rand(1, 3, 64, 64, device="cuda")
    one, two = (illumina.createDepthModel(arch, weights=w) for w in (weights, back))
    a, b = one.forward(frames).clone(), two.forward(frames).clone()
    torch.cuda.synchronize()
    assert bool(torch.isfinite(b).all()) and not torch.equal(a, b)
    one.destroy()
    two.destroy()


def test_refusals(torch):
    import illumina
    p = [torch.zeros(10, device="cuda")]
    bad = [lambda: illumina.createOptimizer([]), lambda: illumina.createOptimizer([torch.zeros(3)]),
           lambda: illumina.createOptimizer([torch.zeros(3, device="cuda", dtype=torch.bfloat16)]),
           lambda: illumina.createOptimizer([torch.zeros(0, device="cuda")]),
           lambda: illumina.createOptimizer(p, momentBits=16), lambda: illumina.createOptimizer(p, decay=[True, False]),
           lambda: illumina.createOptimizer([torch.zeros(4, 4, device="cuda").t()[:2]]),
           lambda: illumina.createOptimizer(p, gradDtype=torch.float16)]
    opt = illumina.createOptimizer(p)
    bad += [lambda: opt.step([]), lambda: opt.step([torch.zeros(9, device="cuda")]),
            lambda: opt.step([torch.zeros(10, device="cuda", dtype=torch.bfloat16)]), lambda: opt.step([torch.zeros(10)]),
            lambda: opt.step([torch.zeros(20, device="cuda")[::2]]),
            lambda: opt.loadState({"step": 1, "m": torch.zeros(3, device="cuda"), "v": opt.v})]
    for i, call in enumerate(bad):
        with pytest.raises(illumina.IlluminaError) as e:
            call()
        assert e.value.status == 1, i
    opt.betas = (1.0, 0.9)
    with pytest.raises(illumina.IlluminaError):
        opt.step([torch.zeros(10, device="cuda")])


@pytest.mark.parametrize("eps", [-1e-8, 1e-39, float("nan")])
def test_refuses_eps_below_the_normal_floats(torch, eps):
    import illumina
    opt = illumina.createOptimizer([torch.zeros(10, device="cuda")], eps=eps)
    with pytest.raises((ValueError, RuntimeError), match="eps"):
        opt.step([torch.zeros(10, device="cuda")])
