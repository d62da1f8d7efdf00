"""AdamW: what a step refuses and keeps of its arguments, and sizes that send its kernels round their loops."""
import pytest

from tests import test_optimizer_gpu as G
from tests.test_optimizer_gpu import torch  # noqa: F401
from tests.test_token_checks_gpu import refused

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
def test_refuses_parameters_that_moved(torch, bits):  # noqa: F811
    import illumina
    p = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (1000, 0, 300)]
    g = [torch.ones(n, device="cuda") for n in (1000, 0, 300)]
    opt = illumina.createOptimizer(p, momentBits=bits)
    opt.step(g)
    old, kept = p[2].data, p[2].detach().clone()
    first = p[0].detach().clone()
    p[2].data = torch.ones(300, device="cuda")
    refused(lambda: opt.step(g), "parameter 2 has moved")
    assert torch.equal(old, kept) and torch.equal(p[0], first) and opt.steps == 1
    p[2].data = old[:200]  # the place of its first 200 elements
    refused(lambda: opt.step(g), "parameter 2 has moved")
    with torch.no_grad():
        p[2].set_(torch.zeros(300, device="cuda"))
    refused(lambda: opt.step(g), "parameter 2 has moved")
    p[2].data = old
    opt.step(g)
    assert opt.steps == 2
    opt.m.set_(opt.m.clone())
    refused(lambda: opt.step(g), "moments have moved")
    if bits == 8:
        refused(opt.moments, "moments have moved")


def test_gradients_made_as_they_are_asked_for(torch):  # noqa: F811
    """Every gradient lives until the step is queued: here none would, and each could take the place of the one before."""
    import illumina

    class Cast:
        def __init__(self, tensors):
            self.tensors = tensors

        def __len__(self):
            return len(self.tensors)

        def __getitem__(self, i):
            return self.tensors[i].bfloat16()

    grads = [torch.full((5000,), 0.01 * (i + 1), device="cuda") for i in range(6)]
    runs = []
    for given in ([g.bfloat16() for g in grads], Cast(grads)):
        p = [torch.ones(5000, device="cuda") for _ in grads]
        opt = illumina.createOptimizer(p, gradDtype=torch.bfloat16)
        opt.step(given)
        runs.append((*p, opt.m.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_an_optimizer_released_during_a_capture(torch):  # noqa: F811
    """Python may collect an optimizer at any time, while a graph is being captured too: the capture goes on."""
    import illumina
    p, g = torch.ones(5000, device="cuda"), torch.ones(5000, device="cuda")
    want = [torch.ones(5000, device="cuda") for _ in range(2)]
    for x in want:
        illumina.createOptimizer([x]).step([g])
    opt = illumina.createOptimizer([p])
    gone = [illumina.createOptimizer([torch.ones(300, device="cuda")]) for _ in range(2)]
    gone[1].step([g[:300]])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gone[0].destroy()  # reports what goes wrong
        gone.pop()         # collected
        opt.step([g])
    graph.replay()
    torch.cuda.synchronize()
    assert opt.steps == 1 and torch.equal(p, want[0])


# chunks of 2048 elements: more than the CTAs of a launch (296 with 32-bit moments, 444 with 8-bit ones) take at once
LARGE = [1, 255, 0, 600001, 256, 700000, 33, 500003, 4097, 700001]
MANY = [(7 * i) % 600 + (5000 if i % 3 == 0 else 0) for i in range(1000)]  # three launches a step, over 700 chunks each


@pytest.mark.parametrize("grad", ["float32", "bfloat16"])
@pytest.mark.parametrize("gap", [0, 1])
def test_32_bit_moments_round_the_loop(torch, monkeypatch, grad, gap):  # noqa: F811
    monkeypatch.setattr(G, "COUNTS", LARGE)
    G.test_32_bit_moments(torch, grad, gap)


@pytest.mark.parametrize("grad", ["float32", "bfloat16"])
@pytest.mark.parametrize("counts", [LARGE, MANY], ids=["large", "many"])
def test_8_bit_moments_round_the_loop_bit_for_bit(torch, monkeypatch, grad, counts):  # noqa: F811
    monkeypatch.setattr(G, "COUNTS", counts)
    G.test_8_bit_moments_bit_for_bit(torch, grad)


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_round_the_loop(torch, monkeypatch, bits):  # noqa: F811
    monkeypatch.setattr(G, "COUNTS", MANY)
    G.test_captured_steps_count_on(torch, bits)


def test_8_bit_roots_are_held_at_one_code(torch):  # noqa: F811
    """What is promised of elements whose gradients stay far below their block's largest: their root is one code, their
    steps are smaller than with 32-bit moments."""
    import illumina
    g = torch.full((512,), 1e-3, device="cuda")
    g[::64] = 1.0
    small = g < 1
    moved = {}
    for bits in (8, 32):
        p = torch.zeros(512, device="cuda")
        opt = illumina.createOptimizer([p], lr=1e-2, weightDecay=0.0, momentBits=bits)
        for _ in range(60):
            opt.step([g])
        moved[bits] = -p
    assert bool((opt.moments()[1][small] < 1.1 * 1e-6).all())  # 32 bits: the gradient's square, at most
    opt = illumina.createOptimizer([torch.zeros(512, device="cuda")], momentBits=8)
    for _ in range(60):
        opt.step([g])
    assert bool((opt.v.view(-1)[small] == 1).all()) and bool((opt.v.view(-1)[~small] >= 254).all())
    # the first step is exact; a later one divides by the root's code instead of the root, m's code being right on average
    mean = float(moved[8][small].mean()) / float(moved[32][small].mean())
    assert 1 / 60 < mean < 0.6
    # the largest elements' codes are a whole scale: they move as with 32 bits, but for the codes' roundings (1/255 a step)
    assert float((moved[8][~small] / moved[32][~small] - 1).abs().max()) < 0.02
