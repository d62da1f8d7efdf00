"""Attention kernels that give up a wait, without a GPU fault: the wait limit is lowered so far that waits give up at once;
roles that gave up leave their loops, the waits that drain copies and products keep the default limit, and the host finds
the device's word set: after a synchronisation, after a replay, or at the next call. Then the default limit gives the
results it gave before."""
import pytest

from tests.test_tokens_gpu import attention_inputs, ops, torch  # noqa: F401

pytestmark = pytest.mark.gpu

# one and two streamed images, shared heads, shares of the keys, padding that is cleared in flight
CASES = [(2, 300, 300, 4, 2, 64, 1, [300, 130], [300, 150]), (1, 100, 4000, 4, 2, 64, 0, None, [3990]),
         (1, 500, 500, 2, 1, 128, 0, None, None)]


@pytest.fixture(autouse=True)
def default_limit(ops):  # noqa: F811
    yield
    ops.setAttentionWaitLimit(0)


def gave_up(call):
    import illumina
    from illumina import _lib
    with pytest.raises(illumina.IlluminaError, match="gave up a bounded wait") as e:
        call()
    assert e.value.status == _lib.TIMEOUT


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_timeouts_are_reported_and_the_next_calls_are_right(torch, ops, case):  # noqa: F811
    q, k, v, dout, masks = attention_inputs(torch, case, "bfloat16")
    out, lse = ops.attention(q, k, v, **masks)
    want = (out, lse, *ops.attentionBackward(dout, q, k, v, out, lse, **masks))
    torch.cuda.synchronize()
    ops.checkAttention()
    for call in (lambda: ops.attention(q, k, v, **masks), lambda: ops.attentionBackward(dout, q, k, v, out, lse, **masks)):
        ops.setAttentionWaitLimit(1)
        call()
        torch.cuda.synchronize()
        ops.setAttentionWaitLimit(0)
        gave_up(ops.checkAttention)
        ops.checkAttention()  # reported once
        ops.setAttentionWaitLimit(1)
        call()
        torch.cuda.synchronize()
        ops.setAttentionWaitLimit(0)
        gave_up(call)  # the next call reports it too
    out2, lse2 = ops.attention(q, k, v, **masks)
    again = (out2, lse2, *ops.attentionBackward(dout, q, k, v, out, lse, **masks))
    torch.cuda.synchronize()
    ops.checkAttention()
    assert all(torch.equal(a, b) for a, b in zip(want, again))


def test_replays_report(torch, ops):  # noqa: F811
    q, k, v, dout, masks = attention_inputs(torch, CASES[0], "bfloat16")
    out, lse = ops.attention(q, k, v, **masks)
    ops.attentionBackward(dout, q, k, v, out, lse, **masks)
    graphs = []
    for limit in (1, 0):
        ops.setAttentionWaitLimit(limit)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ops.attention(q, k, v, **masks)
        graphs.append((graph, held))
    for _ in range(2):
        graphs[0][0].replay()
        torch.cuda.synchronize()
        gave_up(ops.checkAttention)
        graphs[1][0].replay()
        torch.cuda.synchronize()
        ops.checkAttention()
        assert torch.equal(graphs[1][1][0], out) and torch.equal(graphs[1][1][1], lse)


def test_limits_belong_to_a_thread(torch, ops):  # noqa: F811
    import threading
    q, k, v, _, masks = attention_inputs(torch, CASES[0], "bfloat16")
    other = threading.Thread(target=ops.setAttentionWaitLimit, args=(1,))
    other.start()
    other.join()
    ops.attention(q, k, v, **masks)
    torch.cuda.synchronize()
    ops.checkAttention()
