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
