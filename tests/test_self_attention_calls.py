"""Calls of the self-attention and 8-bit cache operators around their kernels: copied plans, saved tensors that come back
in another layout, plans that captured graphs still read, tangents, padded prompts into a cache, empty batches, full
caches.  Tolerances are those of test_self_attention.py, whose formulas are used."""
import copy
import io
import pickle

import pytest
import torch

from tests.test_self_attention import BF, DEV, by_formula, check, packed, rnd

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from star_amd import ops as o
    return o


# ------------------------------------------------------------------------------------------------------ copied plans
def saved(x):
    f = io.BytesIO()
    torch.save(x, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIES = [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x)), saved]


def check_own_addresses(p, q):
    """q is a copy of p with the same contents, and its addresses are those of its own tensors."""
    for n in ("q_tiles", "k_tiles", "starts", "counts"):
        assert getattr(q, n + "_ptr") == getattr(q, n).data_ptr(), n
        assert torch.equal(getattr(q, n), getattr(p, n)), n
    assert q.counts.stride() == p.counts.stride() and q.device == p.device
    assert {n: x for n, x in vars(p).items() if isinstance(x, int) and not n.endswith("_ptr")} == {
        n: x for n, x in vars(q).items() if isinstance(x, int) and not n.endswith("_ptr")}


@pytest.mark.parametrize("how", range(len(COPIES)))
def test_a_copied_plan_points_to_its_own_buffer(ops, how):
    p = ops.PackedSeqs([130, 0, 5], "cpu", q_lengths=[3, 0, 200])
    check_own_addresses(p, COPIES[how](p))
    valid = ops.ValidFrames([50, 0, 130], 130, "cpu")
    plan = valid.seqs()
    check_own_addresses(plan, COPIES[how](valid).seqs())


@pytest.mark.parametrize("how", [1, 2, 3])
def test_a_copied_module_leaves_the_plan_behind(ops, how):
    from star_amd import NuggetSelfAttention
    m = NuggetSelfAttention(128, 2)
    with pytest.raises(ops.StarDeviceError):                   # (the plan is made before the tensors are refused)
        m(torch.zeros(2, 5, 128))
    theirs = COPIES[how](m)
    assert not any(isinstance(x, ops.PackedSeqs) for v in vars(theirs).values() for x in (v.values() if isinstance(v, dict) else v if isinstance(v, tuple) else [v]))
    for a, b in zip(m.parameters(), theirs.parameters()):
        assert torch.equal(a, b) and a is not b


@gpu
def test_a_copied_plan_outlives_the_original(ops):
    keys, H, hd = [130, 64, 3], 2, 64
    q, k, v, _ = packed(keys, None, H, H, hd, BF)
    plan = ops.PackedSeqs(keys, DEV)
    want = ops.causal_attn(q, k, v, plan)
    theirs = copy.deepcopy(plan)
    check_own_addresses(plan, theirs)
    del plan
    torch.full((4096,), -1, dtype=torch.int32, device=DEV)     # (what lay there is somebody else's)
    assert torch.equal(ops.causal_attn(q, k, v, theirs), want)
    cache = [ops.KVCache8(3, H, 192, hd, DEV) for _ in range(2)]
    ops.kv8_append(cache[0], k, v, plan=theirs)
    ops.kv8_append(cache[1], k, v, plan=ops.PackedSeqs(keys, DEV))
    assert all(torch.equal(a, b) for a, b in zip(cache[0].values(), cache[1].values()))
