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


# ------------------------------------------------------------------------------------------------------ saved tensors
def qkv_views(qkv, H, Hkv, hd):
    t = qkv.view(len(qkv), H + 2 * Hkv, hd)
    return t[:, :H], t[:, H:H + Hkv], t[:, H + Hkv:]


@pytest.mark.parametrize("H,Hkv,n", [(4, 2, 9), (1, 1, 1)])
@pytest.mark.parametrize("whole", [False, True])
def test_backward_takes_the_layout_of_the_tensors_that_come_back(ops, monkeypatch, H, Hkv, n, whole):
    """Saved-tensor hooks give back dense copies of views with gaps: what the backward's launch is told is their layout.
    (CPU: the launches are recorded, not made.)"""
    hd = 64
    calls = []
    monkeypatch.setattr(ops, "_launch", lambda fn, what, dev, *args: calls.append((what, args)))
    plan = ops.PackedSeqs([n], "cpu")
    wide = torch.zeros(n, (H + 2 * Hkv) * hd + 64, dtype=BF)
    qkv = wide[:, :(H + 2 * Hkv) * hd].requires_grad_()
    views = qkv_views(qkv.detach(), H, Hkv, hd)
    s = ops._causal_layout(*views, plan, None)
    back = []

    def dense(t):
        back.append(t.clone(memory_format=torch.contiguous_format))
        return back[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, dense):
        if whole:
            o = ops._CausalAttnQKV.apply(qkv, views, plan, s)
        else:
            o = ops._CausalAttn.apply(*(t.requires_grad_() for t in views), plan, s, False)
    o.backward(torch.zeros_like(o))
    (_, fwd), (what, bwd) = calls
    assert what == "star_causal_bwd"
    q, k, v = qkv_views(back[0], H, Hkv, hd) if whole else back[:3]
    s = next(a for a in bwd if isinstance(a, ops.CausalShape))
    assert bwd[:3] == (q.data_ptr(), k.data_ptr(), v.data_ptr())
    for t, sr, sh in ((q, s.q_sr, s.q_sh), (k, s.k_sr, s.k_sh), (v, s.v_sr, s.v_sh)):
        assert [x for x, size in zip((sr, sh), t.shape) if size > 1] == [x for x, size in zip(t.stride()[:2], t.shape) if size > 1]
    assert s.dq_sr == (H + 2 * Hkv if whole else H) * hd


def test_saved_tensors_of_another_type_or_size_are_refused(ops, monkeypatch):
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    plan = ops.PackedSeqs([9], "cpu")
    for other in (lambda t: t.half(), lambda t: t[:-1], lambda t: t.double()):
        q, k, v = (torch.zeros(9, 2, 64, dtype=BF, requires_grad=True) for _ in range(3))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: other(t) if t.dtype == BF else t):
            o = ops._CausalAttn.apply(q, k, v, plan, ops._causal_layout(q, k, v, plan, None), False)
        with pytest.raises((ValueError, TypeError)):
            o.backward(torch.zeros_like(o))


@gpu
@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (4, 1)])
def test_gradients_of_views_under_save_on_cpu(ops, H, Hkv, whole):
    keys, hd = [150, 40, 1], 64
    plan = ops.PackedSeqs(keys, DEV)
    qkv, do = rnd(7, sum(keys), (H + 2 * Hkv) * hd), rnd(8, sum(keys), H, hd)

    def step():
        x = qkv.detach().requires_grad_()
        o = ops.causal_attn_qkv(x, H, Hkv, plan) if whole else ops.causal_attn(*qkv_views(x, H, Hkv, hd), plan)
        return o.detach(), torch.autograd.grad(o, x, do)[0]

    o, g = step()
    want, _ = by_formula(*qkv_views(qkv, H, Hkv, hd), keys, keys, hd ** -0.5, do)
    check(g, torch.cat([want[n][0].flatten(1) for n in ("dq", "dk", "dv")], 1), torch.cat([want[n][1].flatten(1) for n in ("dq", "dk", "dv")], 1))
    with torch.autograd.graph.save_on_cpu():
        o2, g2 = step()
    assert torch.equal(o, o2) and torch.equal(g, g2)
