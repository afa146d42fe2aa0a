"""Calls of the self-attention and 8-bit cache operators around their kernels: copied plans, saved tensors that come back
in another layout, plans that captured graphs still read, tangents, padded prompts into a cache, empty batches, full
caches.  Tolerances are those of test_self_attention.py, whose formulas are used."""
import copy
import gc
import io
import pickle
import random
import sys
import threading
import weakref

import pytest
import torch

from tests.test_self_attention import BF, DEV, FP, by_formula, cached_formula, check, packed, rnd

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

    def plans(x):
        parts = x.values() if isinstance(x, dict) else x if isinstance(x, (tuple, list)) else ()
        return isinstance(x, ops.PackedSeqs) or any(plans(y) for y in parts)

    assert plans(vars(m)) and not plans(vars(theirs))
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


# ------------------------------------------------------------------------------------------------------ kept plans
def recording(monkeypatch, ops, seen):
    """A module on the CPU whose core only records the plan that it was given."""
    from star_amd import NuggetSelfAttention

    def core(qkv, H, Hkv, plan, scale=None):
        seen.append(weakref.ref(plan))
        assert plan.q_rows == len(qkv), "a plan of other lengths"
        return qkv[:, :128].view(-1, 2, 64)

    monkeypatch.setattr(ops, "causal_attn_qkv", core)
    return NuggetSelfAttention(128, 2).eval()


def test_a_captured_shape_keeps_its_plan(ops, monkeypatch):
    """A graph reads the plan's buffer at every replay: calls of other shapes between the replays must not free it."""
    seen = []
    m = recording(monkeypatch, ops, seen)
    x = torch.zeros(2, 5, 128)
    with torch.no_grad():
        m(x)
        monkeypatch.setattr(ops, "capturing", lambda dev: True, raising=False)
        m(x)
        monkeypatch.setattr(ops, "capturing", lambda dev: False)
        for t in range(6, 80):
            m(torch.zeros(1, t, 128))
        gc.collect()
        assert seen[1]() is not None and seen[0]() is seen[1]()
        m(x)
        assert seen[-1]() is seen[1]()
        assert sum(r() is not None for r in seen[2:-1]) <= 32 and seen[-2]() is not None       # the others are bounded
        monkeypatch.setattr(ops, "capturing", lambda dev: True)
        with pytest.raises(RuntimeError, match="before a HIP-graph capture"):
            m(torch.zeros(7, 3, 128))


def test_threads_with_different_shapes_get_their_own_plans(ops, monkeypatch):
    seen, failed = [], []
    m = recording(monkeypatch, ops, seen)

    def work(t):
        try:
            with torch.no_grad():
                for _ in range(300):
                    m(torch.zeros(1, t, 128))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    every = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(t,)) for t in (3, 4, 5, 6)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(every)
    assert not failed, failed[:1]


@gpu
def test_a_captured_module_replays_after_calls_of_other_shapes(ops):
    """Forward and backward captured at one shape, more shapes than are kept in between, memory reused, on two streams."""
    from star_amd import NuggetSelfAttention
    torch.manual_seed(0)
    m = NuggetSelfAttention(256, 4, kv_heads=2).to(DEV, BF)
    x, g = rnd(1, 2, 150, 256), rnd(2, 2, 150, 256)

    def step(x, g):
        leaf = x.detach().requires_grad_()
        y = m(leaf)
        return (y.detach(), *torch.autograd.grad(y, [leaf, *m.parameters()], g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(x, g)
    new = rnd(3, 3, 9, 256)
    with pytest.raises(RuntimeError, match="before a HIP-graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            m(new)
    torch.cuda.synchronize()
    for seed in (10, 20, 30):
        with torch.cuda.stream(side), torch.no_grad():
            others = [m(rnd(seed, 1, t, 256)) for t in range(1, 90, 2)]
            junk = [torch.full((64, 8), -1, dtype=torch.int32, device=DEV) for _ in range(64)]
        torch.cuda.current_stream().wait_stream(side)
        x.copy_(rnd(seed, 2, 150, 256))
        g.copy_(rnd(seed + 1, 2, 150, 256))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(x, g)):
            assert torch.equal(a, b)
        with torch.no_grad():
            for t, o in zip(range(1, 90, 2), others):
                assert torch.equal(o, m(rnd(seed, 1, t, 256)))
        del junk


# ------------------------------------------------------------------------------------------------------ tangents
def refuses_tangents(ops, dev):
    from types import SimpleNamespace
    from torch.autograd import forward_ad
    q, qkv, b = (torch.ones(n, device=dev, dtype=BF) for n in ((4, 2, 64), (4, 384), (1, 5)))
    plan = ops.PackedSeqs([4], dev)
    cache = SimpleNamespace(device=q.device, batch=1, kv_heads=2, head_dim=64, dtype=BF)
    x = q[None].transpose(1, 2)
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: ops.causal_attn(dual(q), q, q, plan), lambda: ops.causal_attn(q, dual(q), q, plan),
                 lambda: ops.causal_attn(q, q, dual(q), plan), lambda: ops.causal_attn_qkv(dual(qkv), 2, 2, plan),
                 lambda: ops.kv8_append(cache, dual(x), x), lambda: ops.kv8_append(cache, x, dual(x)),
                 lambda: ops.kv8_attn(dual(x), cache), lambda: ops.kv8_attn(x, cache, bias=dual(b))]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: ops.causal_attn(t, q, q, plan), (q,), (q,))


def test_tensors_with_a_tangent_are_refused(ops):
    refuses_tangents(ops, "cpu")


@gpu
def test_tensors_with_a_tangent_are_refused_on_the_gpu_and_others_beside_them_run(ops):
    from torch.autograd import forward_ad
    refuses_tangents(ops, DEV)
    q, k, v, _ = packed([9, 70], None, 2, 2, 64, BF)
    plan = ops.PackedSeqs([9, 70], DEV)
    with forward_ad.dual_level():
        assert torch.equal(ops.causal_attn(q, k, v, plan), ops.causal_attn(q.requires_grad_(), k, v, plan).detach())


# ------------------------------------------------------------------------------------------------------ padded prompts
def test_a_padded_prompt_for_a_cache_goes_by_its_lengths(ops, monkeypatch):
    """(CPU: the core and the append only record what they are given.)"""
    seen = []
    m = recording(monkeypatch, ops, seen)
    valid, given = ops.ValidFrames([3, 0, 5], 5, "cpu"), []
    monkeypatch.setattr(ops, "kv8_append", lambda cache, k, v, counts=None, plan=None, at=None: given.append((k.shape, plan, counts)))
    cache = type("Cache", (), dict(dtype=torch.bfloat16))()
    with torch.no_grad():
        m(torch.zeros(3, 5, 128), valid=valid, cache=cache)
        assert given == [((15, 2, 64), valid.seqs(), None)] and seen[0]() is valid.seqs()
        for kw, text in ((dict(valid=valid, plan=valid.seqs()), "not both"), (dict(valid=valid, counts=torch.ones(3)), "counts go")):
            with pytest.raises(ValueError, match=text):
                m(torch.zeros(3, 5, 128), cache=cache, **kw)
        with pytest.raises(ValueError, match="valid is for"):
            m(torch.zeros(3, 4, 128), valid=valid, cache=cache)


@gpu
def test_a_padded_prompt_into_a_cache_equals_the_packed_one(ops):
    """Pad rows, NaN included, neither enter the cache nor the prompt; sequences without a row in it keep what they hold."""
    from star_amd import NuggetSelfAttention
    lens, T, d = [50, 0, 130, 64], 130, 256
    torch.manual_seed(0)
    m = NuggetSelfAttention(d, 4, kv_heads=2).to(DEV, BF).eval()
    x = rnd(1, 4, T, d)
    real = torch.arange(T, device=DEV)[None] < torch.tensor(lens, device=DEV)[:, None]
    with torch.no_grad():
        packed_cache, padded_cache = m.new_cache(4, 192), m.new_cache(4, 192)
        held = rnd(2, 4, 2, 7, 64)
        for cache in (packed_cache, padded_cache):
            ops.kv8_append(cache, held, held, counts=torch.tensor([0, 7, 0, 0], device=DEV))
        want = m(x[real], plan=ops.PackedSeqs(lens, DEV), cache=packed_cache)
        x[~real] = float("nan")
        got = m(x, valid=ops.ValidFrames(lens, T, DEV), cache=padded_cache)
        assert torch.equal(got[real], want) and padded_cache.lens.tolist() == [50, 7, 130, 64]
        for a, b in zip(packed_cache.values(), padded_cache.values()):
            assert torch.equal(a, b)
        x = rnd(3, 4, 2, d)
        assert torch.equal(m(x, cache=padded_cache), m(x, cache=packed_cache))


# ------------------------------------------------------------------------------------------------------ streaming memory
def streamed(B, kmax, dev, dtype=torch.bfloat16, d=128):
    from star_amd import NuggetCrossAttention, NuggetScorer
    from star_amd.streaming import StreamingEncoderKV, StreamingNuggetSegmenter
    torch.manual_seed(0)
    seg = StreamingNuggetSegmenter(NuggetScorer(d).to(dev), B, d, kmax, dev, dtype=dtype)
    return seg, StreamingEncoderKV([NuggetCrossAttention(d, 2).to(dev, dtype)], seg, eight_bit=True)


@pytest.mark.parametrize("before,then", [([5], [3]), ([5], [0]), ([7, 5], [4, 5]), ([7, 5], [9, 4])])
def test_a_count_that_goes_back_is_refused_whether_or_not_a_row_is_projected(ops, monkeypatch, before, then):
    """(CPU: the caches and the segmenter are stand-ins; what extend() takes and keeps is looked at.)"""
    from types import SimpleNamespace
    from star_amd.streaming import StreamingEncoderKV
    kv, given = StreamingEncoderKV.__new__(StreamingEncoderKV), []
    B, d = len(before), 128
    kv.seg = SimpleNamespace(B=B, d=d, kmax=64, device=torch.device("cpu"), state=SimpleNamespace(mem=torch.zeros(B, 64, d)))
    kv.nl, kv.h, kv.w_all, kv.b_all, kv.kv = 1, 2, torch.zeros(d, 2 * d), torch.zeros(2 * d), None
    kv.caches, kv._prev = [SimpleNamespace(dtype=BF)], [0] * B
    monkeypatch.setattr(ops, "kv8_append", lambda cache, k, v, plan=None: given.append(plan.counts.tolist()))
    kv.extend(before)
    with pytest.raises(ValueError, match="went back"):
        kv.extend(then)
    assert kv._prev == before and given == [before]
    kv.extend([c + 1 for c in before])
    assert given == [before, [1] * B]


@gpu
def test_a_refused_extend_leaves_the_caches_as_they_were(ops):
    seg, kv = streamed(1, 150, DEV)
    seg.state.mem.copy_(rnd(1, 1, 150, 128))
    kv.extend([70])
    for back in ([60], [0]):
        with pytest.raises(ValueError, match="went back"):
            kv.extend(back)
    kv.extend([80])
    _, whole = streamed(1, 150, DEV)
    whole.seg.state.mem.copy_(seg.state.mem)
    whole.extend([70])
    whole.extend([80])
    a, b = kv.layers()[0].cache, whole.layers()[0].cache
    assert a.lens.tolist() == [80] and all(torch.equal(x, y) for x, y in zip(a.values(), b.values()))


# ------------------------------------------------------------------------------------------------------ empty batches
EMPTY = [([0], [5]), ([0, 0], [300, 1]), ([5], [0]), ([700, 3], [0, 0]), ([0], [0]), ([], [])]


def empty_batch(ops, keys, queries, dev, padded, monkeypatch=None):
    """No key (query) in the whole batch: o = 0, lse = -inf, gradients 0, whether or not the tensors have rows at all."""
    H, Hkv, hd = 4, 2, 64
    n_q, n_k = (max(1, len(keys)) * 1000,) * 2 if padded else (sum(queries), sum(keys))
    q, k, v = (torch.ones(n, h, hd, dtype=BF, device=dev).requires_grad_() for n, h in ((n_q, H), (n_k, Hkv), (n_k, Hkv)))
    plan = ops.PackedSeqs(keys, dev, q_lengths=queries, padded_to=1000 if padded else None)
    if dev == "cpu":
        o, lse = ops._CausalAttn.apply(q, k, v, plan, ops._causal_layout(q, k, v, plan, None), True)
    else:
        o, lse = ops.causal_attn(q, k, v, plan, need_lse=True)
        with torch.no_grad():
            assert torch.equal(ops.causal_attn(q, k, v, plan), o)
    assert o.shape == q.shape and (o == 0).all() and lse.shape == (H, n_q) and torch.isneginf(lse).all()
    for t, g in zip((q, k, v), torch.autograd.grad(o, (q, k, v), torch.ones_like(o))):
        assert g.shape == t.shape and (g == 0).all()


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("keys,queries", EMPTY)
def test_a_batch_without_keys_or_without_queries_launches_nothing_that_needs_them(ops, monkeypatch, keys, queries, padded):
    """(CPU: the memory that torch.empty gives is poisoned, and a launch may be asked for only if it has nothing to do.)"""
    def launch(fn, what, dev, *args):
        s = next(a for a in args if isinstance(a, ops.CausalShape))
        assert what == "star_causal_fwd" and s.n_q_tiles == 0, (what, s.n_q_tiles, s.n_k_tiles)

    make = torch.empty_like
    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(torch, "empty", lambda size, dtype, device: torch.full(size, 7.0, dtype=dtype, device=device))
    monkeypatch.setattr(torch, "empty_like", lambda t, **kw: make(t, **kw).fill_(7.0))
    empty_batch(ops, keys, queries, "cpu", padded)


@gpu
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("keys,queries", EMPTY)
def test_a_batch_without_keys_or_without_queries(ops, keys, queries, padded):
    empty_batch(ops, keys, queries, DEV, padded)


# ------------------------------------------------------------------------------------------------------ full caches
@gpu
@pytest.mark.parametrize("held,T,L,H,Hkv,hd,dtype", [
    ([63, 10, 64, 62], 64, 3, 4, 2, 64, BF),
    ([5055, 5000, 17], 5056, 4, 4, 4, 128, BF),                # cut into parts
    ([127, 128], 128, 16, 4, 2, 96, FP)])
def test_tokens_that_found_room_see_themselves_when_others_did_not(ops, held, T, L, H, Hkv, hd, dtype):
    """An append that fills the cache in the middle of its tokens: query i is the token at held + i and sees everything up to
    itself that the cache holds."""
    B = len(held)
    cache = ops.KVCache8(B, Hkv, T, hd, DEV, dtype)
    n = torch.tensor(held, device=DEV)

    def fill(at=None):
        new = (rnd(1, B, Hkv, max(held), hd, dtype=dtype), rnd(2, B, Hkv, max(held), hd, dtype=dtype))
        ops.kv8_append(cache, *new, counts=n, at=at)

    def attend(counts, first, q_len):
        q = rnd(5, B, H, L, hd, dtype=dtype)
        o = ops.kv8_attn(q, cache, q_len=q_len)
        k, v = cache.values()
        for i in range(L):
            see = [max(0, min(T, f + i + 1)) if i < c else 0 for f, c in zip(first, counts)]
            want, bound = cached_formula(q[:, :, i:i + 1], k, v, see, False, None, -1, None, hd ** -0.5)
            check(o[:, :, i:i + 1], want, bound, i)

    fill()
    new = rnd(3, B, Hkv, L, hd, dtype=dtype), rnd(4, B, Hkv, L, hd, dtype=dtype)
    counts = [L - b % 2 for b in range(B)]
    c = torch.tensor(counts, device=DEV)
    ops.kv8_append(cache, *new, counts=c)
    assert cache.lens.tolist() == [min(T, h + x) for h, x in zip(held, counts)]
    assert cache.overflow().tolist() == [max(0, h + x - T) for h, x in zip(held, counts)]
    attend(counts, held, c)
    first = [h + x for h, x in zip(held, counts)]              # and the next ones, of which none may fit
    ops.kv8_append(cache, *new)
    attend([L] * B, first, None)
    # positions given: what is missing is counted from there
    fill(at=torch.zeros(B, dtype=torch.int32, device=DEV))
    assert cache.overflow().tolist() == [0] * B
    ops.kv8_append(cache, *new, counts=c, at=n)
    assert cache.overflow().tolist() == [max(0, h + x - T) for h, x in zip(held, counts)]
    attend(counts, held, c)
    back = [h // 64 * 64 for h in held]                        # taken back
    ops.kv8_append(cache, new[0][:, :, :0], new[1][:, :, :0], at=torch.tensor(back, device=DEV))
    assert cache.overflow().tolist() == [0] * B and cache.lens.tolist() == back
    attend([L] * B, [x - L for x in back], None)


@gpu
def test_positions_behind_the_capacity_count_what_is_missing(ops):
    """A program that gives every token's position: overflow() is the part of the sequence that is not held."""
    cache = ops.KVCache8(3, 1, 64, 64, DEV)
    k, v, q = rnd(1, 3, 1, 66, 64), rnd(2, 3, 1, 66, 64), rnd(3, 3, 2, 1, 64)
    at = torch.tensor([60, 62, -5], dtype=torch.int32, device=DEV)
    ops.kv8_append(cache, k[:, :, :60], v[:, :, :60])
    ops.kv8_append(cache, k[:, :, 60:62], v[:, :, 60:62], counts=torch.tensor([0, 2, 2], device=DEV))
    for step in range(6):
        ops.kv8_append(cache, k[:, :, step:step + 1], v[:, :, step:step + 1], at=at + torch.tensor([step, step, 0], device=DEV))
        end = [60 + step + 1, 62 + step + 1, 1]
        assert cache.lens.tolist() == [min(64, n) for n in end]
        assert cache.overflow().tolist() == [max(0, n - 64) for n in end]
        want, bound = cached_formula(q, *cache.values(), cache.lens.tolist(), False, None, -1, None, 0.125)
        check(ops.kv8_attn(q, cache), want, bound, step)
    ops.kv8_append(cache, k[:, :, :2], v[:, :, :2], at=torch.full((3,), 2 ** 31 - 1, device=DEV))
    assert cache.lens.tolist() == [64] * 3 and cache.overflow().tolist() == [2 ** 31 - 1 - 62] * 3


@gpu
def test_tokens_of_a_module_that_fills_its_cache(ops):
    from star_amd import NuggetSelfAttention
    torch.manual_seed(0)
    m = NuggetSelfAttention(256, 4, kv_heads=2).to(DEV, BF).eval()
    x = rnd(1, 2, 70, 256)
    with torch.no_grad():
        small, large = m.new_cache(2, 64), m.new_cache(2, 128)
        for cache in (small, large):
            m(x[:, :62], valid=ops.ValidFrames([62, 61], 62, DEV), cache=cache)
        a, b = (m(x[:, 62:65], cache=cache) for cache in (small, large))
    assert torch.equal(a[0, :2], b[0, :2]) and torch.equal(a[1], b[1]) and small.overflow().tolist() == [1, 0]


# ------------------------------------------------------------------------------------------------------ low logits
@gpu
@pytest.mark.parametrize("low", [-1e30, -2.3e38])
@pytest.mark.parametrize("n,T", [(100, 128), (5000, 5056)])
def test_kv8_attn_rows_whose_every_bias_is_low_give_the_mean(ops, low, n, T):
    """A finite bias takes a key out only beside higher ones: where every bias is the same, the softmax is that without it
    (here every other logit is rounded away by it, which leaves the mean)."""
    hd, H = 64, 4
    cache = ops.KVCache8(2, 2, T, hd, DEV)
    k, v = rnd(1, 2, 2, n, hd), rnd(2, 2, 2, n, hd)
    ops.kv8_append(cache, k, v)
    q = rnd(3, 2, H, 1, hd)
    bias = torch.full((2, T), low, device=DEV)
    bias[1, 5:9] = 0.0
    o = ops.kv8_attn(q, cache, bias=bias)
    kk, vv = cache.values()
    want, bound = cached_formula(torch.stack([torch.zeros_like(q[0]), q[1]]), kk, vv, [n, n], True, None, -1,
                                 torch.stack([torch.zeros_like(bias[0]), bias[1]]), hd ** -0.5)
    check(o, want, bound)


# ------------------------------------------------------------------------------------------------------ types of caches
@gpu
@pytest.mark.parametrize("dtype,held", [(FP, BF), (BF, FP), (torch.float32, FP), (torch.float32, BF)])
def test_a_prompt_and_its_next_part_into_a_cache_of_another_type(ops, dtype, held):
    """The prompt's own output is that without a cache; what follows, a long next part and single tokens, is the formula's on
    the values that the cache stands for."""
    from star_amd import NuggetSelfAttention
    H, Hkv, hd, lens = 4, 2, 64, [60, 1, 129]
    torch.manual_seed(0)
    m = NuggetSelfAttention(H * hd, H, kv_heads=Hkv).to(DEV, dtype).eval()
    seen = []
    m.c_attn.register_forward_hook(lambda mod, args, out: seen.append(out))
    plan, x = ops.PackedSeqs(lens, DEV), rnd(1, sum(lens), H * hd, dtype=dtype)
    with torch.no_grad():
        m.c_proj.weight.copy_(torch.eye(H * hd))
        cache = m.new_cache(3, 350, dtype=held)
        assert torch.equal(m(x, plan=plan, cache=cache), m(x, plan=plan)) and cache.lens.tolist() == lens
        core = seen[0].to(BF) if dtype == torch.float32 else seen[0]
        k = core.to(held).view(-1, H + 2 * Hkv, hd)[:, H:H + Hkv]
        for b, (first, n) in enumerate(zip((0, 60, 61), lens)):
            assert torch.equal(cache.k_tail[b, :, :n % 64], k[first + n // 64 * 64:first + n].transpose(0, 1))
        n = lens
        for L, counts in ((190, [190, 100, 7]), (1, [1, 1, 1])):
            xs = rnd(L, 3, L, H * hd, dtype=dtype)
            seen.clear()
            y = m(xs, cache=cache, counts=torch.tensor(counts, device=DEV))
            n = [a + c for a, c in zip(n, counts)]
            assert cache.lens.tolist() == n
            q = seen[0].view(3, L, -1, hd)[:, :, :H].transpose(1, 2).to(held)
            want, bound = cached_formula(q, *cache.values(), n, True, counts, -1, None, hd ** -0.5)
            u = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2          # (rounded to the module's type once more)
            check(y.view(3, L, H, hd).transpose(1, 2), want, bound + u * (want.abs() + bound) + 2.0 ** -25, L)


@gpu
def test_kv8_attn_lookback_beyond_32_bits(ops):
    """A lookback mask as far as any integer hides nothing, one as far back as any integer is none."""
    cache = ops.KVCache8(1, 2, 128, 64, DEV)
    k, v, q = rnd(1, 1, 2, 100, 64), rnd(2, 1, 2, 100, 64), rnd(3, 1, 4, 3, 64)
    ops.kv8_append(cache, k, v)
    want = ops.kv8_attn(q, cache, causal=False)
    for far in (100, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40, -2 ** 32 + 5):
        assert torch.equal(ops.kv8_attn(q, cache, causal=False, ilk_diag=far), want), far


def test_more_tokens_than_one_call_takes_are_refused_before_they_are_appended(ops, monkeypatch):
    from star_amd import _lib
    appended = []
    m = recording(monkeypatch, ops, [])
    monkeypatch.setattr(m.c_attn, "forward", lambda x: torch.empty(1).expand(x.shape[0], x.shape[1], 384))
    monkeypatch.setattr(ops, "kv8_append", lambda *a, **kw: appended.append(a))
    cache = type("Cache", (), dict(dtype=torch.bfloat16))()
    with torch.no_grad(), pytest.raises(ValueError, match="in parts"):
        m(torch.zeros(1, 1, 128).expand(1, 1 << 23, 128), cache=cache)
    assert not appended
    # (the library's own limit)
    c = _lib.KV8Cache(B=1, Hkv=2, T=128, hd=64, dtype=0)
    for n in ("k_codes", "k_scales", "v_codes", "v_scales", "k_tail", "v_tail", "lens", "dropped", "tickets"):
        setattr(c, n, 16)
    q = _lib.KV8Query(H=2, L=ops.KV8_MOST_ROWS // 2)
    assert _lib.lib().star_kv8_attn(c, 16, None, None, q, 16, None, 0, None) == -1 and b"queries" in _lib.lib().star_last_error()


# ------------------------------------------------------------------------------------------------------ workspaces
def test_every_launch_is_given_the_workspace_that_the_library_asks_for(ops, monkeypatch):
    """The size is not asked for where launches are never cut: the library agrees on both sides of every border.  (CPU: the
    launches are recorded, not made.)"""
    from star_amd import _lib
    L, given = _lib.lib(), []

    def launch(fn, what, dev, *args):
        s = next(a for a in args if isinstance(a, ops.CausalShape))
        size = L.star_causal_fwd_workspace if what == "star_causal_fwd" else L.star_causal_bwd_workspace
        need = size(s)
        given.append((what, need > 0))
        assert args[-1] == need and bool(args[-2]) == (need > 0), (what, args[-1], need, [(n, getattr(s, n)) for n, _ in s._fields_])

    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(ops, "_rows_like", lambda rows, used, heads, hd, t: torch.empty(hd, dtype=t.dtype))
    rng = random.Random(0)
    for _ in range(600):
        hd, Hkv, g = rng.choice([64, 96, 128]), rng.choice([1, 2, 3, 8]), rng.choice([1, 1, 2, 8])
        most = rng.choice([32, 33, 255, 256, 257, 319, 320, 321, 384, 385, 448, 449, 832, 833, 1500])
        keys = [rng.randint(1, most) for _ in range(rng.choice([0, 1, 3, 30, 64, 127]))] + [most]
        queries = rng.choice([None, [min(n, rng.choice([1, 16, 17, 32, 33])) for n in keys]])
        plan = ops.PackedSeqs(keys, "cpu", q_lengths=queries)
        q, k = (torch.empty(hd, dtype=BF).expand(n, h, hd) for n, h in ((plan.q_rows, g * Hkv), (plan.k_rows, Hkv)))
        s = ops._causal_layout(q, k, k, plan, None)
        ops._causal_forward(q, k, k, plan, s, False)
        with torch.no_grad():
            ops._causal_backward(torch.empty(0, dtype=BF), q, k, k, q, torch.empty(1), plan, s, q, k, k)
    assert set(given) == {("star_causal_fwd", False), ("star_causal_fwd", True), ("star_causal_bwd", False), ("star_causal_bwd", True)}
