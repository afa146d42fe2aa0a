"""causal_attn, kv8_append and kv8_attn against their formulas in 64 bits, and what they refuse.

Tolerances follow from where 16-bit roundings enter, u = finfo(dtype).eps / 2 relative to the rounded value (fp16 below
2^-14: 2^-25 absolute):
  o    P is rounded for P V, o on the way out:            u P|V| + u |o|
  dV   P rounded, dV rounded:                             u P^T|dO| + u |dV|
  dQ   dS rounded; delta = rowsum(dO o) is formed from the stored o, off by |dO| (err of o); dQ rounded:
       scale (u |dS| + P |dO|.(err of o)) |K| + u |dQ|;   dK the same with dS^T, |Q|
plus 2^-12 of the magnitudes for fp32 arithmetic: a logit of hd <= 128 fp32 products is off by at most 128 * 2^-24 *
sum|q k| scale, below 2^-12 for the values here (sum|q k| scale < 32).  A weight P under 2^-126, the smallest normal
fp32, may be taken for 0: 2^-126 of absolute error per weight, times what it is multiplied with (|v| for o, |dO| for dV,
|dP| + |delta| for dS)."""
import math

import numpy as np
import pytest
import torch

DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16
F32 = 2.0 ** -12
FLUSH = 2.0 ** -126
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from star_amd import ops as o
    return o


def rnd(seed, *shape, dtype=BF):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == FP else 0.0


def check(got, want, bound, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert over.max().item() <= 0 if over.numel() else True, (what, over.max().item(), bound.max().item())


def formula(q, k, v, scale, do=None, off=0):
    """One sequence, one head, in 64 bits: results and their bounds."""
    u, t = half_step(q.dtype), tiny(q.dtype)
    q, k, v = q.double(), k.double(), v.double()
    i, j = torch.arange(len(q), device=DEV)[:, None], torch.arange(len(k), device=DEV)[None]
    seen = (j <= i + off).expand(len(q), len(k))
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, 1)) * seen if len(k) else s
    lse = torch.logsumexp(s, 1) if len(k) else torch.full((len(q),), -math.inf, dtype=torch.float64, device=DEV)
    o = p @ v
    ob = (u + F32) * (p @ v.abs()) + u * o.abs() + t + (t + FLUSH) * (seen.double() @ v.abs())
    if do is None:
        return dict(o=(o, ob), lse=lse)
    do = do.double()
    dp = do @ v.T
    de = (do * o).sum(1, keepdim=True)
    ds = p * (dp - de)
    db = u * ds.abs() + p * (do.abs() * ob).sum(1, keepdim=True) + F32 * p * (do.abs() @ v.abs().T + (do * o).abs().sum(1, keepdim=True)) + t * seen
    db = db + FLUSH * seen * (dp.abs() + de.abs())
    dq, dk, dv = ds @ k * scale, ds.T @ q * scale, p.T @ do
    return dict(o=(o, ob), lse=lse, dq=(dq, scale * db @ k.abs() + u * dq.abs() + t), dk=(dk, scale * db.T @ q.abs() + u * dk.abs() + t),
                dv=(dv, (u + F32) * (p.T @ do.abs()) + u * dv.abs() + t + (t + FLUSH) * (seen.double().T @ do.abs())))


# ------------------------------------------------------------------------------------------------------ causal_attn
SHAPES = [  # keys, queries (None: the same), H, Hkv, hd, dtype
    ([1], None, 1, 1, 64, BF),
    ([5, 0, 1, 33], None, 2, 2, 128, BF),
    ([63, 64, 65], None, 2, 1, 64, FP),
    ([127, 128, 129, 257], None, 4, 2, 96, BF),
    ([200, 31], None, 3, 3, 96, FP),
    ([300, 1, 130], None, 8, 1, 128, FP),
    ([375], [16], 8, 8, 128, BF),
    ([700, 65, 0], [1, 64, 0], 4, 4, 64, BF),
    ([40, 3, 0], [100, 130, 5], 2, 2, 128, BF),            # more queries than keys: the first see nothing
    ([1000], None, 12, 4, 128, BF),
    ([3, 700, 64, 0, 257], [16, 1, 9, 2, 16], 4, 2, 128, BF),  # few queries each: the waves share them
    ([520, 5, 1], [30, 17, 1], 2, 1, 64, FP),
    ([100, 300], [32, 20], 3, 3, 96, BF),
    # few query tiles over many keys, cut along them and joined
    ([5000, 64, 0, 1030], [16, 7, 0, 1], 2, 1, 128, BF),
    ([3001], [30], 2, 2, 64, FP),
    ([2000, 100], [130, 100], 2, 1, 96, BF),
    ([10, 1500], [200, 60], 1, 1, 128, FP),
    ([450, 20], [40, 20], 2, 2, 128, BF),
    ([2600] * 11, [2] * 11, 12, 12, 64, FP),                   # two workgroups a CU, three parts
    ([20000, 0], [16, 3], 1, 1, 128, BF),                      # so many parts that four waves join a row
    ([185000], [3], 1, 1, 64, FP),                             # more parts a wave than lanes
    # gradients in pieces: of long walks, beside short and empty ones, of the heads' parts, with more queries than keys
    ([2100], None, 2, 1, 64, BF),
    ([1200, 0, 5, 300, 0], [700, 3, 400, 300, 0], 2, 2, 128, FP),
    ([900, 130], None, 6, 2, 96, BF),
    ([200, 1], [1500, 700], 1, 1, 64, BF),
]


def packed(keys, queries, H, Hkv, hd, dtype, seed=0):
    queries = keys if queries is None else queries
    return (rnd(seed, sum(queries), H, hd, dtype=dtype), rnd(seed + 1, sum(keys), Hkv, hd, dtype=dtype),
            rnd(seed + 2, sum(keys), Hkv, hd, dtype=dtype), rnd(seed + 3, sum(queries), H, hd, dtype=dtype))


def by_formula(q, k, v, keys, queries, scale, do=None):
    H, Hkv = q.shape[1], k.shape[1]
    g = H // Hkv
    out = {n: [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for _ in range(2)]
           for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    lse = torch.full((H, len(q)), -math.inf, dtype=torch.float64, device=DEV)
    q0 = k0 = 0
    for nk, nq in zip(keys, queries):
        a, b = slice(q0, q0 + nq), slice(k0, k0 + nk)
        for h in range(H):
            r = formula(q[a, h], k[b, h // g], v[b, h // g], scale, None if do is None else do[a, h], nk - nq)
            lse[h, a] = r.pop("lse")
            for n, (x, e) in r.items():
                where = (a, h) if n in ("o", "dq") else (b, h // g)
                out[n][0][where] += x
                out[n][1][where] += e
        q0, k0 = q0 + nq, k0 + nk
    return out, lse


@gpu
@pytest.mark.parametrize("keys,queries,H,Hkv,hd,dtype", SHAPES)
def test_causal_attn_and_gradients_against_the_formula(ops, keys, queries, H, Hkv, hd, dtype):
    q, k, v, do = packed(keys, queries, H, Hkv, hd, dtype)
    plan = ops.PackedSeqs(keys, DEV, q_lengths=queries)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o, lse = ops.causal_attn(q, k, v, plan, need_lse=True)
    grads = torch.autograd.grad(o, (q, k, v), do)
    want, want_lse = by_formula(q.detach(), k.detach(), v.detach(), keys, keys if queries is None else queries, hd ** -0.5, do)
    check(o, *want["o"], "o")
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    fine = torch.isfinite(want_lse)
    assert (lse.double() - want_lse)[fine].abs().max().item() < F32 if fine.any() else True
    for n, g in zip(("dq", "dk", "dv"), grads):
        check(g, *want[n], n)


@gpu
def test_causal_attn_takes_views_of_one_projection_and_a_scale(ops):
    keys, H, Hkv, hd = [150, 40], 4, 2, 64
    qkv = rnd(7, sum(keys), (H + 2 * Hkv) * hd).requires_grad_()
    q, k, v = (t.view(-1, n, hd) for t, n in zip(qkv.split([H * hd, Hkv * hd, Hkv * hd], 1), (H, Hkv, Hkv)))
    do = rnd(8, sum(keys), H, hd)
    o = ops.causal_attn(q, k, v, ops.PackedSeqs(keys, DEV), scale=0.3)
    g, = torch.autograd.grad(o, qkv, do.expand_as(do))
    want, _ = by_formula(q.detach(), k.detach(), v.detach(), keys, keys, 0.3, do)
    check(o, *want["o"])
    check(g, torch.cat([want[n][0].flatten(1) for n in ("dq", "dk", "dv")], 1), torch.cat([want[n][1].flatten(1) for n in ("dq", "dk", "dv")], 1))


@gpu
def test_causal_attn_qkv_equals_causal_attn_with_its_gradients_side_by_side(ops):
    keys, H, Hkv, hd = [150, 40, 700], 4, 2, 64
    plan = ops.PackedSeqs(keys, DEV)
    qkv = rnd(7, sum(keys), (H + 2 * Hkv) * hd).requires_grad_()
    do = rnd(8, sum(keys), H, hd)
    o1 = ops.causal_attn_qkv(qkv, H, Hkv, plan, scale=0.2)
    g1, = torch.autograd.grad(o1, qkv, do)
    q, k, v = (t.view(-1, n, hd) for t, n in zip(qkv.split([H * hd, Hkv * hd, Hkv * hd], 1), (H, Hkv, Hkv)))
    o2 = ops.causal_attn(q, k, v, plan, scale=0.2)
    g2, = torch.autograd.grad(o2, qkv, do)
    assert torch.equal(o1, o2) and torch.equal(g1, g2)
    with torch.no_grad():
        assert torch.equal(ops.causal_attn_qkv(qkv, H, Hkv, plan, scale=0.2), o1)
    for bad in (qkv[:, :-1], qkv[None]):
        with pytest.raises(ValueError, match="rows, "):
            ops.causal_attn_qkv(bad, H, Hkv, plan)
    with pytest.raises(ValueError, match="as many queries"):
        ops.causal_attn_qkv(qkv, H, Hkv, ops.PackedSeqs([3, 5], DEV, q_lengths=[5, 3]))
    # two sequences on the same key rows: forward only
    both = ops.PackedSeqs([100, 60], DEV, q_lengths=[10, 20], k_starts=[0, 40])
    with torch.no_grad():
        o = ops.causal_attn(q[:30], k, v, both)
        apart = ops.causal_attn(q[:30], torch.cat([k[:100], k[40:100]]), torch.cat([v[:100], v[40:100]]), ops.PackedSeqs([100, 60], DEV, q_lengths=[10, 20]))
    assert torch.equal(o, apart)
    with pytest.raises(ValueError, match="in common"):
        ops.causal_attn(q[:30], k, v, both)


@gpu
def test_causal_attn_strides_and_expanded_gradient(ops):
    """Rows and heads in another order, shared rows (stride 0) and a gradient without memory of its own."""
    keys, H, hd = [70, 129], 2, 64
    n = sum(keys)
    q = rnd(1, H, n, hd).transpose(0, 1)
    k = rnd(2, n, 1, hd).expand(n, H, hd)
    v = rnd(3, n, 2 * H, hd)[:, ::2]
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    do = rnd(4, 1, 1, hd).expand(n, H, hd)
    o = ops.causal_attn(q, k, v, ops.PackedSeqs(keys, DEV))
    grads = torch.autograd.grad(o, (q, k, v), do)
    want, _ = by_formula(q.detach(), k.detach(), v.detach(), keys, keys, hd ** -0.5, do)
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        check(got, *want[name], name)


@gpu
def test_causal_attn_padded_batch_leaves_nothing_between_the_sequences(ops):
    """padded_to: rows in no sequence give 0 and have zero gradients whatever they hold, NaN included."""
    lens, T, H, hd = [50, 0, 130], 130, 2, 128
    q, k, v, do = (rnd(s, 3 * T + 5, H, hd) for s in range(4))
    real = torch.cat([torch.arange(T, device=DEV) < n for n in lens] + [torch.zeros(5, dtype=torch.bool, device=DEV)])
    packed_in = [t[real].clone().requires_grad_() for t in (q, k, v)]
    o1 = ops.causal_attn(*packed_in, ops.PackedSeqs(lens, DEV))
    g1 = torch.autograd.grad(o1, packed_in, do[real])
    for t in (q, k, v, do):
        t[~real] = math.nan
    padded_in = [t.requires_grad_() for t in (q, k, v)]
    o2 = ops.causal_attn(*padded_in, ops.PackedSeqs(lens, DEV, padded_to=T))
    g2 = torch.autograd.grad(o2, padded_in, do)
    for a, b in zip((o1, *g1), (o2, *g2)):
        assert torch.equal(a, b[real])
        assert (b[~real] == 0).all()


@gpu
def test_causal_attn_nothing_crosses_from_the_future_or_from_neighbours(ops):
    """Infinite and NaN keys behind a query, and anything in another sequence, change no bit of it."""
    keys, H, hd = [90, 100], 2, 64
    q, k, v, _ = packed(keys, None, H, H, hd, BF)
    plan = ops.PackedSeqs(keys, DEV)
    base = ops.causal_attn(q, k, v, plan)
    k2, v2 = k.clone(), v.clone()
    k2[80] = math.inf
    k2[81] = math.nan
    k2[90:], v2[90:] = math.nan, math.inf
    got = ops.causal_attn(q, k2, v2, plan)
    assert torch.equal(got[:80], base[:80]) and torch.isnan(got[81:90]).all()
    k3, v3 = k.clone(), v.clone()
    v3[70] = math.nan                                          # reaches its own 64-key tile (keys 64 ..), no further back
    got = ops.causal_attn(q, k3, v3, plan)
    assert torch.equal(got[:64], base[:64]) and torch.equal(got[90:], base[90:]) and torch.isnan(got[70:90]).all()


@gpu
@pytest.mark.parametrize("big", [3.0e4, -3.0e4, 1e-30])
def test_causal_attn_large_and_small_logits(ops, big):
    """Logits far from 0 in either direction, the running maximum rising and falling along the keys."""
    keys, hd = [300], 64
    q, k, v, do = packed(keys, None, 1, 1, hd, BF)
    q = torch.full_like(q, 0.0)
    q[..., 0] = 1.0
    k = torch.zeros_like(k)
    k[:, 0, 0] = (torch.linspace(-1, 1, 300, device=DEV).sign() * big + torch.arange(300, device=DEV) % 7).to(BF)
    plan = ops.PackedSeqs(keys, DEV)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o = ops.causal_attn(q, k, v, plan)
    want, _ = by_formula(q.detach(), k.detach(), v.detach(), keys, keys, hd ** -0.5, None)
    # (one product per logit: the logit is exact to 2^-24 of its size, at most 2^-24 * 3750 = 2.3e-4)
    check(o, want["o"][0], want["o"][1] + 5e-4 * v.detach().double().abs().max())
    for g in torch.autograd.grad(o, (q, k, v), do):
        assert torch.isfinite(g).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rise", [5.0, 11.0, 13.0, 40.0, -40.0])
def test_causal_attn_logits_that_climb_from_tile_to_tile(ops, dtype, rise):
    """Logits that rise (fall) by `rise` in log2 with every 64 keys: the weights of a tile are formed against the maximum of
    an earlier one until their sum would pass 2^12, and rescaled then."""
    n, hd = 400, 64
    q = torch.zeros(n, 1, hd, device=DEV, dtype=dtype)
    k = torch.zeros(n, 1, hd, device=DEV, dtype=dtype)
    q[..., 0] = 1
    tile = torch.arange(n, device=DEV) // 64
    k[:, 0, 0] = (tile * rise * math.log(2) + torch.rand(n, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)).to(dtype)
    v, do = rnd(2, n, 1, hd, dtype=dtype), rnd(3, n, 1, hd, dtype=dtype)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o, lse = ops.causal_attn(q, k, v, ops.PackedSeqs([n], DEV), scale=1.0, need_lse=True)
    want, want_lse = by_formula(q.detach(), k.detach(), v.detach(), [n], [n], 1.0, do)
    check(o, *want["o"])
    assert (lse.double() - want_lse).abs().max().item() < F32
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
        # (logits up to 167: an fp32 logit or log-sum-exp is off by 2^-17 of 1, beyond F32's share by little)
        check(g, want[name][0], want[name][1] * 1.01, name)


@gpu
def test_causal_attn_gradient_against_differences(ops):
    """(loss(x + d) - loss(x - d)) / 2 along random directions, the loss in 64 bits by the formula."""
    keys, H, Hkv, hd = [20, 9], 4, 2, 64
    q, k, v, do = packed(keys, None, H, Hkv, hd, BF)
    plan = ops.PackedSeqs(keys, DEV)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.causal_attn(*leaves, plan), leaves, do)

    def loss(ts):
        total, r = 0.0, 0
        for n in keys:
            for h in range(H):
                x = ts[0][r:r + n, h] @ ts[1][r:r + n, h // 2].T / math.sqrt(hd)
                x = x.masked_fill(torch.ones((n, n), dtype=torch.bool, device=DEV).triu(1), -math.inf)
                total += (torch.softmax(x, 1) @ ts[2][r:r + n, h // 2] * do[r:r + n, h].double()).sum().item()
            r += n
        return total

    for which in range(3):
        x = [t.double() for t in (q, k, v)]
        d = torch.randn(x[which].shape, generator=torch.Generator(device=DEV).manual_seed(9), device=DEV, dtype=torch.float64)
        e = 1e-4
        up, down = list(x), list(x)
        up[which], down[which] = x[which] + e * d, x[which] - e * d
        slope = (loss(up) - loss(down)) / (2 * e)
        got = (grads[which].double() * d).sum().item()
        # three roundings of at most 2^-8 on each of the n products of the sum, independent: 3 * 2^-8 of its 2-norm, and
        # a random sum of n terms stays below 5 of them
        assert abs(got - slope) < 5 * 3 * 2.0 ** -8 * (grads[which].double() * d).norm().item(), which


@gpu
def test_causal_attn_is_reproducible_and_runs_on_another_stream(ops):
    keys, H, Hkv, hd = [500, 77, 260], 4, 2, 128
    q, k, v, do = packed(keys, None, H, Hkv, hd, BF)
    plan = ops.PackedSeqs(keys, DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = ops.causal_attn(*leaves, plan)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    third = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_causal_attn_training_step_under_graph_capture(ops):
    """Forward and backward captured once, replayed on new inputs with eager work in between: the eager bits."""
    keys, H, hd = [130, 64, 3], 2, 64
    plan = ops.PackedSeqs(keys, DEV)
    ins = [t.clone() for t in packed(keys, None, H, H, hd, BF)]

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = ops.causal_attn(*leaves, plan)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*ins)
    for seed in (10, 20, 30):
        new = packed(keys, None, H, H, hd, BF, seed)
        for a, b in zip(ins, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(*new)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------ 8-bit cache
def quantise(x):
    """[64, hd] fp32 -> e4m3 values, scale: the definition in star_nugget.h."""
    x = x.float().cpu()
    fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
    m = fin.max().item()
    e = -126
    while m > 448 * 2.0 ** e:
        e += 1
    s = 2.0 ** e if m > 0 else 1.0
    y = torch.where(torch.isfinite(x), x / s, math.nan)
    return y.to(torch.float8_e4m3fn), s


def same_bytes(a, b):
    """Codes are equal up to the sign of a NaN."""
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    return bool(((a == b) | ((a & 0x7f == 0x7f) & (b & 0x7f == 0x7f))).all())


def check_cache(cache, k, v, lens):
    """k, v: per sequence [n, H, hd], what was appended in all."""
    assert cache.lens.tolist() == list(lens)
    for b, n in enumerate(lens):
        full = n // 64
        for h in range(cache.kv_heads):
            for name, x in (("k", k[b]), ("v", v[b])):
                for blk in range(full):
                    c, s = quantise(x[blk * 64:(blk + 1) * 64, h])
                    got = cache.k_codes[b, h, blk * 64:(blk + 1) * 64] if name == "k" else cache.v_codes[b, h, blk].view(torch.uint8).T.contiguous().view(torch.float8_e4m3fn)
                    assert same_bytes(got.contiguous(), c), (name, b, h, blk)
                    assert getattr(cache, name + "_scales")[b, h, blk].item() == s
                rest = x[full * 64:n, h]
                tail = cache.k_tail[b, h, :len(rest)] if name == "k" else cache.v_tail[b, h, :, :len(rest)].T
                assert torch.equal(tail, rest), (name, b, h)
    assert int(cache._tickets.abs().sum()) == 0


@gpu
@pytest.mark.parametrize("hd,dtype", [(64, BF), (96, FP), (128, BF)])
def test_kv8_append_holds_the_same_however_the_tokens_are_split(ops, hd, dtype):
    lens, H = [0, 1, 63, 64, 65, 200], 2
    k = [rnd(b, n, H, hd, dtype=dtype) * (0.01 + b) for b, n in enumerate(lens)]
    v = [rnd(50 + b, n, H, hd, dtype=dtype) for b, n in enumerate(lens)]
    whole = ops.KVCache8(len(lens), H, 200, hd, DEV, dtype)
    ops.kv8_append(whole, torch.cat(k), torch.cat(v), plan=ops.PackedSeqs(lens, DEV))
    check_cache(whole, k, v, lens)
    for step in (1, 7, 64, 130):
        cache = ops.KVCache8(len(lens), H, 200, hd, DEV, dtype)
        for r in range(0, 200, step):
            cut = [min(max(n - r, 0), step) for n in lens]
            kb, vb = (torch.full((len(lens), H, step, hd), math.nan, dtype=dtype, device=DEV) for _ in range(2))
            for b, n in enumerate(cut):
                kb[b, :, :n], vb[b, :, :n] = k[b][r:r + n].transpose(0, 1), v[b][r:r + n].transpose(0, 1)
            ops.kv8_append(cache, kb, vb, counts=torch.tensor(cut, device=DEV))
        check_cache(cache, k, v, lens)
        assert all(torch.equal(a, b) for a, b in zip(cache.values(), whole.values()))


@gpu
def test_kv8_append_writes_nothing_else_and_counts_what_finds_no_room(ops):
    H, hd = 2, 64
    cache = ops.KVCache8(3, H, 128, hd, DEV)
    for t in cache.tensors().values():
        if t.dtype != torch.int32:
            t.view(torch.uint8).fill_(0x55)
    before = {n: t.clone() for n, t in cache.tensors().items()}
    k, v = rnd(1, 3, H, 150, hd), rnd(2, 3, H, 150, hd)
    ops.kv8_append(cache, k, v, counts=torch.tensor([150, 10, 0], device=DEV))
    assert cache.lens.tolist() == [128, 10, 0] and cache.overflow().tolist() == [22, 0, 0]
    check_cache(cache, [t[:n].contiguous() for t, n in zip(k.transpose(1, 2), (128, 10, 0))], [t[:n].contiguous() for t, n in zip(v.transpose(1, 2), (128, 10, 0))], [128, 10, 0])
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    for n in ("k_codes", "v_codes", "k_scales", "v_scales"):
        assert torch.equal(raw(getattr(cache, n))[1:], raw(before[n])[1:]), n
    assert torch.equal(raw(cache.k_tail[0]), raw(before["k_tail"][0])) and torch.equal(raw(cache.k_tail[1, :, 10:].contiguous()), raw(before["k_tail"][1, :, 10:].contiguous()))
    assert torch.equal(raw(cache.v_tail[1, :, :, 10:].contiguous()), raw(before["v_tail"][1, :, :, 10:].contiguous()))
    ops.kv8_append(cache, k[:, :, :1], v[:, :, :1])
    assert cache.lens.tolist() == [128, 11, 1] and cache.overflow().tolist() == [23, 0, 0]
    cache.reset(torch.tensor([0], device=DEV))
    assert cache.lens.tolist() == [0, 11, 1] and cache.overflow().tolist() == [0, 0, 0]


@gpu
def test_kv8_append_at_takes_tokens_back(ops):
    H, hd = 1, 128
    k, v = rnd(1, 2, H, 100, hd), rnd(2, 2, H, 100, hd)
    cache = ops.KVCache8(2, H, 256, hd, DEV)
    ops.kv8_append(cache, k, v)
    k2, v2 = rnd(3, 2, H, 40, hd), rnd(4, 2, H, 40, hd)
    ops.kv8_append(cache, k2, v2, at=torch.tensor([64, 90], device=DEV))
    ks = [torch.cat([k[b, :, :a], k2[b]], 1).transpose(0, 1).contiguous() for b, a in enumerate((64, 90))]
    vs = [torch.cat([v[b, :, :a], v2[b]], 1).transpose(0, 1).contiguous() for b, a in enumerate((64, 90))]
    check_cache(cache, ks, vs, [104, 130])
    ops.kv8_append(cache, k, v, at=torch.zeros(2, dtype=torch.int64, device=DEV))
    check_cache(cache, list(k.transpose(1, 2).contiguous()), list(v.transpose(1, 2).contiguous()), [100, 100])
    ops.kv8_append(cache, k[:, :, :0], v[:, :, :0], at=torch.tensor([64, 99], device=DEV))      # nothing but taken back
    check_cache(cache, [k[0, :, :64].transpose(0, 1), k[1, :, :99].transpose(0, 1)], [v[0, :, :64].transpose(0, 1), v[1, :, :99].transpose(0, 1)], [64, 99])
    at = torch.tensor([64 + 63, 127], device=DEV)
    ops.kv8_append(cache, k[:, :, :63], v[:, :, :63], counts=torch.tensor([63, 28], device=DEV))
    for i in (0, 1, 2):                                        # the append that completes a block, repeated
        ops.kv8_append(cache, k[:, :, i:i + 1], v[:, :, i:i + 1], at=at)
    ks = [torch.cat([k[0, :, :64], k[0, :, :63], k[0, :, 2:3]], 1), torch.cat([k[1, :, :99], k[1, :, :28], k[1, :, 2:3]], 1)]
    vs = [torch.cat([v[0, :, :64], v[0, :, :63], v[0, :, 2:3]], 1), torch.cat([v[1, :, :99], v[1, :, :28], v[1, :, 2:3]], 1)]
    check_cache(cache, [t.transpose(0, 1) for t in ks], [t.transpose(0, 1) for t in vs], [128, 128])


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_kv8_append_extreme_values(ops, dtype):
    """Zero blocks, single large values, the smallest and largest of the type, infinities and NaN."""
    hd, n = 64, 64 * 7
    x = rnd(5, 1, 1, n, hd, dtype=dtype)
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x[0, 0, :64] = 0
    x[0, 0, 64, 3] = big
    x[0, 0, 128:192] = x[0, 0, 128:192] * small
    x[0, 0, 192, 0], x[0, 0, 193, 1], x[0, 0, 194, 2] = math.inf, -math.inf, math.nan
    x[0, 0, 256:320] = math.inf
    x[0, 0, 320, 5] = -448.0
    x[0, 0, 384, 5] = 450.0
    cache = ops.KVCache8(1, 1, n, hd, DEV, dtype)
    ops.kv8_append(cache, x, -x)
    check_cache(cache, [x[0].transpose(0, 1)], [-x[0].transpose(0, 1)], [n])


def cached_formula(q, k, v, lens, causal, q_len, ilk, bias, scale):
    B, H, L, hd = q.shape
    u, t = half_step(q.dtype), tiny(q.dtype)
    g = H // k.shape[1]
    o, bound = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for b in range(B):
        nq = L if q_len is None else q_len[b]
        n = lens[b]
        i, j = torch.arange(nq, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        seen = torch.ones((nq, n), dtype=torch.bool, device=DEV)
        if causal:
            seen &= j <= n - nq + i
        if ilk >= 0:
            seen &= j <= i + ilk
        for h in range(H):
            s = q[b, h, :nq].double() @ k[b, h // g, :n].double().T * scale
            if bias is not None:
                w = min(n, bias.shape[1])
                s[:, :w] += bias[b, :w].double()
            p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), 1)) if n else s
            vv = v[b, h // g, :n].double()
            o[b, h, :nq] = p @ vv
            # fp16: p is at most 2^8 times the largest weight, V halves exactly but for 2^-25 of subnormals
            bound[b, h, :nq] = (u + F32) * (p @ vv.abs()) + u * o[b, h, :nq].abs() + t * (2 + seen.double() @ vv.abs())
    return o, bound


CACHED = [  # lens, L, H, Hkv, hd, dtype, capacity
    ([375], 1, 8, 8, 128, BF, 384),
    ([0, 1, 63, 64, 65, 129], 1, 4, 2, 64, BF, 192),
    ([700, 64, 5, 1023], 3, 6, 2, 96, FP, 1024),
    ([2000, 17], 16, 8, 1, 128, BF, 2048),                    # 128 rows: two tiles of 16 in a workgroup, four groups
    ([300, 64], 5, 12, 2, 64, FP, 320),                       # 30 rows: two tiles
    ([5000, 4096, 100], 1, 32, 8, 128, FP, 5056),             # cut into parts and joined
    ([30000], 2, 2, 1, 96, BF, 30016),
    ([60000] + [1] * 15, 1, 1, 1, 64, BF, 60032),             # more parts of a row than lanes
    ([300000], 1, 2, 1, 64, FP, 300032),                      # more than threads
    ([2150, 7] * 20, 1, 8, 8, 128, BF, 2176),                 # the card full without parts, long sequences cut all the same
    ([2150 - 9 * i for i in range(40)], 2, 8, 8, 64, BF, 2176),     # much the same length: whole
    ([1500, 1], 8, 8, 1, 64, FP, 1536),                       # 64 rows: cut from 23 blocks of capacity on
    ([64 * (i % 9) + i for i in range(70)], 1, 2, 2, 64, BF, 640),   # more sequences than lanes
]


def filled(ops, lens, Hkv, hd, dtype, T, seed=0):
    cache = ops.KVCache8(len(lens), Hkv, T, hd, DEV, dtype)
    for t in (cache.k_tail, cache.v_tail):
        t.fill_(math.nan)                                      # what lies behind the last token must not matter
    cache.k_codes.view(torch.uint8).fill_(0x7f)
    cache.v_codes.view(torch.uint8).fill_(0x7f)
    if sum(lens):
        ops.kv8_append(cache, rnd(seed, sum(lens), Hkv, hd, dtype=dtype), rnd(seed + 1, sum(lens), Hkv, hd, dtype=dtype),
                       plan=ops.PackedSeqs(lens, DEV))
    return cache


@gpu
@pytest.mark.parametrize("lens,L,H,Hkv,hd,dtype,T", CACHED)
@pytest.mark.parametrize("how", ["causal", "ilk_bias", "all_q_len"])
def test_kv8_attn_against_the_formula(ops, lens, L, H, Hkv, hd, dtype, T, how):
    cache = filled(ops, lens, Hkv, hd, dtype, T)
    k, v = cache.values()
    q = rnd(9, len(lens), H, L, hd, dtype=dtype)
    kw = dict(causal=True, q_len=None, ilk_diag=-1, bias=None)
    if how == "ilk_bias":
        kw.update(causal=False, ilk_diag=37, bias=torch.randn((len(lens), max(1, T - 30)), device=DEV) * 2)
    if how == "all_q_len":
        kw.update(causal=L > 1, q_len=torch.tensor([(b + L) % (L + 1) for b in range(len(lens))], device=DEV))
    o = ops.kv8_attn(q, cache, **kw)
    want, bound = cached_formula(q, k, v, lens, kw["causal"], None if kw["q_len"] is None else kw["q_len"].tolist(), kw["ilk_diag"], kw["bias"], hd ** -0.5)
    check(o, want, bound, how)


@gpu
def test_kv8_attn_masks_of_the_lowest_value(ops):
    """Biases of finfo.min and -inf take keys out; a row that they leave empty gives 0."""
    cache = filled(ops, [100, 100, 100], 2, 64, BF, 128)
    k, v = cache.values()
    q = rnd(3, 3, 4, 1, 64)
    bias = torch.zeros((3, 128), device=DEV)
    bias[0, 10:] = torch.finfo(torch.float32).min
    bias[1, 20:90] = -math.inf
    bias[2] = torch.finfo(torch.float32).min
    o = ops.kv8_attn(q, cache, bias=bias)
    assert (o[2] == 0).all()
    want, bound = cached_formula(q[:2], k[:2], v[:2], [100, 100], True, None, -1, bias[:2].clamp(min=-1e30), 0.125)
    check(o[:2], want, bound)


@gpu
def test_kv8_attn_strides_and_a_largest_fp16_value(ops):
    lens, H, hd = [130, 64], 4, 128
    cache = ops.KVCache8(2, H, 192, hd, DEV, FP)
    v = rnd(2, sum(lens), H, hd, dtype=FP)
    v[3, 0, 0] = 65504.0                                      # held as 65536, which fp16 does not have
    ops.kv8_append(cache, rnd(1, sum(lens), H, hd, dtype=FP), v, plan=ops.PackedSeqs(lens, DEV))
    q = rnd(3, 2, 3, H * hd, dtype=FP).view(2, 3, H, hd).permute(0, 2, 1, 3)
    o = ops.kv8_attn(q, cache, scale=0.01)
    kk, vv = cache.values()
    want, bound = cached_formula(q, kk, vv, lens, True, None, -1, None, 0.01)
    check(o, want, bound)
    assert o.transpose(1, 2).is_contiguous()


@gpu
def test_kv8_attn_non_finite_values_stay_in_their_sequence(ops):
    lens = [200, 200]
    cache = ops.KVCache8(2, 1, 256, 64, DEV)
    k, v = rnd(1, 400, 1, 64), rnd(2, 400, 1, 64)
    plan = ops.PackedSeqs(lens, DEV)
    ops.kv8_append(cache, k, v, plan=plan)
    q = rnd(3, 2, 2, 1, 64)
    base = ops.kv8_attn(q, cache)
    k[150], v[170] = math.nan, math.inf
    ops.kv8_append(cache, k, v, plan=plan, at=torch.zeros(2, dtype=torch.int32, device=DEV))
    got = ops.kv8_attn(q, cache)
    assert torch.isnan(got[0]).all() and torch.equal(got[1], base[1])


# ------------------------------------------------------------------------------------------------------ together
@gpu
@pytest.mark.parametrize("graph", [False, True])
def test_prompt_then_tokens_equals_attention_over_the_held_values(ops, graph):
    """A prompt through causal_attn into the cache, then tokens one by one (append, attend), eager or replayed from one
    captured graph: every token's output is the formula's on the values that the cache stands for."""
    lens, H, Hkv, hd, steps = [100, 62, 1], 4, 2, 128, 5
    cache = ops.KVCache8(3, Hkv, 256, hd, DEV)
    q, k, v, _ = packed(lens, None, H, Hkv, hd, BF)
    plan = ops.PackedSeqs(lens, DEV)
    o = ops.causal_attn(q, k, v, plan)
    ops.kv8_append(cache, k, v, plan=plan)
    want, _ = by_formula(q, k, v, lens, lens, hd ** -0.5)
    check(o, *want["o"])
    new = [tuple(rnd(100 + 3 * s + i, 3, n, 1, hd) for i, n in enumerate((H, Hkv, Hkv))) for s in range(steps)]
    buf = [t.clone() for t in new[0]]

    def step():
        ops.kv8_append(cache, buf[1], buf[2])
        return ops.kv8_attn(buf[0], cache)

    g = None
    if graph:
        kept = {n: t.clone() for n, t in cache.tensors().items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for n, t in cache.tensors().items():
            t.view(torch.uint8).copy_(kept[n].view(torch.uint8))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
    for s in range(steps):
        for a, b in zip(buf, new[s]):
            a.copy_(b)
        if g is None:
            out = step()
        else:
            g.replay()
        n = [x + s + 1 for x in lens]
        assert cache.lens.tolist() == n
        kk, vv = cache.values()
        want, bound = cached_formula(buf[0], kk, vv, n, True, None, -1, None, hd ** -0.5)
        check(out, want, bound, s)


# ------------------------------------------------------------------------------------------------------ refusals
def test_packed_seqs_layout_and_refusals(ops):
    p = ops.PackedSeqs([130, 0, 5], "cpu", q_lengths=[3, 0, 200])
    assert p.seqs.tolist() == [[0, 3, 0, 130], [3, 0, 130, 0], [3, 200, 130, 5]]
    assert (p.q_rows, p.k_rows, p.q_used, p.k_used, p.max_q, p.max_k, p.n) == (203, 135, 203, 135, 200, 130, 3)
    tiles = lambda t: sorted((p.seqs.tolist().index(w[:4]), w[4]) for w in t.tolist())  # noqa: E731
    assert tiles(p.q_tiles) == [(0, 0), (2, 0), (2, 128)]
    assert tiles(p.k_tiles) == [(0, 0), (0, 128), (2, 0)]
    p = ops.PackedSeqs([2, 7], "cpu", padded_to=7)
    assert p.seqs.tolist() == [[0, 2, 0, 2], [7, 7, 7, 7]] and (p.q_rows, p.q_used) == (14, 9)
    p = ops.PackedSeqs([40, 2000, 2000, 500], "cpu")
    assert tiles(p.q_tiles) == sorted((s, f) for s, n in enumerate([40, 2000, 2000, 500]) for f in range(0, n, 128))
    order = [(p.seqs.tolist().index(w[:4]), w[4]) for w in p.q_tiles.tolist()]
    assert order[0] == (1, 1920) and order[-1] == (0, 0)       # the longest walk starts first, the shortest last,
    assert [f for s, f in order if s == 2 and f >= 1024] == list(range(1920, 1023, -128))   # each sequence from its end
    p = ops.PackedSeqs([], "cpu")
    assert p.n == 0 and p.q_rows == 0 and p.q_tiles.shape == (0, 8)
    assert p.starts.numel() == 0
    with pytest.raises(ValueError, match="negative"):
        ops.PackedSeqs([3, -1], "cpu")
    with pytest.raises(ValueError, match="query lengths"):
        ops.PackedSeqs([3, 1], "cpu", q_lengths=[3])
    with pytest.raises(ValueError, match="padded_to"):
        ops.PackedSeqs([3, 9], "cpu", padded_to=8)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.PackedSeqs([2 ** 30] * 2, "cpu", q_lengths=[0, 0])


def test_cpu_tensors_are_refused(ops):
    z = torch.zeros(4, 2, 64, dtype=BF)
    with pytest.raises(ops.StarDeviceError):
        ops.causal_attn(z, z, z, ops.PackedSeqs([4], "cpu"))
    with pytest.raises(ops.StarDeviceError):
        ops.KVCache8(1, 1, 64, 64, "cpu")


def test_the_library_checks_sizes_before_any_launch():
    from star_amd import _lib
    L = _lib.lib()
    S = _lib.CausalShape
    fwd = lambda s, k=16, ws=None, n=0: L.star_causal_fwd(16, k, 16, 16, s, 16, 16, ws, n, None)  # noqa: E731
    bwd = lambda s, ws=None, n=0: L.star_causal_bwd(*[16] * 8, s, 16, 16, 16, 16, ws, n, None)  # noqa: E731
    for kw, text in [(dict(hd=80), b"head dim 80"), (dict(Hkv=3), b"divide"), (dict(dtype=1), b"dtype"), (dict(q_sr=4), b"multiples of 8"),
                     (dict(q_sr=1 << 23), b"row stride"), (dict(q_sr=-8), b"row stride"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"),
                     (dict(scale=math.inf), b"scale"), (dict(scale=math.nan), b"scale"), (dict(max_k=-1), b"negative"),
                     (dict(n_k_tiles=1 << 22), b"tiles x 4 heads"), (dict(n_q_tiles=1 << 22), b"tiles x 4 heads")]:
        s = S(**{**dict(H=4, Hkv=2, hd=64, dtype=0, scale=1, n_q_tiles=1), **kw})
        for call in (fwd, bwd):
            assert call(s) == -1 and text in L.star_last_error(), kw
        assert L.star_causal_fwd_workspace(s) == 0 and L.star_causal_bwd_workspace(s) == 0
    s = S(H=4, Hkv=2, hd=64, dtype=0, scale=1, n_q_tiles=1)
    assert fwd(s, k=24) == -1 and b"aligned" in L.star_last_error()
    assert fwd(s, k=None) == -1 and b"null pointer" in L.star_last_error()
    assert L.star_causal_fwd(None, None, None, None, S(H=4, Hkv=2, hd=64, dtype=0, scale=1), None, None, None, 0, None) == 0
    # cut along the keys: few query tiles, many keys
    need = lambda nq, n, nk: L.star_causal_fwd_workspace(S(H=4, Hkv=2, hd=64, dtype=0, scale=1, n_q_tiles=n, max_q=nq, max_k=nk))  # noqa: E731
    assert need(16, 1, 832) == 0 and need(16, 1, 833) == 4 * 14 * 16 * 66 * 4 and need(16, 64, 100000) == 0
    assert need(33, 1, 320) == 0 and need(33, 1, 321) == 4 * 6 * 128 * 66 * 4
    assert need(17, 2, 10 ** 6) == 2 * 4 * 64 * 32 * 66 * 4 and need(33, 63, 10 ** 6) == 63 * 4 * 2 * 128 * 66 * 4
    s = S(H=4, Hkv=2, hd=64, dtype=0, scale=1, n_q_tiles=1, max_q=16, max_k=4096)
    assert fwd(s) == -3 and b"workspace" in L.star_last_error() and fwd(s, ws=16, n=100) == -3 and fwd(s, ws=24, n=1 << 30) == -3
    # cut by query heads: few key tiles, long walks
    s = S(H=4, Hkv=1, hd=64, dtype=0, k_rows=2000, scale=1, dq_sr=256, dkv_sr=64, n_k_tiles=16, max_q=2000, max_k=2000)
    assert L.star_causal_bwd_workspace(s) == 4 * 8 * 2 * 2000 * 64 * 4     # and each of the 4 heads' walks into 8 pieces
    assert bwd(s) == -3 and b"workspace" in L.star_last_error()
    s.dq_sr = 128
    assert bwd(s) == -1 and b"gradient row" in L.star_last_error()
    s.n_k_tiles = 512
    assert L.star_causal_bwd_workspace(s) == 2 * 2 * 2000 * 64 * 4
    s.n_k_tiles = 1024
    assert L.star_causal_bwd_workspace(s) == 0
    s.n_k_tiles, s.max_q = 16, 96
    assert L.star_causal_bwd_workspace(s) == 0
    # the queries' gradient by tiles of keys: 16 of 16 tiles in pieces of 4 (mean 8; 32 workgroups)
    s.n_q_tiles, s.n_k_tiles, s.H, s.Hkv, s.max_q, s.max_k, s.lse_stride, s.k_rows = 8, 0, 4, 4, 1024, 1024, 1024, 1024
    s.dq_sr, s.dkv_sr = 256, 256
    assert L.star_causal_bwd_workspace(s) == 4 * 1024 * 4 * 64 * 4
    s.max_q = s.max_k = 384
    assert L.star_causal_bwd_workspace(s) == 0
    c = _lib.KV8Cache(B=1, Hkv=2, T=100, hd=64, dtype=0)
    assert L.star_kv8_append(c, 16, 16, 0, 0, 0, 0, 0, 0, None, None, 1, None, 1, None) == -1 and b"capacity 100" in L.star_last_error()
    c = _lib.KV8Cache(B=1, Hkv=2, T=128, hd=64, dtype=0)
    assert L.star_kv8_append(c, 16, 16, 0, 0, 0, 0, 0, 0, None, None, 1, None, 1, None) == -1 and b"null pointer" in L.star_last_error()
    for n in ("k_codes", "k_scales", "v_codes", "v_scales", "k_tail", "v_tail", "lens", "dropped", "tickets"):
        setattr(c, n, 16)
    q = _lib.KV8Query(H=4, L=1 << 22)
    assert L.star_kv8_attn(c, 16, None, None, q, 16, None, 0, None) == -1 and b"4194304 queries" in L.star_last_error()
    assert L.star_kv8_attn_workspace(c, 4, 1 << 22) == 0
    for sr in (1 << 23, -8):
        assert L.star_kv8_append(c, 16, 16, 0, 0, sr, 0, 0, 0, None, None, 1, None, 1, None) == -1 and b"row strides" in L.star_last_error()
    assert L.star_kv8_append(c, 16, 16, 0, 0, 0, 0, 4, 0, None, None, 1, None, 1, None) == -1 and b"multiples of 8" in L.star_last_error()
    assert L.star_kv8_append(c, 16, 16, 0, 0, 0, 0, 0, 0, None, None, 1, None, -1, None) == -1 and b"max_rows" in L.star_last_error()
    q = _lib.KV8Query(H=3, L=1)
    assert L.star_kv8_attn(c, 16, None, None, q, 16, None, 0, None) == -1 and b"divide" in L.star_last_error()
    c.T = 1 << 20
    q = _lib.KV8Query(H=2, L=1)
    need = L.star_kv8_attn_workspace(c, 2, 1)
    assert need > 0 and L.star_kv8_attn(c, 16, None, None, q, 16, None, 0, None) == -3 and b"workspace" in L.star_last_error()
    c.k_tail = 24
    assert L.star_kv8_attn(c, 16, None, None, q, 16, 16, need, None) == -1 and b"aligned" in L.star_last_error()


@gpu
def test_causal_attn_refusals(ops):
    plan = ops.PackedSeqs([10], DEV)
    q = rnd(0, 10, 4, 64)
    bad = [
        (ValueError, "rows, heads", (q[0], q, q)), (ValueError, "do not fit", (q, q, q[:9])), (ValueError, "do not fit", (q, rnd(0, 10, 4, 128), rnd(0, 10, 4, 128))),
        (TypeError, "share one dtype", (q, q.half(), q)), (TypeError, "float32", (q.float(), q.float(), q.float())),
        (ValueError, "divide", (q, q[:, :3], q[:, :3])), (ValueError, "head dim 32", tuple(rnd(0, 10, 4, 32) for _ in range(3))),
        (ValueError, "plan needs", (q[:9], q, q)), (ValueError, "plan needs", (q, q[:9], q[:9])),
        (ValueError, "contiguous head", (rnd(0, 10, 64, 4).transpose(1, 2), q, q)), (ValueError, "aligned", (rnd(0, 10, 4, 68)[..., 4:], q, q)),
        (ValueError, "aligned", (q, rnd(0, 10 * 4 * 64 + 1)[1:].view(10, 4, 64), q)),
    ]
    for err, text, args in bad:
        with pytest.raises(err, match=text):
            ops.causal_attn(*args, plan)
    with pytest.raises(ValueError, match="plan is on cpu"):
        ops.causal_attn(q, q, q, ops.PackedSeqs([10], "cpu"))
    with pytest.raises(ValueError, match="scale"):
        ops.causal_attn(q, q, q, plan, scale=0.0)
    assert ops.causal_attn(q[:0], q[:0], q[:0], ops.PackedSeqs([], DEV)).shape == (0, 4, 64)
    x = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.causal_attn(x, x, x, plan).sum(), x, create_graph=True)


@gpu
def test_kv8_refusals(ops):
    cache = ops.KVCache8(2, 2, 100, 64, DEV)
    assert cache.capacity == 128
    k = rnd(0, 2, 2, 3, 64)
    for err, text, args, kw in [
        (ValueError, "differ", (k, k[:, :, :2]), {}), (TypeError, "takes", (k.half(), k.half()), {}), (ValueError, "expected", (k[:1], k[:1]), {}),
        (ValueError, "counts must be", (k, k), dict(counts=torch.ones(3, dtype=torch.int32, device=DEV))),
        (TypeError, "integers", (k, k), dict(counts=torch.ones(2, device=DEV))),
        (ValueError, "at must be", (k, k), dict(at=torch.ones(1, dtype=torch.int32, device=DEV))),
        (ValueError, "expected", (k, k), dict(plan=ops.PackedSeqs([1, 2], DEV))),
        (ValueError, "plan of 1", (k[0].transpose(0, 1).contiguous(),) * 2, dict(plan=ops.PackedSeqs([3], DEV))),
        (ValueError, "plan needs", (k[0].transpose(0, 1).contiguous(),) * 2, dict(plan=ops.PackedSeqs([3, 1], DEV))),
        (ValueError, "counts go", (k[0].transpose(0, 1).contiguous(),) * 2, dict(plan=ops.PackedSeqs([1, 1], DEV), counts=torch.ones(2, dtype=torch.int32, device=DEV))),
        (ValueError, "aligned", (rnd(0, 2, 2, 3, 68)[..., 4:],) * 2, {}),
        (ops.StarDeviceError, "GPU only", (k.cpu(), k.cpu()), {}),
    ]:
        with pytest.raises(err, match=text):
            ops.kv8_append(cache, *args, **kw)
    assert cache.lens.tolist() == [0, 0]
    ops.kv8_append(cache, k[:, :, :0], k[:, :, :0])
    q = rnd(1, 2, 4, 1, 64)
    for err, text, args, kw in [
        (ValueError, "multiple of 2", (q[:, :3],), {}), (ValueError, "multiple", (q[:1],), {}), (TypeError, "holds", (q.half(),), {}),
        (ValueError, "bias", (q,), dict(bias=torch.zeros(2, 129, device=DEV))), (ValueError, "q_len must be", (q,), dict(q_len=torch.ones(3, dtype=torch.int32, device=DEV))),
        (ValueError, "aligned", (rnd(0, 2, 4, 1, 68)[..., 4:],), {}),
    ]:
        with pytest.raises(err, match=text):
            ops.kv8_attn(*args, cache, **kw)
    with pytest.raises(Exception, match="no backward"):
        ops.kv8_attn(q.clone().requires_grad_(), cache)
    assert (ops.kv8_attn(q, cache) == 0).all() and ops.kv8_attn(q[:, :, :0], cache).shape == (2, 4, 0, 64)
    parts = cache.tensors()
    with pytest.raises(ValueError, match="expected the tensors"):
        ops.KVCache8.from_tensors(k_codes=parts["k_codes"])
    with pytest.raises(ValueError, match="lens"):
        ops.KVCache8.from_tensors(**{**parts, "lens": parts["lens"].long()})
    with pytest.raises(ValueError, match="contiguous"):
        ops.KVCache8.from_tensors(**{**parts, "k_tail": parts["k_tail"].transpose(2, 3).contiguous().transpose(2, 3)})
    with pytest.raises(TypeError, match="float32"):
        ops.KVCache8(1, 1, 64, 64, DEV, torch.float32)
    with pytest.raises(ValueError):
        ops.KVCache8(1, 0, 64, 64, DEV)
