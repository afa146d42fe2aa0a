"""NuggetSelfAttention (training, prompt, token by token) and the 8-bit form of StreamingEncoderKV with
NuggetCrossAttention: the modules against the formulas of their cores on the projections that they themselves made.
c_proj is the identity here, which passes 16-bit values through unchanged."""
import math

import pytest
import torch

from tests.test_self_attention import BF, DEV, by_formula, cached_formula, check, rnd

gpu = pytest.mark.gpu


def module(H, Hkv, hd, dtype=BF, **kw):
    from star_amd import NuggetSelfAttention
    torch.manual_seed(H * hd + Hkv)
    m = NuggetSelfAttention(H * hd, H, kv_heads=Hkv, **kw).to(DEV, dtype)
    with torch.no_grad():
        m.c_attn.weight.mul_(2.0)
        m.c_attn.bias.normal_()
        m.c_proj.weight.copy_(torch.eye(H * hd))
    seen = []
    m.c_attn.register_forward_hook(lambda mod, args, out: seen.append(out))
    return m, seen


def split(qkv, H, Hkv, hd):
    t = qkv.detach().reshape(-1, H + 2 * Hkv, hd)
    return t[:, :H], t[:, H:H + Hkv], t[:, H + Hkv:]


@gpu
@pytest.mark.parametrize("how", ["packed", "padded", "plain"])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 4, 96), (8, 2, 64)])
def test_training_in_every_layout(how, H, Hkv, hd):
    from star_amd import ops
    lens, T, d = ([40, 150, 0, 77], 150, H * hd) if how != "plain" else ([90, 90], 90, H * hd)
    m, seen = module(H, Hkv, hd)
    if how == "packed":
        x, kw = rnd(1, sum(lens), d), dict(plan=ops.PackedSeqs(lens, DEV))
        rows = torch.ones(sum(lens), dtype=torch.bool, device=DEV)
    else:
        x, kw = rnd(1, len(lens), T, d), dict(valid=ops.ValidFrames(lens, T, DEV)) if how == "padded" else {}
        rows = (torch.arange(T, device=DEV)[None] < torch.tensor(lens, device=DEV)[:, None]).flatten()
    x.requires_grad_()
    y = m(x, **kw)
    assert y.shape == x.shape
    seen[0].retain_grad()
    g = rnd(2, *y.shape)
    y.backward(g)
    q, k, v = (t[rows] for t in split(seen[0], H, Hkv, hd))
    do = g.reshape(-1, H, hd)[rows]
    want, _ = by_formula(q, k, v, lens, lens, hd ** -0.5, do)
    check(y.reshape(-1, H, hd)[rows], *want["o"])
    assert (y.reshape(-1, d)[~rows] == 0).all()
    grad = seen[0].grad
    for name, t in zip(("dq", "dk", "dv"), split(grad, H, Hkv, hd)):
        check(t[rows], *want[name], name)
    assert (grad.reshape(len(rows), -1)[~rows] == 0).all()
    assert all(torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in m.parameters()) and torch.isfinite(x.grad).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_other_types_and_the_inverse_layer_scale(dtype):
    from star_amd import ops
    m, seen = module(2, 2, 64, dtype, layer_idx=2, scale_attn_by_inverse_layer_idx=True)
    lens = [33, 70]
    x = rnd(1, sum(lens), 128, dtype=dtype)
    y = m(x, plan=ops.PackedSeqs(lens, DEV))
    assert y.dtype == dtype
    core = seen[0].to(BF) if dtype == torch.float32 else seen[0]
    want, _ = by_formula(*split(core, 2, 2, 64), lens, lens, 0.125 / 3, None)
    check(y.detach().view(-1, 2, 64), *want["o"])


@gpu
def test_prompt_and_tokens_through_the_cache():
    """The prompt's output is the training path's; every later output is the formula's on the held values, with a
    sequence that pauses and one that takes two tokens at once."""
    from star_amd import ops
    H, Hkv, hd, lens = 4, 2, 64, [60, 1, 129]
    m, seen = module(H, Hkv, hd)
    m.eval()
    plan = ops.PackedSeqs(lens, DEV)
    x = rnd(1, sum(lens), H * hd)
    with torch.no_grad():
        cache = m.new_cache(3, 200)
        y = m(x, plan=plan, cache=cache)
        assert torch.equal(y, m(x, plan=plan)) and cache.lens.tolist() == lens
        n = list(lens)
        for step, counts in enumerate([[2, 2, 2], [1, 0, 2], [2, 1, 1]]):
            xs = rnd(10 + step, 3, 2, H * hd)
            seen.clear()
            y = m(xs, cache=cache, counts=torch.tensor(counts, device=DEV))
            n = [a + c for a, c in zip(n, counts)]
            assert cache.lens.tolist() == n
            q = seen[0].view(3, 2, -1, hd)[:, :, :H].transpose(1, 2)
            want, bound = cached_formula(q, *cache.values(), n, True, counts, -1, None, hd ** -0.5)
            check(y.view(3, 2, H, hd).transpose(1, 2), want, bound, step)
    with pytest.raises(ValueError, match="no_grad"):
        m(xs, cache=cache)


@gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_streaming_memory_in_8_bits(dtype):
    """StreamingEncoderKV(eight_bit=True), extended chunk by chunk, against the 16-bit buffers of the same memory, and
    NuggetCrossAttention on it against the formula on the held values."""
    from star_amd import NuggetCrossAttention, NuggetScorer, ops
    from star_amd.streaming import StreamingEncoderKV, StreamingNuggetSegmenter
    B, d, h, kmax, nl = 3, 256, 4, 150, 2
    torch.manual_seed(0)
    seg = StreamingNuggetSegmenter(NuggetScorer(d).to(DEV), B, d, kmax, DEV, dtype=dtype)
    mods = [NuggetCrossAttention(d, h, layer_idx=i).to(DEV, dtype).eval() for i in range(nl)]
    with torch.no_grad():
        for m in mods:
            m.c_attn.weight.mul_(3.0)
            m.c_proj.weight.copy_(torch.eye(d))
    seg.state.mem.copy_(rnd(1, B, kmax, d).to(dtype))
    scores = torch.randn(B, kmax, device=DEV)
    wide, held = StreamingEncoderKV(mods, seg), StreamingEncoderKV(mods, seg, eight_bit=True)
    for counts in ([5, 0, 20], [70, 3, 64], [70, 66, 150]):
        wide.extend(counts)
        held.extend(counts)
        seg.state.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        x = rnd(sum(counts), B, 1, d).to(dtype)
        for l, m in enumerate(mods):
            cache, kv = held.layers()[l].cache, wide.layers()[l]
            assert cache.lens.tolist() == counts
            live = (torch.arange(kmax, device=DEV)[None] < torch.tensor(counts, device=DEV)[:, None])[:, None, :, None]
            for got, ref in zip(cache.values(), (kv.key, kv.value)):
                ref = torch.where(live, ref.double(), 0.0)
                got = got.double()[:, :, :kmax]
                # e4m3: half a step, 2^-4 of the value, at most 2^-10 of the scale near zero, the scale at most max / 224;
                # 2^-7 more for another order of the projection's sums and its rounding to 16 bits
                bound = (2.0 ** -4 + 2.0 ** -7) * ref.abs() + 2.0 ** -10 * ref.abs().amax() / 224 + 2.0 ** -7 * 2.0 ** -4 * ref.abs().amax()
                assert ((got - ref).abs() <= bound).all()
            for token in (0, 40):
                with torch.no_grad():
                    y, present = m(x, encoder_kv=held.layers()[l], scorer_logits=scores, limit_cross_attn=True, query_offset=token)
                    q = m._split_heads(m.q_attn(x)).to(cache.dtype)
                assert present is None and y.dtype == dtype
                want, bound = cached_formula(q, *cache.values(), counts, False, None, token + 2, scores, (d // h) ** -0.5)
                check(y.view(B, 1, h, d // h).transpose(1, 2), want, bound, (counts, l, token))
            with torch.no_grad():                              # an additive mask changes nothing that lens does not
                assert torch.equal(m(x, encoder_kv=held.layers()[l], encoder_attention_mask=wide.encoder_attention_mask())[0],
                                   m(x, encoder_kv=held.layers()[l])[0])
    with pytest.raises(ValueError, match="went back"):
        held.extend([0, 66, 150])
    held.reset([0])
    assert held.layers()[0].cache.lens.tolist() == [0, 66, 150]
    held.extend([4, 66, 150])
    assert held.layers()[1].cache.lens.tolist() == [4, 66, 150]
    for kw in (dict(output_attentions=True), dict(use_cache=True), dict(head_mask=torch.ones(1, h, 1, 1, device=DEV))):
        with pytest.raises(ValueError, match="8-bit"), torch.no_grad():
            mods[0](x, encoder_kv=held.layers()[0], **kw)
    with pytest.raises(Exception, match="no backward"):
        mods[0](x, encoder_kv=held.layers()[0])


def test_module_refusals():
    from star_amd import NuggetSelfAttention, ops
    with pytest.raises(ValueError, match="divisible"):
        NuggetSelfAttention(100, 3)
    with pytest.raises(ValueError, match="divide"):
        NuggetSelfAttention(256, 4, kv_heads=3)
    with pytest.raises(NotImplementedError, match="attn_pdrop"):
        NuggetSelfAttention(256, 4, attn_pdrop=0.1)
    m = NuggetSelfAttention(256, 4, kv_heads=2)
    assert m.c_attn.weight.shape == (256, 512) and m.scale == 64 ** -0.5
    assert sorted(m.state_dict()) == ["c_attn.bias", "c_attn.weight", "c_proj.bias", "c_proj.weight"]
    x = torch.zeros(2, 5, 256)
    with pytest.raises(ValueError, match="counts"):
        m(x, counts=torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="or a plan"):
        m(x[0])
    with pytest.raises(ValueError, match="not both"):
        m(x[0], plan=ops.PackedSeqs([5], "cpu"), valid=ops.ValidFrames([5], 5, "cpu"))
    with pytest.raises(ValueError, match="valid is for"):
        m(x, valid=ops.ValidFrames([5], 5, "cpu"))
    with pytest.raises(ops.StarDeviceError):
        m(x)
    with pytest.raises(ValueError, match="key starts"):
        ops.PackedSeqs([1, 2], "cpu", k_starts=[0])
    p = ops.PackedSeqs([1, 2], "cpu", k_starts=[7, 3])
    assert p.seqs.tolist() == [[0, 1, 7, 1], [1, 2, 3, 2]] and p.k_rows == 8
