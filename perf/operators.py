"""Cases of the self-attention and 8-bit cache operators: what a pass of each reads, writes and computes, in plain torch
and through star_amd.ops.

  attn    ops.causal_attn     causal attention of packed sequences, forward
  train   ops.causal_attn     the same, forward and backward
  append  ops.kv8_append      keys and values into the 8-bit cache
  cached  ops.kv8_attn        attention of a few new tokens over the 8-bit cache

Sequences are packed one behind the other, [rows, heads, head dim].  Query i of a sequence with nq queries and nk keys
sees the keys j <= i + nk - nq.  The cache keeps blocks of 64 tokens of one head as e4m3 values times one power of two
(K [B,H,T,hd], V transposed inside its block [B,H,T/64,hd,64]) and the newest, unfinished block as it came.
"""
import math
import random

import torch

own = False
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
F8 = torch.float8_e4m3fn
BLK = 64


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one utterance of a live stream: a chunk of 16 new frames over all the frames so far (latency)
        dict(name="attn_stream_chunk", kind="attn", B=1, lo=375, hi=375, nq=16, H=8, Hkv=8, hd=128, type="bf16", lens=1),
        # semantic encoder on a speech batch with utterances of very different lengths
        dict(name="attn_speech_batch", kind="attn", B=64, lo=40, hi=1500, nq=0, H=8, Hkv=8, hd=128, type="bf16", lens=2),
        # twelve heads of 64, fp16
        dict(name="attn_heads64_fp16", kind="attn", B=16, lo=512, hi=1999, nq=0, H=12, Hkv=12, hd=64, type="fp16", lens=3),
        # one long recording, grouped heads, odd length
        dict(name="attn_long_grouped", kind="attn", B=1, lo=12001, hi=12001, nq=0, H=16, Hkv=4, hd=128, type="bf16", lens=4),
        # text decoder training: 32 transcripts of up to 128 tokens, 8 heads of 96
        dict(name="train_transcripts", kind="train", B=32, lo=20, hi=128, nq=0, H=8, Hkv=8, hd=96, type="bf16", lens=5),
        # semantic encoder training: 32 utterances of 1500 frames, width 1024
        dict(name="train_speech_batch", kind="train", B=32, lo=1500, hi=1500, nq=0, H=8, Hkv=8, hd=128, type="bf16", lens=6),
        # training on one long sequence with grouped heads
        dict(name="train_long_grouped", kind="train", B=1, lo=8191, hi=8191, nq=0, H=16, Hkv=4, hd=128, type="bf16", lens=7),
        # generation: one token of each of 64 sequences into the cache (latency)
        dict(name="append_token", kind="append", B=64, lo=0, hi=4095, n=1, Hkv=8, hd=128, type="bf16", lens=8, T=4096),
        # 32 prompts of different lengths into an empty cache
        dict(name="append_prompts", kind="append", B=32, lo=30, hi=4000, n=0, Hkv=8, hd=128, type="bf16", lens=9, T=4096),
        # one token of one utterance over its nugget memory, with the scorer's logits and the lookback mask (latency)
        dict(name="cached_nuggets", kind="cached", B=1, lo=375, hi=375, L=1, H=8, Hkv=8, hd=128, type="bf16", lens=10, T=384, nugget=True),
        # generation: one token of each of 64 sequences, grouped heads
        dict(name="cached_batch", kind="cached", B=64, lo=100, hi=4096, L=1, H=32, Hkv=8, hd=128, type="bf16", lens=11, T=4096, nugget=False),
        # four tokens at once over very long sequences
        dict(name="cached_long", kind="cached", B=4, lo=60001, hi=131072, L=4, H=32, Hkv=8, hd=128, type="bf16", lens=12, T=131072, nugget=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    c = dict(kind=rng.choice(["attn", "train", "append", "cached"]), hd=rng.choice([64, 96, 128]),
             type=rng.choice(["bf16", "bf16", "fp16"]), lens=rng.randrange(1 << 20))
    c["Hkv"] = rng.choice([1, 2, 4, 8, 12])
    g = rng.choice([1, 1, 2, 4, 8])
    if c["kind"] == "append":
        c["T"] = T = 64 * _log(rng, 2, 256)
        c["n"] = rng.choice([0, 1])
        c["B"] = max(1, min(_log(rng, 1, 96), (1 << 27) // (T * c["Hkv"] * c["hd"])))
        c["lo"], c["hi"] = (rng.randrange(0, T // 2), T - 1)
    elif c["kind"] == "cached":
        c["H"] = c["Hkv"] * g
        c["T"] = T = 64 * _log(rng, 1, 1024)
        c["L"] = rng.choice([1, 1, 2, 5, 16])
        c["B"] = max(1, min(_log(rng, 1, 96), (1 << 28) // (T * c["Hkv"] * c["hd"])))
        c["hi"] = rng.randrange(max(c["L"], T // 2), T + 1)
        c["lo"] = rng.randrange(c["L"], c["hi"] + 1)
        c["nugget"] = rng.random() < 0.3
    else:
        c["H"] = c["Hkv"] * g
        c["hi"] = _log(rng, 16, 6000)
        c["lo"] = rng.randrange(1, c["hi"] + 1)
        most = (1 << 30) // (c["H"] * c["hi"] * c["hi"])
        c["B"] = max(1, min(_log(rng, 1, 64), most))
        c["nq"] = 0 if c["kind"] == "train" else rng.choice([0, 0, rng.randrange(1, 100)])
    return c


def _lengths(case):
    """Keys (tokens in the cache) of every sequence; the longest is `hi`."""
    rng = random.Random(case["lens"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    lens[rng.randrange(case["B"])] = case["hi"]
    return lens


def _queries(case):
    return [min(case["nq"], n) if case["nq"] else n for n in _lengths(case)]


# ------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dt)

    lens = _lengths(case)
    hd, Hkv = case["hd"], case["Hkv"]
    s = dict(case=case)
    if case["kind"] in ("attn", "train"):
        nq = _queries(case)
        s["q"], s["k"], s["v"] = normal(sum(nq), case["H"], hd), normal(sum(lens), Hkv, hd), normal(sum(lens), Hkv, hd)
        if case["kind"] == "train":
            s["do"] = normal(sum(nq), case["H"], hd)
        s["nq"], s["nk"] = _ints(nq), _ints(lens)
        s["most_q"], s["most_k"] = max(nq), max(lens)
        if own:
            from star_amd import ops
            s["plan"] = ops.PackedSeqs(lens, DEV, q_lengths=nq)
        return s
    B, T = case["B"], case["T"]
    if case["kind"] == "append" and case["n"] == 0:            # prompts into an empty cache
        s["parts"] = _empty_cache(B, Hkv, T, hd, dt)
        s["at"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        s["k"], s["v"] = normal(sum(lens), Hkv, hd), normal(sum(lens), Hkv, hd)
        s["n"], s["most"] = _ints(lens), max(lens)
        if own:
            from star_amd import ops
            s["plan"] = ops.PackedSeqs(lens, DEV)
    else:
        s["parts"] = _filled_cache(lens, Hkv, T, hd, dt, gen)
        if case["kind"] == "append":
            s["at"] = s["parts"]["lens"].clone()
            s["k"], s["v"] = normal(B, Hkv, case["n"], hd), normal(B, Hkv, case["n"], hd)
            s["n"] = torch.full((B,), case["n"], dtype=torch.int32, device=DEV)
        else:
            s["q"] = normal(B, case["H"], case["L"], hd)
            if case["nugget"]:
                s["bias"] = torch.randn((B, T), generator=gen, device=DEV, dtype=torch.float32) * 2
    if own:
        from star_amd import ops
        s["cache"] = ops.KVCache8.from_tensors(**s["parts"])
    return s


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _empty_cache(B, H, T, hd, dt):
    z = lambda *shape, dtype: torch.zeros(shape, dtype=dtype, device=DEV)  # noqa: E731
    return dict(k_codes=z(B, H, T, hd, dtype=torch.uint8).view(F8), k_scales=z(B, H, T // BLK, dtype=torch.float32),
                v_codes=z(B, H, T // BLK, hd, BLK, dtype=torch.uint8).view(F8), v_scales=z(B, H, T // BLK, dtype=torch.float32),
                k_tail=z(B, H, BLK, hd, dtype=dt), v_tail=z(B, H, hd, BLK, dtype=dt), lens=z(B, dtype=torch.int32))


def _filled_cache(lens, H, T, hd, dt, gen):
    """A cache that holds `lens` tokens of normal keys and values, a few dimensions of the keys larger than the others."""
    B = len(lens)
    parts = _empty_cache(B, H, T, hd, dt)
    parts["lens"] = _ints(lens)
    gain = 1 + 3 * (torch.rand((H, 1, hd), generator=gen, device=DEV) < 0.05).float()
    for b in range(B):
        for codes, scales, tail, g in (("k_codes", "k_scales", "k_tail", gain), ("v_codes", "v_scales", "v_tail", 1.0)):
            x = (torch.randn((H, T, hd), generator=gen, device=DEV) * g).to(dt).float().view(H, T // BLK, BLK, hd)
            c, s = _quantise(x)
            full = lens[b] // BLK
            if codes == "v_codes":
                c, x = c.view(torch.uint8).transpose(2, 3).contiguous().view(F8), x.transpose(2, 3)
                parts[codes][b, :, :full] = c[:, :full]
            else:
                parts[codes][b, :, :full * BLK] = c.reshape(H, T, hd)[:, :full * BLK]
            parts[scales][b, :, :full] = s[:, :full]
            if full < T // BLK:
                parts[tail][b] = x[:, full].to(dt)
    return parts


def _quantise(x):
    """x [..., 64, hd] fp32 -> e4m3 values, power-of-two scales [...]: the smallest 2^e with max|x| <= 448 * 2^e."""
    m = x.abs().amax(dim=(-1, -2))
    mant, e = torch.frexp(m)                                   # m = mant * 2^e, 0.5 <= mant < 1; 448 = 0.875 * 2^9
    e = torch.where(mant <= 0.875, e - 9, e - 8)
    s = torch.where(m > 0, torch.ldexp(torch.ones_like(m), e), torch.ones_like(m))
    return (x / s[..., None, None]).to(F8), s


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attn": _own_attn, "train": _own_train, "append": _own_append, "cached": _own_cached}[kind](state)
    return {"attn": _plain_attn, "train": _plain_train, "append": _plain_append, "cached": _plain_cached}[kind](state)


def _own_attn(s):
    from star_amd import ops
    return ops.causal_attn(s["q"], s["k"], s["v"], s["plan"])


def _own_train(s):
    from star_amd import ops
    q, k, v = (s[n].detach().requires_grad_() for n in "qkv")
    o = ops.causal_attn(q, k, v, s["plan"])
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
    return dict(o=o.detach(), dq=dq, dk=dk, dv=dv)


def _own_append(s):
    from star_amd import ops
    ops.kv8_append(s["cache"], s["k"], s["v"], plan=s.get("plan"), at=s["at"])
    return s["cache"].tensors()


def _own_cached(s):
    from star_amd import ops
    if s["case"]["nugget"]:
        return ops.kv8_attn(s["q"], s["cache"], causal=False, ilk_diag=s["case"]["hi"] // 2, bias=s["bias"])
    return ops.kv8_attn(s["q"], s["cache"])


def _rows(n, most):
    """Packed rows of sequences of n[b] rows -> their indices in a padded [B, most] layout (clamped) and, back, the
    sequence and place of every packed row."""
    start = torch.cumsum(n, 0) - n
    place = torch.arange(most, device=n.device)
    pad = (start[:, None] + torch.minimum(place[None, :], (n - 1).clamp(min=0)[:, None])).long()
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n)
    return pad, seq, torch.arange(len(seq), device=n.device) - start[seq]


def _padded_probs(s):
    c = s["case"]
    g = c["H"] // c["Hkv"]
    pad_q, seq_q, at_q = _rows(s["nq"], s["most_q"])
    pad_k, seq_k, at_k = _rows(s["nk"], s["most_k"])
    q = s["q"].float()[pad_q].unflatten(2, (c["Hkv"], g)).permute(0, 2, 3, 1, 4).contiguous()   # [B,Hkv,g,Q,hd]
    k = s["k"].float()[pad_k].permute(0, 2, 1, 3)[:, :, None].contiguous()                      # [B,Hkv,1,K,hd]
    v = s["v"].float()[pad_k].permute(0, 2, 1, 3)[:, :, None].contiguous()
    i = torch.arange(s["most_q"], device=DEV)[:, None]
    j = torch.arange(s["most_k"], device=DEV)[None, :]
    seen = (j <= i + (s["nk"] - s["nq"])[:, None, None]) & (j < s["nk"][:, None, None])
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * c["hd"] ** -0.5
    x = torch.where(seen[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    p = x / x.sum(-1, keepdim=True)
    return q, k, v, p, seq_q, at_q, seq_k, at_k


def _plain_attn(s):
    q, k, v, p, seq_q, at_q, _, _ = _padded_probs(s)
    o = torch.matmul(p, v).flatten(1, 2)
    return o[seq_q, :, at_q].to(s["q"].dtype)


def _plain_train(s):
    c = s["case"]
    q, k, v, p, seq_q, at_q, seq_k, at_k = _padded_probs(s)
    o = torch.matmul(p, v)
    do = torch.zeros((c["B"], s["most_q"], c["H"], c["hd"]), device=DEV)
    do[seq_q, at_q] = s["do"].float()
    do = do.unflatten(2, (c["Hkv"], -1)).permute(0, 2, 3, 1, 4).contiguous()
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = p * (torch.matmul(do, v.transpose(-1, -2).contiguous()) - (do * o).sum(-1, keepdim=True)) * c["hd"] ** -0.5
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2)
    dt = s["q"].dtype
    return dict(o=o.flatten(1, 2)[seq_q, :, at_q].to(dt), dq=dq.flatten(1, 2)[seq_q, :, at_q].to(dt),
                dk=dk[seq_k, :, at_k].to(dt), dv=dv[seq_k, :, at_k].to(dt))


def _plain_append(s):
    p, at, n = s["parts"], s["at"].long(), s["n"].long()
    B, H, T, hd = p["k_codes"].shape
    most = s.get("most", s["k"].shape[2])
    base = at // BLK                                           # the block that is open before the call
    nb = -(-(most + BLK - 1) // BLK)                           # blocks that a sequence can reach, the open one included
    place = torch.arange(nb * BLK, device=DEV)
    row = place[None, :] - (at % BLK)[:, None]                 # row of the new tokens at this place; < 0: it is in the tail
    batch = torch.arange(B, device=DEV)
    if s["k"].dim() == 3:
        src = (torch.cumsum(n, 0) - n)[:, None] + torch.minimum(row.clamp(min=0), (n - 1).clamp(min=0)[:, None])
        new_k, new_v = s["k"][src], s["v"][src]                # [B, places, H, hd]
    else:
        src = row.clamp(0, most - 1)
        new_k, new_v = (s[x].permute(0, 2, 1, 3)[batch[:, None], src] for x in ("k", "v"))
    old = place.clamp(max=BLK - 1)
    old_k, old_v = p["k_tail"].permute(0, 2, 1, 3)[:, old], p["v_tail"].permute(0, 3, 1, 2)[:, old]
    end = at + n
    done = (base[:, None] + torch.arange(nb, device=DEV) + 1) * BLK <= end[:, None]             # [B, nb]
    blk = (base[:, None] + torch.arange(nb, device=DEV)).clamp(max=T // BLK - 1)
    keep = (row >= 0)[..., None, None]
    last = end // BLK - base                                   # the block that is open after the call
    in_tail = (last[:, None] * BLK + torch.arange(BLK, device=DEV))                             # its places
    fresh = (torch.gather(row, 1, in_tail.clamp(max=nb * BLK - 1)) >= 0) & (base[:, None] * BLK + in_tail < end[:, None])
    b_done, j_done = torch.nonzero(done, as_tuple=True)
    for name, new, before in (("k", new_k, old_k), ("v", new_v, old_v)):
        x = torch.where(keep, new, before)                     # [B, places, H, hd]
        codes, scales = _quantise(x.float().view(B, nb, BLK, H, hd).permute(0, 1, 3, 2, 4))      # [B, nb, H, 64, hd]
        at_blk = blk[b_done, j_done]
        p[name + "_scales"][b_done, :, at_blk] = scales[b_done, j_done]
        bytes_ = codes.view(torch.uint8)[b_done, j_done]
        tail = x[batch[:, None], in_tail.clamp(max=nb * BLK - 1)].permute(0, 2, 1, 3)           # [B, H, 64, hd]
        to = p[name + "_tail"]
        if name == "k":
            p["k_codes"].view(torch.uint8).view(B, H, T // BLK, BLK, hd)[b_done, :, at_blk] = bytes_
            to.copy_(torch.where(fresh[:, None, :, None], tail, to))
        else:
            p["v_codes"].view(torch.uint8)[b_done, :, at_blk] = bytes_.transpose(-1, -2)
            to.copy_(torch.where(fresh[:, None, None, :], tail.transpose(-1, -2), to))
    p["lens"].copy_(end)
    return p


def _values(p, as_type):
    """The keys and values that a cache stands for, [B,H,T,hd]."""
    B, H, T, hd = p["k_codes"].shape
    blocks = torch.arange(T // BLK, device=DEV)
    is_tail = (blocks[None, :] == (p["lens"] // BLK)[:, None])[:, None, :, None, None]
    k = p["k_codes"].to(as_type).view(B, H, T // BLK, BLK, hd) * p["k_scales"].to(as_type)[..., None, None]
    k = torch.where(is_tail, p["k_tail"].to(as_type)[:, :, None], k)
    v = p["v_codes"].to(as_type) * p["v_scales"].to(as_type)[..., None, None]
    v = torch.where(is_tail, p["v_tail"].to(as_type)[:, :, None], v)
    return k.view(B, H, T, hd), v.transpose(-1, -2).reshape(B, H, T, hd)


def _plain_cached(s):
    c, p = s["case"], s["parts"]
    k, v = _values(p, torch.float32)
    B, Hkv, T, hd = k.shape
    q = s["q"].float().reshape(B, Hkv, -1, hd)                 # rows: (head of the group, token)
    x = torch.matmul(q, k.transpose(-1, -2)).view(B, c["H"], c["L"], T) * hd ** -0.5
    i = torch.arange(c["L"], device=DEV)[:, None]
    j = torch.arange(T, device=DEV)[None, :]
    n = p["lens"][:, None, None]
    seen = (j < n) & (j <= i + (c["hi"] // 2 if c["nugget"] else n - c["L"]))
    if c["nugget"]:
        x = x + s["bias"][:, None, None, :]
    x = torch.where(seen[:, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    return torch.matmul(x.view(B, Hkv, -1, T), v).view(B, c["H"], c["L"], hd).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    lens = _lengths(case)
    hd, Hkv = case["hd"], case["Hkv"]
    if case["kind"] in ("attn", "train"):
        nq = _queries(case)
        H = case["H"]
        pairs = sum(a * n - a * (a - 1) // 2 for a, n in zip(nq, lens))
        rows = 2 * hd * (2 * H * sum(nq) + 2 * Hkv * sum(lens))
        if case["kind"] == "attn":
            return dict(bytes=rows, flops=4 * hd * H * pairs)
        # q, k, v, dO read, o, dq, dk, dv written; QK', PV, dP, dV, dQ, dK
        return dict(bytes=2 * rows, flops=12 * hd * H * pairs)
    if case["kind"] == "append":
        if case["n"] == 0:
            full = [n // BLK * BLK for n in lens]
            read, eight, tail = sum(lens), sum(full), sum(lens) - sum(full)
        else:
            done = sum((n + 1) % BLK == 0 for n in lens)
            read, eight, tail = case["B"] + done * (BLK - 1), done * BLK, case["B"] - done
        return dict(bytes=2 * Hkv * (hd * (2 * read + eight + 2 * tail) + 4 * eight // BLK) + 8 * case["B"],
                    flops=4 * Hkv * hd * eight)
    H, L = case["H"], case["L"]
    if case["nugget"]:
        seen = [min(n, case["hi"] // 2 + L) for n in lens]
        pairs = sum(min(n, case["hi"] // 2 + i + 1) for n in lens for i in range(L))
    else:
        seen = lens
        pairs = sum(n - L + i + 1 for n in lens for i in range(L))
    cache = 0
    for n, top in zip(lens, seen):
        full = min(top, n // BLK * BLK)
        cache += hd * (full + 2 * (top - full)) + 4 * -(-full // BLK)
    return dict(bytes=2 * Hkv * cache + 4 * hd * H * L * case["B"] + (4 * sum(seen) if case["nugget"] else 0),
                flops=4 * hd * H * pairs)


# ------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        return _exact_append(case, s)
    if kind == "cached":
        return _exact_cached(case, s)
    g = case["H"] // case["Hkv"]
    out = {n: [] for n in ("o", "dq", "dk", "dv")}
    q0 = k0 = 0
    for nq, nk in zip(_queries(case), _lengths(case)):
        q = s["q"][q0:q0 + nq].double()
        k, v = (s[n][k0:k0 + nk].double() for n in "kv")
        hidden = torch.ones((nq, nk), dtype=torch.bool, device=DEV).triu(nk - nq + 1)
        parts = {n: [] for n in out}
        for h in range(case["H"]):
            kh, vh, qh = k[:, h // g], v[:, h // g], q[:, h]
            p = torch.softmax((qh @ kh.T / math.sqrt(case["hd"])).masked_fill(hidden, -math.inf), -1)
            oh = p @ vh
            parts["o"].append(oh)
            if kind == "train":
                do = s["do"][q0:q0 + nq, h].double()
                ds = p * (do @ vh.T - (do * oh).sum(1, keepdim=True)) / math.sqrt(case["hd"])
                parts["dq"].append(ds @ kh)
                for name, x in (("dk", ds.T @ qh), ("dv", p.T @ do)):
                    if h % g == 0:
                        parts[name].append(x)
                    else:
                        parts[name][-1] += x
        for n in out:
            if parts[n]:
                out[n].append(torch.stack(parts[n], 1))
        q0, k0 = q0 + nq, k0 + nk
    if kind == "attn":
        return torch.cat(out["o"])
    return {n: torch.cat(x) for n, x in out.items()}


def _exact_append(case, s):
    p = {n: x.clone() if n == "lens" else x.double() for n, x in s["parts"].items()}
    row = 0
    for b in range(case["B"]):
        a, n = int(s["at"][b]), int(s["n"][b])
        for name in "kv":
            if s["k"].dim() == 3:
                new = s[name][row:row + n].double().transpose(0, 1)
            else:
                new = s[name][b].double()
            tail = p[name + "_tail"][b] if name == "k" else p[name + "_tail"][b].transpose(1, 2)
            x = torch.cat([tail[:, :a % BLK], new], 1)          # tokens from the open block's first on
            first, j = a // BLK, 0
            while x.shape[1] - j >= BLK:
                part = x[:, j:j + BLK]
                m = part.abs().amax((1, 2))
                e = torch.ceil(torch.log2(m / 448))
                scale = torch.where(m > 0, 2.0 ** e, 1.0)
                c = _e4m3(part / scale[:, None, None])
                blk = first + j // BLK
                p[name + "_scales"][b, :, blk] = scale
                if name == "k":
                    p["k_codes"][b, :, blk * BLK:(blk + 1) * BLK] = c
                else:
                    p["v_codes"][b, :, blk] = c.transpose(1, 2)
                j += BLK
            rest = x[:, j:]
            if name == "k":
                p["k_tail"][b, :, :rest.shape[1]] = rest
            else:
                p["v_tail"][b, :, :, :rest.shape[1]] = rest.transpose(1, 2)
        p["lens"][b] = a + n
        row += n
    return p


def _e4m3(x):
    """The e4m3 value nearest to x, |x| <= 448, ties to the even mantissa: steps of 2^(e-3) for 2^e <= |x|, e >= -6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = 2.0 ** (e - 3)
    return torch.round(x / step) * step


def _exact_cached(case, s):
    p = s["parts"]
    B, g, L = case["B"], case["H"] // case["Hkv"], case["L"]
    out = torch.zeros((B, case["H"], L, case["hd"]), dtype=torch.float64, device=DEV)
    k, v = None, None
    for b in range(B):
        n = int(p["lens"][b])
        k, v = _values({x: y[b:b + 1] for x, y in p.items()}, torch.float64)
        k, v = k[0, :, :n], v[0, :, :n]
        for i in range(L):
            top = min(n, i + case["hi"] // 2 + 1) if case["nugget"] else n - L + i + 1
            q = s["q"][b, :, i].double().view(case["Hkv"], g, -1)
            x = q @ k[:, :top].transpose(1, 2) / math.sqrt(case["hd"])
            if case["nugget"]:
                x = x + s["bias"][b, :top].double()
            out[b, :, i] = (torch.softmax(x, -1) @ v[:, :top]).flatten(0, 1)
    return out
