"""Drop-in mirror of the reference's nugget operators (same names, arguments and return values).

The reference has no plugin interface; its boundary is these Python signatures:

  reference (src/models/...)                               here
  -------------------------------------------------------  ------------------------------------------
  nugget_model = Sequential(Linear, ReLU, Linear)          NuggetScorer                (w2v_asr.py:113-117)
  W2VASRModel.apply_nugget_compression (w2v_asr.py:208)    NuggetOpsMixin.apply_nugget_compression
  W2VASRModel.add_nugget_type_embedding (w2v_asr.py:316)   NuggetOpsMixin.add_nugget_type_embedding
  W2VSimulModel.resize (w2v_simul.py:504)                  NuggetOpsMixin.resize
  W2VSimulModel.apply_threshold_yield_nugget (:376)        NuggetOpsMixin.apply_threshold_yield_nugget
  W2VSimulModel.get_valid_mask_indices (:196)              NuggetOpsMixin.get_valid_mask_indices
  semantic_repr[arange(B)[:,None], nugget_indices]         gather_nuggets              (w2v_asr.py:566-567)
  MyGPT2Attention._attn (my_transformer.py:535)            score_biased_attn / NuggetCrossAttention._attn
  MyGPT2Attention.forward, cross branch (:490-533)         NuggetCrossAttention.forward
  MyGPT2Attention.forward, self branch (:490-533)          NuggetSelfAttention.forward (causal, lengths for masks)

A maintainer of the reference makes `W2VASRModel` / `W2VSimulModel` inherit `NuggetOpsMixin` (first in
the MRO), builds `self.nugget_model = NuggetScorer(hidden_size)` and uses `NuggetCrossAttention` for
`MyGPT2Block.crossattention`; parameter names (`nugget_model.0.weight`, `crossattention.c_attn.weight`,
...) are unchanged, so checkpoints and the trainers' optimizer grouping keep working.
Everything runs in the HIP kernels of libstar_nugget.so; there is no CPU path.
"""
from __future__ import annotations

import threading
from typing import Optional

import torch
from torch import nn

from . import ops
from ._lib import StarNuggetError


# ------------------------------------------------------------------------------------------ a1
class NuggetScorer(nn.Sequential):
    """nn.Sequential(nn.Linear(d, d), nn.ReLU(inplace=True), nn.Linear(d, 1)) with a fused HIP forward/backward.
    state_dict keys: 0.weight, 0.bias, 2.weight, 2.bias -- identical to the reference module."""

    def __init__(self, hidden_size: int):
        super().__init__(nn.Linear(hidden_size, hidden_size), nn.ReLU(inplace=True), nn.Linear(hidden_size, 1))
        self.active_rows = ops.ActiveRows()

    def set_active_rows(self, rows: Optional[torch.Tensor]):
        """Optional, SINGLE-USE: frames (flattened b*T+t) that can receive a score gradient in the backward of the
        most recent forward (or of the next one, when called before any forward); None = dense.  The hint is
        consumed by that backward; every other forward/backward of this module runs dense (ops.ActiveRows)."""
        self.active_rows.set(rows)

    def forward(self, x: torch.Tensor, valid: Optional["ops.ValidFrames"] = None) -> torch.Tensor:  # [B,T,d] -> [B,T,1]
        """valid (optional, not in the reference): ops.ValidFrames of the padded batch -- pad frames get score 0 and
        row tiles made of padding only are not computed.  Every consumer of the scores on the path masks pad frames
        (w2v_asr.py:214-216, w2v_simul.py:421), so results do not change."""
        s = ops.scorer(x, self[0].weight, self[0].bias, self[2].weight, self[2].bias, self.active_rows, valid)
        return s.to(x.dtype if x.dtype != torch.bfloat16 else torch.float32).unsqueeze(-1)


# ------------------------------------------------------------------------------------------ a4
def gather_nuggets(semantic_repr: torch.Tensor, nugget_indices: torch.Tensor) -> torch.Tensor:
    """semantic_repr[torch.arange(B)[:, None], nugget_indices]; -1 indexes the last frame, as in the reference."""
    return ops.gather_rows(semantic_repr, nugget_indices)


def gather_nuggets_layernorm(hidden: torch.Tensor, nugget_indices: torch.Tensor, ln_f: nn.LayerNorm) -> torch.Tensor:
    """ln_f(hidden)[torch.arange(B)[:, None], nugget_indices] for the semantic encoder's final LayerNorm
    (my_transformer.py:945, then w2v_asr.py:566-567): call the encoder without its ln_f and pass the
    un-normalised last hidden state here -- only the nugget rows are normalised and written."""
    if tuple(ln_f.normalized_shape) != (hidden.shape[-1],) or ln_f.weight is None or ln_f.bias is None:
        raise ValueError("gather_nuggets_layernorm: ln_f must be an affine LayerNorm over the last dimension")
    return ops.gather_layernorm(hidden, nugget_indices, ln_f.weight, ln_f.bias, ln_f.eps)


# ------------------------------------------------------------------------------------------ a2, a3, a6, a7
class NuggetOpsMixin:
    """Methods with the reference's names and signatures; expects `self.nugget_compress_rate` and
    `self.nugget_model` like the reference classes."""

    def apply_nugget_compression(self, encoder_repr, attn_mask, nugget_scores=None, n_nugget=None):
        """-> (nugget_mask [B,K] bool, indices_ascending [B,K] int64, scores_gather [B,K])  (w2v_asr.py:208-244).
        Like the reference this reads max(k_b) back to the host to size the outputs."""
        if nugget_scores is None:
            nugget_scores = self.nugget_model(encoder_repr).squeeze(-1)
        rate = None if n_nugget is not None else self.nugget_compress_rate
        nmask, idx, sg = ops.topk_select(nugget_scores, attn_mask=attn_mask, rate=rate, n_nugget=n_nugget,
                                         want_table=False)
        return nmask, idx, sg

    @staticmethod
    def add_nugget_type_embedding(inputs_embed, nugget_indices, nugget_mask):
        """-> (type_ind_table [B,T] int64, nugget_position [B,K] int64 with pads = -1)  (w2v_asr.py:316-323).
        The fused path (`select_nuggets`) gets both from the select kernel for free."""
        return ops.type_table(nugget_indices, nugget_mask, inputs_embed.shape[1])

    def select_nuggets(self, nugget_scores, attn_mask=None, lengths=None, K: Optional[int] = None):
        """Fused apply_nugget_compression + add_nugget_type_embedding: one kernel, no host sync when K is given.
        -> (nugget_mask, indices_ascending, scores_gather, type_ind_table, nugget_position)."""
        return ops.topk_select(nugget_scores, attn_mask=attn_mask, lengths=lengths,
                               rate=self.nugget_compress_rate, K=K, want_table=True)

    def resize(self, alphas, target_lengths, noise=0.0, threshold=1.0):
        """w2v_simul.py:504-535, differentiable w.r.t. alphas like the reference's (lm_cif_training sends the
        lm_loss gradient through it).  noise must be 0 (the only value the reference ever passes)."""
        if noise != 0.0:
            raise NotImplementedError("resize: noise != 0 is never used by the reference and is not implemented")
        return ops.cif_resize(alphas, target_lengths, threshold=threshold)

    @staticmethod
    def add_type_embedding(inputs_embed: torch.Tensor, type_ind_table: torch.Tensor, type_embed):
        """`inputs_embed + self.semantic_encoder.type_embed(type_ind_table)` (w2v_asr.py:383,400,456,560;
        w2v_simul.py:432) in one pass; `type_embed` is the nn.Embedding(2, d) module or its weight."""
        weight = type_embed.weight if isinstance(type_embed, nn.Module) else type_embed
        return ops.type_embed_add(inputs_embed, type_ind_table, weight)

    @staticmethod
    def cif_weighted_aggregate(alphas: torch.Tensor, semantic_repr: torch.Tensor, threshold: float = 1.0):
        """The integrate-and-fire frame loop of lm_cif_training (w2v_simul.py:558-606; w2v_asr.py:681-722) as one
        call: -> (cif_repr [B,Kf,d], cif_attn_mask [B,Kf] fp32 0/1, fired positions [B,Kf] int64 with -1 pads),
        Kf = max number of fires (read back to size the outputs, as the reference does with num_fires.max())."""
        cif, mask, idx, counts, mx = ops.cif_aggregate(alphas, semantic_repr, threshold=threshold)
        kf = max(int(mx.item()), 0)
        return cif[:, :kf], mask[:, :kf].to(torch.float32), idx[:, :kf]

    def segment_nuggets(self, full_nugget_scores, target_lengths, frame_lengths, cap=None):
        """Optional fast path of lm_nugget_training's segmenter (w2v_simul.py:419-431) when the frame lengths are
        known as a tensor: quantity loss, resize, apply_threshold_yield_nugget, the score gather and
        add_nugget_type_embedding in one launch and without a device->host sync.  Returns (alphas, quantity_loss,
        resized_alphas, nugget_indices [B,cap] (-1 padded), nugget_mask, counts, max_count, nugget_scores,
        type_ind_table, nugget_index_to_save); cap defaults to T (the reference's width is max_count)."""
        return ops.cif_segment(full_nugget_scores, target_lengths, frame_lengths, cap=cap)

    @staticmethod
    def get_valid_mask_indices(mask: torch.Tensor, padding_value: int = -1):
        """w2v_simul.py:196-220: ascending positions of the True entries, padded; -> (indices, max_valid, n)."""
        assert len(mask.shape) <= 2, f"Only supports 1D or 2D tensors - got {len(mask.shape)}."
        m2 = mask if mask.dim() == 2 else mask.unsqueeze(0)
        # a fire scan over a 0/1 "alpha" fires exactly at the True positions; lengths = T+1 (> T) makes every frame
        # count and switches the forced last-frame fire off (star_cif_fire_scan keeps the length unclamped for that)
        idx, _, counts, mx, _ = ops.cif_fire_scan(m2.to(torch.float32), lengths=torch.full(
            (m2.shape[0],), m2.shape[1] + 1, dtype=torch.int32, device=m2.device))
        max_valid = int(mx.item())
        idx = idx[:, :max_valid]
        if padding_value != -1:
            idx = torch.where(idx < 0, torch.full_like(idx, padding_value), idx)
        if mask.dim() == 1:
            idx = idx[0]
        return idx, max_valid, counts.to(torch.int64) if mask.dim() == 2 else counts.to(torch.int64)[0]

    def apply_threshold_yield_nugget(self, alphas, attn_mask, build_block_mask: bool = True):
        """-> (nugget_mask [B,Kf] bool, nugget_indices [B,Kf] int64 (-1 padded), block_attn_mask [B,T,T] fp32)
        (w2v_simul.py:376-403).  One device->host read of the fire count sizes the outputs (the reference
        does the same through `.item()`).  The [B,T,T] block mask is unused by the live model
        (`use_soft = False`, w2v_simul.py:440-444): pass build_block_mask=False to skip its T*T*B*4 bytes."""
        idx, nmask, counts, mx, _ = ops.cif_fire_scan(alphas, attn_mask=attn_mask)
        kf = int(mx.item())
        block = None
        if build_block_mask:
            block = ops.cif_block_mask(idx, counts, attn_mask=attn_mask)
        return nmask[:, :kf], idx[:, :kf], block


# ------------------------------------------------------------------------------------------ a8
def _additive_bias(attention_mask, scorer_logits, B, K):
    """The additive [B,1,1,K] encoder mask and the scorer logits [B,Kb<=K] as one per-key bias, fp32 [B,<=K] or None."""
    bias = None
    if attention_mask is not None:
        if attention_mask.shape[-1] != K or attention_mask.numel() != B * K:
            raise ValueError(f"attention_mask must broadcast as [B,1,1,K]; got {tuple(attention_mask.shape)}")
        bias = attention_mask.reshape(B, K).to(torch.float32)
    if scorer_logits is not None:
        s = scorer_logits.to(torch.float32)
        if s.shape[1] > K:
            raise ValueError(f"scorer_logits has {s.shape[1]} columns but there are only {K} keys")
        if bias is None:
            bias = s            # prefix-bias variant (my_transformer.py:114-125): the kernel takes bias_len <= K
        else:
            if s.shape[1] < K:
                s = torch.nn.functional.pad(s, (0, K - s.shape[1]))   # the pad mask covers all K keys
            bias = bias + s
    return bias


def _attn_scale(head_dim, scale_attn_weights, scale_attn_by_inverse_layer_idx, layer_idx):
    scale = 1.0
    if scale_attn_weights:
        scale = scale / (head_dim ** 0.5)
    if scale_attn_by_inverse_layer_idx:
        scale = scale / float(layer_idx + 1)
    return scale


def score_biased_cached_attn(query, cache, attention_mask=None, scorer_logits=None, limit_cross_attn=False,
                             scale_attn_weights=True, scale_attn_by_inverse_layer_idx=False, layer_idx=0, query_offset=0):
    """score_biased_attn for generation over an 8-bit cache of the memory's keys and values (ops.KVCache8): the same
    masks and biases on the tokens that the cache holds (its device-side lens; attention_mask and scorer_logits may end
    before or behind them).  query [B,h,L,hd]; returns [B,h,L,hd] in query's dtype.  No dropout, weights or gradient."""
    scale = _attn_scale(query.shape[-1], scale_attn_weights, scale_attn_by_inverse_layer_idx, layer_idx)
    K = cache.capacity if attention_mask is None else attention_mask.shape[-1]
    if scorer_logits is not None and scorer_logits.dim() == 3:
        raise ValueError("score_biased_cached_attn: give the [B,K] scorer logits themselves, not a share_scorer_logits() view")
    bias = _additive_bias(attention_mask, scorer_logits, query.shape[0], K)
    # (like the core, the cached attention computes on 16-bit operands: an fp32 query is rounded on entry)
    out = ops.kv8_attn(query.to(cache.dtype), cache, causal=False, ilk_diag=2 + int(query_offset) if limit_cross_attn else -1,
                       bias=bias, scale=scale)
    return out.to(query.dtype)


def score_biased_attn(query, key, value, attention_mask=None, head_mask=None, scorer_logits=None,
                      limit_cross_attn=False, scale_attn_weights=True, scale_attn_by_inverse_layer_idx=False,
                      layer_idx=0, key_lengths=None, output_attentions=False, dropout_p=0.0, dropout_rng=None,
                      kv_grad=None, query_offset=0):
    """MyGPT2Attention._attn for cross-attention (my_transformer.py:535-603); dropout_p is the probability of
    `self.attn_dropout` (my_transformer.py:595; pass 0 in eval mode), applied inside the kernels.  kv_grad: the
    gradient slot that came with key / value from share_encoder_kv() (optional).  query_offset (not in the reference):
    the target position of the FIRST query row -- a decoding loop that feeds one token at a time passes the token's
    index, so that the infinite-lookback mask of my_transformer.py:566 (key j visible to row i iff j <= i + 2) is
    evaluated at the token's true row instead of row 0.

    query [B,h,L,hd], key/value [B,h,K,hd]; attention_mask is the additive [B,1,1,K] encoder mask produced
    by invert_attention_mask (0 / finfo.min); scorer_logits [B,Kb<=K].  Returns (attn_output, attn_weights or
    None).  The additive mask and the scorer logits are folded into one per-key bias vector, which is what the
    kernel consumes; `key_lengths` (optional, [B]) lets the kernel skip fully padded key tiles."""
    if head_mask is not None:
        # my_transformer.py:598-599: `attn_weights = attn_weights * head_mask` after the dropout.  In the form HF's
        # get_head_mask gives a block ([1, h, 1, 1] or [B, h, 1, 1]: one factor per head) the factor commutes with
        # P.V, so it scales the core's output (and the returned weights) per head; masks that vary over queries or
        # keys would have to enter the kernel and are not built (the reference's own trainers pass None)
        h = query.shape[1]
        if head_mask.dim() != 4 or head_mask.shape[1] not in (1, h) or head_mask.shape[2:] != (1, 1) \
                or head_mask.shape[0] not in (1, query.shape[0]):
            raise NotImplementedError(f"head_mask {tuple(head_mask.shape)}: only per-head factors ([1 or B, 1 or h, 1, 1], "
                                      "what get_head_mask produces) are supported")
        out, probs = score_biased_attn(query, key, value, attention_mask, None, scorer_logits, limit_cross_attn,
                                       scale_attn_weights, scale_attn_by_inverse_layer_idx, layer_idx, key_lengths,
                                       output_attentions, dropout_p, dropout_rng, kv_grad, query_offset)
        out = out * head_mask.to(out.dtype)
        if probs is not None:
            probs = probs * head_mask.to(probs.dtype)
        return out, probs
    scale = _attn_scale(value.size(-1), scale_attn_weights, scale_attn_by_inverse_layer_idx, layer_idx)
    B, K = query.shape[0], key.shape[2]
    if scorer_logits is not None and scorer_logits.dim() == 3:
        # a per-layer view from share_scorer_logits(): the encoder mask is already folded in
        if scorer_logits.shape[2] > K:
            raise ValueError(f"shared scorer_logits cover {scorer_logits.shape[2]} keys but there are {K}")
        return ops.xattn(query, key, value, bias=scorer_logits, key_len=key_lengths,
                         ilk_diag=2 + int(query_offset) if limit_cross_attn else -1, scale=scale, need_probs=output_attentions,
                         dropout_p=dropout_p, dropout_rng=dropout_rng, kv_grad=kv_grad)
    bias = _additive_bias(attention_mask, scorer_logits, B, K)
    out, probs = ops.xattn(query, key, value, bias=bias, key_len=key_lengths,
                           ilk_diag=2 + int(query_offset) if limit_cross_attn else -1, scale=scale, need_probs=output_attentions,
                           dropout_p=dropout_p, dropout_rng=dropout_rng, kv_grad=kv_grad)
    return out, probs


def share_scorer_logits(scorer_logits, n_layers: int, n_heads: int, attention_mask=None, n_keys=None):
    """The reference hands the same scorer_logits [B,Kb] (and the same additive encoder mask [B,1,1,K]) to every
    decoder block (my_transformer.py:917-928), so autograd reduces the bias gradient over heads once per layer and
    then adds the layers up.  Call this once per forward (in MyGPT2Model.forward, before the block loop) and pass
    element i of the result as `scorer_logits` of block i: mask and logits are folded into one bias, every layer
    gets a [B,h,K] broadcast view of it, and the backward sums all layers' per-head partials in one launch.
    Blocks that receive such a view ignore their `encoder_attention_mask` (it is already inside)."""
    s = scorer_logits.to(torch.float32)
    B = s.shape[0]
    K = n_keys if n_keys is not None else (attention_mask.shape[-1] if attention_mask is not None else s.shape[1])
    if s.shape[1] > K:
        raise ValueError(f"scorer_logits has {s.shape[1]} columns but there are only {K} keys")
    if attention_mask is not None:
        if attention_mask.shape[-1] != K or attention_mask.numel() != B * K:
            raise ValueError(f"attention_mask must broadcast as [B,1,1,K]; got {tuple(attention_mask.shape)}")
        if s.shape[1] < K:
            s = torch.nn.functional.pad(s, (0, K - s.shape[1]))
        s = attention_mask.reshape(B, K).to(torch.float32) + s
    return ops.share_bias(s, n_layers, n_heads)


class EncoderKV:
    """One decoder layer's share of share_encoder_kv(): key / value [B,h,K,hd] and the slot its dK / dV go to.  Or, in
    `cache`, an 8-bit cache that holds them (streaming.StreamingEncoderKV with eight_bit=True)."""
    __slots__ = ("key", "value", "grad_slot", "cache")

    def __init__(self, key, value, grad_slot, cache=None):
        self.key, self.value, self.grad_slot, self.cache = key, value, grad_slot, cache


def share_encoder_kv(attn_modules, encoder_hidden_states):
    """K / V of every decoder layer's cross-attention in one projection.

    The reference runs `c_attn(encoder_hidden_states)` inside every block (my_transformer.py:500-501) on the SAME
    encoder memory (my_transformer.py:917-928) -- nl GEMMs with N = 2d each, and again for every generated token
    (my_transformer.py:724-733, 1079-1099).  Call this once per forward, before the block loop, with the blocks'
    cross-attention modules (anything with a Conv1D-layout `c_attn`), and pass element i as `encoder_kv=` of block i's
    NuggetCrossAttention: one [B*K, d] x [d, nl*2d] GEMM forward, two GEMMs backward over all layers, and the
    attention backwards write dK / dV straight into the shared gradient buffer.  Under no_grad the result is the
    K/V cache of all layers: keep it for the whole generation."""
    mods = list(attn_modules)
    if not mods:
        raise ValueError("share_encoder_kv: no attention modules")
    dt = encoder_hidden_states.dtype
    heads = {m.num_heads for m in mods}
    if len(heads) != 1:
        raise ValueError("share_encoder_kv: the layers must have the same number of heads")
    h = heads.pop()
    if encoder_hidden_states.is_cuda and dt == torch.bfloat16 and encoder_hidden_states.dim() == 3:
        # bf16 memory on the GPU: one launch of this library's GEMM (bias in the epilogue) on the transposed weights of
        # all layers, which are rebuilt only when a weight has changed (once per optimizer step in training, never
        # during generation) -- no per-call concatenation
        wt_all, b_all = _kv_weight_cache(mods, dt)
        B, Kn, d = encoder_hidden_states.shape
        kv = ops.shared_conv1d(encoder_hidden_states.reshape(B * Kn, d), wt_all, b_all,
                               [m.c_attn.weight for m in mods], [m.c_attn.bias for m in mods]).view(B, Kn, -1)
        return [EncoderKV(k, v, slot) for k, v, slot in ops.split_kv(kv, len(mods), h)]
    w_all = torch.cat([m.c_attn.weight for m in mods], dim=1).to(dt)
    b_all = torch.cat([m.c_attn.bias for m in mods], dim=0).to(dt)
    return [EncoderKV(k, v, slot) for k, v, slot in ops.share_kv(encoder_hidden_states, w_all, b_all, len(mods), h)]


_KV_WEIGHTS = {}


def _kv_weight_cache(mods, dt):
    """(wt_all [nl*2d, d] bf16 = the layers' c_attn weights transposed, side by side; b_all [nl*2d] fp32), rebuilt when
    any of the parameters has changed (address or version counter)."""
    key = tuple(id(m) for m in mods)
    tag = tuple((m.c_attn.weight.data_ptr(), m.c_attn.weight._version, m.c_attn.bias.data_ptr(), m.c_attn.bias._version)
                for m in mods) + (dt,)
    ent = _KV_WEIGHTS.get(key)
    if ent is None or ent[0] != tag:
        with torch.no_grad():
            # (concatenate the contiguous [in, out] weights, then ONE transposing copy: a cat of transposed views is a
            # strided gather, 45 us against 13 + 12 at nl = 4, d = 1024)
            ws = [m.c_attn.weight.detach() for m in mods]
            w0 = ws[0]
            if (w0.is_cuda and dt == torch.bfloat16 and len(ws) <= ops.TN_MAX_BATCH and w0.shape[0] % 64 == 0
                    and w0.shape[1] % 64 == 0 and w0.dtype in (torch.bfloat16, torch.float32)
                    and all(w.shape == w0.shape and w.dtype == w0.dtype and w.is_contiguous() and w.data_ptr() % 32 == 0
                            for w in ws)):
                wt_all = ops.transpose_cat_bf16(ws)          # one launch (cat + strided copy: 14 + 40 us at nl = 4)
            else:
                wt_all = torch.cat([w.to(dt) for w in ws], dim=1).t().contiguous()
            b_all = torch.cat([m.c_attn.bias.detach() for m in mods], dim=0).to(torch.float32)   # (cat, then ONE cast)
        ent = (tag, wt_all, b_all)
        if len(_KV_WEIGHTS) > 64:
            _KV_WEIGHTS.clear()
        _KV_WEIGHTS[key] = ent
    return ent[1], ent[2]


def clear_kv_weight_cache():
    """Drop the transposed c_attn weights kept by share_encoder_kv() (they are rebuilt at the next call)."""
    _KV_WEIGHTS.clear()


def defer_projection_weight_grads(modules, enable: bool = True):
    """Batch the weight gradients of the small projections (q_attn, c_proj of every NuggetCrossAttention found in
    `modules`, an iterable of modules or one module) into ONE launch at the end of each backward pass
    (ops._DeferredWeightGrads).  A training loop that calls loss.backward() sees the same
    .grad tensors as before, up to the summation order of the fp32 accumulation; torch.autograd.grad() callers and
    gradient hooks on these weights (hook-based DDP) must leave it off -- star_amd.dist reduces .grad after backward
    and works with it."""
    mods = [modules] if isinstance(modules, nn.Module) else list(modules)
    n = 0
    for m in mods:
        for sub in m.modules():
            if isinstance(sub, NuggetCrossAttention):
                sub.q_attn.defer_weight_grad = sub.c_proj.defer_weight_grad = bool(enable)
                n += 1
    return n


class Conv1D(nn.Module):
    """HF GPT-2's Conv1D (transformers 4.34 pytorch_utils.Conv1D): y = x @ weight + bias, weight [in, out]."""

    def __init__(self, nf: int, nx: int):
        super().__init__()
        self.nf = nf
        self.weight = nn.Parameter(torch.empty(nx, nf))
        self.bias = nn.Parameter(torch.zeros(nf))
        nn.init.normal_(self.weight, std=0.02)
        # opt-in (defer_projection_weight_grads): the weight gradient is formed at the end of the backward pass, in one
        # launch with those of the other deferred projections, and written straight to weight.grad
        self.defer_weight_grad = False

    def forward(self, x):
        if x.is_cuda and x.dtype == self.weight.dtype:
            # same arithmetic (hipBLASLt GEMMs through torch); the bias gradient comes from star_colsum
            return ops.conv1d(x, self.weight, self.bias, defer_weight_grad=self.defer_weight_grad)
        size_out = x.size()[:-1] + (self.nf,)
        x = torch.addmm(self.bias, x.view(-1, x.size(-1)), self.weight)
        return x.view(size_out)


class NuggetCrossAttention(nn.Module):
    """Cross-attention branch of MyGPT2Attention.forward (my_transformer.py:490-533) with the fused core.
    Parameters: q_attn, c_attn, c_proj (Conv1D layout) as in GPT2Attention(is_cross_attention=True)."""

    def __init__(self, hidden_size: int, num_heads: int, layer_idx: int = 0, scale_attn_weights: bool = True,
                 scale_attn_by_inverse_layer_idx: bool = False, resid_pdrop: float = 0.0, attn_pdrop: float = 0.0):
        super().__init__()
        # dropout on the attention probabilities (GPT2Config.attn_pdrop, 0.1 in the reference's decoder config,
        # w2v_asr.py:134-145; my_transformer.py:595) runs inside the fused core, in training mode only
        self.attn_pdrop = float(attn_pdrop)
        if not 0.0 <= self.attn_pdrop < 1.0:
            raise ValueError(f"attn_pdrop = {attn_pdrop} not in [0, 1)")
        if hidden_size % num_heads:
            raise ValueError("`embed_dim` must be divisible by num_heads")
        self.embed_dim, self.num_heads, self.head_dim = hidden_size, num_heads, hidden_size // num_heads
        self.split_size = hidden_size
        self.layer_idx = layer_idx
        self.scale_attn_weights = scale_attn_weights
        self.scale_attn_by_inverse_layer_idx = scale_attn_by_inverse_layer_idx
        self.is_cross_attention = True
        self.c_attn = Conv1D(2 * hidden_size, hidden_size)
        self.q_attn = Conv1D(hidden_size, hidden_size)
        self.c_proj = Conv1D(hidden_size, hidden_size)
        self.resid_dropout = nn.Dropout(resid_pdrop)
        self._kv_cache = None        # (tag, key, value) of the last encoder memory seen under no_grad / eval

    def clear_kv_cache(self):
        self._kv_cache = None

    def _encoder_kv(self, encoder_hidden_states):
        """K/V of the encoder memory.  During generation the reference recomputes c_attn(encoder_hidden_states) for
        every decoded token (my_transformer.py:724-733,1079-1099) although the memory does not change; here, in eval
        mode under no_grad, the projected heads are kept while the memory tensor and the projection weights are the
        very same objects at the same version."""
        cacheable = (not self.training) and (not torch.is_grad_enabled())
        tag = None
        if cacheable:
            e, w, bb = encoder_hidden_states, self.c_attn.weight, self.c_attn.bias
            tag = (e.data_ptr(), tuple(e.shape), e.dtype, e._version, w.data_ptr(), w._version, bb.data_ptr(), bb._version)
            if self._kv_cache is not None and self._kv_cache[0] == tag:
                return self._kv_cache[1], self._kv_cache[2]
        key, value = self.c_attn(encoder_hidden_states).split(self.split_size, dim=2)
        key, value = self._split_heads(key), self._split_heads(value)
        # the memory tensor itself is kept alive with the entry, so its address cannot be handed to another tensor
        self._kv_cache = (tag, key, value, encoder_hidden_states) if cacheable else None
        return key, value

    def _encoder_kv_train(self, encoder_hidden_states):
        """Grad-enabled form of the same projection: split + split_heads through ops.split_kv, so that the attention
        backward writes dK / dV into the two halves of ONE [B,K,2d] gradient (what c_attn's backward consumes)
        instead of two gapped tensors that autograd then concatenates."""
        self._kv_cache = None                           # grad-enabled calls never cache
        return ops.split_kv(self.c_attn(encoder_hidden_states), 1, self.num_heads)[0]

    def _split_heads(self, t):
        return t.view(t.shape[0], t.shape[1], self.num_heads, self.head_dim).permute(0, 2, 1, 3)

    def _attn(self, query, key, value, attention_mask=None, head_mask=None, scorer_logits=None,
              limit_cross_attn=False, output_attentions=False, kv_grad=None, query_offset=0):
        return score_biased_attn(query, key, value, attention_mask, head_mask, scorer_logits, limit_cross_attn,
                                 self.scale_attn_weights, self.scale_attn_by_inverse_layer_idx, self.layer_idx,
                                 output_attentions=output_attentions,
                                 dropout_p=self.attn_pdrop if self.training else 0.0, kv_grad=kv_grad,
                                 query_offset=query_offset)

    def forward(self, hidden_states, layer_past=None, attention_mask=None, head_mask=None,
                encoder_hidden_states=None, encoder_attention_mask=None, use_cache=False, output_attentions=False,
                scorer_logits=None, limit_cross_attn=False, encoder_kv=None, query_offset=0):
        """encoder_kv (not in the reference): this layer's element of share_encoder_kv() (or of a
        streaming.StreamingEncoderKV); encoder_hidden_states is then not projected again.  query_offset (not in the
        reference): target position of the first row of hidden_states, for token-by-token decoding under
        limit_cross_attn (score_biased_attn)."""
        if encoder_hidden_states is None and encoder_kv is None:
            raise ValueError("NuggetCrossAttention is the cross-attention module: encoder_hidden_states is required")
        query = self._split_heads(self.q_attn(hidden_states))
        kv_grad = None
        if encoder_kv is not None and encoder_kv.cache is not None:
            if head_mask is not None or output_attentions or use_cache or layer_past is not None:
                raise ValueError("an 8-bit encoder_kv takes no head_mask, output_attentions, use_cache or layer_past")
            if self.training and self.attn_pdrop > 0.0:
                raise ValueError("an 8-bit encoder_kv is for generation: attention dropout does not run on it")
            out = score_biased_cached_attn(query, encoder_kv.cache, encoder_attention_mask, scorer_logits,
                                           bool(limit_cross_attn), self.scale_attn_weights,
                                           self.scale_attn_by_inverse_layer_idx, self.layer_idx, query_offset)
            return self.resid_dropout(self.c_proj(out.permute(0, 2, 1, 3).flatten(2))), None
        if encoder_kv is not None:
            key, value = encoder_kv.key, encoder_kv.value
            kv_grad = encoder_kv.grad_slot if layer_past is None else None
        elif torch.is_grad_enabled() and encoder_hidden_states.dim() == 3 and layer_past is None:
            key, value, kv_grad = self._encoder_kv_train(encoder_hidden_states)
        else:
            key, value = self._encoder_kv(encoder_hidden_states)
        if layer_past is not None:
            past_key, past_value = layer_past
            key = torch.cat((past_key, key), dim=-2)
            value = torch.cat((past_value, value), dim=-2)
        present = (key, value) if use_cache else None
        attn_output, attn_weights = self._attn(query, key, value, encoder_attention_mask, head_mask, scorer_logits,
                                               limit_cross_attn=bool(limit_cross_attn),
                                               output_attentions=output_attentions, kv_grad=kv_grad,
                                               query_offset=query_offset)
        # merge heads: the kernel already wrote [B, L, h, hd] memory order
        b, h, l, hd = attn_output.shape
        attn_output = attn_output.permute(0, 2, 1, 3).reshape(b, l, h * hd)
        attn_output = self.resid_dropout(self.c_proj(attn_output))
        outputs = (attn_output, present)
        if output_attentions:
            outputs += (attn_weights,)
        return outputs


class NuggetSelfAttention(nn.Module):
    """Self-attention branch of MyGPT2Attention.forward (my_transformer.py:490-533), causal: the attention of the
    semantic encoder over the frames and of the decoder over its own tokens.  Parameters c_attn and c_proj (Conv1D
    layout) as in GPT2Attention; kv_heads < num_heads (not in the reference) shares every key head between
    num_heads // kv_heads query heads, c_attn is then [hidden, (num_heads + 2 kv_heads) * head_dim].

    The core runs on 16-bit operands with fp32 softmax and sums, as NuggetCrossAttention's does: fp32 activations are
    rounded to bfloat16 for it.  The softmax is never padded, so no additive attention_mask is taken: give the lengths.
    The plan of an unpadded or padded batch is made at its first call: make that before a HIP-graph capture (a new shape is
    refused in one).  Plans of unpadded batches are kept for the last 32 shapes, and as long as the module for a shape that
    was captured, since a graph reads its plan at every replay.

        attn(x)                                  x [B,T,d], every row T frames
        attn(x, valid=frames)                    x [B,T,d] padded, frames an ops.ValidFrames; pad rows see nothing
        attn(x, plan=plan)                       x [rows,d] packed, plan an ops.PackedSeqs
        attn(x, plan=plan, cache=cache)          the same prompt, whose keys and values also go into an ops.KVCache8
        attn(x, valid=frames, cache=cache)       the same, padded; pad rows do not go into the cache
        attn(x, cache=cache, counts=n)           x [B,L,d]: the next (at most L) tokens of every sequence of the cache

    A prompt attends to itself alone: the cache must hold nothing yet of the sequences that it has rows for (those of length 0
    keep what they have).  What follows on held tokens, a prompt's next part too, goes in by the last form."""

    def __init__(self, hidden_size: int, num_heads: int, layer_idx: int = 0, scale_attn_weights: bool = True,
                 scale_attn_by_inverse_layer_idx: bool = False, resid_pdrop: float = 0.0, attn_pdrop: float = 0.0,
                 kv_heads: Optional[int] = None):
        super().__init__()
        if hidden_size % num_heads:
            raise ValueError("`embed_dim` must be divisible by num_heads")
        self.embed_dim, self.num_heads, self.head_dim = hidden_size, num_heads, hidden_size // num_heads
        self.kv_heads = num_heads if kv_heads is None else int(kv_heads)
        if self.kv_heads < 1 or num_heads % self.kv_heads:
            raise ValueError(f"{num_heads} query heads do not divide into {kv_heads} key heads")
        if attn_pdrop:
            raise NotImplementedError("NuggetSelfAttention: attention-probability dropout is not built (attn_pdrop must be 0)")
        self.layer_idx = layer_idx
        self.scale = _attn_scale(self.head_dim, scale_attn_weights, scale_attn_by_inverse_layer_idx, layer_idx)
        self.c_attn = Conv1D((num_heads + 2 * self.kv_heads) * self.head_dim, hidden_size)
        self.c_proj = Conv1D(hidden_size, hidden_size)
        self.resid_dropout = nn.Dropout(resid_pdrop)
        self._plans, self._captured = {}, {}     # (B, T, device) -> (plan, streams it was used on): unpadded batches

    def __getstate__(self):
        return {**self.__dict__, "_plans": {}, "_captured": {}}     # (a copied or saved module makes its plans itself)

    _PLANS, _LOCK = 32, threading.Lock()

    def _plan_of(self, B, T, device):
        """The plan of B sequences of T frames.  One that is dropped from _plans may still be read by work on any stream it was
        used on, which is recorded for the allocator; one that a capture has seen is never dropped."""
        key = (B, T, device)
        kept, capture = self._captured.get(key) or self._plans.get(key), ops.capturing(device)
        if kept is None:
            if capture:
                raise StarNuggetError(f"NuggetSelfAttention: call it once with [{B},{T},{self.embed_dim}] before a HIP-graph "
                                      "capture (the plan of a new shape is copied to the device)")
            kept = ops.PackedSeqs([T] * B, device), set()
            with self._LOCK:
                while len(self._plans) >= self._PLANS:
                    self._plans.pop(next(iter(self._plans)))
                self._plans[key] = kept
        plan, streams = kept
        if capture:
            self._captured[key] = kept
        elif plan.device.type == "cuda":
            raw = ops._raw_stream(plan.device.index)
            if raw not in streams:
                plan.record_stream(torch.cuda.current_stream(plan.device))
                streams.add(raw)
        return plan

    def new_cache(self, batch: int, max_tokens: int, device=None, dtype=torch.bfloat16):
        """An empty 8-bit cache for this layer."""
        return ops.KVCache8(batch, self.kv_heads, max_tokens, self.head_dim, device or self.c_attn.weight.device, dtype)

    def forward(self, hidden_states, plan=None, valid=None, cache=None, counts=None):
        if cache is not None and plan is None and valid is None:
            return self._next_tokens(hidden_states, cache, counts)
        if counts is not None:
            raise ValueError("NuggetSelfAttention: counts go with the next tokens of a cache")
        if plan is None:
            if hidden_states.dim() != 3:
                raise ValueError(f"NuggetSelfAttention: [B,T,{self.embed_dim}] or a plan expected, got {tuple(hidden_states.shape)}")
            B, T, _ = hidden_states.shape
            if valid is not None:
                if not valid.matches(hidden_states):
                    raise ValueError(f"NuggetSelfAttention: valid is for [{valid.B},{valid.T},d], got {tuple(hidden_states.shape)}")
                plan = valid.seqs()
            else:
                plan = self._plan_of(B, T, hidden_states.device)
        elif valid is not None:
            raise ValueError("NuggetSelfAttention: give plan or valid, not both")
        qkv = self.c_attn(hidden_states).reshape(-1, self.c_attn.nf)
        core = qkv.to(torch.bfloat16) if qkv.dtype == torch.float32 else qkv
        out = ops.causal_attn_qkv(core, self.num_heads, self.kv_heads, plan, scale=self.scale)
        if cache is not None:
            _, k, v = ops._qkv_views(core.detach().to(cache.dtype), self.num_heads, self.kv_heads, self.head_dim)
            ops.kv8_append(cache, k, v, plan=plan)
        out = out.flatten(1).to(qkv.dtype).view(hidden_states.shape)
        return self.resid_dropout(self.c_proj(out))

    def _next_tokens(self, hidden_states, cache, counts):
        if torch.is_grad_enabled():
            raise ValueError("NuggetSelfAttention: nothing is differentiated through a cache; call it under torch.no_grad()")
        if hidden_states.dim() != 3:
            raise ValueError(f"NuggetSelfAttention: [B,L,{self.embed_dim}] expected with a cache, got {tuple(hidden_states.shape)}")
        B, L, _ = hidden_states.shape
        if B * self.num_heads * L >= ops.KV8_MOST_ROWS:            # (refused before anything is appended)
            raise ValueError(f"NuggetSelfAttention: {B} sequences x {self.num_heads} heads x {L} tokens at once; give them in parts")
        qkv = self.c_attn(hidden_states)
        core = qkv.to(cache.dtype).unflatten(2, (-1, self.head_dim)).transpose(1, 2)       # [B, heads, L, hd]
        q, k, v = core.split([self.num_heads, self.kv_heads, self.kv_heads], dim=1)
        ops.kv8_append(cache, k, v, counts=counts)
        out = ops.kv8_attn(q, cache, q_len=counts, scale=self.scale)
        return self.resid_dropout(self.c_proj(out.transpose(1, 2).flatten(2).to(qkv.dtype)))
