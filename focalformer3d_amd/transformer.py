"""Box-level deformable transformer decoder on MI355X.

Host-side mirror of the third-party classes the reference builds from config type strings
(FocalFormer3D_L.py:285-313 -> focal_decoder.py:16,304):

    DeformableDetrTransformerDecoder   (mmdet 2.14.0  mmdet/models/utils/transformer.py)
    DetrTransformerDecoderLayer        (mmcv 1.3.18   mmcv/cnn/bricks/transformer.py BaseTransformerLayer)
    MultiheadAttention, FFN            (mmcv 1.3.18   mmcv/cnn/bricks/transformer.py)
    MultiScaleDeformableAttention      (mmcv 1.3.18   mmcv/ops/multi_scale_deform_attn.py)

Same constructor arguments, same ``forward`` signatures, same parameter names (state-dict layout of
SURVEY.md Appendix B), so the reference's ``decoder_cfg`` dict and checkpoints load unchanged.  Their
source is not part of /root/reference; behaviour follows the published algorithm.

MI355X design: the inference path (eval semantics: dropout is the identity) runs batch-first on
contiguous (B, N, C) activations so every projection is one hipBLASLt GEMM on MFMA, the deformable
gather is the hand-written ``ff3d_msda_fused_fwd`` kernel (softmax + sampling-location prologue fused, LDS
staged), and the two small projections that share an input (sampling offsets + attention logits) are one
GEMM.  The ``forward`` methods keep the mmcv (num_query, bs, C) calling convention; the ``forward_bf``
methods are the batch-first fast path the head drives directly.

Training mode (``module.train()``) takes a separate, differentiable route through the same parameters:
the projections / LayerNorms / dropouts are the framework's autograd ops (plain library GEMMs), self-attention is
``nn.MultiheadAttention`` itself (attention masks of the ground-truth query groups, FD:849-858), and the deformable gather is
``autograd.MultiScaleDeformableAttnFunction`` = ``ff3d_msda_fwd`` / ``ff3d_msda_bwd``.
"""
import copy
import os
import warnings

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .layers import weight_signature
from .registry import (ATTENTION, FEEDFORWARD_NETWORK, TRANSFORMER_LAYER, TRANSFORMER_LAYER_SEQUENCE,
                       build_attention, build_feedforward_network, build_transformer_layer, register)


# Row count below which the decoder's projections go to the vendor GEMM.  0 since round 6 (third session): the own kernels serve every
# row count in eager steps too - as captured / overlapping replays always did (runtime.PipelinedHead).  Rounds 3-5 kept eager steps of
# fewer than 1 536 rows on hipBLASLt because one launch is level there (9.4 us for the small-M form of the own kernel against 8.7 at
# 600 rows, profiles/r03_m_bench_b1_kernel_stats_last_step.txt) - but an eager one-frame step is bound by the HOST's launch rate, and the
# own route's fused steps (projection + add + LayerNorm, q | k | v, the one-launch feed-forward) are 90 launches against 142:
# 2.28 - 2.34 ms against 3.28 - 3.42 ms per one-frame eager step, level at four frames (profiles/r06_mr0_eager_small_batch.txt; whole GPU
# suite green with either setting).  No eval-mode projection with K % 32 == 0 reaches a vendor GEMM any more; FF3D_LIN_MIN_ROWS=1536
# restores the old dispatch.
LIN_F16X3_MIN_ROWS = int(os.environ.get('FF3D_LIN_MIN_ROWS', '0'))
_NORMALIZERS = {}                    # (level shapes, dtype, device) -> (L, 2) offset normaliser of the training route


def _cached(m, name, weight, bias, make):
    """Per-module cache of a weight-derived operand (bf16 copies, split-fp16 planes), keyed on the parameter versions."""
    cache = m.__dict__.setdefault(name, {})
    key = weight_signature((weight,) if bias is None else (weight, bias)) + (tuple(weight.shape), weight.storage_offset())
    if key not in cache:
        if len(cache) > 16:                                 # stale versions of updated weights
            cache.clear()
        cache[key] = make()
    return cache[key]


def _own_linear(m, x, weight):
    """Does this projection of module ``m`` run on the own split-fp16 kernel (csrc/linear.hip)?"""
    use = getattr(m, 'lin_f16x3', None)
    if use is None:
        use = ops.ATTN_F16X3
    return bool(use and x.is_cuda and weight.shape[1] % 32 == 0 and not torch.is_grad_enabled()
                and x.numel() // x.shape[-1] >= LIN_F16X3_MIN_ROWS)


def _split_w(m, weight, bias):
    return _cached(m, '_f16_w', weight, bias, lambda: ops.split_weight_f16(weight.detach(), bias=bias))


def _lin32(m, x, weight, bias, relu=False):
    """fp32-class dense projection of module ``m``: the row-scaled split-fp16 MFMA kernel (ops.linear_f16x3; dense mode
    'f16x3', the default) or the vendor fp32 GEMM (``m.lin_f16x3 = False`` / FF3D_DENSE_MODE=vendor)."""
    if _own_linear(m, x, weight):
        return ops.linear_f16x3(x, _split_w(m, weight, bias), None if bias is None else bias.detach(), relu)
    ops.note_vendor('fp32 linear', x.numel() // x.shape[-1], weight.shape[0], weight.shape[1])
    return ops.linear_relu(x, weight, bias) if relu else F.linear(x, weight, bias)


# one launch for [projection + identity add + LayerNorm (+ query_pos)] of a post-norm decoder-layer step (FF3D_LIN_LN=0: the
# projection and ops.add_layer_norm as two launches).  Only while the small-M kernel serves it (<= 4 096 rows = 6 frames): a block
# of the fused form owns whole 256-column rows and streams all of W, which at 19 200 rows costs 68 us against 34 + 20 for the
# 128-column tiles + the LayerNorm kernel (profiles/r03_n_bench_b32_kernel_stats_last_step.txt); at 600 - 2 400 rows the two
# forms are level (profiles/r03_m_small_batch_ab.txt) and the fused one saves 18 launches per step.
LIN_LN_FUSED = os.environ.get('FF3D_LIN_LN', '1') != '0'
LIN_LN_MAX_ROWS = int(os.environ.get('FF3D_LIN_LN_MAX_ROWS', '4096'))
# Round 6 (third session): the fused step with a LONG K at few rows (fc2 of the feed-forward step: K = 1024) as K slices - a plain
# projection whose column blocks are the 256-wide K slices (4 x the blocks, each streaming a quarter of the weight) + the slice-order sum
# inside the LayerNorm launch: 11.5 / 13.7 / 20.2 us against 23.4 / 23.7 / 24.4 us at 600 / 1 200 / 2 400 rows; routed up to 2 560 rows
# (four frames: the pipelined 4-frame step 3.302 vs 3.330 ms, three alternations; profiles/r06_ksl_*).  FF3D_LIN_LN_KSLICES=0: off.
LIN_LN_KSLICES = os.environ.get('FF3D_LIN_LN_KSLICES', '1') != '0'
LIN_LN_KSLICES_MAX_ROWS = int(os.environ.get('FF3D_LIN_LN_KSLICES_MAX_ROWS', '2560'))
# q | k | v of the self-attention in one launch (FF3D_QKV_FUSED=0: two)
QKV_FUSED = os.environ.get('FF3D_QKV_FUSED', '1') != '0'


# Round 5: beyond LIN_LN_MAX_ROWS the fused step runs on the ROW-OWNING kernel (ops.linear_rows, csrc/linrows.hip: a block owns
# 16 * MT rows x 256 columns, the grid is one round of the chip - 19 200 rows = 240 blocks), which also serves every projection
# of the bf16 mode.  FF3D_LIN_ROWS: 'ln' (default) = the fused LayerNorm steps; 'all' = also the plain N % 256 == 0 projections
# of the fp32-class mode; '0' = never (rounds 3-4: linear.hip's 64 x 128 tiles + the add + LayerNorm kernel).
LIN_ROWS = os.environ.get('FF3D_LIN_ROWS', 'ln')


# Round 5: the feed-forward step [fc1 + ReLU + fc2 + identity + LayerNorm (+ query_pos)] as one launch from FFN_FUSED_MIN_ROWS rows
# (ops.ffn_rows; below that its 80-row blocks do not fill the chip and the two small-M launches are ahead).  FF3D_FFN_FUSED=0: two
# launches (rounds 3-5: linear.hip + linrows.hip).
FFN_FUSED = os.environ.get('FF3D_FFN_FUSED', '1') != '0'
FFN_FUSED_MIN_ROWS = int(os.environ.get('FF3D_FFN_FUSED_MIN_ROWS', '8192'))


def _bf16_w(m, weight, bias):
    return _cached(m, '_bf16_rows_w', weight, bias, lambda: ops.bf16_weight(weight.detach(), None if bias is None else bias.detach()))


def _own_bf16(m, x, weight):
    """bf16 mode: does this projection run on the own bf16 MFMA kernel (csrc/linrows.hip, one-plane instance)?"""
    return bool(getattr(m, 'gemm_dtype', torch.float32) == torch.bfloat16 and getattr(m, 'lin_f16x3', ops.ATTN_F16X3)
                and x.is_cuda and x.dtype == torch.float32 and weight.shape[1] % 32 == 0 and not torch.is_grad_enabled())


def _lin_add_ln(m, o, weight, bias, residual, norm, pos=None):
    """LayerNorm(residual + o @ weight^T + bias) (+ pos as a second result when given)."""
    fusable = (LIN_LN_FUSED and weight.shape[0] == 256 and residual.is_contiguous() and (pos is None or pos.is_contiguous())
               and o.stride(-1) == 1)
    if fusable and _own_bf16(m, o, weight):
        return ops.linear_rows(o, _bf16_w(m, weight, bias), residual=residual, gamma=norm.weight, beta=norm.bias, eps=norm.eps, pos=pos)
    if fusable and getattr(m, 'gemm_dtype', torch.float32) == torch.float32 and _own_linear(m, o, weight):
        rows, K = o.numel() // o.shape[-1], weight.shape[1]
        if LIN_LN_KSLICES and K >= 1024 and K % 256 == 0 and K // 256 <= 16 and rows <= LIN_LN_KSLICES_MAX_ROWS:
            # long K, few rows (fc2 of the feed-forward step at 1 - 4 frames): K slices of 256 as extra column blocks + the slice-order sum
            # inside the LayerNorm launch (ops.linear_kslices_f16x3): each row-owning block of the fused form streams the whole weight
            ks = K // 256
            wk = _cached(m, '_f16_wk', weight, None, lambda: ops.kslice_weight(weight, ks))
            parts = ops.linear_kslices_f16x3(o, wk, ks, 256)
            return ops.sum_add_layer_norm(parts, ks, None if bias is None else bias.detach(), residual, norm.weight, norm.bias, norm.eps, pos)
        if o.numel() // o.shape[-1] <= LIN_LN_MAX_ROWS:
            return ops.linear_add_ln_f16x3(o, _split_w(m, weight, bias), None if bias is None else bias.detach(), residual,
                                           norm.weight, norm.bias, norm.eps, pos)
        if LIN_ROWS != '0':
            return ops.linear_rows(o, _split_w(m, weight, bias), None if bias is None else bias.detach(), residual=residual,
                                   gamma=norm.weight, beta=norm.bias, eps=norm.eps, pos=pos)
    return ops.add_layer_norm(residual, _lin(m, o, weight, bias), norm.weight, norm.bias, norm.eps, pos)


def _lin(m, x, weight, bias, relu=False):
    """Dense projection of module ``m``: fp32-class (parity path, _lin32) or bf16 operands on MFMA when the owning head was
    switched with ``set_gemm_dtype('bf16')`` ('bf16 QKV/FFN on MFMA'); fp32 result."""
    if getattr(m, 'gemm_dtype', torch.float32) == torch.bfloat16:
        if _own_bf16(m, x, weight) and x.stride(-1) == 1:
            # round 5: own one-plane bf16 MFMA kernel - fp32 rows in (rounded while staged), fp32 rows out (holding bf16 values): no
            # cast launch on either side, no vendor GEMM (rounds 1-4: F.linear on hipBLASLt between two casts)
            return ops.linear_rows(x, _bf16_w(m, weight, bias), relu=relu)
        ops.note_vendor('bf16 linear', x.numel() // x.shape[-1], weight.shape[0], weight.shape[1])
        w16, b16 = _cached(m, '_bf16_w', weight, bias,
                           lambda: (weight.detach().to(torch.bfloat16), None if bias is None else bias.detach().to(torch.bfloat16)))
        y = F.linear(x.to(torch.bfloat16), w16, b16)
        return (F.relu_(y) if relu else y).float()
    if (LIN_ROWS == 'all' and weight.shape[0] % 256 == 0 and x.stride(-1) == 1 and _own_linear(m, x, weight)
            and x.numel() // x.shape[-1] > LIN_LN_MAX_ROWS):
        return ops.linear_rows(x, _split_w(m, weight, bias), None if bias is None else bias.detach(), relu)
    return _lin32(m, x, weight, bias, relu)


class DeviceLevels:
    """mmcv's level tables as it passes them: ``spatial_shapes`` (L,2) / ``level_start_index`` (L) int64 DEVICE tensors
    (FD:837-841).  Kept on the device end to end (ff3d_msda_fwd_dev): reading them on the host would synchronise and break
    graph capture of the drop-in route."""

    def __init__(self, spatial_shapes, level_start_index=None):
        self.spatial_shapes = spatial_shapes.contiguous()
        if level_start_index is None:
            hw = spatial_shapes[:, 0] * spatial_shapes[:, 1]
            level_start_index = torch.cat([hw.new_zeros(1), hw.cumsum(0)[:-1]])
        self.level_start_index = level_start_index.contiguous()


def _level_hw(spatial_shapes, level_start_index=None):
    if isinstance(spatial_shapes, torch.Tensor):
        if spatial_shapes.is_cuda:                        # mmcv passes a (L,2) int64 device tensor (FD:840)
            return DeviceLevels(spatial_shapes, level_start_index)
        return [tuple(int(v) for v in r) for r in spatial_shapes.tolist()]
    return [tuple(int(v) for v in r) for r in spatial_shapes]


class PosTable:
    """Value mode 'gather_first' with the positional part split off (FocalDecoder): ``value_cl`` is the UN-embedded pyramid (shared by
    the decoder stages and by the RoI sampler), and ``table`` (1, Nv, heads, Dh) = value_proj(bev_pos_embed) + bias of ONE layer - weights
    and grid only, the same for every frame.  sum_k w_k (W (raw_k + pos_k) + b) = W (sum_k w_k raw_k) + sum_k w_k (W pos_k + b): the
    second sum is the ordinary gather of head slices over the table (every frame's queries as one frame's), zero outside the map."""

    def __init__(self, table):
        self.table = table


def _per_level_ref(reference_points, num_levels):
    """(B, Nq, 2) stays; (B, Nq, 1, 2) -> (B, Nq, 2) (one point for every level); (B, Nq, L, 2) stays per level."""
    if reference_points.dim() == 4 and reference_points.shape[2] == 1:
        return reference_points[:, :, 0]
    if reference_points.dim() == 4 and num_levels is not None and reference_points.shape[2] != num_levels:
        raise ValueError(f'reference_points carry {reference_points.shape[2]} levels, the attention has {num_levels}')
    return reference_points


def _frame_mask(attn_mask, B, heads, N):
    """An attention mask as nn.MultiheadAttention takes it - (N, N), (B, N, N) or (B*heads, N, N), True / negative = blocked - as one
    (B, N, N) boolean mask per frame, or None."""
    if attn_mask is None:
        return None
    if attn_mask.dtype != torch.bool:
        attn_mask = attn_mask < 0                           # additive float form: -inf = blocked
    if attn_mask.dim() == 2:
        return attn_mask[None].expand(B, -1, -1)
    if attn_mask.shape[0] == B and heads > 1:               # one mask per frame (what train_forward.py passes): used as it is
        return attn_mask
    m4 = attn_mask.reshape(B, heads, N, N)                  # (B*heads, N, N): FD:856 repeats one mask per frame over the heads
    # a per-head mask is not supported by the kernel.  The check costs a B*heads*N*N compare and a host sync, so
    # it runs once per mask tensor (the six layers of a step share one), not once per layer; a mask that is a
    # broadcast view over the heads (stride 0) needs no check at all
    # (the verdict rides on the tensor OBJECT together with the version it was reached at - a (data_ptr, _version)
    #  key in a module global could be matched by a NEW mask the allocator placed at the same address)
    if heads > 1 and m4.stride(1) != 0 and getattr(attn_mask, '_ff3d_head_uniform', None) != attn_mask._version:
        if not bool((m4 == m4[:, :1]).all()):
            raise NotImplementedError('per-head attention masks (FocalFormer3D builds one mask per frame)')
        attn_mask._ff3d_head_uniform = attn_mask._version
    return m4[:, 0]


@register(ATTENTION)
class MultiheadAttention(nn.Module):
    """mmcv ``MultiheadAttention``: wraps ``nn.MultiheadAttention`` (parameters under ``.attn``), adds the
    positional encodings to query/key (not to value) and the residual."""

    def __init__(self, embed_dims, num_heads, attn_drop=0., proj_drop=0.,
                 dropout_layer=dict(type='Dropout', drop_prob=0.), init_cfg=None, batch_first=False, **kwargs):
        super().__init__()
        dropout_layer = dict(dropout_layer) if dropout_layer else None
        if 'dropout' in kwargs:                            # deprecated spelling used by the reference configs: both the
            attn_drop = kwargs.pop('dropout')              # attention dropout and the output dropout (Appendix A.2)
            dropout_layer = dict(type='Dropout', drop_prob=attn_drop)
        self.embed_dims, self.num_heads, self.batch_first = embed_dims, num_heads, batch_first
        self.attn = nn.MultiheadAttention(embed_dims, num_heads, attn_drop)
        self.proj_drop = nn.Dropout(proj_drop)
        if dropout_layer and dropout_layer.get('type', 'Dropout') != 'Dropout':
            raise NotImplementedError("dropout_layer: only type='Dropout' (DropPath is not used by the FocalFormer3D configs)")
        self.dropout_layer = nn.Dropout(dropout_layer.get('drop_prob', 0.)) if dropout_layer else nn.Identity()

    def invalidate_cache(self):
        self.__dict__.pop('_bf16_w', None)
        self.__dict__.pop('_bf16_rows_w', None)
        self.__dict__.pop('_f16_w', None)

    def core_bf(self, x, xp, attn_mask=None):
        """attn(q = k = xp, v = x) before the output projection; x, xp = x + pos: (B, N, C)."""
        B, N, C = x.shape
        w, b = self.attn.in_proj_weight, self.attn.in_proj_bias
        if attn_mask is not None:
            raise NotImplementedError('attention masks only occur on the training path (FD:849-858): module.train()')
        f16x3 = getattr(self, 'attn_f16x3', None)
        if (QKV_FUSED and (2 * C) % 128 == 0 and getattr(self, 'gemm_dtype', torch.float32) == torch.float32
                and _own_linear(self, xp, w) and x.is_contiguous() and xp.is_contiguous()):
            qkv = ops.linear_f16x3(xp, _split_w(self, w, b), None if b is None else b.detach(), x2=x, n_split=2 * C)
            return ops.self_attention(qkv[:, :, :C], qkv[:, :, C:2 * C], qkv[:, :, 2 * C:], self.num_heads, f16x3=f16x3)
        if ((2 * C) % 256 == 0 and _own_bf16(self, xp, w) and x.is_contiguous() and xp.is_contiguous()):
            qkv = ops.linear_rows(xp, _bf16_w(self, w, b), x2=x, n_split=2 * C)         # bf16 mode: q | k | v in one launch
            return ops.self_attention(qkv[:, :, :C], qkv[:, :, C:2 * C], qkv[:, :, 2 * C:], self.num_heads, f16x3=f16x3)
        qk = _lin(self, xp, w[:2 * C], b[:2 * C])                  # (B, N, 2C): q | k column blocks
        v = _lin(self, x, w[2 * C:], b[2 * C:])
        return ops.self_attention(qk[:, :, :C], qk[:, :, C:], v, self.num_heads, f16x3=f16x3)   # fused flash kernel (split-fp16 | fp32 MFMA)

    def delta_bf(self, x, xp, attn_mask=None):
        """out_proj(attn(q = k = xp, v = x)) without the residual; x, xp = x + pos: (B, N, C)."""
        return _lin(self, self.core_bf(x, xp, attn_mask), self.attn.out_proj.weight, self.attn.out_proj.bias)

    def forward_train_bf(self, x, pos=None, attn_mask=None):
        """Appendix A.2, differentiable: identity + dropout_layer(proj_drop(nn.MultiheadAttention(q = k = x + pos, v = x))).
        attn_mask: (N, N), (B, N, N) or (B*heads, N, N), True / -inf = blocked (FD:851-856).  The in / out projections are the framework's
        linear ops on ``self.attn``'s parameters; the masked, dropout-carrying scaled-dot-product core is
        ``MaskedSelfAttentionFunction`` (ff3d_mha_train_fwd / _bwd) - round 2 sent it to torch's fused SDPA (AOTriton) kernels,
        which ``train_sdpa = 'torch'`` / FF3D_TRAIN_SDPA=torch (or 'math') still selects."""
        mode = getattr(self, 'train_sdpa', os.environ.get('FF3D_TRAIN_SDPA', 'hip'))
        B, N, C = x.shape
        heads, a = self.num_heads, self.attn
        if mode == 'hip' and x.is_cuda and C // heads in (4, 8, 16, 32, 64) and a.in_proj_weight is not None:
            from .autograd import MaskedSelfAttentionFunction
            xp = x if pos is None else x + pos
            w, b = a.in_proj_weight, a.in_proj_bias
            qk = F.linear(xp, w[:2 * C], None if b is None else b[:2 * C])
            v = F.linear(x, w[2 * C:], None if b is None else b[2 * C:])
            mask = _frame_mask(attn_mask, B, heads, N)
            p_drop = a.dropout if a.training else 0.0           # (nn.MultiheadAttention's own flag, as its forward uses it)
            o = MaskedSelfAttentionFunction.apply(qk[..., :C], qk[..., C:], v, heads, mask, p_drop)
            out = F.linear(o, a.out_proj.weight, a.out_proj.bias)
            return x + self.dropout_layer(self.proj_drop(out))
        qk = (x if pos is None else x + pos).transpose(0, 1)
        if attn_mask is not None and attn_mask.dim() == 3 and attn_mask.shape[0] == B and heads > 1:
            attn_mask = attn_mask[:, None].expand(-1, heads, -1, -1).flatten(0, 1)          # nn.MultiheadAttention: (B*heads, N, N)
        if mode == 'math' and x.is_cuda:
            from torch.nn.attention import SDPBackend, sdpa_kernel
            with sdpa_kernel(SDPBackend.MATH):
                out = self.attn(qk, qk, x.transpose(0, 1), attn_mask=attn_mask, need_weights=False)[0]
        else:
            out = self.attn(qk, qk, x.transpose(0, 1), attn_mask=attn_mask, need_weights=False)[0]
        return x + self.dropout_layer(self.proj_drop(out.transpose(0, 1)))

    def forward_bf(self, x, pos=None, attn_mask=None):
        """Self-attention, batch-first: x, pos (B, N, C) -> (B, N, C) = x + out_proj(attn(x+pos, x+pos, x))."""
        if self.training:
            return self.forward_train_bf(x, pos, attn_mask)
        return x + self.delta_bf(x, x if pos is None else x + pos, attn_mask)

    def forward(self, query, key=None, value=None, identity=None, query_pos=None, key_pos=None, attn_mask=None,
                key_padding_mask=None, **kwargs):
        if (key is not None and key is not query) or (value is not None and value is not query) \
                or identity is not None or key_padding_mask is not None:
            raise NotImplementedError('only the self-attention use of the decoder layer is implemented '
                                      "(operation 'self_attn' of FocalFormer3D's decoder_cfg)")
        if key_pos is not None and key_pos is not query_pos:
            raise NotImplementedError('key_pos must equal query_pos for self-attention')
        if self.batch_first:
            return self.forward_bf(query, query_pos, attn_mask)
        out = self.forward_bf(query.transpose(0, 1).contiguous(),
                              None if query_pos is None else query_pos.transpose(0, 1).contiguous(), attn_mask)
        return out.transpose(0, 1)


@register(ATTENTION)
class DifferentialAttention(nn.Module):
    """Self-attention whose weights are the difference of two softmax maps, in the place and with the calling conventions of
    ``MultiheadAttention`` (``attn_cfgs=[dict(type='DifferentialAttention', embed_dims=..., num_heads=...), ...]``):

        identity + out_proj(concat_h (1 - lambda_init) * RMSNorm(softmax(q1 k1^T / sqrt(d)) v - lam softmax(q2 k2^T / sqrt(d)) v))
        lam = exp(<lambda_q1, lambda_k1>) - exp(<lambda_q2, lambda_k2>) + lambda_init

    with q = k = x + pos, v = x projected to ``num_heads`` heads of 2 d columns ([map 1 | map 2] of q and k) and to ``kv_heads`` (default:
    as many) heads of k and v; d = embed_dims / num_heads / 2 is 8, 16, 32 or 64.  The core is ``ops.diff_attention`` (evaluation) /
    ``autograd.differential_attention`` (training), fp32 or 16-bit as the input is.  Attention masks: one per frame, True / negative =
    blocked; ``key_padding_mask`` (B, N), True = no key.  There is no dropout on the attention weights."""

    def __init__(self, embed_dims, num_heads, kv_heads=None, lambda_init=0.8, eps=1e-5, attn_drop=0., proj_drop=0.,
                 dropout_layer=dict(type='Dropout', drop_prob=0.), init_cfg=None, batch_first=False, **kwargs):
        super().__init__()
        dropout_layer = dict(dropout_layer) if dropout_layer else None
        if 'dropout' in kwargs:                            # the decoder configs' spelling: the output dropout
            dropout_layer = dict(type='Dropout', drop_prob=kwargs.pop('dropout'))
        if attn_drop:
            raise NotImplementedError('DifferentialAttention has no dropout on its attention weights (attn_drop)')
        if dropout_layer and dropout_layer.get('type', 'Dropout') != 'Dropout':
            raise NotImplementedError("dropout_layer: only type='Dropout'")
        kv_heads = num_heads if kv_heads is None else kv_heads
        d = embed_dims // (2 * num_heads)
        if embed_dims != 2 * d * num_heads or d not in (8, 16, 32, 64) or kv_heads < 1 or num_heads % kv_heads:
            raise ValueError(f'DifferentialAttention: embed_dims {embed_dims}, {num_heads} heads over {kv_heads}: expected heads of '
                             '16, 32, 64 or 128 columns and a multiple of kv_heads')
        self.embed_dims, self.num_heads, self.kv_heads, self.batch_first = embed_dims, num_heads, kv_heads, batch_first
        self.lambda_init, self.eps = float(lambda_init), float(eps)
        self.q_proj = nn.Linear(embed_dims, embed_dims)
        self.k_proj = nn.Linear(embed_dims, kv_heads * 2 * d)
        self.v_proj = nn.Linear(embed_dims, kv_heads * 2 * d)
        self.out_proj = nn.Linear(embed_dims, embed_dims)
        self.lambda_q1, self.lambda_k1, self.lambda_q2, self.lambda_k2 = (nn.Parameter(torch.randn(d) * 0.1) for _ in range(4))
        self.head_norm = nn.Parameter(torch.ones(2 * d))
        self.proj_drop = nn.Dropout(proj_drop)
        self.dropout_layer = nn.Dropout(dropout_layer.get('drop_prob', 0.)) if dropout_layer else nn.Identity()

    def invalidate_cache(self):
        for name in ('_bf16_w', '_bf16_rows_w', '_f16_w'):
            self.__dict__.pop(name, None)

    def _project(self, x, linear):
        from .autograd import is_dual
        if x.dtype != torch.float32 or torch.is_grad_enabled() or not x.is_contiguous() or x.numel() == 0 or is_dual(x, linear.weight, linear.bias):
            return F.linear(x, linear.weight, linear.bias)
        return _lin(self, x, linear.weight, linear.bias)

    def lam(self):
        """The weight of the second map, (num_heads,) - one value per layer, shared by its heads."""
        a = torch.exp((self.lambda_q1.float() * self.lambda_k1.float()).sum())
        b = torch.exp((self.lambda_q2.float() * self.lambda_k2.float()).sum())
        return (a - b + self.lambda_init).to(self.lambda_q1.dtype).expand(self.num_heads)

    def forward_bf(self, x, pos=None, attn_mask=None, key_padding_mask=None):
        """x, pos (B, N, C) -> (B, N, C)."""
        from .autograd import differential_attention
        B, N, C = x.shape
        xp = x if pos is None else x + pos
        mask = _frame_mask(attn_mask, B, self.num_heads, N)
        if key_padding_mask is not None:
            pad = key_padding_mask.bool()[:, None, :].expand(B, N, N)
            mask = pad if mask is None else mask | pad
        q = self._project(xp, self.q_proj)                 # (under autocast the projections' type is not the parameters')
        o = differential_attention(q, self._project(xp, self.k_proj), self._project(x, self.v_proj), self.lam().to(q.dtype), self.num_heads,
                                   kv_heads=self.kv_heads, mask=mask)
        heads = o.view(B, N, self.num_heads, C // self.num_heads)
        o = F.rms_norm(heads, heads.shape[-1:], self.head_norm.to(o.dtype), self.eps) * (1.0 - self.lambda_init)
        out = self._project(o.reshape(B, N, C), self.out_proj)
        return x + self.dropout_layer(self.proj_drop(out))

    def forward(self, query, key=None, value=None, identity=None, query_pos=None, key_pos=None, attn_mask=None,
                key_padding_mask=None, **kwargs):
        if (key is not None and key is not query) or (value is not None and value is not query) or identity is not None:
            raise NotImplementedError("only the self-attention use of the decoder layer is implemented (operation 'self_attn')")
        if key_pos is not None and key_pos is not query_pos:
            raise NotImplementedError('key_pos must equal query_pos for self-attention')
        if self.batch_first:
            return self.forward_bf(query, query_pos, attn_mask, key_padding_mask)
        out = self.forward_bf(query.transpose(0, 1).contiguous(),
                              None if query_pos is None else query_pos.transpose(0, 1).contiguous(), attn_mask, key_padding_mask)
        return out.transpose(0, 1)


@register(ATTENTION)
class MultiScaleDeformableAttention(nn.Module):
    """mmcv ``MultiScaleDeformableAttention`` with the gather on the HIP kernel."""

    def __init__(self, embed_dims=256, num_heads=8, num_levels=4, num_points=4, im2col_step=64, dropout=0.1,
                 batch_first=False, norm_cfg=None, init_cfg=None, **kwargs):
        super().__init__()
        if embed_dims % num_heads != 0:
            raise ValueError(f'embed_dims must be divisible by num_heads, but got {embed_dims} and {num_heads}')
        self.embed_dims, self.num_heads = embed_dims, num_heads
        self.num_levels, self.num_points = num_levels, num_points
        self.im2col_step, self.batch_first = im2col_step, batch_first
        self.sampling_offsets = nn.Linear(embed_dims, num_heads * num_levels * num_points * 2)
        self.attention_weights = nn.Linear(embed_dims, num_heads * num_levels * num_points)
        self.value_proj = nn.Linear(embed_dims, embed_dims)
        self.output_proj = nn.Linear(embed_dims, embed_dims)
        self.dropout = nn.Dropout(dropout)
        self._fused = None
        self.init_weights()

    def init_weights(self):
        """mmcv's own init: zero offset weights, a ring of directions as offset bias, zero attention
        logits, xavier projections."""
        import math
        nn.init.constant_(self.sampling_offsets.weight, 0.)
        thetas = torch.arange(self.num_heads, dtype=torch.float32) * (2.0 * math.pi / self.num_heads)
        grid = torch.stack([thetas.cos(), thetas.sin()], -1)
        grid = (grid / grid.abs().max(-1, keepdim=True)[0]).view(self.num_heads, 1, 1, 2) \
            .repeat(1, self.num_levels, self.num_points, 1)
        for i in range(self.num_points):
            grid[:, :, i, :] *= i + 1
        with torch.no_grad():
            self.sampling_offsets.bias.copy_(grid.view(-1))
        nn.init.constant_(self.attention_weights.weight, 0.)
        nn.init.constant_(self.attention_weights.bias, 0.)
        nn.init.xavier_uniform_(self.value_proj.weight)
        nn.init.constant_(self.value_proj.bias, 0.)
        nn.init.xavier_uniform_(self.output_proj.weight)
        nn.init.constant_(self.output_proj.bias, 0.)

    def invalidate_cache(self):
        self._fused = None
        self.__dict__.pop('_bf16_w', None)
        self.__dict__.pop('_bf16_rows_w', None)
        self.__dict__.pop('_f16_w', None)

    def _fused_offlog(self):
        sig = weight_signature((self.sampling_offsets.weight, self.attention_weights.weight, self.sampling_offsets.bias,
                                self.attention_weights.bias))
        if self._fused is None or self._fused[0] != sig:
            # the split-fp16 planes of the OLD concatenation are keyed on (data_ptr, _version) of a derived tensor that is about to
            # be freed: a later rebuild could be handed the same address at version 0 again (ABA) and match the stale entry
            self.__dict__.pop('_f16_w', None)
            self.__dict__.pop('_bf16_w', None)
            self.__dict__.pop('_bf16_rows_w', None)
            with torch.no_grad():
                self._fused = (sig, torch.cat([self.sampling_offsets.weight, self.attention_weights.weight], 0).contiguous(),
                               torch.cat([self.sampling_offsets.bias, self.attention_weights.bias], 0).contiguous())
        return self._fused[1:]

    def _gather_first_groups(self):
        """Column groups of the gathered rows = diagonal blocks of the projection: 2 when the two halves of the output are whole
        128-column tiles of the dual linear kernel (C = 256: out[:, :128] from heads 0-3, out[:, 128:] from heads 4-7), else 1."""
        return 2 if (self.embed_dims == 256 and self.num_heads % 2 == 0) else 1

    def _gather_first_weight(self, with_bias=True):
        """(C, hpg * C + 32) fp32, hpg = heads / groups: value_proj as a block-diagonal map over the per-head C-wide gathered rows + the
        bias on the per-head weight-sum columns (ops.msda_gather_rows' layout); output rows of group g multiply column group g of the
        gathered rows (the dual linear kernel: columns from C / 2 on read the second group).  Cached per weight version."""
        sig = weight_signature((self.value_proj.weight, self.value_proj.bias)) + (bool(with_bias),)
        c = self.__dict__.get('_gf_w')
        if c is None or c[0] != sig:
            with torch.no_grad():
                C_, M, G = self.embed_dims, self.num_heads, self._gather_first_groups()
                Dh, hpg = C_ // M, M // G
                w = self.value_proj.weight.detach().new_zeros(C_, hpg * C_ + 32)
                for h in range(M):
                    hl = h % hpg
                    w[h * Dh:(h + 1) * Dh, hl * C_:(hl + 1) * C_] = self.value_proj.weight[h * Dh:(h + 1) * Dh]
                    if with_bias:              # (with a PosTable the bias lives in the table: the weight-sum columns meet zeros)
                        w[h * Dh:(h + 1) * Dh, hpg * C_ + hl] = self.value_proj.bias[h * Dh:(h + 1) * Dh]
            self.__dict__.pop('_f16_w_gf', None)
            c = self.__dict__['_gf_w'] = (sig, w.contiguous())
        return c[1]

    def pos_table(self, pos_embed):
        """(1, Nv, heads, Dh) fp32 = value_proj(pos_embed) + bias for a (Nv, C) positional embedding (computed in fp64 once per call
        site; the caller caches it per weight version and grid)."""
        with torch.no_grad():
            t = (pos_embed.double() @ self.value_proj.weight.double().t() + self.value_proj.bias.double()).float()
        return t.view(1, t.shape[0], self.num_heads, -1).contiguous()

    def gather_first_ok(self, value_cl, reference_points, level_hw):
        """The opt-in value mode 'gather_first' (VERDICT r05 #4 (ii)): gather the UN-projected rows, project afterwards."""
        return (getattr(self, 'value_mode', 'project_first') == 'gather_first' and torch.is_tensor(value_cl) and value_cl.is_cuda
                and value_cl.dtype == torch.float32 and value_cl.dim() == 3 and self.embed_dims in (64, 128, 256)
                and self.num_heads <= 32 and not isinstance(level_hw, DeviceLevels) and reference_points.dim() == 3
                and not torch.is_grad_enabled())      # (bf16 mode too: the projection of the gathered rows then runs fp32-class)

    def project_value(self, value_cl):
        """value (B, Nv, C) channels-last -> (B, Nv, heads, Dh)."""
        B, Nv, C = value_cl.shape
        if getattr(self, 'gemm_dtype', torch.float32) == torch.bfloat16:   # bf16 value: half the gather bytes too
            ops.note_vendor('value_proj (per layer)', B * Nv, C, C)
            return F.linear(value_cl.to(torch.bfloat16), self.value_proj.weight.to(torch.bfloat16),
                            self.value_proj.bias.to(torch.bfloat16)).view(B, Nv, self.num_heads, -1)
        ops.note_vendor('value_proj (per layer)', B * Nv, C, C)
        if self.training and torch.is_grad_enabled():    # training: weight / bias gradient on the own TN kernel (csrc/wgrad.hip)
            from .autograd import train_linear
            return train_linear(value_cl, self.value_proj.weight, self.value_proj.bias).view(B, Nv, self.num_heads, -1)
        return F.linear(value_cl, self.value_proj.weight, self.value_proj.bias).view(B, Nv, self.num_heads, -1)

    def gather_bf(self, xp, value_cl, reference_points, level_hw, value_projected=None):
        """The deformable gather before the output projection; xp = query + query_pos (B, Nq, C)."""
        B, Nq, C = xp.shape
        if isinstance(level_hw, DeviceLevels) or reference_points.dim() == 4:
            return self._gather_dev_tables(xp, value_cl, reference_points, level_hw, value_projected)
        w, b = self._fused_offlog()
        both = _lin32(self, xp, w, b).view(B * Nq, -1)           # (sampling offsets | attention logits: fp32-class in either mode)
        n_off = self.num_heads * self.num_levels * self.num_points * 2
        table = value_projected.table if isinstance(value_projected, PosTable) else None
        if (value_projected is None or table is not None) and self.gather_first_ok(value_cl, reference_points, level_hw):
            # sum_k w_k (W v_k + b) = W (sum_k w_k v_k) + b sum_k w_k: the gather reads the un-projected C-wide rows per head, the
            # projection runs over B*Nq rows instead of B*Nv (one block-diagonal GEMM, K = heads * C + 32)
            G = self._gather_first_groups()
            rows = ops.msda_gather_rows(value_cl.contiguous(), level_hw, reference_points.contiguous(), both[:, :n_off], both[:, n_off:],
                                        self.num_points, self.num_heads, groups=G)
            wbig = self._gather_first_weight(with_bias=table is None)
            ws = _cached(self, '_f16_w_gf', wbig, None, lambda: ops.split_weight_f16(wbig))
            Kg = wbig.shape[1]
            rows = rows.view(B, Nq, -1)
            if G == 2:                       # columns 0 .. C/2 - 1 from group 0's K columns, C/2 .. from group 1's (one launch)
                out = ops.linear_f16x3(rows[:, :, :Kg], ws, None, False, x2=rows[:, :, Kg:], n_split=C // 2)
            else:
                out = ops.linear_f16x3(rows, ws, None, False)
            if table is not None:
                # + sum_k w_k (W pos_k + b): the ordinary head-slice gather over the frame-independent table, all B * Nq queries as
                # the queries of its single "frame" (the 43 MB table lives in L2 / MALL)
                out = out.view(B, Nq, C) + ops.msda_fused_fwd(table, level_hw, reference_points.reshape(1, B * Nq, 2), both[:, :n_off],
                                                              both[:, n_off:], self.num_points).view(B, Nq, C)
            return out
        v = value_projected if value_projected is not None else self.project_value(value_cl)
        return ops.msda_fused_fwd(v, level_hw, reference_points.contiguous(), both[:, :n_off], both[:, n_off:],
                                  self.num_points)

    def delta_bf(self, xp, value_cl, reference_points, level_hw, value_projected=None):
        """output_proj(gather) without the residual; xp = query + query_pos (B, Nq, C)."""
        return _lin(self, self.gather_bf(xp, value_cl, reference_points, level_hw, value_projected),
                    self.output_proj.weight, self.output_proj.bias)

    def forward_train_bf(self, x, value_cl, pos, reference_points, level_hw, value_projected=None):
        """Appendix A.3, differentiable: mmcv's op sequence on the framework's autograd ops around the HIP gather
        (MultiScaleDeformableAttnFunction: ff3d_msda_fwd / ff3d_msda_bwd); dropout(output_proj(gather)) + identity.
        ``value_projected`` (B, Nv, heads, Dh): this layer's column block of the decoder's batched value projection."""
        from .autograd import MultiScaleDeformableAttnFunction
        B, Nq, C = x.shape
        M, L, P = self.num_heads, self.num_levels, self.num_points
        xp = x if pos is None else x + pos
        if isinstance(level_hw, DeviceLevels):
            level_hw = [tuple(int(v) for v in r) for r in level_hw.spatial_shapes.tolist()]
        from .autograd import train_linear      # (weight / bias gradient over the B * Nv rows on the own TN kernel, csrc/wgrad.hip)
        value = value_projected if value_projected is not None else \
            train_linear(value_cl, self.value_proj.weight, self.value_proj.bias).view(B, value_cl.shape[1], M, -1)
        off = self.sampling_offsets(xp).view(B, Nq, M, L, P, 2)
        attn = self.attention_weights(xp).view(B, Nq, M, L * P).softmax(-1).view(B, Nq, M, L, P)
        nkey = (tuple(level_hw), off.dtype, off.device)  # (W_l, H_l) on the device: built once (a blocking host-to-device copy per call)
        if nkey not in _NORMALIZERS:
            _NORMALIZERS[nkey] = torch.tensor([[w, h] for h, w in level_hw], dtype=off.dtype, device=off.device)
        normalizer = _NORMALIZERS[nkey]
        ref = reference_points[:, :, None, None, None, :] if reference_points.dim() == 3 else reference_points[:, :, None, :, None, :]
        loc = ref + off / normalizer[None, None, None, :, None, :]
        o = MultiScaleDeformableAttnFunction.apply(value, level_hw, None, loc, attn, self.im2col_step)
        return self.dropout(self.output_proj(o)) + x

    def forward_bf(self, x, value_cl, pos, reference_points, level_hw, value_projected=None):
        """x, pos (B, Nq, C); value_cl (B, Nv, C); reference_points (B, Nq, 2) normalised -> (B, Nq, C)."""
        if self.training:
            return self.forward_train_bf(x, value_cl, pos, reference_points, level_hw, value_projected)
        return x + self.delta_bf(x if pos is None else x + pos, value_cl, reference_points, level_hw, value_projected)

    def forward(self, query, key=None, value=None, identity=None, query_pos=None, key_padding_mask=None,
                reference_points=None, spatial_shapes=None, level_start_index=None, **kwargs):
        if value is None:
            value = query
        if key_padding_mask is not None:
            raise NotImplementedError('key_padding_mask is None at the reference call site (FD:864)')
        if identity is not None and identity is not query:
            raise NotImplementedError('identity != query is not used by the decoder layer')
        if reference_points.shape[-1] != 2:
            raise NotImplementedError('4-d reference boxes are not used by FocalFormer3D')
        if not self.batch_first:
            query = query.permute(1, 0, 2)
            value = value.permute(1, 0, 2)
            if query_pos is not None:
                query_pos = query_pos.permute(1, 0, 2)
        reference_points = _per_level_ref(reference_points, self.num_levels)
        query, value = query.contiguous(), value.contiguous()
        query_pos = None if query_pos is None else query_pos.contiguous()
        out = self.forward_bf(query, value, query_pos, reference_points, _level_hw(spatial_shapes, level_start_index))
        return out if self.batch_first else out.permute(1, 0, 2)

    def _gather_dev_tables(self, xp, value_cl, reference_points, levels, value_projected=None):
        """mmcv MultiScaleDeformableAttention.forward's own op sequence (offset normaliser from the device shape table,
        softmax over L*P) feeding the gather kernel with device level tables; before output_proj."""
        B, Nq, C = xp.shape
        M, L, P = self.num_heads, self.num_levels, self.num_points
        w, b = self._fused_offlog()
        both = _lin32(self, xp, w, b)
        n_off = M * L * P * 2
        off = both[..., :n_off].reshape(B, Nq, M, L, P, 2)
        attn = both[..., n_off:].reshape(B, Nq, M, L * P).softmax(-1).view(B, Nq, M, L, P).contiguous()
        dev = isinstance(levels, DeviceLevels)
        shapes = levels.spatial_shapes if dev else torch.as_tensor(levels, dtype=torch.long, device=off.device)
        normalizer = torch.stack([shapes[..., 1], shapes[..., 0]], -1).to(off.dtype)                       # (W_l, H_l)
        # (B, Nq, 2): one reference point per query; (B, Nq, L, 2): one per level = reference point x valid ratio of that level,
        # as mmdet's decoder hands it to every layer (a ratio of exactly 1 leaves the value bit for bit)
        ref = reference_points[:, :, None, None, None, :] if reference_points.dim() == 3 else reference_points[:, :, None, :, None, :]
        loc = (ref + off / normalizer[None, None, None, :, None, :]).contiguous()
        v = value_projected if value_projected is not None else self.project_value(value_cl)
        if not v.is_contiguous():
            v = v.contiguous()                              # column block of the batched value_proj GEMM
        if dev:
            return ops.msda_fwd_dev(v, shapes, levels.level_start_index, loc, attn)
        return ops.msda_fwd(v, levels, loc, attn)


@register(FEEDFORWARD_NETWORK)
class FFN(nn.Module):
    """mmcv ``FFN``: Linear-act-(drop) x (num_fcs-1), Linear, (drop), residual."""

    def __init__(self, embed_dims=256, feedforward_channels=1024, num_fcs=2, act_cfg=dict(type='ReLU', inplace=True),
                 ffn_drop=0., dropout_layer=None, add_identity=True, init_cfg=None, **kwargs):
        super().__init__()
        assert num_fcs >= 2
        if act_cfg.get('type', 'ReLU') != 'ReLU':
            raise NotImplementedError('only ReLU FFNs are used by the FocalFormer3D configs')
        self.embed_dims, self.feedforward_channels, self.add_identity = embed_dims, feedforward_channels, add_identity
        layers, cin = [], embed_dims
        for _ in range(num_fcs - 1):
            layers.append(nn.Sequential(nn.Linear(cin, feedforward_channels), nn.ReLU(inplace=True), nn.Dropout(ffn_drop)))
            cin = feedforward_channels
        layers.append(nn.Linear(feedforward_channels, embed_dims))
        layers.append(nn.Dropout(ffn_drop))
        self.layers = nn.Sequential(*layers)

    def invalidate_cache(self):
        self.__dict__.pop('_bf16_w', None)
        self.__dict__.pop('_bf16_rows_w', None)
        self.__dict__.pop('_f16_w', None)
        self.__dict__.pop('_f16_tiled', None)

    def hidden(self, x):
        """Everything before the last Linear -> (hidden activation, last Linear)."""
        y, last = x, None
        for m in self.layers:
            if isinstance(m, nn.Sequential):
                y = _lin(self, y, m[0].weight, m[0].bias, relu=True)   # GEMM with fused bias + ReLU epilogue
            elif isinstance(m, nn.Linear):
                last = m
        return y, last

    def delta(self, x):
        y, last = self.hidden(x)
        return _lin(self, y, last.weight, last.bias)

    def fused_add_ln(self, x, norm, pos=None):
        """Round 5: LayerNorm(x + fc2(relu(fc1(x)))) (+ pos) as ONE launch (ops.ffn_rows, csrc/ffnrows.hip) - the hidden activation
        stays on the CU.  -> the result (a pair with ``pos``), or None where the fused kernel does not apply (more than two fcs, another
        width, the bf16 mode, autograd, fewer than FFN_FUSED_MIN_ROWS rows): the caller runs the two-launch form."""
        fcs = [m for m in self.layers if isinstance(m, (nn.Sequential, nn.Linear))]
        if not (FFN_FUSED and len(fcs) == 2 and isinstance(fcs[0], nn.Sequential) and self.add_identity and self.embed_dims == 256
                and self.feedforward_channels % 128 == 0 and getattr(self, 'gemm_dtype', torch.float32) == torch.float32
                and x.is_contiguous() and (pos is None or pos.is_contiguous()) and _own_linear(self, x, fcs[0][0].weight)
                and x.numel() // x.shape[-1] >= FFN_FUSED_MIN_ROWS):
            return None
        fc1, fc2 = fcs[0][0], fcs[1]
        w1 = _cached(self, '_f16_tiled', fc1.weight, fc1.bias, lambda: ops.tile_weight_f16(fc1.weight.detach(), bias=fc1.bias))
        w2 = _cached(self, '_f16_tiled', fc2.weight, fc2.bias, lambda: ops.tile_weight_f16(fc2.weight.detach(), bias=fc2.bias))
        b1 = fc1.bias if fc1.bias is not None else x.new_zeros(fc1.weight.shape[0])
        return ops.ffn_rows(x, w1, b1.detach(), w2, None if fc2.bias is None else fc2.bias.detach(), x, norm.weight, norm.bias,
                            norm.eps, pos)

    def forward(self, x, identity=None):
        y = self.layers(x) if self.training else self.delta(x)      # training: Linear / ReLU / Dropout modules under autograd
        if not self.add_identity:
            return y
        return (x if identity is None else identity) + y


@register(FEEDFORWARD_NETWORK)
class GatedFFN(nn.Module):
    """Gated feed-forward step in the place of ``FFN`` (``ffn_cfgs=dict(type='GatedFFN', feedforward_channels=..., ...)``):
    identity + fc_out(act(fc_g(x)) * fc_u(x)), both inner projections, the activation and the product in one kernel
    (``ops.gated_linear`` / ``autograd.gated_linear``).  ``in_proj`` holds the gate's rows, then the value's.
    act_cfg type: SiLU (default), GELU, ReLU or Sigmoid."""

    def __init__(self, embed_dims=256, feedforward_channels=1024, num_fcs=2, act_cfg=dict(type='SiLU'), ffn_drop=0., dropout_layer=None,
                 add_identity=True, init_cfg=None, **kwargs):
        super().__init__()
        if num_fcs != 2:
            raise NotImplementedError('GatedFFN: one gated projection and one output projection (num_fcs=2)')
        if dropout_layer and dropout_layer.get('drop_prob', 0.):
            raise NotImplementedError('GatedFFN: ffn_drop is its dropout (dropout_layer)')
        self.act = act_cfg.get('type', 'SiLU').lower()
        if self.act not in ops._ACTS:
            raise NotImplementedError(f"act_cfg: type {act_cfg.get('type')!r} (SiLU, GELU, ReLU or Sigmoid)")
        self.embed_dims, self.feedforward_channels, self.add_identity = embed_dims, feedforward_channels, add_identity
        self.in_proj = nn.Linear(embed_dims, 2 * feedforward_channels)
        self.out_proj = nn.Linear(feedforward_channels, embed_dims)
        self.drop = nn.Dropout(ffn_drop)

    def invalidate_cache(self):
        for name in ('_bf16_w', '_bf16_rows_w', '_f16_w', '_f16_tiled', '_f16_wk'):
            self.__dict__.pop(name, None)

    def hidden(self, x):
        """Everything before the last Linear -> (hidden activation, last Linear)."""
        from .autograd import gated_linear, is_dual
        w, b = self.in_proj.weight, self.in_proj.bias
        if torch.is_grad_enabled() or is_dual(x, w, b):
            if x.is_cuda and x.dtype != torch.float64 and torch.is_autocast_enabled('cuda'):     # as the Linear layers around it
                x = x.to(torch.get_autocast_dtype('cuda'))
            return gated_linear(x, w.to(x.dtype), b.to(x.dtype), self.act), self.out_proj
        if x.dtype == torch.float32 and getattr(self, 'gemm_dtype', torch.float32) == torch.bfloat16:
            # bf16 mode: operands on the bf16 matrix cores, fp32 rows out
            w16, b16 = _cached(self, '_bf16_w', w, b, lambda: (w.detach().to(torch.bfloat16), b.detach().to(torch.bfloat16)))
            return ops.gated_linear(x.to(torch.bfloat16), w16, b16, self.act).float(), self.out_proj
        # (fp32 rows stay fp32 here, as in FFN; 16-bit ones come from projections under autocast)
        return ops.gated_linear(x, w.detach().to(x.dtype), b.detach().to(x.dtype), self.act), self.out_proj

    def delta(self, x):
        y, last = self.hidden(x)
        own = y.dtype == torch.float32 and y.numel() > 0
        return _lin(self, y, last.weight, last.bias) if own else F.linear(y, last.weight, last.bias)

    def fused_add_ln(self, x, norm, pos=None):
        """There is no one-launch form: the caller runs the projection and the fused add + LayerNorm."""
        return None

    def forward(self, x, identity=None):
        if self.training or torch.is_grad_enabled():
            y, last = self.hidden(x)
            y = self.drop(last(self.drop(y)))
        else:
            y = self.delta(x)
        if not self.add_identity:
            return y
        return (x if identity is None else identity) + y


@register(TRANSFORMER_LAYER)
class DetrTransformerDecoderLayer(nn.Module):
    """mmcv ``BaseTransformerLayer`` / mmdet ``DetrTransformerDecoderLayer`` (post-norm order used by the
    reference: 'self_attn','norm','cross_attn','norm','ffn','norm')."""

    def __init__(self, attn_cfgs=None, ffn_cfgs=dict(type='FFN', embed_dims=256, feedforward_channels=1024, num_fcs=2,
                                                     ffn_drop=0., act_cfg=dict(type='ReLU', inplace=True)),
                 operation_order=None, norm_cfg=dict(type='LN'), init_cfg=None, batch_first=False, **kwargs):
        super().__init__()
        ffn_cfgs = copy.deepcopy(ffn_cfgs)
        for old, new in dict(feedforward_channels='feedforward_channels', ffn_dropout='ffn_drop',
                             ffn_num_fcs='num_fcs').items():
            if old in kwargs:                              # deprecated spellings used by the reference configs
                ffn_cfgs[new] = kwargs.pop(old)
        assert set(operation_order) <= {'self_attn', 'norm', 'ffn', 'cross_attn'}
        if norm_cfg.get('type', 'LN') != 'LN':
            raise NotImplementedError('LayerNorm only')
        num_attn = operation_order.count('self_attn') + operation_order.count('cross_attn')
        if isinstance(attn_cfgs, dict):
            attn_cfgs = [copy.deepcopy(attn_cfgs) for _ in range(num_attn)]
        assert num_attn == len(attn_cfgs)
        self.batch_first, self.operation_order = batch_first, tuple(operation_order)
        self.pre_norm = operation_order[0] == 'norm'
        self.attentions = nn.ModuleList()
        for cfg in attn_cfgs:
            cfg = copy.deepcopy(cfg)
            cfg.setdefault('batch_first', batch_first)
            self.attentions.append(build_attention(cfg))
        self.embed_dims = self.attentions[0].embed_dims
        num_ffns = operation_order.count('ffn')
        if isinstance(ffn_cfgs, dict):
            ffn_cfgs = [copy.deepcopy(ffn_cfgs) for _ in range(num_ffns)]
        self.ffns = nn.ModuleList()
        for cfg in ffn_cfgs:
            cfg = copy.deepcopy(cfg)
            cfg.setdefault('type', 'FFN')
            cfg['embed_dims'] = self.embed_dims
            self.ffns.append(build_feedforward_network(cfg))
        self.norms = nn.ModuleList([nn.LayerNorm(self.embed_dims) for _ in range(operation_order.count('norm'))])

    _POST_NORM = ('self_attn', 'norm', 'cross_attn', 'norm', 'ffn', 'norm')

    def forward_fused(self, x, xp, value_cl, pos, reference_points, level_hw, value_projected=None, want_xp=True):
        """The reference's post-norm layer with every residual add + LayerNorm (+ the following `+ query_pos`)
        in one kernel: 3 fused launches instead of 8 elementwise / norm launches.  xp = x + pos."""
        n0, n1, n2 = self.norms
        sa, ca, ffn = self.attentions[0], self.attentions[1], self.ffns[0]
        # each step: [output projection + identity + LayerNorm (+ query_pos)] in one launch where the own dense kernel applies
        # (_lin_add_ln), else the projection followed by the fused add + LayerNorm kernel
        x, xp = _lin_add_ln(sa, sa.core_bf(x, xp), sa.attn.out_proj.weight, sa.attn.out_proj.bias, x, n0, pos)
        o = ca.gather_bf(xp, value_cl, reference_points, level_hw, value_projected)
        x = _lin_add_ln(ca, o, ca.output_proj.weight, ca.output_proj.bias, x, n1)
        fused = ffn.fused_add_ln(x, n2, pos if want_xp else None)
        if fused is not None:
            return fused if want_xp else (fused, None)
        h, last = ffn.hidden(x)
        if want_xp:
            return _lin_add_ln(ffn, h, last.weight, last.bias, x, n2, pos)
        return _lin_add_ln(ffn, h, last.weight, last.bias, x, n2), None

    def can_fuse(self):
        return (self.operation_order == self._POST_NORM and isinstance(self.attentions[0], MultiheadAttention)
                and isinstance(self.attentions[1], MultiScaleDeformableAttention) and self.ffns[0].add_identity)

    def forward_bf(self, x, value_cl, pos, reference_points, level_hw, attn_mask=None, value_projected=None):
        if not self.training and attn_mask is None and pos is not None and self.can_fuse():
            return self.forward_fused(x, x + pos, value_cl, pos, reference_points, level_hw, value_projected, False)[0]
        ai = ni = fi = 0
        for op in self.operation_order:
            if op == 'self_attn':
                x = self.attentions[ai].forward_bf(x, pos, attn_mask)
                ai += 1
            elif op == 'cross_attn':
                x = self.attentions[ai].forward_bf(x, value_cl, pos, reference_points, level_hw, value_projected)
                ai += 1
            elif op == 'norm':
                n = self.norms[ni]
                x = F.layer_norm(x, (x.shape[-1],), n.weight, n.bias, n.eps)
                ni += 1
            else:
                x = self.ffns[fi](x)
                fi += 1
        return x

    def forward(self, query, key=None, value=None, query_pos=None, key_pos=None, attn_masks=None,
                query_key_padding_mask=None, key_padding_mask=None, reference_points=None, spatial_shapes=None,
                level_start_index=None, **kwargs):
        if self.pre_norm:
            raise NotImplementedError('pre-norm order is not used by the FocalFormer3D configs')
        if isinstance(attn_masks, (list, tuple)):
            attn_masks = attn_masks[0]
        elif attn_masks is not None:
            warnings.warn(f'Use same attn_mask in all attentions in {type(self).__name__}')
        bf = (lambda t: t) if self.batch_first else (lambda t: None if t is None else t.transpose(0, 1).contiguous())
        ref = _per_level_ref(reference_points, None)
        out = self.forward_bf(bf(query), bf(value), bf(query_pos), ref, _level_hw(spatial_shapes, level_start_index), attn_masks)
        return out if self.batch_first else out.transpose(0, 1)


@register(TRANSFORMER_LAYER_SEQUENCE)
class DeformableDetrTransformerDecoder(nn.Module):
    """mmdet ``DeformableDetrTransformerDecoder`` (reg_branches None, as called at FD:927-933)."""

    def __init__(self, transformerlayers=None, num_layers=None, return_intermediate=False, init_cfg=None, **kwargs):
        super().__init__()
        if isinstance(transformerlayers, dict):
            transformerlayers = [copy.deepcopy(transformerlayers) for _ in range(num_layers)]
        assert len(transformerlayers) == num_layers
        if return_intermediate:
            raise NotImplementedError('return_intermediate=False in every FocalFormer3D config')
        self.num_layers, self.return_intermediate = num_layers, return_intermediate
        self.layers = nn.ModuleList([build_transformer_layer(c) for c in transformerlayers])
        self.embed_dims = self.layers[0].embed_dims
        self.batch_value_proj = True       # one (B*Nv, C) x (C, n_layers*C) GEMM for all layers' value_proj
        self._vcat, self._vcat_sig = None, None

    def invalidate_cache(self):
        self._vcat = None
        self._vcat_rows = None

    def set_value_mode(self, mode):
        """'project_first' (default: value_proj over every BEV cell, then the HBM-bound gather of Dh-wide head slices - the form
        north_star names) or 'gather_first' (opt-in: the gather reads un-projected C-wide rows per head, value_proj runs on the
        gathered B*Nq rows; mathematically the same operator, fp32-class; trades the 2 x 2 ms value GEMM of the 32-frame step for a
        gather that requests 8 x the bytes, served by L2 / MALL)."""
        assert mode in ('project_first', 'gather_first')
        for a in (self._cross_attns() or []):
            a.value_mode = mode

    def set_gemm_dtype(self, dtype):
        """torch.float32 (default, parity path) or torch.bfloat16 for the decoder's dense projections."""
        self._vcat = None
        for m in self.modules():
            m.gemm_dtype = dtype
            m.__dict__.pop('_bf16_w', None)
            m.__dict__.pop('_bf16_rows_w', None)
            m.__dict__.pop('_f16_w', None)
            m.__dict__.pop('_f16_tiled', None)

    def _cross_attns(self):
        out = []
        for layer in self.layers:
            ms = [a for a in layer.attentions if isinstance(a, MultiScaleDeformableAttention)]
            if len(ms) != 1:
                return None
            out.append(ms[0])
        return out

    def value_weights(self):
        """(W (n_layers*C, C), b (n_layers*C)) fp32: the value_proj of every layer stacked (None when a layer has no
        single MSDA cross-attention)."""
        cross = self._cross_attns()
        if cross is None:
            return None
        dt = getattr(self, 'gemm_dtype', torch.float32)
        sig = weight_signature([t for a in cross for t in (a.value_proj.weight, a.value_proj.bias)]) + (dt,)
        if self._vcat is None or self._vcat_sig != sig:
            with torch.no_grad():
                self._vcat = (torch.cat([a.value_proj.weight for a in cross], 0).to(dt).contiguous(),
                              torch.cat([a.value_proj.bias for a in cross], 0).to(dt).contiguous())
            self._vcat_sig = sig
        return self._vcat

    def project_values(self, value_cl):
        """All layers' value_proj as ONE GEMM over the stage's value tensor ((B, Nv, C) fp32, or the (hi, lo') Pair ->
        split-fp16 MFMA GEMM): list of per-layer (B, Nv, heads, Dh) column-block views, or None when the layers cannot be
        batched.  Independent of the queries, so the caller may run it ahead of time / on another stream."""
        cross = self._cross_attns() if self.batch_value_proj else None
        if cross is None or len(cross) < 2:
            return None
        dt = getattr(self, 'gemm_dtype', torch.float32)
        self.value_weights()
        if torch.is_tensor(value_cl) and value_cl.dtype == torch.bfloat16:
            # bf16 mode on the own kernels (round 5): the value arrives as ONE bf16 plane (+ zero row) from bev_flatten, the projected
            # value leaves as bf16 rows - weight-stationary one-plane MFMA GEMM (ff3d_gemm_bf16), no cast launch, no vendor GEMM
            B, Nv, C = value_cl.shape
            if getattr(self, '_vcat_rows', None) is None or self._vcat_rows[0] is not self._vcat:
                with torch.no_grad():
                    w32 = torch.cat([a.value_proj.weight for a in cross], 0)
                    b32 = torch.cat([a.value_proj.bias for a in cross], 0)
                self._vcat_rows = (self._vcat, ops.bf16_weight(w32, b32))
            allv = ops.gemm_bf16(value_cl.view(B * Nv, C), self._vcat_rows[1], out_bf16=True)
        elif isinstance(value_cl, tuple):               # (hi, lo') fp16 pair -> split-fp16 MFMA GEMM (splitmm.hip)
            B, Nv, C = value_cl[0].shape
            if getattr(self, '_vcat_split', None) is None or self._vcat_split[0] is not self._vcat:
                self._vcat_split = (self._vcat, ops.split_weight_f16(self._vcat[0].float(), bias=self._vcat[1]))
            allv = ops.gemm_f16x3(ops.as_pair(value_cl).view(B * Nv, C), self._vcat_split[1], self._vcat[1].float())
        else:
            B, Nv, C = value_cl.shape
            ops.note_vendor('value_proj', B * Nv, self._vcat[0].shape[0], C)
            allv = F.linear(value_cl.to(dt), *self._vcat)
        allv = allv.view(B, Nv, len(cross), cross[0].num_heads, -1)
        return [allv[:, :, i] for i in range(len(cross))]

    def forward_bf(self, x, value_cl, pos, reference_points, level_hw, attn_mask=None, vals=None):
        """Batch-first fast path: x, pos (B, Nq, C); value_cl (B, Nv, C); reference_points (B, Nq, 2).
        Every layer's value_proj reads the same value tensor (it is never refined, FD:927-933), so the
        projections of all layers run as ONE GEMM (the big input is read once, N = n_layers*C keeps the
        MFMA tiles full); each layer's gather then reads its (heads, Dh) column block in place.  ``vals``: the per-layer
        projected values when the caller already ran that GEMM (FocalDecoder fuses it across decoder stages)."""
        if self.training:                                # differentiable route: per-layer modules under autograd
            # (tried in round 6: the layers' value_proj as ONE linear over the stacked weights under autograd too - 41.8 vs 41.2 ms of
            #  kernels per step and a slower wall clock: the N = 768 forms of the three GEMMs gain 0.3 ms, the copies that make the
            #  layers' column blocks contiguous for the gather and stack their gradients cost 0.4 ms, the weight-gradient kernel is
            #  slower at six tiles per row slice than three launches at two; profiles/r06_train_step_kernels.txt)
            for layer in self.layers:
                x = layer.forward_bf(x, value_cl, pos, reference_points, level_hw, attn_mask)
            return x
        gather_first = (not isinstance(level_hw, DeviceLevels) and self._cross_attns() is not None
                        and all(a.gather_first_ok(value_cl, reference_points, level_hw) for a in self._cross_attns()))
        if vals is not None and not gather_first and any(isinstance(v, PosTable) for v in vals):
            raise RuntimeError("PosTable values need the 'gather_first' value mode")
        if vals is None:
            # (device level tables = the mmcv drop-in route: per-layer projections, the gather kernel wants a dense value;
            #  value mode 'gather_first': nothing is projected per cell)
            vals = self.project_values(value_cl) if not (isinstance(level_hw, DeviceLevels) or gather_first) else None
            if vals is None:
                vals = [None] * len(self.layers)
        if attn_mask is None and pos is not None and all(l.can_fuse() for l in self.layers):
            x, pos = x.contiguous(), pos.contiguous()
            xp = x + pos
            for i, (layer, v) in enumerate(zip(self.layers, vals)):
                x, xp = layer.forward_fused(x, xp, value_cl, pos, reference_points, level_hw, v,
                                            want_xp=i + 1 < len(self.layers))
            return x
        for layer, v in zip(self.layers, vals):
            x = layer.forward_bf(x, value_cl, pos, reference_points, level_hw, attn_mask, value_projected=v)
        return x

    def forward(self, query, *args, key=None, value=None, query_pos=None, reference_points=None, valid_ratios=None,
                reg_branches=None, spatial_shapes=None, level_start_index=None, key_padding_mask=None,
                attn_masks=None, **kwargs):
        if reg_branches is not None:
            raise NotImplementedError('reg_branches is None at the reference call site (FD:927-933)')
        if reference_points.shape[-1] != 2:
            raise NotImplementedError('4-d reference boxes are not used by FocalFormer3D')
        # mmdet: reference_points_input = reference_points[:, :, None] * valid_ratios[:, None], one point per level.  The head's
        # own fast path calls forward_bf with (B, Nq, 2) points (valid_ratios is all ones at FD:863); this drop-in route honours
        # whatever ratios it is given, without reading them on the host.
        ref_in = reference_points
        if valid_ratios is not None:
            ref_in = reference_points[:, :, None] * valid_ratios[:, None].to(reference_points.dtype)
        out = self.forward_bf(query.transpose(0, 1).contiguous(), value.transpose(0, 1).contiguous(),
                              None if query_pos is None else query_pos.transpose(0, 1).contiguous(),
                              _per_level_ref(ref_in, None), _level_hw(spatial_shapes, level_start_index), attn_masks)
        return out.transpose(0, 1), reference_points
