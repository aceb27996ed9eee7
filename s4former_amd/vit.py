"""VisionTransformer backbone with the reference's constructor, forward signature, return convention and
state-dict keys (reference mmseg/models/backbones/vit.py:237-264,479-570 and models/utils/embed.py), running on
the C-ABI HIP kernels (functional.PatchEmbedFn / LayerFn).

The torch.nn modules instantiated here (Conv2d, LayerNorm, Linear, MultiheadAttention) are parameter CONTAINERS:
they give the reference's parameter names and default initialisers; their own forward() is never called on the
product path.
"""
import math
import os
import warnings

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import runtime
from ._lib import F32, S4FError
from .base_module import BaseModule, ModuleList, constant_init, kaiming_init, trunc_normal_
from .functional import LayerFn, LayerOpt, PatchEmbedFn
from .params import ParamStore
from .registry import BACKBONES


def to_2tuple(x):
    return tuple(x) if isinstance(x, (tuple, list)) else (x, x)


class PatchEmbed(BaseModule):
    """Image to patch embedding (reference models/utils/embed.py:83-204), Conv2d k = s = patch_size."""

    def __init__(self, in_channels=3, embed_dims=768, conv_type='Conv2d', kernel_size=16, stride=None, padding='corner',
                 dilation=1, bias=True, norm_cfg=None, input_size=None, init_cfg=None):
        super().__init__(init_cfg=init_cfg)
        self.embed_dims = embed_dims
        if stride is None:
            stride = kernel_size
        kernel_size, stride = to_2tuple(kernel_size), to_2tuple(stride)
        assert kernel_size == stride, 'only non-overlapping patches are on the hot path'
        assert norm_cfg is None, 'patch_norm is not used by the SETR configs'
        self.kernel_size = kernel_size
        self.padding = padding
        self.projection = nn.Conv2d(in_channels, embed_dims, kernel_size, stride, 0, dilation, bias=bias)
        self.norm = None
        self.init_input_size = to_2tuple(input_size) if input_size else None
        if input_size:
            self.init_out_size = (self.init_input_size[0] // stride[0], self.init_input_size[1] // stride[1])
        else:
            self.init_out_size = None

    def pad(self, x):
        """AdaptivePadding 'corner' (embed.py:58-80): zero-pad bottom/right to a multiple of the patch size."""
        ph, pw = self.kernel_size
        H, W = x.shape[-2:]
        pad_h, pad_w = (ph - H % ph) % ph, (pw - W % pw) % pw
        if pad_h or pad_w:
            if self.padding == 'corner':
                x = F.pad(x, [0, pad_w, 0, pad_h])
            else:
                x = F.pad(x, [pad_w // 2, pad_w - pad_w // 2, pad_h // 2, pad_h - pad_h // 2])
        return x


class _Gain(BaseModule):
    """gain of an RMS norm: parameter path `weight`"""

    def __init__(self, dims):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dims))


class _AttnContainer(BaseModule):
    """mmcv MultiheadAttention wrapper: parameter path `attn.attn.*` (nn.MultiheadAttention container); qk_norm adds `attn.q_norm.weight`
    and `attn.k_norm.weight` [64], shared by the heads."""

    def __init__(self, embed_dims, num_heads, bias=True, qk_norm=False):
        super().__init__()
        self.embed_dims, self.num_heads = embed_dims, num_heads
        self.attn = nn.MultiheadAttention(embed_dims, num_heads, 0.0, bias=bias)
        if qk_norm:
            self.q_norm, self.k_norm = _Gain(embed_dims // num_heads), _Gain(embed_dims // num_heads)
        self.self_attn = None       # Q7: the patched mmcv stored head-averaged weights here (visualisation only)


class _FFNContainer(BaseModule):
    """mmcv FFN: parameter paths `ffn.layers.0.0.*`, `ffn.layers.1.*`."""

    def __init__(self, embed_dims, feedforward_channels):
        super().__init__()
        self.layers = nn.Sequential(
            nn.Sequential(nn.Linear(embed_dims, feedforward_channels), nn.GELU(), nn.Dropout(0.0)),
            nn.Linear(feedforward_channels, embed_dims), nn.Dropout(0.0))


class TransformerEncoderLayer(BaseModule):
    """reference vit.py:28-127.  forward(x, attn_mask) with attn_mask given in the rank-1 form
    (bias_u [B,N], row_flag [B,N] | None, weight) or None.  qk_norm, act_q8 and the rotation tables given to forward are options beyond the
    reference (VisionTransformer has their description)."""

    def __init__(self, embed_dims, num_heads, feedforward_channels, drop_rate=0., attn_drop_rate=0., drop_path_rate=0.,
                 num_fcs=2, qkv_bias=True, act_cfg=dict(type='GELU'), norm_cfg=dict(type='LN'), batch_first=True,
                 attn_cfg=dict(), ffn_cfg=dict(), with_cp=False, qk_norm=False, act_q8=False):
        super().__init__()
        if drop_rate or attn_drop_rate or drop_path_rate:
            raise S4FError('dropout / drop-path are 0 in every SETR config; the fused layer has no dropout')
        assert num_fcs == 2 and act_cfg.get('type') == 'GELU' and norm_cfg.get('type') == 'LN'
        assert embed_dims % num_heads == 0 and embed_dims // num_heads == 64, 'the attention kernels are built for head dim 64'
        self.embed_dims, self.num_heads = embed_dims, num_heads
        self.eps = float(norm_cfg.get('eps', 1e-5))
        self.ln1 = nn.LayerNorm(embed_dims, eps=self.eps)
        self.attn = _AttnContainer(embed_dims, num_heads, bias=qkv_bias, qk_norm=qk_norm)
        self.ln2 = nn.LayerNorm(embed_dims, eps=self.eps)
        self.ffn = _FFNContainer(embed_dims, feedforward_channels)
        self.qk_norm, self.act_q8 = bool(qk_norm), bool(act_q8)
        self._store = None

    @property
    def norm1(self):
        return self.ln1

    @property
    def norm2(self):
        return self.ln2

    def _params(self):
        ps = self.__dict__.get('_params_cache')
        if ps is None or ps[0] is not self.ln1.weight:
            ps = self.__dict__['_params_cache'] = self._build_params()
        return ps

    def _build_params(self):
        a, f = self.attn.attn, self.ffn.layers
        gains = (self.attn.q_norm.weight, self.attn.k_norm.weight) if self.qk_norm else ()
        return (self.ln1.weight, self.ln1.bias, a.in_proj_weight, a.in_proj_bias, a.out_proj.weight, a.out_proj.bias,
                self.ln2.weight, self.ln2.bias, f[0][0].weight, f[0][0].bias, f[1].weight, f[1].bias) + gains

    def forward(self, x, attn_mask=None, rope=None):
        store = self._store
        if store is None:
            raise S4FError('TransformerEncoderLayer must be run through VisionTransformer (it owns the ParamStore)')
        bu = rf = None
        bw = 0.0
        if attn_mask is not None:
            bu, rf, bw = attn_mask
        opt = None
        grad = torch.is_grad_enabled()                       # (inside LayerFn it never is)
        if self.qk_norm or rope is not None or (self.act_q8 and grad):
            cos, sin = rope if rope is not None else (None, None)
            opt = LayerOpt(self.qk_norm, cos, sin, self.act_q8, grad)
        return LayerFn.apply(x, bu, rf, float(bw), self.num_heads, self.eps, store, opt, *self._params())


# patch grids whose rotation tables a backbone keeps (256 bytes a token); the tables of further ones are made for each call
ROPE_GRIDS = 64


def axial_rope_tables(h, w, theta, device):
    """cos and sin fp32 [1 + h w, 32] of the rotation of queries and keys on an h x w patch grid: pairs 0..15 of a head turn with the patch's
    row, pairs 16..31 with its column, by theta^(-i / 16) radians a patch; the cls token is not turned.  Angles in 64 bits."""
    freq = float(theta) ** (-torch.arange(16, dtype=torch.float64) / 16)
    y, x = torch.meshgrid(torch.arange(h, dtype=torch.float64), torch.arange(w, dtype=torch.float64), indexing='ij')
    ang = torch.cat([y.reshape(-1, 1) * freq, x.reshape(-1, 1) * freq], -1)
    ang = torch.cat([torch.zeros(1, 32, dtype=torch.float64), ang])
    return ang.cos().float().to(device), ang.sin().float().to(device)


@BACKBONES.register_module()
class VisionTransformer(BaseModule):
    """reference vit.py:129-577 (DeiT-B / ViT for SETR).

    Options beyond the reference, all off by default (a student and its teacher take the same ones):
      qk_norm      RMS norm of every query and key head in front of the attention, with a learned gain [64] each for queries and keys
                   shared by the heads: bounds the attention logits, which bf16 training of larger models needs
      rope_theta   (e.g. 100.) queries and keys are turned by the row and column of their patch (axial_rope_tables), in addition to
                   the learned position embedding: attention sees relative positions
      act_q8       what only the backward pass reads of a layer's activations is kept in 8 bits (kernels.act_pack) and its weight
                   gradients are computed from that: 19 instead of 36 bytes a token and channel in bf16 mode.  The forward pass is
                   not changed; gradients carry the rounding of the kept activations."""

    def __init__(self, img_size=224, patch_size=16, in_channels=3, embed_dims=768, num_layers=12, num_heads=12, mlp_ratio=4,
                 out_indices=-1, qkv_bias=True, drop_rate=0., attn_drop_rate=0., drop_path_rate=0., with_cls_token=True,
                 output_cls_token=False, norm_cfg=dict(type='LN'), act_cfg=dict(type='GELU'), patch_norm=False,
                 final_norm=False, interpolate_mode='bicubic', num_fcs=2, norm_eval=False, with_cp=False, pretrained=None,
                 init_cfg=None, no_pos_embed=False, feature_ps_indices=0, w_PatchRelativeAttention=False,
                 qk_norm=False, rope_theta=None, act_q8=False):
        super().__init__(init_cfg=init_cfg)
        if isinstance(img_size, int):
            img_size = to_2tuple(img_size)
        elif isinstance(img_size, tuple):
            if len(img_size) == 1:
                img_size = to_2tuple(img_size[0])
            assert len(img_size) == 2, f'The size of image should have length 1 or 2, but got {len(img_size)}'
        if output_cls_token:
            assert with_cls_token is True, f'with_cls_token must be True if set output_cls_token to True, but got {with_cls_token}'
        assert not (init_cfg and pretrained), 'init_cfg and pretrained cannot be set at the same time'
        if isinstance(pretrained, str):
            warnings.warn('DeprecationWarning: pretrained is deprecated, please use "init_cfg" instead')
            self.init_cfg = dict(type='Pretrained', checkpoint=pretrained)
        elif pretrained is not None:
            raise TypeError('pretrained must be a str or None')
        if patch_size != 16 or in_channels != 3:
            raise S4FError('the patch-embed kernels are built for 16x16 RGB patches')
        if not with_cls_token or patch_norm or w_PatchRelativeAttention or with_cp:
            raise S4FError('with_cls_token=False / patch_norm / PatchRelativeAttention / with_cp are outside the SETR hot path')
        if rope_theta is not None and not 1.0 <= float(rope_theta) < math.inf:
            raise S4FError(f'rope_theta must be a finite number of at least 1, got {rope_theta}')
        self.qk_norm, self.act_q8 = bool(qk_norm), bool(act_q8)
        self.rope_theta = None if rope_theta is None else float(rope_theta)
        self._rope_tables = {}       # (h, w, device) -> (cos, sin)
        self.img_size, self.patch_size = tuple(img_size), patch_size
        self.interpolate_mode, self.norm_eval, self.with_cp = interpolate_mode, norm_eval, with_cp
        self.pretrained, self.num_heads, self.embed_dims = pretrained, num_heads, embed_dims
        self.no_pos_embed = no_pos_embed
        self.w_PatchRelativeAttention = False

        self.patch_embed = PatchEmbed(in_channels=in_channels, embed_dims=embed_dims, conv_type='Conv2d',
                                      kernel_size=patch_size, stride=patch_size, padding='corner', norm_cfg=None)
        num_patches = (img_size[0] // patch_size) * (img_size[1] // patch_size)
        self.with_cls_token, self.output_cls_token = with_cls_token, output_cls_token
        self.cls_token = nn.Parameter(torch.zeros(1, 1, embed_dims))
        self.pos_embed = nn.Parameter(torch.zeros(1, num_patches + 1, embed_dims))
        if drop_rate:
            raise S4FError('drop_rate must be 0 on the fused path')
        self.drop_after_pos = nn.Dropout(p=drop_rate)
        if isinstance(out_indices, int):
            if out_indices == -1:
                out_indices = num_layers - 1
            self.out_indices = [out_indices]
        elif isinstance(out_indices, (list, tuple)):
            self.out_indices = list(out_indices)
        else:
            raise TypeError('out_indices must be type of int, list or tuple')
        self.layers = ModuleList([
            TransformerEncoderLayer(embed_dims=embed_dims, num_heads=num_heads, feedforward_channels=mlp_ratio * embed_dims,
                                    attn_drop_rate=attn_drop_rate, drop_rate=drop_rate, drop_path_rate=0., num_fcs=num_fcs,
                                    qkv_bias=qkv_bias, act_cfg=act_cfg, norm_cfg=norm_cfg, with_cp=with_cp, batch_first=True,
                                    qk_norm=qk_norm, act_q8=act_q8)
            for _ in range(num_layers)])
        self.final_norm = final_norm
        if final_norm:
            raise S4FError('final_norm=True is not used by the SETR configs')
        self.multi_self_attn = None
        self._store = None          # set by the segmentor, or created lazily for a stand-alone backbone
        self._store_owner = False

    # ------------------------------------------------------------------ weights
    def init_weights(self):
        ck = self.init_cfg.get('checkpoint') if isinstance(self.init_cfg, dict) else None
        if isinstance(self.init_cfg, dict) and self.init_cfg.get('type') == 'Pretrained' and ck and os.path.exists(ck):
            # vit.py:369-393 (+ the README's mmcls key mapping when the file still has mmcls' names: checkpoint.py)
            from .checkpoint import load_backbone_pretrained
            load_backbone_pretrained(self, ck, convert='auto', strict=False)
            return
        if isinstance(self.init_cfg, dict) and self.init_cfg.get('type') == 'Pretrained':
            # the reference raises in CheckpointLoader.load_checkpoint; a silent random initialisation of student and teacher
            # behind a mistyped path is not an option (init_cfg allow_missing=True asks for it explicitly)
            if not self.init_cfg.get('allow_missing', False):
                raise FileNotFoundError(f'init_cfg checkpoint {ck!r} does not exist')
            warnings.warn(f'checkpoint {ck!r} not found: falling back to the random (jax_impl) initialisation')
        # vit.py:396-414
        trunc_normal_(self.pos_embed, std=.02)
        trunc_normal_(self.cls_token, std=.02)
        for n, m in self.named_modules():
            if isinstance(m, nn.Linear):
                trunc_normal_(m.weight, std=.02)
                if m.bias is not None:
                    if 'ffn' in n:
                        nn.init.normal_(m.bias, mean=0., std=1e-6)
                    else:
                        nn.init.constant_(m.bias, 0)
            elif isinstance(m, nn.Conv2d):
                kaiming_init(m, mode='fan_in', bias=0.)
            elif isinstance(m, (nn.modules.batchnorm._BatchNorm, nn.GroupNorm, nn.LayerNorm)):
                constant_init(m, val=1.0, bias=0.)
        if self._store is not None:
            self._store.mark_dirty()

    @staticmethod
    def resize_pos_embed(pos_embed, input_shpae, pos_shape, mode, no_pos_embed=False):
        """vit.py:447-477 (checkpoint-load / inference path; plain torch, not on the training hot path)."""
        assert pos_embed.ndim == 3, 'shape of pos_embed must be [B, L, C]'
        pos_h, pos_w = pos_shape
        cls_token_weight = pos_embed[:, 0:1]
        pos_embed_weight = pos_embed[:, (-1 * pos_h * pos_w):]
        pos_embed_weight = pos_embed_weight.reshape(1, pos_h, pos_w, pos_embed.shape[2]).permute(0, 3, 1, 2)
        pos_embed_weight = F.interpolate(pos_embed_weight, size=input_shpae, align_corners=False, mode=mode)
        pos_embed_weight = torch.flatten(pos_embed_weight, 2).transpose(1, 2)
        if no_pos_embed:
            pos_embed_weight = torch.zeros_like(pos_embed_weight)
        return torch.cat((cls_token_weight, pos_embed_weight), dim=1)

    # ------------------------------------------------------------------ store plumbing
    def _attach_store(self, store):
        self._store = store
        for layer in self.layers:
            layer._store = store

    def _ensure_store(self, device):
        if self._store is None:
            self._store_owner = True
            self._attach_store(ParamStore([('backbone', self, '')], with_grad=True))
        if self._store_owner:
            self._store.ensure(device, runtime.compute_dtype())
            self._store.ensure_grads()
            self._store.sync_shadow()
        return self._store

    @staticmethod
    def _rank1_mask(attn_mask, attn_mask_weight, adaptive_attn_mask):
        """vit.py:519-535 in rank-1 form: bias[b,i,j] = weight * u_j * flag_i (never materialised)."""
        B = attn_mask.size(0)
        u = attn_mask.reshape(B, -1).to(torch.float32)
        u = torch.cat((torch.zeros([B, 1], device=u.device), u), -1).contiguous()
        flag = None
        if adaptive_attn_mask:
            # if the patch is more confident than half (<half), it is not encouraged to change
            # u takes the values k / 256: the k-th smallest is often TIED with its neighbours, and which of the tied patches
            # torch.topk returns is implementation-defined (CPU: libstdc++ nth_element; GPU: radix select) - tied patches are
            # equally (un)confident, so either choice is the reference's semantics.  The selection stays on the device (no host
            # round trip in the step); the golden fixtures use batches whose top-k boundary is free of ties.  S4F_TOPK_TIES=cpu
            # reproduces the reference CPU path's choice for a tied batch (debugging aid: a host sync per step).
            k = int(0.5 * (u.size(-1) - 1))
            if os.environ.get('S4F_TOPK_TIES', 'device') == 'cpu':
                idx = (torch.topk(u[:, 1:].cpu(), k, dim=-1, largest=False)[1] + 1).to(u.device)
            else:
                idx = torch.topk(u[:, 1:], k, dim=-1, largest=False)[1] + 1
            flag = torch.ones_like(u)
            flag[torch.arange(B, device=u.device).unsqueeze(1), idx] = 0
        return u, flag, float(attn_mask_weight)

    # ------------------------------------------------------------------ forward
    def forward(self, inputs, no_pos_embed=False, avg_pos_emd=False, duplicate_pos_emd=False, use_fdrop=False,
                attn_mask=None, attn_mask_weight=0.0, adaptive_attn_mask=False):
        if no_pos_embed or avg_pos_emd or duplicate_pos_emd or use_fdrop:
            raise S4FError('position-embedding ablations / fdrop are outside the hot path (SURVEY §8)')
        mask = None
        if attn_mask is not None and self.with_cls_token:
            mask = self._rank1_mask(attn_mask, attn_mask_weight, adaptive_attn_mask)
        return self.forward_rank1(inputs, mask)

    def _rope(self, hw, device):
        if self.rope_theta is None:
            return None
        key = (*hw, torch.device(device))
        tab = self._rope_tables.get(key)
        if tab is None:
            tab = axial_rope_tables(*hw, self.rope_theta, device)
            if len(self._rope_tables) < ROPE_GRIDS:          # (a kept table is never dropped: another stream or a graph may read it)
                self._rope_tables[key] = tab
        return tab

    def forward_rank1(self, inputs, mask=None, tap_groups=None):
        """forward with the PASA mask already in rank-1 form (bias_u [B,N], row_flag [B,N] | None, weight) | None.
        The segmentor uses this to push several image groups (supervised, masked / plain unlabeled) through the
        backbone in ONE pass: every backbone op is per image, rows of images without a mask carry u = 0."""
        if not inputs.is_cuda:
            raise S4FError('VisionTransformer runs on the HIP kernels only: move the model and inputs to the GPU')
        store = self._ensure_store(inputs.device)
        x = self.patch_embed.pad(inputs.to(torch.float32)).contiguous()
        B, _, H, W = x.shape
        hw_shape = (H // self.patch_size, W // self.patch_size)
        pe = self.patch_embed.projection
        tokens = PatchEmbedFn.apply(x, pe.weight, pe.bias, self.cls_token, self.pos_embed, store)
        outs = []
        rope = self._rope(hw_shape, x.device)
        wait = self.__dict__.pop('_pre_layer_wait', None)   # (layer index, event): the part of this (teacher) model's weights that
        for i, layer in enumerate(self.layers):             # the EMA updates on the side stream (encoder_decoder.update_ema_variables)
            if wait is not None and i == wait[0]:
                torch.cuda.current_stream().wait_event(wait[1])
            tokens = layer(tokens, mask, rope)
            if i in self.out_indices:
                parts = None
                if tap_groups is not None:
                    tokens, parts = self._split_tap(tokens, tap_groups, chain=i + 1 < len(self.layers))
                o = self.tap_view(tokens, hw_shape)
                if parts is not None:
                    (o[0] if isinstance(o, list) else o)._s4f_parts = (tuple(tap_groups), parts)
                outs.append(o)
        self.multi_self_attn = [[], hw_shape]
        return tuple(outs)

    def tap_view(self, tokens, hw_shape):
        """[B, C, h, w] view of the patch tokens (vit.py:555-562 without the copy); the token tensor rides along so
        that the SETR head can read it token-major"""
        B, _, C = tokens.shape
        out = tokens[:, 1:].reshape(B, hw_shape[0], hw_shape[1], C).permute(0, 3, 1, 2)
        out._s4f_tokens = tokens
        out._s4f_grid = hw_shape
        if self.output_cls_token:
            out = [out, tokens[:, 0]]
        return out

    def split_taps(self, outs, a, b):
        """taps of the images [a, b) of a multi-group pass"""
        res = []
        for o in outs:
            t = o._s4f_tokens[a:b]
            res.append(self.tap_view(t, o._s4f_grid))
        return tuple(res)

    @staticmethod
    def _split_tap(tok, bounds, chain):
        """(tokens for the chain, group views) of one tap; None for the views when the shared-gradient node does not apply"""
        from .functional import TAP_SPLIT, TapSplitFn, _TapGrad
        if not (TAP_SPLIT and tok.requires_grad and torch.is_grad_enabled() and tok.is_cuda):
            return tok, None
        holder = _TapGrad(tok, bounds)
        res = TapSplitFn.apply(tok, holder, chain)
        nxt, parts = (res[0], res[1:]) if chain else (tok, res)
        for gi, t in enumerate(parts):
            t._s4f_tapdst = (holder, gi)
        return nxt, parts

    def split_taps_multi(self, outs, bounds):
        """taps of several image groups [a, b) of a multi-group pass at once: list (per group) of tap tuples.  With gradients
        the groups of a tap share ONE gradient buffer that the heads write directly (functional.TapSplitFn); a pass that was
        given `tap_groups` has made the split where the tap leaves the chain (forward_rank1)."""
        bounds = tuple((int(a), int(b)) for a, b in bounds)
        res = [[] for _ in bounds]
        for o in outs:
            o0 = o[0] if isinstance(o, list) else o
            pre = getattr(o0, '_s4f_parts', None)
            if pre is not None and pre[0] == bounds:
                parts = pre[1]
            else:
                _, parts = self._split_tap(o0._s4f_tokens, bounds, chain=False)
                if parts is None:
                    parts = [o0._s4f_tokens[a:b] for a, b in bounds]
            for gi, t in enumerate(parts):
                res[gi].append(self.tap_view(t, o0._s4f_grid))
        return [tuple(r) for r in res]

    def train(self, mode=True):
        super().train(mode)
        return self
