"""Window attention of a Swin block.  `attention`: with its gradients (csrc/window_train.hip; a Swin student).  The rest: without an autograd graph (the frozen teacher of BASELINE config 4) as ONE kernel over the qkv Linear's
output (csrc/window_attn.hip; reference mmseg/models/backbones/swin_transformer.py:119-153): relative position bias and shift mask are read
from small packed tables inside the kernel, q / k / v are not permuted and the output comes out token-major for the projection."""
from __future__ import annotations

import math
import os

import torch

from . import _lib
from .ops import _DT, _addressless, _launch, _ptr, _require_gpu, _stream_ptr, _transformed

ENABLED = os.environ.get('SEGDISTILL_WINDOW_ATTN', '1') == '1'       # A/B: 0 = F.scaled_dot_product_attention with a materialised additive tensor


def supported(qkv, n, heads, head_dim):
    """qkv: the qkv Linear's output [windows, N, 3*heads*D]."""
    return bool(ENABLED and qkv.is_cuda and qkv.dtype == torch.float32 and qkv.numel() > 0 and qkv.dim() == 3
                and _lib.lib().sd_window_attn_supported(int(n), int(head_dim)))


def pack_tables(tables, pad_key=0.0, want_flags=False):
    """[n, 49, 49] additive tables in the reference's orientation ([query, key]) -> ([n, 4096] in the MFMA kernel's accumulator layout,
    int32 flags [n] = table has a nonzero entry, or None)."""
    t = tables.detach().float().contiguous()
    n = t.shape[0]
    assert t.shape[1:] == (49, 49)
    L = _lib.lib()
    packed = torch.empty(n, int(L.sd_window_attn_packed_floats()), dtype=torch.float32, device=t.device)
    flags = torch.empty(n, dtype=torch.int32, device=t.device) if want_flags else None
    _lib.check(L.sd_window_attn_pack(t.data_ptr(), packed.data_ptr(), None if flags is None else flags.data_ptr(), n, 49, float(pad_key), _stream_ptr()),
               'sd_window_attn_pack')
    return packed, flags


def forward_packed(qkv, bias_p, mask_p, mask_flags, heads, scale):
    """qkv [windows, 49, 3*heads*32] (contiguous fp32); bias_p = pack_tables(bias [heads, 49, 49], -inf)[0]; mask_p, mask_flags =
    pack_tables(mask [nW, 49, 49], 0, True) or (None, None) -> [windows, 49, heads*32]."""
    bw, n, c3 = qkv.shape
    c = c3 // 3
    assert qkv.is_contiguous() and bias_p.shape[0] == heads
    out = torch.empty(bw, n, c, dtype=qkv.dtype, device=qkv.device)
    rc = _lib.lib().sd_window_attn_fwd_packed(qkv.data_ptr(), bias_p.data_ptr(), None if mask_p is None else mask_p.data_ptr(),
                                              None if mask_p is None else mask_flags.data_ptr(), out.data_ptr(), _DT[qkv.dtype], bw,
                                              0 if mask_p is None else mask_p.shape[0], heads, n, c // heads, float(scale), _stream_ptr())
    _lib.check(rc, 'sd_window_attn_fwd_packed')
    return out


def train_supported(qkv, n, head_dim):
    """The training kernels take this qkv Linear output [windows, N, 3*heads*head_dim]: fp32 or bf16, windows of up to 64 tokens, head_dim 32; and no transform
    (torch.func, forward mode) is on."""
    return bool(ENABLED and qkv.is_cuda and qkv.dtype in _DT and qkv.dim() == 3 and not _transformed()
                and _lib.lib().sd_window_attn_train_supported(int(n), int(head_dim)))


def _version(t):
    """the counter of writes in place; None where there is none (no tensor, or one made in inference mode)"""
    return None if t is None or t.is_inference() else t._version


def _probabilities(qkv, bias, mask, heads, scale):
    """q, k, v [windows, heads, N, D] and the softmax of their scores, in fp32 (fp64 where qkv is) by torch operators"""
    bw, n, c3 = qkv.shape
    wide = torch.promote_types(qkv.dtype, torch.float32)
    q, k, v = (t.contiguous() for t in qkv.to(wide).reshape(bw, n, 3, heads, c3 // 3 // heads).permute(2, 0, 3, 1, 4))
    s = q @ k.transpose(-2, -1).contiguous() * scale + bias.to(wide)
    if mask is not None:
        s = (s.view(bw // mask.shape[0], mask.shape[0], heads, n, n) + mask.detach().to(wide).unsqueeze(1)).view(bw, heads, n, n)
    nothing = (s == -math.inf).all(-1, keepdim=True)
    return q, k, v, torch.softmax(s.masked_fill(nothing, 0.), -1).masked_fill(nothing, 0.)


def plain_attention(qkv, bias, mask, heads, scale):
    """`attention` by torch operators that every transform (torch.func, forward mode) knows.  (The library's fused attention is not one of them: per-sample
    gradients of its additive tensor are wrong from the second sample on.)"""
    with torch.autocast(qkv.device.type, enabled=False):
        _, _, v, p = _probabilities(qkv, bias, mask, heads, scale)
        return (p @ v).transpose(1, 2).reshape(qkv.shape[0], qkv.shape[1], -1).to(qkv.dtype)


def _plain_gradients(qkv, bias, mask, heads, scale, grad_out):
    """The gradients (csrc/window_train.hip) by torch operators in fp32, which differentiate further and take batches of gradients."""
    bw, n, c3 = qkv.shape
    with torch.autocast(qkv.device.type, enabled=False):
        q, k, v, p = _probabilities(qkv, bias, mask, heads, scale)
        g = grad_out.float().reshape(bw, n, heads, -1).transpose(1, 2).contiguous()
        dp = g @ v.transpose(-2, -1).contiguous()
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dqkv = torch.stack([ds @ k * scale, ds.transpose(-2, -1).contiguous() @ q * scale, p.transpose(-2, -1).contiguous() @ g])
        return dqkv.permute(1, 3, 0, 2, 4).reshape(bw, n, c3).to(qkv.dtype), ds.sum(0).to(bias.dtype)


class _WindowAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, bias, mask, heads, scale):
        bw, n, c3 = qkv.shape
        nw, dt, L = (0 if mask is None else mask.shape[0]), _DT[qkv.dtype], _lib.lib()
        b = bias.detach().to(torch.float32).contiguous()
        m = None if mask is None else mask.to(torch.float32).contiguous()
        floats = L.sd_window_attn_train_packed_floats(heads, nw, n)
        packed = torch.empty(floats, dtype=torch.float32, device=qkv.device)
        out = torch.empty(bw, n, c3 // 3, dtype=qkv.dtype, device=qkv.device)
        rc = _launch(qkv.device, L.sd_window_attn_train_fwd, qkv.data_ptr(), b.data_ptr(), _ptr(m), packed.data_ptr(), floats, out.data_ptr(), dt, bw, nw, heads,
                     n, c3 // 3 // heads, scale)
        _lib.check(rc, 'sd_window_attn_train_fwd')
        ctx.save_for_backward(qkv, packed)
        ctx.meta = (nw, heads, scale, bias.dtype)
        ctx.tables = (bias, mask, _version(bias), _version(mask))          # `packed` has what the kernel needs: these may change, unless a graph is asked for
        return out

    @staticmethod
    def backward(ctx, grad_out):
        qkv, packed = ctx.saved_tensors
        nw, heads, scale, bias_dtype = ctx.meta
        if torch.is_grad_enabled() or _addressless(grad_out):
            bias, mask, *versions = ctx.tables
            if versions != [_version(bias), _version(mask)]:
                raise RuntimeError('window_attn.attention: bias or mask was modified by an inplace operation between the forward and a backward with a graph of its own')
            return (*_plain_gradients(qkv, bias, mask, heads, scale, grad_out), None, None, None)
        bw, n, c3 = qkv.shape
        L, dt = _lib.lib(), _DT[qkv.dtype]
        go = grad_out.to(qkv.dtype).contiguous()
        if go.data_ptr() % 16:
            go = go.clone()
        dqkv = torch.empty_like(qkv)
        dbias = torch.empty(heads, n, n, dtype=torch.float32, device=qkv.device)
        ws_bytes = L.sd_window_attn_train_workspace_bytes(dt, bw, heads, n)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
        rc = _launch(qkv.device, L.sd_window_attn_train_bwd, qkv.data_ptr(), packed.data_ptr(), packed.numel(), go.data_ptr(), dqkv.data_ptr(), dbias.data_ptr(), dt,
                     bw, nw, heads, n, c3 // 3 // heads, scale, ws.data_ptr(), ws_bytes)
        _lib.check(rc, 'sd_window_attn_train_bwd')
        return dqkv, dbias.to(bias_dtype), None, None, None


def attention(qkv, bias, mask, heads, scale):
    """softmax(scale * q k^T + bias[head] + mask[window % nW]) v for every window and head, with gradients for qkv and bias.

    qkv [windows, N, 3*heads*32] (fp32 or bf16) as the qkv Linear leaves it, N <= 64; bias [heads, N, N]; mask [nW, N, N] additive, without a gradient
    (windows of one image are contiguous and nW divides their number), or None -> [windows, N, heads*32].  A query row that bias + mask leave at -inf
    everywhere has output 0 and no gradient.  A gradient with a graph of its own (create_graph), or for a batch of gradients at once, is taken by torch
    operators."""
    _require_gpu(qkv, bias)
    heads = int(heads)
    if qkv.dim() != 3 or heads <= 0 or qkv.shape[2] % (3 * heads):
        raise ValueError(f'attention: qkv must be [windows, N, 3 * heads * head_dim], got {tuple(qkv.shape)} for {heads} heads')
    bw, n, c3 = qkv.shape
    if qkv.dtype not in _DT:
        raise TypeError(f'attention: unsupported dtype {qkv.dtype}')
    if not _lib.lib().sd_window_attn_train_supported(n, c3 // 3 // heads):
        raise ValueError(f'attention: windows of {n} tokens with head_dim {c3 // 3 // heads} are not supported (1 .. 64 tokens, head_dim 32)')
    if tuple(bias.shape) != (heads, n, n) or not bias.is_floating_point():
        raise ValueError(f'attention: bias must be a floating [{heads}, {n}, {n}], got {bias.dtype} {tuple(bias.shape)}')
    if mask is not None:
        if mask.dim() != 3 or tuple(mask.shape[1:]) != (n, n) or mask.shape[0] == 0 or bw % mask.shape[0] or not mask.is_floating_point():
            raise ValueError(f'attention: mask must be a floating [nW, {n}, {n}] with nW dividing {bw}, got {mask.dtype} {tuple(mask.shape)}')
        if mask.requires_grad:
            raise ValueError('attention: the mask has no gradient')
    if any(t is not None and t.device != qkv.device for t in (bias, mask)):
        raise ValueError('attention: operands on different devices')
    if bw == 0:
        return qkv[..., :c3 // 3] * bias.sum().to(qkv.dtype)           # empty, and so are its gradients
    qkv = qkv.contiguous()
    if qkv.data_ptr() % 16:
        qkv = qkv.clone()
    return _WindowAttentionFunction.apply(qkv, bias, mask, heads, float(scale))
