"""A learned position bias by buckets and its gradient (csrc/rel_bias.hip; reference mmseg/models/backbones/swin_transformer.py:133-135, where the buckets
are the (dy, dx) offsets of a window's tokens).  Autograd of `table[index]` scatters with atomics, in an order of its own each time; here the pairs are
ordered by bucket once (`BucketPlan`) and the gradient is a sum over each bucket's pairs in that order."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .ops import _DT, _addressless, _launch, _no_double_backward, _ptr, _require_gpu, _transformed


CHUNK = 512          # sd_bucket_bias_chunk(): the pairs of one bucket that one wave sums (a plan is built without the library)


class BucketPlan(nn.Module):
    """The (query, key) pairs of `index` [Nq, Nk] (integers in [0, num_buckets)) in the order the gradient sums them.  Built once per index: it reads the
    index on the host.  A module without parameters or state-dict entries, so that a model that holds one moves it along.  A captured graph reads the plan's
    memory: `update` gives it another index, and the plan has to live as long as the graph."""

    def __init__(self, index, num_buckets):
        super().__init__()
        if index.dim() != 2 or index.is_floating_point() or index.is_complex() or index.dtype == torch.bool or index.numel() == 0:
            raise ValueError(f'BucketPlan: index must be a non-empty integer [Nq, Nk], got {index.dtype} {tuple(index.shape)}')
        nb = int(num_buckets)
        if index.numel() > 2 ** 31 - 1:
            raise ValueError('BucketPlan: more than 2^31 - 1 pairs')
        with torch.inference_mode(False):                                    # buffers that a backward may keep, wherever the plan is built
            self._order(index, nb)

    def _order(self, index, nb):
        flat = index.detach().reshape(-1).long()
        lo, hi = torch.stack(torch.aminmax(flat)).tolist()
        if lo < 0 or hi >= nb:
            raise ValueError(f'BucketPlan: index holds {lo} .. {hi}, outside [0, {nb})')
        order = torch.sort(flat, stable=True).indices
        count = torch.bincount(flat, minlength=nb)
        chunks = ((count + CHUNK - 1) // CHUNK).clamp(min=1)               # an empty bucket: one empty chunk
        first = torch.cumsum(chunks, 0)
        bucket_chunk = torch.cat([first.new_zeros(1), first])
        owner = torch.repeat_interleave(torch.arange(nb, device=flat.device), chunks)
        within = torch.arange(owner.numel(), device=flat.device) - bucket_chunk[owner]
        start = (torch.cumsum(count, 0) - count)[owner] + within * CHUNK
        self.num_buckets, self.num_chunks, self.num_pairs, self.shape = nb, owner.numel(), flat.numel(), tuple(index.shape)
        self.register_buffer('index', flat.int().view(index.shape), persistent=False)
        self.register_buffer('order', order.int(), persistent=False)
        self.register_buffer('chunk_start', torch.cat([start, start.new_tensor([flat.numel()])]).int(), persistent=False)
        self.register_buffer('bucket_chunk', bucket_chunk.int(), persistent=False)
        first_pair = order[start.clamp(max=flat.numel() - 1)]
        self.register_buffer('chunk_order', torch.sort(first_pair, stable=True).indices.int(), persistent=False)

    def update(self, index):
        """Take another index of the same shape and number of buckets, written where the old one is: a captured graph that reads this plan reads the new
        one.  False, and nothing written, if the new index needs another number of chunks or lies on another device (then: a new plan)."""
        new = BucketPlan(index, self.num_buckets)
        if new.shape != self.shape or new.num_chunks != self.num_chunks or new.index.device != self.index.device:
            return False
        with torch.no_grad():
            for name, b in self.named_buffers():
                b.copy_(getattr(new, name))
        return True

    def extra_repr(self):
        return f'{self.shape[0]} x {self.shape[1]} pairs in {self.num_buckets} buckets'


class _BucketBiasFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, plan, create_graph):
        nb, heads = table.shape
        held = tuple(plan._buffers[n] for n in ('index', 'order', 'chunk_start', 'chunk_order', 'bucket_chunk'))
        out = torch.empty((heads,) + plan.shape, dtype=table.dtype, device=table.device)
        rc = _launch(table.device, _lib.lib().sd_bucket_bias_fwd, table.data_ptr(), held[0].data_ptr(), out.data_ptr(), _DT[table.dtype], nb, heads, plan.num_pairs)
        _lib.check(rc, 'sd_bucket_bias_fwd')
        ctx.plan, ctx.create_graph = plan, create_graph
        ctx.save_for_backward(*held)                   # (the plan may move meanwhile, or be updated: an error)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        plan = ctx.plan
        index, order, start, by_pair, bucket = ctx.saved_tensors
        if ctx.create_graph and (torch.is_grad_enabled() or _addressless(grad_out)):
            d = grad_out.reshape(grad_out.shape[0], -1).t().float()
            return d.new_zeros(plan.num_buckets, d.shape[1]).index_add(0, index.reshape(-1), d).to(grad_out.dtype), None, None
        _no_double_backward('bucket_bias')
        nb, chunks = plan.num_buckets, plan.num_chunks
        d = grad_out.contiguous()
        heads = d.shape[0]
        L = _lib.lib()
        dtable = torch.empty(nb, heads, dtype=d.dtype, device=d.device)
        ws_bytes = L.sd_bucket_bias_workspace_bytes(nb, chunks, heads) if chunks > nb else 0
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=d.device) if ws_bytes else None
        rc = _launch(d.device, L.sd_bucket_bias_bwd, d.data_ptr(), order.data_ptr(), start.data_ptr(), by_pair.data_ptr(), bucket.data_ptr(),
                     dtable.data_ptr(), _DT[d.dtype], nb, chunks, heads, plan.num_pairs, _ptr(ws), ws_bytes)
        _lib.check(rc, 'sd_bucket_bias_bwd')
        return dtable, None, None


def supported(table):
    """bucket_bias takes a table of this type on this device, and no transform (torch.func, forward mode) is on."""
    return table.is_cuda and table.dtype in _DT and not _transformed()


def bucket_bias(table, plan, create_graph=False):
    """table [num_buckets, heads] (fp32 or bf16) -> bias [heads, Nq, Nk] = table[index].permute(2, 0, 1), with a deterministic gradient for the table.
    create_graph: the gradient may be asked for with a graph of its own, or for a batch of gradients at once (then by torch operators); without, that is an
    error."""
    _require_gpu(table)
    if table.dtype not in _DT:
        raise TypeError(f'bucket_bias: unsupported dtype {table.dtype}')
    if table.dim() != 2 or table.shape[0] != plan.num_buckets or table.shape[1] == 0:
        raise ValueError(f'bucket_bias: table {tuple(table.shape)} does not fit a plan of {plan.num_buckets} buckets')
    if plan._buffers['index'].device != table.device:
        raise ValueError(f'bucket_bias: the plan is on {plan.index.device}, the table on {table.device}')
    return _BucketBiasFunction.apply(table.contiguous(), plan, create_graph)
