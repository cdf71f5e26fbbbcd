"""Argument checks of the top-logit, bucketed-bias and trainable window-attention entry points: the C entry points return their error before any launch
(so a GPU is not needed, and the pointers are never followed), the plan of a bucket map is checked where it is built, CPU tensors are refused."""
import math

import pytest
import torch

NULL, P = None, 4096                 # a pointer value that is 16-byte aligned and never followed
OK, E_NULL, E_SHAPE, E_DTYPE, E_WS, E_ALIGN, E_UNSUP = 0, -1, -2, -3, -4, -5, -6


@pytest.fixture(scope='module')
def L():
    from segdistill_amd import _lib
    return _lib.lib()


def test_topk_select_refusals(L):
    def call(x=P, v=P, i=P, r=P, dt=0, B=2, C=10, p=1, k=3, tau=1.0):
        return L.sd_topk_select(x, v, i, r, dt, B, C, p, k, tau, NULL)
    assert L.sd_topk_max_entries() == 128 and L.sd_topk_max_classes() == 262144
    for a in 'xvir':
        assert call(**{a: NULL}) == E_NULL
    assert call(dt=2) == E_DTYPE and call(dt=-1) == E_DTYPE
    for kw in (dict(B=0), dict(B=-1), dict(C=0), dict(p=0), dict(k=0), dict(k=11), dict(tau=0.0), dict(tau=-1.0), dict(tau=math.nan), dict(tau=math.inf), dict(B=2 ** 31),
               dict(p=2 ** 31)):
        assert call(**kw) == E_SHAPE, kw
    assert call(C=300, k=129) == E_UNSUP and call(C=262145) == E_UNSUP
    assert call(x=P + 2) == E_ALIGN and call(i=P + 2) == E_ALIGN and call(r=P + 1) == E_ALIGN and call(dt=1, v=P + 1) == E_ALIGN
    assert call(B=2 ** 31 - 1, C=5000) == E_SHAPE and call(B=2 ** 20, p=2 ** 20) == E_SHAPE              # more workgroups than a launch holds


def test_topk_kl_refusals(L):
    ws = L.sd_topk_kl_workspace_bytes(2, 10, 6, 3)
    assert ws >= 16 and L.sd_topk_kl_workspace_bytes(0, 10, 6, 3) == 0 and L.sd_topk_kl_workspace_bytes(2, 10, 6, 129) == 0

    def fwd(S=P, v=P, i=P, r=NULL, ok=NULL, dt=0, vdt=0, B=2, C=10, p=6, k=3, tau=1.0, st=P, n=P, loss=P, w=P, wb=ws):
        return L.sd_topk_kl_fwd(S, v, i, r, ok, dt, vdt, B, C, p, k, tau, 1.0, st, n, loss, w, wb, NULL)

    def bwd(S=P, v=P, i=P, r=NULL, ok=NULL, dt=0, vdt=0, B=2, C=10, p=6, k=3, tau=1.0, st=P, n=P, up=P, d=P):
        return L.sd_topk_kl_bwd(S, v, i, r, ok, dt, vdt, B, C, p, k, tau, 1.0, st, n, up, d, NULL)
    for f, names in ((fwd, ('S', 'v', 'i', 'st', 'n', 'loss', 'w')), (bwd, ('S', 'v', 'i', 'st', 'n', 'up', 'd'))):
        for a in names:
            assert f(**{a: NULL}) == E_NULL, a
        assert f(dt=2) == E_DTYPE and f(vdt=3) == E_DTYPE
        for kw in (dict(B=0), dict(C=-1), dict(p=0), dict(k=0), dict(tau=0.0), dict(tau=math.nan)):
            assert f(**kw) == E_SHAPE, kw
        assert f(k=129) == E_UNSUP and f(C=262145, p=1) == E_UNSUP and f(C=8000) == E_UNSUP       # class planes: bits of 8000 classes per pixel do not fit LDS
        assert f(S=P + 1) == E_ALIGN and f(st=P + 4) == E_ALIGN and f(vdt=1, v=P + 1) == E_ALIGN and f(r=P + 2) == E_ALIGN
    assert fwd(wb=ws - 1) == E_WS and fwd(w=P + 4) == E_WS and bwd(d=P + 2) == E_ALIGN
    assert L.sd_topk_kl_supported(8, 150, 16384, 128) and L.sd_topk_kl_supported(4, 262144, 1, 128) and not L.sd_topk_kl_supported(2 ** 40, 150, 1, 3)
    for C in (1, 31, 32, 33, 150, 1760):                                     # what is called supported fits the LDS that a launch may ask for
        for k in (1, 10, 64, 128):
            assert L.sd_topk_kl_supported(1, C, 7, k)


def test_bucket_bias_refusals(L):
    c = L.sd_bucket_bias_chunk()
    from segdistill_amd import rel_bias
    assert c == rel_bias.CHUNK and L.sd_bucket_bias_workspace_bytes(7, 7, 3) == 0 and L.sd_bucket_bias_workspace_bytes(7, 9, 3) == 9 * 3 * 4

    def fwd(t=P, i=P, o=P, dt=0, nb=7, h=3, n=100):
        return L.sd_bucket_bias_fwd(t, i, o, dt, nb, h, n, NULL)

    def bwd(d=P, o=P, cs=P, co=P, bc=P, t=P, dt=0, nb=7, ch=9, h=3, n=100, w=P, wb=9 * 3 * 4):
        return L.sd_bucket_bias_bwd(d, o, cs, co, bc, t, dt, nb, ch, h, n, w, wb, NULL)
    assert fwd(t=NULL) == fwd(i=NULL) == fwd(o=NULL) == E_NULL and fwd(dt=9) == E_DTYPE
    assert fwd(nb=0) == fwd(h=0) == fwd(n=0) == fwd(n=2 ** 31) == fwd(h=65536) == E_SHAPE and fwd(t=P + 2) == E_ALIGN and fwd(i=P + 2) == E_ALIGN
    for a in ('d', 'o', 'cs', 'co', 'bc', 't'):
        assert bwd(**{a: NULL}) == E_NULL
    assert bwd(dt=9) == E_DTYPE and bwd(ch=6) == E_SHAPE and bwd(nb=0) == E_SHAPE and bwd(w=NULL) == E_WS and bwd(wb=4) == E_WS and bwd(d=P + 2) == E_ALIGN


def test_window_attention_refusals(L):
    ok = L.sd_window_attn_train_supported
    assert ok(1, 32) and ok(49, 32) and ok(64, 32) and not ok(0, 32) and not ok(65, 32) and not ok(49, 64)
    ws, pk = L.sd_window_attn_train_workspace_bytes(0, 6, 3, 49), L.sd_window_attn_train_packed_floats(3, 2, 49)
    assert ws > 0 and L.sd_window_attn_train_workspace_bytes(0, 6, 3, 65) == 0 and L.sd_window_attn_train_workspace_bytes(0, 0, 3, 49) == 0
    assert L.sd_window_attn_train_workspace_bytes(2, 6, 3, 49) == 0 and pk == 5 * 4096 + 2 * 4 and L.sd_window_attn_train_packed_floats(3, -1, 49) == 0

    def fwd(q=P, b=P, m=NULL, k=P, kf=pk, o=P, dt=0, w=6, nw=0, h=3, n=49, d=32):
        return L.sd_window_attn_train_fwd(q, b, m, k, kf, o, dt, w, nw, h, n, d, 1.0, NULL)

    def bwd(q=P, k=P, kf=pk, g=P, dq=P, db=P, dt=0, w=6, nw=0, h=3, n=49, d=32, s=P, sb=ws):
        return L.sd_window_attn_train_bwd(q, k, kf, g, dq, db, dt, w, nw, h, n, d, 1.0, s, sb, NULL)
    for f, names in ((fwd, 'qbko'), (bwd, ('q', 'k', 'g', 'dq', 'db'))):
        for a in names:
            assert f(**{a: NULL}) == E_NULL, a
        assert f(dt=2) == E_DTYPE and f(n=65) == E_UNSUP and f(n=0) == E_UNSUP and f(d=16) == E_UNSUP
        assert f(w=0) == f(h=0) == f(w=2 ** 40) == f(nw=4) == f(nw=-1) == E_SHAPE and f(kf=10) == E_WS and f(nw=3) == E_WS
        assert f(q=P + 4) == E_ALIGN and f(k=P + 4) == E_ALIGN
    assert fwd(nw=2) == E_NULL and fwd(nw=2, m=P + 2) == E_ALIGN and fwd(b=P + 2) == E_ALIGN
    assert bwd(s=NULL) == E_WS and bwd(sb=ws - 1) == E_WS and bwd(s=P + 8) == E_WS and bwd(g=P + 8) == E_ALIGN and fwd(o=P + 8) == E_ALIGN


def test_bucket_plan_orders_every_pair_once_and_refuses_bad_maps():
    from segdistill_amd import rel_bias
    g = torch.Generator().manual_seed(0)
    index = (torch.rand(70, 60, generator=g) ** 2 * 6).long()
    index[index == 3] = 2
    plan = rel_bias.BucketPlan(index, 8)                                    # buckets 3, 6 and 7 are empty
    assert sorted(plan.order.tolist()) == list(range(4200)) and plan.bucket_chunk[0] == 0 and plan.bucket_chunk[-1] == plan.chunk_start.numel() - 1
    assert sorted(plan.chunk_order.tolist()) == list(range(plan.chunk_start.numel() - 1))
    for b in range(8):
        lo, hi = plan.bucket_chunk[b].item(), plan.bucket_chunk[b + 1].item()
        assert hi > lo
        cuts = plan.chunk_start[lo:hi + 1].tolist()
        assert all(0 <= y - x <= 512 for x, y in zip(cuts, cuts[1:]))
        mine = plan.order[cuts[0]:cuts[-1]].tolist()
        assert mine == (index.view(-1) == b).nonzero().view(-1).tolist()
    for bad in (index + 3, index - 1, index.float(), index > 2, index.view(-1), index[:0]):
        with pytest.raises(ValueError):
            rel_bias.BucketPlan(bad, 8)


def test_cpu_tensors_are_refused():
    from segdistill_amd import ops, rel_bias, window_attn
    from segdistill_amd.distillation.losses import TopKLoss
    x = torch.zeros(2, 5)
    with pytest.raises(RuntimeError, match='GPU only'):
        ops.topk_logits(x, 2)
    with pytest.raises(RuntimeError, match='GPU only'):
        ops.topk_kl(x, x[:, :2], torch.zeros(2, 2, dtype=torch.int32), tau=1.0, alpha=1.0)
    with pytest.raises(RuntimeError, match='GPU only'):
        rel_bias.bucket_bias(torch.zeros(3, 2), rel_bias.BucketPlan(torch.zeros(2, 2, dtype=torch.long), 3))
    with pytest.raises(RuntimeError, match='GPU only'):
        window_attn.attention(torch.zeros(1, 4, 96), torch.zeros(1, 4, 4), None, 1, 1.0)
    with pytest.raises(RuntimeError, match='GPU only'):
        TopKLoss(k=2)(torch.zeros(1, 3, 2, 2), torch.zeros(1, 3, 2, 2), torch.zeros(1, 1, 4, 4), 1)


def test_temperatures_whose_reciprocal_is_no_normal_number_are_refused(L):
    from segdistill_amd import ops
    for tau in (1e-39, 3e-39, 2e38, 3.4e38):
        assert L.sd_topk_select(P, P, P, P, 0, 2, 10, 1, 3, tau, NULL) == E_SHAPE
        assert L.sd_topk_kl_fwd(P, P, P, NULL, NULL, 0, 0, 2, 10, 6, 3, tau, 1.0, P, P, P, P, 1 << 20, NULL) == E_SHAPE
    for tau in (1e-38, 1e38, 0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match='tau'):
            ops._check_tau(tau)
    assert ops._check_tau(1) == 1.0 and ops._check_tau(1e-3) == 1e-3


def test_window_attention_built_on_the_meta_device_gets_its_plan_with_the_loaded_index():
    from segdistill_amd.backbones.swin import WindowAttention
    real = WindowAttention(64, (3, 4), 2)
    for assign in (False, True):
        with torch.device('meta'):
            att = WindowAttention(64, (3, 4), 2)
        assert att.bias_plan is None and set(att.state_dict()) == set(real.state_dict())
        if not assign:
            att.to_empty(device='cpu')
        att.load_state_dict(real.state_dict(), assign=assign)
        for name, t in real.bias_plan.named_buffers():
            assert torch.equal(t, dict(att.bias_plan.named_buffers())[name]), name
    x = torch.randn(4, 12, 64)
    assert torch.equal(att(x), real(x))


def test_more_masks_than_one_launch_packs_are_refused(L):
    for w, h, want in ((1 << 24, 1, E_SHAPE), ((1 << 24) - 1, 1, E_SHAPE), ((1 << 24) - 2, 1, E_WS), ((1 << 24) - 2, 2, E_SHAPE)):
        assert L.sd_window_attn_train_fwd(P, P, P, P, 10, P, 0, w, w, h, 1, 32, 1.0, NULL) == want, (w, h)
        assert L.sd_window_attn_train_bwd(P, P, 10, P, P, P, 0, w, w, h, 1, 32, 1.0, P, 1 << 40, NULL) == want, (w, h)
