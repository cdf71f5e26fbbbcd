"""A Swin student: the attention of a trainable block on csrc/window_train.hip with the bias table through csrc/rel_bias.hip, against the same modules in
fp64 on the CPU, and a KD step of such a student against its teacher's top logits (TopKLoss), eager and as a replayed graph."""
import copy
import math
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu


def _layer(ws, dim=96, heads=3):
    from segdistill_amd.backbones.swin import BasicLayer
    torch.manual_seed(3)
    layer = BasicLayer(dim=dim, depth=2, num_heads=heads, window_size=ws)
    for blk in layer.blocks:
        torch.nn.init.normal_(blk.attn.relative_position_bias_table, std=0.5)
    return layer.train()


@pytest.mark.parametrize('ws,hw,amp', [(7, (28, 28), False), (7, (30, 26), False), (5, (12, 13), False), (8, (16, 24), False), (7, (30, 26), True), (9, (18, 20), False)])
def test_trainable_stage_matches_the_modules_in_fp64(ws, hw, amp, monkeypatch):
    """unshifted + shifted block, whole and padded windows, window sizes 5 / 7 / 8 on the kernel (9: 81 tokens, the library's attention with the bucketed
    bias).  Two blocks with their Linears, norms and GELU: fp32 2e-5 of the largest value, bf16 autocast 4e-2."""
    from segdistill_amd import rel_bias, window_attn
    layer = _layer(ws)
    ref = copy.deepcopy(layer).double()
    layer = layer.cuda()
    calls, gathers = [], []
    real, bias = window_attn.attention, rel_bias.bucket_bias
    monkeypatch.setattr(window_attn, 'attention', lambda *a: (calls.append(a[0].dtype), real(*a))[1])
    monkeypatch.setattr(rel_bias, 'bucket_bias', lambda *a: (gathers.append(1), bias(*a))[1])
    h, w = hw
    x = torch.randn(2, h * w, 96)
    d = torch.randn(2, h * w, 96)
    xg = x.cuda().requires_grad_()
    with torch.autocast('cuda', dtype=torch.bfloat16, enabled=amp):
        y = layer(xg, h, w)[0]
    y.backward(d.cuda().to(y.dtype))
    assert calls == ([] if ws == 9 else [torch.bfloat16 if amp else torch.float32] * 2) and len(gathers) == 2
    xr = x.double().requires_grad_()
    yr = ref(xr, h, w)[0]
    yr.backward(d.double())
    tol = 4e-2 if amp else 2e-5
    assert float((y.double().cpu() - yr).abs().max() / yr.abs().max()) < tol
    assert float((xg.grad.double().cpu() - xr.grad).abs().max() / xr.grad.abs().max()) < tol
    for (n, p), (_, q) in zip(layer.named_parameters(), ref.named_parameters()):
        assert p.grad is not None, n
        # key biases do not move a softmax: their third of the qkv bias gradient is rounding alone
        a, b = p.grad.double().cpu(), q.grad
        assert float((a - b).abs().max()) < tol * float(b.abs().max()), n


def test_table_gradient_is_the_same_each_time_and_the_switch_still_works(monkeypatch):
    from segdistill_amd import window_attn
    layer = _layer(7).cuda()
    x = torch.randn(2, 30 * 26, 96, device='cuda')

    def grads():
        layer.zero_grad()
        layer(x, 30, 26)[0].square().sum().backward()
        return [b.attn.relative_position_bias_table.grad.clone() for b in layer.blocks]
    a, b = grads(), grads()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    monkeypatch.setattr(window_attn, 'ENABLED', False)
    c = grads()
    assert all(float((p - q).abs().max()) < 2e-5 * float(q.abs().max()) for p, q in zip(a, c))


def test_a_loaded_index_gives_the_plan():
    from segdistill_amd.backbones.swin import WindowAttention
    att = WindowAttention(64, (4, 4), 2).cuda()
    sd = att.state_dict()
    assert set(sd) == {'relative_position_bias_table', 'relative_position_index', 'qkv.weight', 'qkv.bias', 'proj.weight', 'proj.bias'}
    sd['relative_position_index'] = sd['relative_position_index'].flip(0)
    att.load_state_dict(sd)
    assert torch.equal(att.bias_plan.index.long(), sd['relative_position_index']) and att.bias_plan.index.is_cuda


def test_a_type_that_the_kernels_do_not_take_keeps_the_modules_path():
    from segdistill_amd import rel_bias
    from segdistill_amd.backbones.swin import WindowAttention
    torch.manual_seed(1)
    att = WindowAttention(64, (4, 4), 2).double()
    x = torch.randn(6, 16, 64, dtype=torch.float64)
    ref = copy.deepcopy(att)
    ref(x).square().sum().backward()
    att.cuda()
    assert not rel_bias.supported(att.relative_position_bias_table) and not rel_bias.supported(att.relative_position_bias_table.half())
    att(x.cuda()).square().sum().backward()
    for (n, p), q in zip(att.named_parameters(), ref.parameters()):
        assert float((p.grad.cpu() - q.grad).abs().max()) <= 1e-12 * float(q.grad.abs().max()), n


def _model():
    import segdistill_amd
    from segdistill_amd.builder import build_segmentor
    from segdistill_amd.segmentors import sd_module
    segdistill_amd.register_all()

    def seg(depths):
        return dict(type='EncoderDecoder', pretrained=None,
                    backbone=dict(type='SwinTransformer', embed_dim=64, depths=depths, num_heads=[2, 4], window_size=7, drop_path_rate=0., out_indices=(0, 1)),
                    decode_head=dict(type='FCNHead', in_channels=128, in_index=1, channels=128, num_convs=0, concat_input=False, dropout_ratio=1e-12, num_classes=19,
                                     norm_cfg=dict(type='SyncBN', requires_grad=True), align_corners=False,
                                     loss_decode=dict(type='CrossEntropyLoss', use_sigmoid=False, loss_weight=1.0)))
    cfg = dict(type='SDModule', cfg_s=seg([2, 2]), cfg_t=seg([2, 4]),
               distillation=[dict(student_layer='decode_head.conv_seg', teacher_layer='decode_head.conv_seg', loss_name='TopKLoss',
                                  loss_config=dict(k=5, alpha=3, tau=2, ignore_index=255, warmup_config={'mode': 'linear', 'warmup_iters': 2}))],
               t_pretrain=None, train_cfg=dict(), test_cfg=dict(mode='whole'))
    sd_module.SYNTHETIC_WEIGHTS_OK = True
    try:
        with warnings.catch_warnings():
            warnings.simplefilter('ignore')
            torch.manual_seed(0)
            m = build_segmentor(cfg)
    finally:
        sd_module.SYNTHETIC_WEIGHTS_OK = False
    for p in m.teacher.decode_head.conv_seg.parameters():
        p.data.mul_(30)                       # a teacher that has opinions
    return m.cuda()


def test_kd_step_of_a_swin_student_against_top_logits_eager_and_replayed():
    from segdistill_amd.engine import KDTrainer, SyntheticADE
    opt, sched = dict(type='AdamW', lr=6e-5, betas=(0.9, 0.999), weight_decay=0.01), dict(policy='poly', power=1.0, min_lr=0.0, by_epoch=False)
    ref = _model()
    gra = copy.deepcopy(ref)
    taps = {}
    inner = ref.distillation_loss.forward

    def spy(sf, tf, gt, step, *rest):
        taps.update(s=sf['decode_head.conv_seg'].detach().double().cpu(), t=tf['decode_head.conv_seg'].detach().double().cpu(), gt=gt.cpu())
        return inner(sf, tf, gt, step, *rest)
    ref.distillation_loss.forward = spy
    te, tg = KDTrainer(ref, opt, sched), KDTrainer(gra, opt, sched)
    de, dg = (SyntheticADE(2, size=(112, 120), num_classes=19, device='cuda:0', pool=3, seed=1) for _ in range(2))
    assert tg.enable_graph(dict(img=dg._pool[0][0], img_metas=None, gt_semantic_seg=dg._pool[0][1])), getattr(tg, 'graph_error', None)
    for it in range(4):
        te.step(de.next())
        torch.cuda.synchronize()
        tg.step(dg.next())
        ve, vg = te.log_values(), tg.log_values()
        key = [k for k in ve if k.startswith('loss_')]
        assert list(ve) == list(vg) and len(key) == 1
        # the definition on the taps that the eager step saw
        alpha = ref.distillation_loss.criteria[0].alpha
        s, t = (x.permute(0, 2, 3, 1).reshape(-1, 19) / 2 for x in (taps['s'], taps['t']))
        keep = torch.nn.functional.interpolate(taps['gt'].float(), size=taps['s'].shape[2:], mode='nearest').reshape(-1) != 255
        lp, lq = torch.log_softmax(t, 1), torch.log_softmax(s, 1)
        top = t.topk(5, 1).indices
        low = torch.ones_like(t, dtype=torch.bool).scatter(1, top, False)
        terms = (lp.exp() * (lp - lq)).gather(1, top).sum(1)
        pr, qr = ((l.masked_fill(~low, -math.inf)).logsumexp(1) for l in (lp, lq))
        want = float(alpha * (terms + pr.exp() * (pr - qr))[keep].mean())
        assert want > 0 and ve[key[0]] == pytest.approx(want, rel=1e-4)
        for k in ve:
            if 'acc' not in k:
                assert vg[k] == pytest.approx(ve[k], abs=3e-4 * max(1.0, abs(ve[k]))), (it, k)
    tables = [b.attn.relative_position_bias_table for l in ref.student.backbone.layers for b in l.blocks]
    assert all(p.grad is not None and float(p.grad.abs().sum()) > 0 for p in tables)


def test_a_captured_step_reads_the_index_that_was_loaded_after_its_capture(monkeypatch):
    """the capture has the plan's addresses: a checkpoint (with another index, and bias tables large enough to show it) loaded into a replaying trainer and an
    eager one, then equal losses and table gradients"""
    from segdistill_amd.engine import KDTrainer, SyntheticADE
    opt, sched = dict(type='AdamW', lr=6e-5, betas=(0.9, 0.999), weight_decay=0.01), dict(policy='poly', power=1.0, min_lr=0.0, by_epoch=False)
    ref = _model()
    gra = copy.deepcopy(ref)
    te, tg = KDTrainer(ref, opt, sched), KDTrainer(gra, opt, sched)
    de, dg = (SyntheticADE(2, size=(112, 120), num_classes=19, device='cuda:0', pool=3, seed=1) for _ in range(2))
    from segdistill_amd import rel_bias
    gathers, bias = [], rel_bias.bucket_bias
    monkeypatch.setattr(rel_bias, 'bucket_bias', lambda *a: (gathers.append(torch.cuda.is_current_stream_capturing()), bias(*a))[1])
    assert tg.enable_graph(dict(img=dg._pool[0][0], img_metas=None, gt_semantic_seg=dg._pool[0][1])), getattr(tg, 'graph_error', None)
    assert gathers == [False] * 8 + [True] * 4                             # two warm-up steps and the capture of four blocks
    graph = tg._graph

    def steps(n):
        for _ in range(n):
            te.step(de.next())
            torch.cuda.synchronize()
            tg.step(dg.next())
            ve, vg = te.log_values(), tg.log_values()
            for k in ve:
                if 'acc' not in k:
                    assert vg[k] == pytest.approx(ve[k], abs=3e-4 * max(1.0, abs(ve[k]))), k
    steps(2)
    sd = te.state_dict()
    sd['state_dict'] = {k: v.clone() for k, v in sd['state_dict'].items()}
    torch.manual_seed(4)
    for k, v in sd['state_dict'].items():
        if k.endswith('relative_position_bias_table'):
            v.normal_(std=3.0)
    plain = copy.deepcopy(sd)
    for k, v in sd['state_dict'].items():
        if k.endswith('relative_position_index'):
            sd['state_dict'][k] = v.flip(0)
    for state in (plain, sd):
        te.load_state_dict(copy.deepcopy(state)), tg.load_state_dict(copy.deepcopy(state))
        junk = [torch.full((n,), -1, dtype=torch.int32, device='cuda') for n in (49, 169, 170, 2401) * 40]          # over whatever a load may have freed
        assert tg._graph is graph
        steps(2)
        del junk
    # a stale index would give unrelated gradients of the tables (a relative difference of 1 and more); two trainers differ by the order of the sums in library
    # kernels and by what two optimizer steps of 6e-5 make of it
    for m in (ref, gra):
        for blk in (b for l in m.student.backbone.layers for b in l.blocks):
            assert torch.equal(blk.attn.bias_plan.index.long(), blk.attn.relative_position_index)
            assert torch.equal(blk.attn.relative_position_index[0], blk.attn.relative_position_index.new_tensor(_first_row_flipped()))
    tables = [[b.attn.relative_position_bias_table for l in m.student.backbone.layers for b in l.blocks] for m in (ref, gra)]
    for a, b in zip(*tables):
        assert float((a.grad - b.grad).norm()) <= 2e-2 * float(a.grad.norm()) and float(a.grad.norm()) > 0


def _first_row_flipped():
    """the last token's row of a 7 x 7 window's index: (dy + 6) * 13 + dx + 6 from (6, 6)"""
    return [(6 - y + 6) * 13 + 6 - x + 6 for y in range(7) for x in range(7)]


def test_the_bias_follows_an_index_that_was_changed_by_hand():
    """the plan of the step before: an index written in place, replaced, and changed while it cannot be read (in a capture)"""
    from segdistill_amd.backbones.swin import WindowAttention
    torch.manual_seed(5)
    att = WindowAttention(64, (4, 5), 2).cuda()
    torch.nn.init.normal_(att.relative_position_bias_table)
    table = att.relative_position_bias_table

    def check(index):
        out = att._bias(20, 2)
        assert torch.equal(out, table.detach()[index.reshape(-1)].view(20, 20, 2).permute(2, 0, 1))
        d = torch.randn_like(out)
        want, size = (torch.zeros(63, 2, dtype=torch.float64).index_add_(0, index.reshape(-1).cpu(), x.double().cpu().reshape(2, -1).t()) for x in (d, d.abs()))
        # at most 20 pairs of a bucket, a tree of six levels: within 15 steps of 2^-24 of the sum of magnitudes, as every bucket of one chunk
        assert ((torch.autograd.grad(out, table, d)[0].double().cpu() - want).abs() <= 15 * 2.0 ** -24 * size).all()
    index = att.relative_position_index
    check(index)
    index.copy_(index.flip(0).clone())
    check(index)
    att.relative_position_index = index.roll(1, 0)
    check(index.roll(1, 0))
    now = att.relative_position_index
    now.copy_(index)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        att.relative_position_index.copy_(index.roll(3, 1))
        out = att._bias(20, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, table.detach()[index.roll(3, 1).reshape(-1)].view(20, 20, 2).permute(2, 0, 1))
    check(index.roll(3, 1))


def _attention_twice(seed=6):
    """a trainable window attention, and the same in fp64 on the CPU"""
    from segdistill_amd.backbones.swin import WindowAttention
    torch.manual_seed(seed)
    att = WindowAttention(64, (4, 4), 2)
    torch.nn.init.normal_(att.relative_position_bias_table)
    ref = copy.deepcopy(att).double()
    x = torch.randn(6, 16, 64)
    mask = torch.where(torch.rand(3, 16, 16) < 0.2, -100.0, 0.0)
    mask[1, 3] = -100.0
    return att.cuda(), ref, x, mask


def _close(got, want, what=''):
    """two Linears, a softmax and their derivatives in fp32: 1e-4 of the largest value is two hundred times what their sums of 64 to 192 terms round by"""
    got = got.detach().double().cpu()
    assert got.shape == want.shape and float((got - want).abs().max()) <= 1e-4 * float(want.abs().max()), what


def test_gradients_with_a_graph_of_their_own():
    """create_graph through a trainable block: first and second derivatives against fp64"""
    att, ref, x, mask = _attention_twice()
    both = []
    for a, inp, m in ((att, x.cuda(), mask.cuda()), (ref, x.double(), mask.double())):
        inp.requires_grad_()
        names = [n for n, _ in a.named_parameters()]
        params = list(a.parameters())
        first = torch.autograd.grad(a(inp, m).square().sum(), [inp] + params, create_graph=True)
        second = torch.autograd.grad(sum(g.square().sum() for g in first), [inp] + params)
        both.append((first, second))
    for k, (got, want) in enumerate(zip(both[0], both[1])):
        for n, g, w in zip(['x'] + names, got, want):
            _close(g, w.detach(), (k, n))
    # and a gradient without a graph is the kernel's, as before
    xg = x.cuda().requires_grad_()
    plain = torch.autograd.grad(att(xg, mask.cuda()).square().sum(), [xg] + list(att.parameters()))
    for g, w in zip(plain, both[1][0]):
        _close(g, w.detach())


def test_transforms_take_torch_operators():
    """torch.func.grad, per-sample gradients, vmap, a batch of gradients at once; the forward mode against the backward: w . J v = J^T w . v"""
    att, ref, x, mask = _attention_twice(7)
    out = []
    for a, inp, m in ((att, x.cuda(), mask.cuda()), (ref, x.double(), mask.double())):
        params = {n: p.detach() for n, p in a.named_parameters()}

        def loss(p, y):
            return torch.func.functional_call(a, p, (y, m)).square().sum()
        pair = torch.stack([inp, inp.flip(0)])
        one = torch.func.grad(loss)(params, inp)
        per = torch.func.vmap(torch.func.grad(loss), in_dims=(None, 0))(params, pair)
        mapped = torch.func.vmap(lambda y: a(y, m))(pair)
        leaf = inp.clone().requires_grad_()
        y = a(leaf, m)
        ds = torch.stack([torch.ones_like(y), y.detach(), y.detach().flip(0)])
        batch = torch.autograd.grad(y, [leaf] + list(a.parameters()), ds, is_grads_batched=True)
        if a is att:
            tangent = torch.func.jvp(lambda z: a(z, m), (inp,), (pair[1],))[1]
            assert tangent.shape == y.shape
            along = (tangent.double() * ds[1].double()).sum().view(1)
        else:
            along = (batch[0][1] * pair[1]).sum().view(1)
        out.append((list(one.values()), list(per.values()), [mapped], list(batch), [along]))
    wide = copy.deepcopy(ref).cuda()
    got = torch.func.vmap(lambda y: wide(y, mask.double().cuda()))(pair.cuda())
    assert float((got.cpu() - mapped).abs().max()) <= 1e-13 * float(mapped.abs().max())
    for got, want in zip(*out):
        for g, w in zip(got, want):
            _close(g, w.detach())


def test_tables_may_change_behind_a_forward_unless_a_graph_is_asked_for():
    from segdistill_amd import window_attn
    g = torch.Generator(device='cuda').manual_seed(8)
    qkv = torch.randn(4, 9, 192, device='cuda', generator=g, requires_grad=True)
    bias, mask = torch.randn(2, 9, 9, device='cuda', generator=g), torch.zeros(2, 9, 9, device='cuda')
    with torch.inference_mode():
        cached = mask.clone()                                               # as one that an evaluation left behind
    out = window_attn.attention(qkv, bias, mask, 2, 0.2)
    want = torch.autograd.grad(out, qkv, torch.ones_like(out), retain_graph=True)[0]
    with_graph = torch.autograd.grad(window_attn.attention(qkv, bias, cached, 2, 0.2), qkv, torch.ones_like(out), create_graph=True)[0]
    assert float((with_graph - want).abs().max()) <= 1e-5 * float(want.abs().max())
    mask.fill_(3.0)
    bias.zero_()
    assert torch.equal(torch.autograd.grad(out, qkv, torch.ones_like(out), retain_graph=True)[0], want)
    with pytest.raises(RuntimeError, match='modified'):
        torch.autograd.grad(out, qkv, torch.ones_like(out), create_graph=True)
