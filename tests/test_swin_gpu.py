"""Frozen Swin (the config-4 teacher) fast paths of round 3 -- pad + cyclic shift + window partition as ONE cached row gather (window reverse +
un-shift + un-pad as another), and the relative-position bias + shift mask + batch repeat cached per block -- against the literal module chain:
pure data movement and a cached copy of the same tensor, so the feature pyramids must be identical."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('size', [(224, 224), (160, 200)])       # windows that divide the map, and maps that need padding on both axes
def test_frozen_swin_gather_path_equals_the_module_chain(size):
    import segdistill_amd
    from segdistill_amd.backbones import swin
    segdistill_amd.register_all()
    torch.manual_seed(0)
    net = swin.SwinTransformer(embed_dim=32, depths=(2, 2, 2), num_heads=(2, 4, 8), window_size=7, out_indices=(0, 1, 2)).cuda().eval()
    for p in net.parameters():
        p.requires_grad = False
    img = torch.randn(2, 3, *size, device='cuda:0')
    outs = {}
    for flag in (True, False):
        swin._GATHER_WINDOWS = flag
        try:
            with torch.no_grad():
                outs[flag] = [f.clone() for f in net(img)]
                again = net(img)                       # second call: the cached bias tensors are used
            for a, b in zip(outs[flag], again):
                assert torch.equal(a, b)
        finally:
            swin._GATHER_WINDOWS = True
    for a, b in zip(outs[True], outs[False]):
        assert a.shape == b.shape and float((a - b).abs().max()) <= 1e-6 * float(b.abs().max())
    # round 4: the fused block form (norm1 + window partition in one kernel, window reverse + residual + norm2 in another, the MLP residual
    # folded into the next block's first kernel) against the separate kernels: the same arithmetic on the same values
    fused = outs[True]
    swin._FUSE_NORMS = False
    try:
        with torch.no_grad():
            plain = net(img)
    finally:
        swin._FUSE_NORMS = True
    for a, b in zip(fused, plain):
        assert a.shape == b.shape and float((a - b).abs().max()) <= 2e-6 * float(b.abs().max())
    blk = net.layers[0].blocks[0]
    blk.H = blk.W = 8
    assert blk.fusable(torch.zeros(1, 64, 32, device='cuda:0'))
    # a tapped block is called as a module and hands its hook the complete block output (the KD Extractor's contract)
    seen = []
    h = net.layers[1].blocks[1].register_forward_hook(lambda m, i, o: seen.append(o.detach().clone()))
    try:
        with torch.no_grad():
            hooked = net(img)
    finally:
        h.remove()
    assert len(seen) == 1 and not net.layers[1].blocks[1]._forward_hooks
    for a, b in zip(fused, hooked):
        assert float((a - b).abs().max()) <= 2e-6 * float(b.abs().max())
    with torch.no_grad():                              # the hooked block's output is what the next stage consumed
        swin._FUSE_NORMS = False
        try:
            seen2 = []
            h = net.layers[1].blocks[1].register_forward_hook(lambda m, i, o: seen2.append(o.detach().clone()))
            net(img)
            h.remove()
        finally:
            swin._FUSE_NORMS = True
    assert float((seen[0] - seen2[0]).abs().max()) <= 2e-6 * float(seen2[0].abs().max())
    # a trainable Swin keeps the autograd-friendly chain (index_select's backward would be an atomic scatter)
    for p in net.parameters():
        p.requires_grad = True
    x = img.clone().requires_grad_(True)
    feats = net.train()(x)
    sum(f.mean() for f in feats).backward()
    assert x.grad is not None and torch.isfinite(x.grad).all()


def test_partially_frozen_swin_keeps_the_gradients_of_its_trainable_parts():
    """frozen patch embedding and norms, TRAINABLE attention (qkv, proj, relative-position table) and MLP, grad mode on, input without
    a graph -- the no-graph block kernels (forward_fused, the packed window attention) must step aside: the gradients of the trainable parameters
    equal those of the literal module chain (fast paths switched off)."""
    import segdistill_amd
    from segdistill_amd.backbones import swin
    segdistill_amd.register_all()
    torch.manual_seed(0)
    net = swin.SwinTransformer(embed_dim=32, depths=(2, 2), num_heads=(2, 4), window_size=7, out_indices=(0, 1)).cuda().eval()
    for name, p in net.named_parameters():
        p.requires_grad = ('attn.' in name) or ('mlp.' in name)
    assert any(p.requires_grad for p in net.parameters()) and not all(p.requires_grad for p in net.parameters())
    img = torch.randn(2, 3, 112, 120, device='cuda:0')
    grads = {}
    for fast in (True, False):
        swin._GATHER_WINDOWS = swin._FUSE_NORMS = fast
        try:
            for p in net.parameters():
                p.grad = None
            sum(f.square().mean() for f in net(img)).backward()
            grads[fast] = {n: p.grad.clone() for n, p in net.named_parameters() if p.requires_grad}
        finally:
            swin._GATHER_WINDOWS = swin._FUSE_NORMS = True
    assert grads[True].keys() == grads[False].keys() and len(grads[True]) > 0
    for n in grads[False]:
        a, b = grads[True][n], grads[False][n]
        assert a is not None and float(b.abs().max()) > 0, n
        assert float((a - b).abs().max()) <= 2e-4 * float(b.abs().max()) + 1e-9, n


@pytest.mark.parametrize('ws', [(7, 7), (5, 5)])
def test_a_captured_frozen_block_keeps_its_tables(ws):
    """what a frozen window attention caches -- packed bias and mask (7 x 7), the additive tensor (other windows) -- is read by a captured forward: it outlives a
    forward with another mask, and follows a checkpoint that is loaded after the capture"""
    from segdistill_amd.backbones.swin import WindowAttention
    torch.manual_seed(11)
    att = WindowAttention(64, ws, 2).cuda().eval().requires_grad_(False)
    torch.nn.init.normal_(att.relative_position_bias_table)
    n = ws[0] * ws[1]
    x = torch.randn(8, n, 64, device='cuda')
    masks = [torch.where(torch.rand(4, n, n, device='cuda') < 0.3, -100.0, 0.0) for _ in range(2)]
    sd = {k: v.clone() for k, v in att.state_dict().items()}
    sd['relative_position_bias_table'] = sd['relative_position_bias_table'].normal_(std=3.0)
    other = WindowAttention(64, ws, 2).cuda().eval().requires_grad_(False)
    other.load_state_dict(sd)
    with torch.no_grad():
        want, loaded = att(x, masks[0]).clone(), other(x, masks[0]).clone()
        assert float((want - loaded).abs().max()) > 0.01
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            att(x, masks[0])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = att(x, masks[0])

        def replay():
            junk = [torch.full((k,), float('nan'), device='cuda') for k in (4 * 4096, 2 * 4096, 8 * 2 * n * n, 2 * n * n) * 20]
            graph.replay()
            torch.cuda.synchronize()
            del junk
            return out
        assert torch.equal(replay(), want)
        att(x, masks[1])
        assert torch.equal(replay(), want)
        att.load_state_dict(sd)
        assert torch.equal(replay(), loaded)
        assert torch.equal(att(x, masks[0]), loaded) and torch.equal(replay(), loaded)


@pytest.mark.parametrize('ws', [(7, 7), (5, 5)])
def test_a_frozen_block_tells_masks_apart_that_share_an_address(ws):
    """each mask goes before the next one comes, to the same memory; and masks made in inference mode, as an evaluation leaves them.  (Sums of at most 64 terms
    in fp32, two Linears and a softmax: within 1e-5 of the largest value.)"""
    from segdistill_amd.backbones.swin import WindowAttention
    torch.manual_seed(12)
    att = WindowAttention(64, ws, 2).cuda().eval().requires_grad_(False)
    n = ws[0] * ws[1]
    x = torch.randn(8, n, 64, device='cuda')
    ref = WindowAttention(64, ws, 2).double().eval()
    ref.load_state_dict({k: v.cpu() for k, v in att.state_dict().items()})
    with torch.no_grad():
        for turn in range(6):
            with torch.inference_mode(turn >= 4):
                mask = torch.where(torch.rand(4, n, n, device='cuda') < 0.5, -100.0, 0.0)
            got = att(x, mask).double().cpu()
            want = ref(x.double().cpu(), mask.double().cpu())
            assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max()), turn
            del mask
