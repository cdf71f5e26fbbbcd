"""The bucketed position bias (csrc/rel_bias.hip) against indexing, and its gradient against sums in fp64.

The forward copies: equal bits.  The gradient sums at most 512 elements of a bucket in fp32 (eight per lane, then a tree of six levels: 14 additions on any
path), the chunks in fp64: off by at most 15 u sum |d|, u = 2^-24, and half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _window_index(wh, ww):
    ys, xs = torch.meshgrid(torch.arange(wh), torch.arange(ww), indexing='ij')
    y, x = ys.flatten(), xs.flatten()
    return (y[:, None] - y[None, :] + wh - 1) * (2 * ww - 1) + (x[:, None] - x[None, :] + ww - 1)


def _check(index, nb, heads, dtype, seed=0):
    from segdistill_amd import rel_bias
    g = torch.Generator(device='cuda').manual_seed(seed)
    plan = rel_bias.BucketPlan(index.cuda(), nb)
    table = torch.randn(nb, heads, device='cuda', generator=g).to(dtype).requires_grad_()
    out = rel_bias.bucket_bias(table, plan)
    assert out.dtype == dtype and torch.equal(out, table.detach()[index.cuda().long()].permute(2, 0, 1))
    d = torch.randn(out.shape, device='cuda', generator=g).to(dtype)
    (got,) = torch.autograd.grad(out, table, d, retain_graph=True)
    flat = index.reshape(-1).long()
    dd = d.double().cpu().reshape(heads, -1).t()
    ref = torch.zeros(nb, heads, dtype=torch.float64).index_add_(0, flat, dd)
    mag = torch.zeros(nb, heads, dtype=torch.float64).index_add_(0, flat, dd.abs())
    lim = 15 * U * mag + torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 1e-3)
    assert ((got.double().cpu() - ref).abs() <= lim).all()
    assert (got.double().cpu()[mag == 0] == 0).all()
    assert torch.equal(got, torch.autograd.grad(out, table, d)[0])
    return plan, table


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('wh,ww,heads', [(1, 1, 1), (2, 3, 3), (7, 7, 4), (7, 7, 32), (5, 8, 9), (12, 12, 6), (14, 3, 8)])
def test_window_buckets(wh, ww, heads, dtype):
    _check(_window_index(wh, ww), (2 * wh - 1) * (2 * ww - 1), heads, dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('nq,nk,nb,heads', [(1, 1, 3, 2), (1, 700, 4, 5), (33, 65, 1, 3), (64, 512, 7, 16), (100, 513, 2, 1), (301, 299, 200, 12), (1000, 1001, 32, 8)])
def test_long_buckets_ragged_sizes_and_empty_buckets(nq, nk, nb, heads, dtype):
    g = torch.Generator().manual_seed(nq)
    index = (torch.rand(nq, nk, generator=g) ** 3 * nb).long().clamp(max=nb - 1)
    if nb > 3:
        index[index == 2] = 1                                   # an empty bucket, between others
        index[index == nb - 1] = 0                              # and at the end
    _check(index.to(torch.int32) if nq % 2 else index, nb, heads, dtype)


def test_gradient_arrives_in_any_layout_and_the_plan_moves_with_its_module():
    from segdistill_amd import rel_bias
    index = _window_index(4, 4)
    plan = rel_bias.BucketPlan(index, 49).cuda()                # built on the host, moved like a module
    assert not plan.state_dict() and not list(plan.parameters())
    table = torch.randn(49, 3, device='cuda', requires_grad=True)
    out = rel_bias.bucket_bias(table, plan)
    d = torch.randn(3, 16, 16, device='cuda')
    a = torch.autograd.grad(out, table, d, retain_graph=True)[0]
    b = torch.autograd.grad(out, table, d.permute(2, 1, 0).contiguous().permute(2, 1, 0), retain_graph=True)[0]
    assert torch.equal(a, b)
    c = torch.autograd.grad(out.sum(), table, retain_graph=True)[0]          # an expanded gradient
    assert torch.equal(c, torch.bincount(index.view(-1), minlength=49).float().cuda().unsqueeze(1).expand(49, 3))
    t2 = table.detach().t().contiguous().t().requires_grad_()                # a strided table
    assert torch.equal(rel_bias.bucket_bias(t2, plan), out)


def test_replayed_in_a_graph():
    from segdistill_amd import rel_bias
    g = torch.Generator(device='cuda').manual_seed(2)
    index = torch.randint(0, 5, (60, 70))
    plan = rel_bias.BucketPlan(index.cuda(), 5)
    sets = [(torch.randn(5, 4, device='cuda', generator=g), torch.randn(4, 60, 70, device='cuda', generator=g)) for _ in range(3)]

    def step(t, d):
        out = rel_bias.bucket_bias(t, plan)
        return out.detach(), torch.autograd.grad(out, t, d)[0]

    eager = [step(t.clone().requires_grad_(), d) for t, d in sets]
    t_in, d_in = sets[0][0].clone().requires_grad_(), sets[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(t_in, d_in)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(t_in, d_in)
    for (t, d), want in zip(sets[::-1], eager[::-1]):
        with torch.no_grad():
            t_in.copy_(t), d_in.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step(t.clone().requires_grad_(), d)


def test_refusals():
    from segdistill_amd import rel_bias
    plan = rel_bias.BucketPlan(_window_index(2, 2), 9)
    with pytest.raises(ValueError, match='the plan is on'):
        rel_bias.bucket_bias(torch.zeros(9, 2, device='cuda'), plan)
    plan.cuda()
    for bad in (torch.zeros(8, 2, device='cuda'), torch.zeros(9, device='cuda'), torch.zeros(9, 0, device='cuda')):
        with pytest.raises(ValueError):
            rel_bias.bucket_bias(bad, plan)
    with pytest.raises(TypeError):
        rel_bias.bucket_bias(torch.zeros(9, 2, device='cuda').half(), plan)


def test_the_plan_may_move_between_forward_and_backward():
    from segdistill_amd import rel_bias
    plan = rel_bias.BucketPlan(_window_index(4, 4), 49).cuda()
    table = torch.randn(49, 3, device='cuda', requires_grad=True)
    out = rel_bias.bucket_bias(table, plan)
    want = torch.autograd.grad(out, table, torch.ones_like(out), retain_graph=True)[0]
    plan.cpu()
    assert torch.equal(torch.autograd.grad(out, table, torch.ones_like(out), retain_graph=True)[0], want)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(out, table, torch.ones_like(out), create_graph=True)


def test_offsets_past_32_bits():
    """a bias of 2.2e9 elements: every head against a call on that head alone"""
    from segdistill_amd import rel_bias
    n, heads = 8192, 33
    d = (torch.arange(n, device='cuda').unsqueeze(1) - torch.arange(n, device='cuda')).abs()
    plan = rel_bias.BucketPlan(torch.minimum(d, torch.full_like(d, 31)), 32)
    g = torch.Generator(device='cuda').manual_seed(4)
    table = torch.randn(32, heads, device='cuda', generator=g).to(torch.bfloat16).requires_grad_()
    grad = torch.empty(heads, n, n, device='cuda', dtype=torch.bfloat16).normal_(generator=g)
    assert grad.numel() > 2 ** 31
    out = rel_bias.bucket_bias(table, plan)
    dtable = torch.autograd.grad(out, table, grad)[0]
    for h in (0, 31, 32):
        t = table.detach()[:, h:h + 1].contiguous().requires_grad_()
        one = rel_bias.bucket_bias(t, plan)
        assert torch.equal(one[0], out[h]) and torch.equal(one[0, 5], t.detach()[plan.index[5].long(), 0])
        assert torch.equal(torch.autograd.grad(one, t, grad[h:h + 1])[0][:, 0], dtable[:, h])


def test_the_last_chunk_of_as_many_pairs_as_there_may_be():
    """2^31 - 1 pairs: the last chunk starts 188 pairs before the end, and 512 from there is beyond a 32-bit integer.  The plan as the C entry takes it, the
    pairs in their own order: all but 700 in one bucket, the rest in the other.  704 and 0 are exact in bf16, and so is every sum on the way."""
    from segdistill_amd import _lib
    L, pairs, last = _lib.lib(), 2 ** 31 - 1, 700
    order = torch.arange(pairs, device='cuda', dtype=torch.int32)
    first = torch.arange(0, pairs - last, 512, device='cuda')
    start = torch.cat([first, torch.tensor([pairs - last, pairs - last + 512, pairs], device='cuda')]).int()
    chunks = start.numel() - 1
    bucket = torch.tensor([0, first.numel(), chunks], device='cuda', dtype=torch.int32)
    assert int(start[-1] - start[-2]) == 188
    dbias = torch.zeros(pairs, device='cuda', dtype=torch.bfloat16)
    dbias[-last:] = 1
    dbias[-4:] = 2
    out = torch.full((2, 1), float('nan'), device='cuda', dtype=torch.bfloat16)
    size = L.sd_bucket_bias_workspace_bytes(2, chunks, 1)
    work = torch.empty(size, dtype=torch.uint8, device='cuda')
    by_pair = torch.arange(chunks, device='cuda', dtype=torch.int32)
    rc = L.sd_bucket_bias_bwd(dbias.data_ptr(), order.data_ptr(), start.data_ptr(), by_pair.data_ptr(), bucket.data_ptr(), out.data_ptr(), 1, 2, chunks, 1, pairs,
                              work.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert out.flatten().tolist() == [0.0, 704.0]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('ws,heads', [(4, 3), (7, 4), (12, 6), (22, 2)])
def test_a_bucket_of_one_chunk_is_rounded_once(ws, heads, dtype):
    """up to 512 pairs are summed in 64 bits: nothing but the result's half step is left (and 2^-44 of the magnitudes, 512 additions of 2^-53)"""
    from segdistill_amd import rel_bias
    index, nb = _window_index(ws, ws), (2 * ws - 1) ** 2
    plan = rel_bias.BucketPlan(index.cuda(), nb)
    assert plan.num_chunks == nb
    g = torch.Generator(device='cuda').manual_seed(ws)
    table = torch.zeros(nb, heads, device='cuda', dtype=dtype, requires_grad=True)
    d = torch.randn(heads, ws * ws, ws * ws, device='cuda', generator=g).to(dtype)
    got = torch.autograd.grad(rel_bias.bucket_bias(table, plan), table, d)[0].double().cpu()
    dd = d.double().cpu().reshape(heads, -1).t()
    ref, mag = (torch.zeros(nb, heads, dtype=torch.float64).index_add_(0, index.reshape(-1), x) for x in (dd, dd.abs()))
    # to bf16 by way of fp32: its half step besides
    lim = (torch.finfo(dtype).eps / 2 + (0 if dtype == torch.float32 else U)) * ref.abs() + 2.0 ** -44 * mag
    assert ((got - ref).abs() <= lim).all()
