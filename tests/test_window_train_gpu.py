"""Window attention with gradients (csrc/window_train.hip) against reference mmseg/models/backbones/swin_transformer.py:119-153 and its autograd in fp64.

Tolerances.  u = 2^-24.  Every product sums at most 64 terms in fp32 and every probability carries the rounding of its score (32 terms) and of one
exponential; rounding errors of either sign add up like their root, so results are held to 8 (sqrt(32) + sqrt(64)) u = 6.5e-6 of the largest value.
Under bf16 storage the products take P and dS rounded to half the bits twice over (two terms: 2^-16 relative), within the same bound; what is stored adds
half a step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TOL = 8 * (32 ** 0.5 + 64 ** 0.5) * U


def _ref(qkv, bias, mask, heads, scale, dout):
    bw, n, c3 = qkv.shape
    qkv, bias = qkv.detach().double().cpu().requires_grad_(), bias.detach().double().cpu().requires_grad_()
    q, k, v = qkv.view(bw, n, 3, heads, 32).permute(2, 0, 3, 1, 4)
    s = (q * scale) @ k.transpose(-2, -1) + bias
    if mask is not None:
        nw = mask.shape[0]
        s = (s.view(bw // nw, nw, heads, n, n) + mask.double().cpu().unsqueeze(1)).view(bw, heads, n, n)
    dead = (s == -math.inf).all(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0)
    out = (p @ v).transpose(1, 2).reshape(bw, n, c3 // 3)
    return (out.detach(),) + torch.autograd.grad(out, (qkv, bias), dout.double().cpu())


def _close(got, ref, what):
    got, lim = got.double().cpu(), TOL * float(ref.abs().max()) + torch.finfo(got.dtype).eps / 2 * (1 + 1e-3) * ref.abs()
    assert torch.isfinite(got).all(), what
    over = ((got - ref).abs() - lim).max()
    assert float(over) <= 0, (what, float(over), float((got - ref).abs().max()), float(ref.abs().max()))


def _check(qkv, bias, mask, heads, scale, dout):
    from segdistill_amd import window_attn
    qkv, bias = qkv.detach().requires_grad_(), bias.detach().requires_grad_()
    out = window_attn.attention(qkv, bias, mask, heads, scale)
    got = (out.detach(),) + torch.autograd.grad(out, (qkv, bias), dout, retain_graph=True)
    assert got[0].dtype == got[1].dtype == qkv.dtype and got[2].dtype == bias.dtype
    for g, r, what in zip(got, _ref(qkv, bias, mask, heads, scale, dout), ('out', 'dqkv', 'dbias')):
        _close(g, r, what)
    again = torch.autograd.grad(out, (qkv, bias), dout)
    assert torch.equal(again[0], got[1]) and torch.equal(again[1], got[2])
    return got


def _inputs(windows, n, heads, dtype, seed, nw=0, fill=-100.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    qkv = (torch.randn(windows, n, 3 * heads * 32, device='cuda', generator=g) * 1.3).to(dtype)
    bias = torch.randn(heads, n, n, device='cuda', generator=g)                  # not symmetric: catches a transposition
    dout = torch.randn(windows, n, heads * 32, device='cuda', generator=g).to(dtype)
    mask = None
    if nw:
        mask = torch.where(torch.rand(nw, n, n, device='cuda', generator=g) < 0.3, fill, 0.0)
        mask[:, torch.arange(n), torch.arange(n)] = 0.0
        if nw > 1:
            mask[0] = 0.0
    return qkv, bias, mask, dout


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('windows,n,heads,nw', [(1, 1, 1, 0), (3, 2, 5, 3), (5, 7, 1, 0), (8, 16, 3, 4), (2, 25, 4, 1), (7, 31, 2, 7), (4, 32, 3, 2), (3, 33, 3, 0), (6, 40, 6, 3),
                                                (24, 49, 4, 4), (50, 49, 16, 25), (9, 49, 32, 9), (1, 56, 2, 0), (5, 64, 3, 5), (900, 49, 3, 0), (361, 64, 1, 361), (2100, 4, 2, 0)])
def test_attention_and_its_gradients(windows, n, heads, nw, dtype):
    _check(*_with(_inputs(windows, n, heads, dtype, windows * 7 + n, nw), heads))


def _with(x, heads, scale=32 ** -0.5):
    return x[0], x[1], x[2], heads, scale, x[3]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n', range(1, 65))
def test_every_window_size(n, dtype):
    _check(*_with(_inputs(4, n, 2, dtype, 500 + n, 2), 2))


@pytest.mark.parametrize('query', [0, 17, 48])
def test_masks_that_say_something_to_one_query(query):
    qkv, bias, _, dout = _inputs(6, 49, 2, torch.float32, query)
    mask = torch.zeros(3, 49, 49, device='cuda')
    mask[1, query, 5:40] = -math.inf
    mask[2, query, 48] = 3.0
    _check(qkv, bias, mask, 2, 32 ** -0.5, dout)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n', [5, 49, 64])
def test_masks_that_leave_nothing(n, dtype):
    """rows, then whole windows, at -inf: output 0, no gradient; a mask at the type's lowest value is a mask, not an empty row"""
    qkv, bias, mask, dout = _inputs(6, n, 2, dtype, n, nw=3, fill=-math.inf)
    mask[1, 2] = -math.inf
    mask[2] = -math.inf
    out, dqkv, dbias = _check(qkv, bias, mask, 2, 0.2, dout)
    assert (out[1, 2] == 0).all() and (out[2] == 0).all() and (out[5] == 0).all() and (dqkv[2] == 0).all()
    low = torch.where(mask == -math.inf, torch.finfo(torch.float32).min, 0.0)
    out, _, _ = _check(qkv, bias, low, 2, 0.2, dout)
    mean = qkv.float().view(6, n, 3, 64)[2, :, 2].mean(0)
    assert float((out[2].float() - mean).abs().max()) < 0.02


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_large_scores_and_a_zero_gradient(dtype):
    qkv, bias, mask, dout = _inputs(4, 49, 2, dtype, 3)
    from segdistill_amd import window_attn
    big = (qkv * 8).detach().requires_grad_()
    out = window_attn.attention(big, bias * 30, None, 2, 1.0)
    assert torch.isfinite(out).all() and torch.isfinite(torch.autograd.grad(out, big, dout)[0]).all()
    x, b = qkv.clone().requires_grad_(), bias.clone().requires_grad_()
    out = window_attn.attention(x, b, None, 2, 0.2)
    g = torch.autograd.grad(out, (x, b), torch.zeros_like(dout))
    assert (g[0] == 0).all() and (g[1] == 0).all()


def test_gradient_against_differences():
    """central differences along random directions of unit size per element, h = 2^-6: cubic term below h^2 of the value's scale, the sum over outputs is
    good to 1e-5 of its terms"""
    from segdistill_amd import window_attn
    qkv, bias, mask, dout = _inputs(3, 20, 2, torch.float32, 5, nw=3)
    x, b = qkv.clone().requires_grad_(), bias.clone().requires_grad_()
    gx, gb = torch.autograd.grad(window_attn.attention(x, b, mask, 2, 0.2), (x, b), dout)
    g = torch.Generator(device='cuda').manual_seed(6)
    h = 2.0 ** -6

    def f(q, c):
        with torch.no_grad():
            return float((window_attn.attention(q, c, mask, 2, 0.2).double() * dout.double()).sum())
    for _ in range(4):
        dx, dbi = torch.randn(qkv.shape, device='cuda', generator=g), torch.randn(bias.shape, device='cuda', generator=g)
        for (q0, q1, c0, c1, want) in ((qkv + h * dx, qkv - h * dx, bias, bias, (gx.double() * dx.double()).sum()), (qkv, qkv, bias + h * dbi, bias - h * dbi, (gb.double() * dbi.double()).sum())):
            diff = (f(q0, c0) - f(q1, c1)) / (2 * h)
            assert abs(diff - float(want)) <= 0.02 * float(dout.abs().sum()) ** 0.5 + 1e-3 * abs(float(want))


def test_strided_operands_offsets_and_bias_types():
    from segdistill_amd import window_attn
    qkv, bias, mask, dout = _inputs(4, 49, 3, torch.float32, 8, nw=2)
    base = _check(qkv, bias, mask, 3, 0.2, dout)
    buf = torch.empty(qkv.numel() + 1, device='cuda')
    buf[1:] = qkv.reshape(-1)
    shifted = buf[1:].view(qkv.shape)                                     # 4 bytes off a 16-byte boundary
    got = _check(shifted, bias.transpose(1, 2).contiguous().transpose(1, 2), mask, 3, 0.2, dout.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(base, got))
    _check(qkv, bias.bfloat16(), mask, 3, 0.2, dout)
    x = qkv.clone().requires_grad_()
    out = window_attn.attention(x, bias, mask, 3, 0.2)
    assert torch.equal(torch.autograd.grad(out.sum(), x)[0], torch.autograd.grad(window_attn.attention(x, bias, mask, 3, 0.2), x, torch.ones_like(out))[0])
    e = torch.empty(0, 49, 3 * 96, device='cuda', requires_grad=True)
    b = bias.clone().requires_grad_()
    ge, gb = torch.autograd.grad(window_attn.attention(e, b, None, 3, 0.2).sum(), (e, b))
    assert ge.shape == e.shape and (gb == 0).all()


def test_replayed_in_a_graph_and_on_a_side_stream():
    from segdistill_amd import window_attn
    sets = [_inputs(6, 49, 3, torch.bfloat16, 20 + i, nw=3) for i in range(3)]

    def step(q, b, m, d):
        out = window_attn.attention(q, b, m, 3, 0.2)
        return (out.detach(),) + torch.autograd.grad(out, (q, b), d)

    eager = [step(q.clone().requires_grad_(), b.clone().requires_grad_(), m, d) for q, b, m, d in sets]
    ins = [t.clone() for t in sets[0]]
    ins[0].requires_grad_(), ins[1].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*ins)
    for given, want in zip(sets[::-1], eager[::-1]):
        with torch.no_grad():
            for a, b in zip(ins, given):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step(given[0].clone().requires_grad_(), given[1].clone().requires_grad_(), given[2], given[3])


def test_refusals():
    from segdistill_amd import window_attn
    qkv, bias, mask, _ = _inputs(4, 9, 2, torch.float32, 1, nw=2)

    def call(q=qkv, b=bias, m=mask, h=2):
        return window_attn.attention(q, b, m, h, 0.2)
    assert call().shape == (4, 9, 64)
    for kw in (dict(h=3), dict(h=0), dict(b=bias[:1]), dict(b=bias.long()), dict(m=mask[:, :8, :8]), dict(m=torch.zeros(3, 9, 9, device='cuda')), dict(m=mask.long()),
               dict(m=mask.clone().requires_grad_()), dict(q=qkv[0]), dict(q=torch.zeros(2, 65, 192, device='cuda'), b=torch.zeros(2, 65, 65, device='cuda'), m=None),
               dict(q=torch.zeros(2, 9, 96, device='cuda')), dict(b=bias.cpu()), dict(m=mask.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            call(**kw)
    with pytest.raises(TypeError):
        call(q=qkv.half())


def test_offsets_past_32_bits():
    """qkv of 2.3e9 elements: the last windows against a call on them alone (their operands are the same, and so is every operation)"""
    from segdistill_amd import window_attn
    windows, n, heads = 160000, 49, 3
    g = torch.Generator(device='cuda').manual_seed(9)
    qkv = torch.empty(windows, n, 3 * heads * 32, device='cuda', dtype=torch.bfloat16).normal_(generator=g).requires_grad_()
    dout = torch.empty(windows, n, heads * 32, device='cuda', dtype=torch.bfloat16).normal_(generator=g)
    bias = torch.randn(heads, n, n, device='cuda', generator=g)
    assert qkv.numel() > 2 ** 31
    out = window_attn.attention(qkv, bias, None, heads, 32 ** -0.5)
    dqkv = torch.autograd.grad(out, qkv, dout)[0]
    for at in (slice(0, 5), slice(windows - 7, windows)):
        q = qkv.detach()[at].clone().requires_grad_()
        o = window_attn.attention(q, bias, None, heads, 32 ** -0.5)
        assert torch.equal(o, out[at]) and torch.equal(torch.autograd.grad(o, q, dout[at])[0], dqkv[at])
