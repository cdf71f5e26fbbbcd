"""Distillation from a teacher's top logits (csrc/topk_select.hip, csrc/topk_kl.hip): the selection against a stable sort, the criterion and its gradient
against the definition in fp64 (class softmax of reference mmseg/models/distillation/losses.py:47-49,108-112 with the teacher's unlisted classes folded
into one) and against differences.

Tolerances.  u = 2^-24.  A softmax term 2^((x - m) c2) carries the rounding of its argument, at most |argument| u twice (difference, product), and one
step of the exponential; sums run over V / 64 folds per thread at worst and a tree of at most ten levels.  With arguments within +-64 a probability is
good to rel(V) = (V / 64 + 160) u.  Stored results add half a step of their type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rel(V):
    return (V / 64 + 160) * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _by_rows(x):
    """[B, C, H, W] -> [B*H*W, C]; classes last -> [rows, C]"""
    return x.permute(0, 2, 3, 1).reshape(-1, x.shape[1]) if x.dim() == 4 else x.reshape(-1, x.shape[-1])


def _sorted_ref(x, k, tau):
    r = _by_rows(x).double().cpu()
    r = torch.where(r == 0, torch.zeros_like(r), r)
    v, i = torch.sort(torch.where(r.isnan(), torch.full_like(r, math.inf), r), dim=1, descending=True, stable=True)
    low = r.gather(1, i)[:, k:]
    rest = tau * torch.logsumexp(low / tau, 1) if low.shape[1] else torch.full((r.shape[0],), -math.inf, dtype=torch.float64)
    return r.gather(1, i)[:, :k], i[:, :k], rest


def _check_select(x, k, tau, rest_tol=None):
    from segdistill_amd import ops
    v, i, rest = ops.topk_logits(x, k, tau=tau)
    assert v.dtype == x.dtype and i.dtype == torch.int32 and rest.dtype == torch.float32
    V = x.shape[1] if x.dim() == 4 else x.shape[-1]
    rv, ri, rr = _sorted_ref(x, k, tau)
    gv, gi, gr = _by_rows(v).double().cpu(), _by_rows(i).long().cpu(), rest.double().cpu().reshape(-1)
    assert torch.equal(gi, ri)
    assert torch.equal(torch.nan_to_num(gv, nan=7e37), torch.nan_to_num(rv, nan=7e37))
    fin = torch.isfinite(rr)
    assert torch.equal(fin, torch.isfinite(gr)) and torch.equal(gr[~fin], rr[~fin])
    err = (gr - rr).abs()[fin]
    # rest = m + tau log s: s good to rel(V), the logarithm and the two roundings of the result
    tol = tau * (rel(V) + 32 * U) + 4 * U * (rr.abs()[fin] + x.double().abs()[torch.isfinite(x)].max().item() if fin.any() else 0)
    assert (err <= tol).all(), float((err - tol).max())
    again = ops.topk_logits(x, k, tau=tau)
    assert all(torch.equal(a.nan_to_num(nan=1e30), b.nan_to_num(nan=1e30)) for a, b in zip((v, i, rest), again))
    return v, i, rest


ROWS = [(1, 1, 1), (3, 2, 1), (5, 7, 7), (4, 19, 5), (37, 150, 10), (9, 255, 32), (2, 256, 33), (3, 2048, 32), (3, 2049, 16), (2, 5000, 128), (3, 32003, 16), (2, 65536, 64),
        (1, 131071, 100), (1, 262144, 8)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('R,V,k', ROWS)
def test_select_rows(R, V, k, dtype):
    g = torch.Generator(device='cuda').manual_seed(R * 1000 + V)
    x = (torch.randn(R, V, device='cuda', generator=g) * 2.5).to(dtype)
    _check_select(x, k, 1.0 if V % 2 else 4.0)


PLANES = [(1, 1, 1, 2, 1), (2, 3, 1, 5, 3), (2, 19, 13, 17, 5), (1, 150, 16, 33, 10), (2, 150, 8, 8, 16), (1, 64, 9, 9, 64), (1, 200, 5, 60, 33), (1, 300, 3, 7, 128),
          (3, 21, 16, 16, 1), (1, 40, 20, 20, 17)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,C,H,W,k', PLANES)
def test_select_planes(B, C, H, W, k, dtype):
    g = torch.Generator(device='cuda').manual_seed(C * 1000 + H)
    x = (torch.randn(B, C, H, W, device='cuda', generator=g) * 2.5).to(dtype)
    _check_select(x, k, 2.0)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(3, 700), (2, 5003), (2, 40000), (2, 70, 5, 9)])
@pytest.mark.parametrize('kind', ['constant', 'levels', 'ascending', 'descending', 'zeros', 'minus_inf', 'lowest', 'nan', 'one_inf'])
def test_select_adverse_rows(shape, kind, dtype):
    """ties (the lowest class wins), sorted rows, signed zeros, rows of -inf or of the type's lowest value, NaN, one infinity"""
    g = torch.Generator(device='cuda').manual_seed(5)
    n = shape[1]
    ramp = (torch.arange(n, device='cuda').float() / 16).view((1, n) + (1,) * (len(shape) - 2)).expand(shape)
    rand = torch.rand(shape, device='cuda', generator=g)
    x = {'constant': torch.full(shape, 1.5, device='cuda'),
         'levels': torch.floor(rand * 3),
         'ascending': ramp, 'descending': -ramp,
         'zeros': torch.where(rand < 0.5, 0.0, -0.0),
         'minus_inf': torch.where(rand < 0.004, 1.0, -math.inf),
         'lowest': torch.where(rand < 0.004, 1.0, torch.finfo(dtype).min),
         'nan': torch.where(rand < 0.002, math.nan, rand),
         'one_inf': rand}[kind].to(dtype).contiguous()
    k = 12
    if kind == 'one_inf':
        x.view(shape[0], n, -1)[:, n // 2] = math.inf
    if kind == 'nan':
        x.view(shape[0], n, -1)[:, n // 3] = math.nan
        assert int(x.isnan().view(shape[0], n, -1).sum(1).max()) <= 200
        k = 30 if n < 6000 else 128
        if int(x.isnan().view(shape[0], n, -1).sum(1).max()) > k:        # NaN left over: the rest is NaN, which the comparison below does not take
            x = torch.where(x.isnan() & (torch.arange(n, device='cuda').view((1, n) + (1,) * (len(shape) - 2)) != n // 3), torch.zeros_like(x), x)
    _check_select(x, k, 1.0)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(3, 700), (2, 5003), (2, 40000), (2, 70, 5, 9), (2, 300, 3, 4)])
@pytest.mark.parametrize('count', [12, 13, 40, 70])
def test_infinities_and_nan_that_are_left_over(shape, count, dtype):
    """more infinities than entries: the rest is their sum, inf; more NaN than entries: NaN; infinities behind NaN: inf"""
    from segdistill_amd import ops
    g = torch.Generator(device='cuda').manual_seed(count)
    n, k = shape[1], 12
    x = torch.randn(shape, device='cuda', generator=g).to(dtype)
    at = torch.randperm(n, device='cuda', generator=g)[:count]
    x[:, at] = math.inf
    _, _, rest = _check_select(x, k, 1.0)                                            # count = k: the finite ones are what is left
    assert bool(torch.isposinf(rest).all()) == (count > k)
    x[:, at[:k]] = math.nan
    v, i, rest = ops.topk_logits(x, k)
    assert v.isnan().all() and (i.sort(1).values == at[:k].sort().values.view((1, k) + (1,) * (len(shape) - 2))).all()
    assert bool(torch.isposinf(rest).all()) == (count > k)
    x[:, at] = math.nan
    v, i, rest = ops.topk_logits(x, k)
    assert v.isnan().all() and bool(rest.isnan().all()) == (count > k)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [40, 700, 2049, 5003, 30001, 40000, 140001])
@pytest.mark.parametrize('kind', ['tiny tau', 'huge logits', 'huge positive logits'])
def test_rest_where_a_logit_over_tau_leaves_fp32(V, kind, dtype):
    """logits whose quotient by tau is beyond 2^128: 2^((x - bound) / tau) is 0 or 1 all the same, and the rest is the largest logit left over"""
    g = torch.Generator(device='cuda').manual_seed(V)
    rand = torch.rand(3, V, device='cuda', generator=g)
    if kind == 'tiny tau':
        tau, x = 1e-37, -30.0 - torch.floor(rand * 60) / 4                          # levels of a quarter, each many times over in a long row
    else:
        tau, x = 1.0, torch.where(rand < 24 / V, -2.5e38, -3e38)
        if kind == 'huge positive logits':
            x = -x
    for k in (1, 7, 30):
        _check_select(x.to(dtype), k, tau)


def test_more_rows_than_one_launch_holds():
    from segdistill_amd import ops
    rows = 4 * 0xffffff + 37                                                         # four rows per workgroup, 2^24 - 1 workgroups
    x = torch.randn(rows, 2, device='cuda', generator=torch.Generator(device='cuda').manual_seed(3))
    v, i, rest = ops.topk_logits(x, 1)
    second = (x[:, 1] > x[:, 0])
    assert torch.equal(v[:, 0], x.amax(1)) and torch.equal(i[:, 0], second.int())
    # rest = b + log s with s = 2^(a c2 - b c2) of the one that is left, a, relative to b >= a.  In steps of U: the shift b c2 rounds by |b|, c2 and the
    # argument by 2 |a - b|, the exponential by 2, the logarithm by 2 |a - b|, the result by |a|: at most |a| + |b| + 4 |a - b| + 2 <= 5 (|a| + |b|) + 2
    low = x.amin(1)
    assert ((rest - low).abs() <= U * (5 * x.abs().sum(1) + 2)).all()


def test_select_takes_strided_and_offset_views():
    g = torch.Generator(device='cuda').manual_seed(6)
    base = torch.randn(1 + 3 * 4001, device='cuda', generator=g)
    _check_select(base[1:].view(3, 4001), 20, 1.0)                                  # rows that start 4 bytes off a 16-byte boundary
    _check_select(base[:12000].to(torch.bfloat16)[3:3 + 3 * 1501].view(3, 1501), 9, 1.0)
    _check_select(base[:12000].view(2, 60, 10, 10).to(memory_format=torch.channels_last), 9, 1.0)
    _check_select(base[:12000].view(3, 8, 500), 9, 1.0)                             # [B, N, C]


# ---- the criterion ------------------------------------------------------------------------------------------------------------------------------
def _kl_ref(S, values, index, rest, tau, alpha, valid):
    """The definition in fp64 on rows [R, C] -> (loss, dS, q, P, terms): P = the teacher's probability per class (duplicates summed), terms = sum p (|log p| + |log q|)."""
    S = _by_rows(S.detach()).double().cpu()
    v, i = _by_rows(values).double().cpu(), _by_rows(index).long().cpu()
    R, C = S.shape
    live = (i >= 0) & (i < C)
    ii = torch.where(live, i, torch.zeros_like(i))
    t = torch.where(live, v, torch.full_like(v, -math.inf))
    if rest is not None:
        t = torch.cat([t, rest.double().cpu().reshape(-1, 1)], 1)
    says = (t > -math.inf).any(1)
    t = torch.where(says.unsqueeze(1), t, torch.zeros_like(t))
    logp = torch.log_softmax(t / tau, 1)
    p = torch.where(says.unsqueeze(1), logp.exp(), torch.zeros_like(logp))
    member = torch.zeros(R, C, dtype=torch.bool)
    for j in range(i.shape[1]):
        member[torch.arange(R)[live[:, j]], i[live[:, j], j]] = True
    m = S.amax(1, keepdim=True)
    e = torch.exp((S - m) / tau)
    q = e / e.sum(1, keepdim=True)
    logq = (S - m) / tau - torch.log(e.sum(1, keepdim=True))
    P = torch.zeros(R, C, dtype=torch.float64)
    k = i.shape[1]
    pk = torch.where(live, p[:, :k], torch.zeros_like(p[:, :k]))
    for j in range(k):
        P[torch.arange(R), ii[:, j]] += pk[:, j]
    lq = logq.gather(1, ii)
    term = torch.where(pk > 0, pk * (logp[:, :k] - lq), torch.zeros_like(pk))
    size = torch.where(pk > 0, pk * (logp[:, :k].abs() + lq.abs()), torch.zeros_like(pk)).sum(1)
    kl = term.sum(1)
    d = torch.where(member, q - P, q)
    if rest is not None:
        low = torch.where(member, torch.full_like(S, -math.inf), S)
        lq_r = torch.logsumexp(low / tau, 1) - torch.logsumexp(S / tau, 1)
        pr = p[:, -1]
        kl = kl + torch.where(pr > 0, pr * (logp[:, -1] - lq_r), torch.zeros_like(pr))
        size = size + torch.where(pr > 0, pr * (logp[:, -1].abs() + lq_r.abs()), torch.zeros_like(pr))
        ur = torch.softmax(torch.where(member.all(1, keepdim=True), S, low) / tau, 1)
        d = torch.where(member, d, (lq_r.exp() - pr).unsqueeze(1) * ur)
        P = torch.where(member, P, pr.unsqueeze(1) * ur)
    ok = torch.ones(R, dtype=torch.bool) if valid is None else valid.cpu().reshape(-1).bool()
    n = int(ok.sum())
    keep = (ok & says).unsqueeze(1)
    d = torch.where(keep, d, torch.zeros_like(d)) * (alpha / (tau * max(n, 1)))
    kl = torch.where(keep[:, 0], kl, torch.zeros_like(kl))
    size = torch.where(keep[:, 0], size, torch.zeros_like(size))
    return alpha * kl.sum() / max(n, 1), d, (q + P) * (alpha / (tau * max(n, 1))), alpha * size.sum() / max(n, 1)


def _check_kl(S, values, index, rest, tau, alpha, valid, up=0.7):
    from segdistill_amd import ops
    S = S.detach().requires_grad_()
    loss = ops.topk_kl(S, values, index, rest, tau=tau, alpha=alpha, valid=valid)
    (loss * up).backward()
    rl, rd, size, lsize = _kl_ref(S, values, index, rest, tau, alpha, valid)
    C = S.shape[1] if S.dim() == 4 else S.shape[-1]
    tol = 2 * rel(C)
    if torch.isfinite(rl):
        assert abs(float(loss) - float(rl)) <= tol * float(lsize) + 4 * U * abs(float(rl)) + 2 * tol * alpha, (float(loss), float(rl))
    else:
        assert float(loss) == float(rl)
    got, ref = _by_rows(S.grad).double().cpu(), rd * up
    lim = tol * up * size + (half_step(S.dtype) + 8 * U) * ref.abs() + 1e-30
    over = ((got - ref).abs() - lim).max()
    assert torch.isfinite(got).all() and over <= 0, (float(over), float((got - ref).abs().max()))
    g1 = S.grad.clone()
    S.grad = None
    (ops.topk_kl(S, values, index, rest, tau=tau, alpha=alpha, valid=valid) * up).backward()
    assert torch.equal(g1, S.grad)
    return float(loss), g1


KL = [  # shape, k, tau, alpha
    ((1, 2), 1, 1.0, 1.0), ((5, 7), 7, 2.0, 3.0), ((33, 19), 5, 1.0, 1.0), ((3, 4, 150), 10, 4.0, 3.0), ((6, 2048), 64, 1.0, 1.0), ((3, 2049), 100, 1.0, 1.0), ((2, 32003), 16, 2.0, 1.0),
    ((1, 131072), 128, 1.0, 1.0), ((1, 3, 2, 2), 1, 1.0, 1.0), ((2, 19, 13, 17), 5, 2.0, 1.0), ((2, 150, 12, 31), 10, 4.0, 3.0), ((1, 33, 9, 9), 33, 1.0, 1.0), ((1, 700, 5, 7), 128, 1.0, 1.0),
    ((1, 256, 8, 40), 64, 1.0, 2.0)]


def _teacher(S, k, tau, g, dtype):
    from segdistill_amd import ops
    return ops.topk_logits((0.7 * S.float() + torch.randn(S.shape, device='cuda', generator=g) * 1.5).to(dtype), k, tau=tau)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('with_rest', [True, False])
@pytest.mark.parametrize('drop', [0.0, 0.4])
@pytest.mark.parametrize('shape,k,tau,alpha', KL)
def test_criterion_and_gradient(shape, k, tau, alpha, drop, with_rest, dtype):
    g = torch.Generator(device='cuda').manual_seed(sum(shape) + k)
    S = (torch.randn(shape, device='cuda', generator=g) * 2).to(dtype)
    v, i, r = _teacher(S, k, tau, g, dtype)
    rows = (shape[0],) + shape[2:] if len(shape) == 4 else shape[:-1]
    valid = torch.rand(rows, device='cuda', generator=g) >= drop if drop else None
    _check_kl(S, v, i, r if with_rest else None, tau, alpha, valid)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(16384, 30), (65536, 12), (66001, 12), (2047, 2052), (2049, 2052), (16411, 2052), (2050, 8193), (1023, 8200), (256, 33001), (257, 33001), (255, 66001), (1025, 33001)])
def test_waves_per_row_and_rows_per_workgroup(shape, dtype):
    """either side of the sizes where a row goes to more waves, or a workgroup to a second row"""
    g = torch.Generator(device='cuda').manual_seed(shape[0])
    S = (torch.randn(shape, device='cuda', generator=g) * 2).to(dtype)
    v, i, r = _teacher(S, 6, 1.0, g, dtype)
    _check_kl(S, v, i, r, 1.0, 1.0, torch.rand(shape[0], device='cuda', generator=g) >= 0.3)


@pytest.mark.parametrize('shape', [(9, 40), (4, 3001), (2, 40, 3, 5)])
@pytest.mark.parametrize('with_rest', [True, False])
def test_entries_absent_doubled_and_without_weight(shape, with_rest):
    """indices outside the classes are no entries; a class listed twice; entries at -inf; a row without a single entry; an fp32 student with bf16 values"""
    g = torch.Generator(device='cuda').manual_seed(3)
    S = torch.randn(shape, device='cuda', generator=g) * 2
    v, i, r = _teacher(S, 8, 1.0, g, torch.bfloat16)
    iv, vv = (t.movedim(1, -1) if t.dim() == 4 else t for t in (i, v))          # views with the entries last
    iv[..., 3] = iv[..., 1]
    iv[..., 5] = iv[..., 1]
    iv[..., 6] = -1
    iv[..., 7] = shape[1] + 5
    vv[..., 2] = -math.inf
    iv.reshape(-1, 8)                                                            # (views only)
    flat = i.view(-1, 8) if i.dim() == 2 else None
    if flat is not None:
        flat[1] = -1
        if r is not None:
            r.view(-1)[1] = -math.inf
    _check_kl(S, v, i, r if with_rest else None, 1.0, 2.0, None)
    if flat is not None:
        from segdistill_amd import ops
        T = S.detach().requires_grad_()
        ops.topk_kl(T, v, i, r if with_rest else None, tau=1.0, alpha=2.0).backward()
        assert (T.grad[1] == 0).all()
    _check_kl(S, v, i.long(), r if with_rest else None, 1.0, 2.0, None)


@pytest.mark.parametrize('shape', [(6, 50), (3, 4000), (2, 50, 2, 3)])
def test_masked_rows_may_hold_anything_and_no_row_may_be_left(shape):
    from segdistill_amd import ops
    g = torch.Generator(device='cuda').manual_seed(4)
    S = torch.randn(shape, device='cuda', generator=g)
    v, i, r = _teacher(S, 4, 1.0, g, torch.float32)
    rows = (shape[0],) + shape[2:] if len(shape) == 4 else shape[:-1]
    valid = torch.rand(rows, device='cuda', generator=g) < 0.5
    valid.view(-1)[0], valid.view(-1)[1] = True, False
    clean = _check_kl(S, v, i, r, 1.0, 1.0, valid)
    bad = (~valid).unsqueeze(1).expand(shape) if S.dim() == 4 else (~valid).unsqueeze(-1).expand(shape)
    S2 = torch.where(bad, torch.full_like(S, math.nan), S).requires_grad_()
    v2 = torch.where((~valid).unsqueeze(1 if S.dim() == 4 else -1), torch.full_like(v, math.inf), v)
    loss = ops.topk_kl(S2, v2, i, torch.where(valid, r, torch.full_like(r, math.nan)), tau=1.0, alpha=1.0, valid=valid)
    loss.backward()
    up = 0.7
    assert float(loss) == clean[0] and torch.allclose(S2.grad * up, clean[1], rtol=4 * U, atol=0) and (S2.grad[bad] == 0).all()
    S3 = torch.full_like(S, math.nan).requires_grad_()
    loss = ops.topk_kl(S3, v, i, r, tau=1.0, alpha=1.0, valid=torch.zeros_like(valid))
    loss.backward()
    assert float(loss) == 0 and (S3.grad == 0).all()


@pytest.mark.parametrize('shape', [(6, 50), (3, 4000), (2, 50, 2, 3)])
@pytest.mark.parametrize('low', [-math.inf, torch.finfo(torch.float32).min])
def test_students_whose_other_classes_are_masked_out(shape, low):
    """logits at -inf / the lowest value: for some classes outside the entries, and for all of them"""
    from segdistill_amd import ops
    g = torch.Generator(device='cuda').manual_seed(8)
    S = torch.randn(shape, device='cuda', generator=g)
    v, i, r = _teacher(S, 4, 1.0, g, torch.float32)
    cd = 1 if S.dim() == 4 else -1
    member = torch.zeros_like(S, dtype=torch.bool).scatter(cd, i.long(), True)
    some = torch.where(~member & (torch.rand(shape, device='cuda', generator=g) < 0.5), torch.full_like(S, low), S)
    _check_kl(some, v, i, r, 1.0, 1.0, None)
    every = torch.where(member, S, torch.full_like(S, low))
    _check_kl(every, v, i, None, 1.0, 1.0, None)
    if low == -math.inf:
        loss = ops.topk_kl(every, v, i, r, tau=1.0, alpha=1.0)
        assert float(loss) == math.inf                                     # the teacher gives the others weight, the student none


def test_a_confident_student_keeps_the_digits_of_the_rest():
    """q_rest = 2e-9: total minus listed would have none left"""
    S = torch.zeros(4, 300, device='cuda')
    S[:, 7] = 26.0
    v, i = torch.tensor([[5.0, 1.0]], device='cuda').repeat(4, 1), torch.tensor([[7, 9]], device='cuda', dtype=torch.int32).repeat(4, 1)
    _check_kl(S, v, i, torch.full((4,), -2.0, device='cuda'), 1.0, 1.0, None)
    S[:, 7] = 300.0                                                         # and beyond the exponent range
    _check_kl(S, v, i, torch.full((4,), -2.0, device='cuda'), 1.0, 1.0, None)


@pytest.mark.parametrize('shape,k', [((3, 40), 6), ((2, 12, 2, 3), 3)])
@pytest.mark.parametrize('with_rest', [True, False])
def test_gradient_against_differences(shape, k, with_rest):
    """central differences with step h = 2^-5: the cubic term is at most alpha h^2 / 6 per row (third derivatives of a log-partition are below 1), the loss
    is good to 2^-20 alpha, which the difference divides by 2 h"""
    from segdistill_amd import ops
    g = torch.Generator(device='cuda').manual_seed(9)
    S = torch.randn(shape, device='cuda', generator=g)
    v, i, r = _teacher(S, k, 1.0, g, torch.float32)
    r = r if with_rest else None
    S.requires_grad_()
    ops.topk_kl(S, v, i, r, tau=1.0, alpha=1.0).backward()
    h = 2.0 ** -5
    rows = S.numel() // shape[1]
    with torch.no_grad():
        for at in torch.randperm(S.numel(), generator=torch.Generator().manual_seed(1))[:24].tolist():
            d = torch.zeros(S.numel(), device='cuda')
            d[at] = h
            d = d.view(shape)
            diff = (float(ops.topk_kl(S + d, v, i, r, tau=1.0, alpha=1.0)) - float(ops.topk_kl(S - d, v, i, r, tau=1.0, alpha=1.0))) / (2 * h)
            assert abs(diff - float(S.grad.view(-1)[at])) <= h * h / 6 / rows + 2.0 ** -20 / h, at


def test_strided_operands_and_offset_rows():
    g = torch.Generator(device='cuda').manual_seed(10)
    base = torch.randn(1 + 4 * 4099, device='cuda', generator=g)
    S = base[1:].view(4, 4099)
    v, i, r = _teacher(S, 9, 1.0, g, torch.float32)
    a = _check_kl(S, v, i, r, 1.0, 1.0, None)
    wide = torch.empty(4, 18, device='cuda', dtype=torch.int32)
    wide[:, ::2] = i
    b = _check_kl(S.t().contiguous().t(), v.t().contiguous().t(), wide[:, ::2], r, 1.0, 1.0, None)
    assert torch.allclose(a[1], b[1], rtol=1e-4, atol=1e-9)
    S4 = base[:2 * 20 * 9 * 7].view(2, 20, 9, 7)
    v, i, r = _teacher(S4, 3, 1.0, g, torch.float32)
    _check_kl(S4.to(memory_format=torch.channels_last), v, i, r, 1.0, 1.0, None)


def test_runs_on_the_current_stream_and_in_a_replayed_graph():
    """selection, criterion and gradient captured once and replayed on new inputs, with eager work between the replays; and on a side stream"""
    from segdistill_amd import ops
    g = torch.Generator(device='cuda').manual_seed(11)

    def inputs(n):
        return [(torch.randn(2, 40, 9, 11, device='cuda', generator=g), torch.randn(2, 40, 9, 11, device='cuda', generator=g)) for _ in range(n)]

    def step(s, t):
        v, i, r = ops.topk_logits(t, 5, tau=2.0)
        loss = ops.topk_kl(s, v, i, r, tau=2.0, alpha=3.0)
        return loss.detach(), torch.autograd.grad(loss, s)[0]

    sets = inputs(4)
    eager = [step(s.clone().requires_grad_(), t) for s, t in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s_in, t_in = torch.empty_like(sets[0][0]).requires_grad_(), torch.empty_like(sets[0][1])
    with torch.no_grad():
        s_in.copy_(sets[0][0]), t_in.copy_(sets[0][1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            on_side = step(s_in, t_in)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(s_in, t_in)
    for (s, t), want in zip(sets[::-1], eager[::-1]):
        with torch.no_grad():
            s_in.copy_(s), t_in.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step(s.clone().requires_grad_(), t)


def test_offsets_past_32_bits():
    """rows whose first element lies beyond 2^31 elements (bf16: 4.6 GB of logits)"""
    from segdistill_amd import ops
    R, V = 17600, 131072
    x = torch.empty(R, V, device='cuda', dtype=torch.bfloat16)
    x.fill_(-3.0)
    at = torch.arange(R, device='cuda') * 7 % V
    x[torch.arange(R, device='cuda'), at] = 5.0
    v, i, r = ops.topk_logits(x, 2, tau=1.0)
    assert torch.equal(i[:, 0].long(), at) and torch.equal(i[:, 1].long(), (at == 0).long()) and (v[:, 0] == 5).all() and (v[:, 1] == -3).all()
    assert float((r - (-3 + math.log(V - 2))).abs().max()) < 1e-4
    x.requires_grad_()
    loss = ops.topk_kl(x, v, i, r, tau=1.0, alpha=1.0)
    (d,) = torch.autograd.grad(loss, x)
    assert abs(float(loss)) < 1e-6 and float(d[-1].abs().max()) < 1e-8 and float(d[0].abs().max()) < 1e-8


def _poisoned(like):
    """the address of memory that holds NaN, free again: the next tensor of that size"""
    torch.cuda.synchronize()
    t = torch.full_like(like, math.nan)
    return t.data_ptr()


def _parts_agree(S, v, i, r, valid, tau, parts):
    """topk_kl of all of S against the same on `parts`, equal pieces of it: the loss is their mean; the gradient of a piece alone is as many times larger, up to
    the rounding of the two results (half a step of bf16 each) and of the 32-bit factors before it.  The gradient is written where NaN was."""
    from segdistill_amd import ops
    S.requires_grad_()
    loss = ops.topk_kl(S, v, i, r, tau=tau, alpha=1.0, valid=valid)
    at = _poisoned(S.detach())
    (d,) = torch.autograd.grad(loss, S)
    assert d.data_ptr() == at
    mean = 0.0
    for p in parts:
        s = S.detach()[p].clone().requires_grad_()
        one = ops.topk_kl(s, v[p], i[p], r[p], tau=tau, alpha=1.0, valid=None if valid is None else valid[p])
        (g,) = torch.autograd.grad(one, s)
        mean += float(one.detach()) / len(parts)
        a, b = d[p].float() * len(parts), g.float()
        assert bool(((a - b).abs() <= (2 ** -7 + 16 * U) * b.abs()).all()), p
        assert float(b.abs().amax()) > 0
    assert abs(float(loss.detach()) - mean) <= 4 * U * mean and mean > 0.1


def test_rows_past_32_bits_against_their_parts():
    """2.3e9 logits in rows (bf16): selection and criterion, every row of the gradient, against calls on eighths"""
    from segdistill_amd import ops
    R, V = 17600, 131072
    g = torch.Generator(device='cuda').manual_seed(21)
    S = torch.empty(R, V, device='cuda', dtype=torch.bfloat16).normal_(std=2.0, generator=g)
    parts = [slice(a, a + R // 8) for a in range(0, R, R // 8)]
    top = ops.topk_logits(S, 5, tau=2.0)
    for p in (parts[0], parts[-1]):
        assert all(torch.equal(a[p], b) for a, b in zip(top, ops.topk_logits(S[p].clone(), 5, tau=2.0)))
    assert int(top[1][-1].long().unique().numel()) == 5 and torch.equal(top[0][-1], S[-1][top[1][-1].long()])
    i = torch.randint(0, V, (R, 6), device='cuda', generator=g, dtype=torch.int32)
    v = torch.randn(R, 6, device='cuda', generator=g) * 3
    _parts_agree(S, v, i, torch.randn(R, device='cuda', generator=g) + 9.0, None, 2.0, parts)


def test_planes_past_32_bits_against_their_images():
    """2.9e9 logits in class planes (bf16), the last image wholly beyond 2^31"""
    from segdistill_amd import ops
    B, C, H = 4, 150, 2200
    g = torch.Generator(device='cuda').manual_seed(22)
    S = torch.empty(B, C, H, H, device='cuda', dtype=torch.bfloat16).normal_(std=2.0, generator=g)
    T = torch.empty(B, C, H, H, device='cuda', dtype=torch.bfloat16).normal_(std=3.0, generator=g)
    assert 3 * C * H * H > 2 ** 31
    v, i, r = ops.topk_logits(T, 5, tau=2.0)
    images = [slice(b, b + 1) for b in range(B)]
    for p in images:
        assert all(torch.equal(a[p], b) for a, b in zip((v, i, r), ops.topk_logits(T[p].clone(), 5, tau=2.0)))
    del T
    # as many valid pixels in every image, so that a part's mean is over exactly a quarter of them
    keep = torch.rand(1, H, H, device='cuda', generator=g) < 0.8
    valid = torch.cat([keep.roll(n, 2) for n in range(B)])
    _parts_agree(S, v, i, r, valid, 2.0, images)


def test_criterion_module_in_the_distillation_loss():
    """TopKLoss by its registered name: selection on the teacher tap, criterion on the student tap, ignored labels left out, a teacher of another size"""
    from segdistill_amd.distillation.opts import DistillationLoss
    g = torch.Generator(device='cuda').manual_seed(12)
    for ignore, tsize in ((None, 16), (255, 16), (255, 24)):
        cfg = [dict(student_layer='head', teacher_layer='head', loss_name='TopKLoss', loss_config=dict(k=6, alpha=3.0, tau=2.0, ignore_index=ignore))]
        crit = DistillationLoss(cfg)
        s = torch.randn(2, 19, 16, 16, device='cuda', generator=g).requires_grad_()
        t = torch.randn(2, 19, tsize, tsize, device='cuda', generator=g)
        gt = torch.randint(0, 19, (2, 1, 64, 64), device='cuda', generator=g)
        gt[torch.rand(gt.shape, device='cuda', generator=g) < 0.3] = 255
        out = crit({'head': s}, {'head': t}, gt, 1)
        assert list(out) == ['loss_head<->head_other']
        tt = t if tsize == 16 else torch.nn.functional.interpolate(t, size=(16, 16), mode='bilinear', align_corners=False)
        valid = None if ignore is None else (torch.nn.functional.interpolate(gt.float(), size=(16, 16), mode='nearest')[:, 0] != ignore)
        v, i, r = _sorted_ref(tt, 6, 2.0)
        rl, rd, size, lsize = _kl_ref(s, v, i, r, 2.0, 3.0, valid)
        assert abs(float(out['loss_head<->head_other']) - float(rl)) <= 1e-4 * float(lsize)      # (a resized teacher differs by the resize's rounding)
        out['loss_head<->head_other'].backward()
        assert float((_by_rows(s.grad).double().cpu() - rd).norm() / rd.norm()) < 1e-4


def test_refusals():
    from segdistill_amd import ops
    x = torch.zeros(3, 10, device='cuda')
    for bad, err in ((dict(k=0), ValueError), (dict(k=11), ValueError), (dict(k=2, tau=0.0), ValueError), (dict(k=2, tau=math.nan), ValueError)):
        with pytest.raises(err):
            ops.topk_logits(x, **bad)
    with pytest.raises(ValueError):
        ops.topk_logits(torch.zeros(3, 200, device='cuda'), 129)
    with pytest.raises(ValueError):
        ops.topk_logits(x[0], 2)
    with pytest.raises(TypeError):
        ops.topk_logits(x.half(), 2)
    v, i, r = ops.topk_logits(x, 2)
    ok = torch.ones(3, dtype=torch.bool, device='cuda')

    def call(S=x, v=v, i=i, r=r, tau=1.0, valid=ok):
        return ops.topk_kl(S, v, i, r, tau=tau, alpha=1.0, valid=valid)
    assert float(call()) == pytest.approx(0.0, abs=1e-6)
    for kw in (dict(v=v[:2]), dict(i=i[:, :1]), dict(r=r[:2]), dict(valid=ok[:2]), dict(tau=-1.0), dict(v=v.view(3, 2, 1)), dict(S=x.view(3, 10, 1)), dict(r=r.cpu())):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(i=i.float()), dict(v=v.half()), dict(S=x.half()), dict(r=r.double()), dict(valid=ok.int())):
        with pytest.raises(TypeError):
            call(**kw)
    with pytest.raises(ValueError):                                                 # bits of 8000 classes per pixel
        ops.topk_kl(torch.zeros(1, 8000, 2, 2, device='cuda'), torch.zeros(1, 1, 2, 2, device='cuda'), torch.zeros(1, 1, 2, 2, device='cuda', dtype=torch.int32), tau=1.0, alpha=1.0)
    e = torch.zeros(0, 10, device='cuda', requires_grad=True)
    ve, ie, re = ops.topk_logits(e.detach(), 2)
    assert ve.shape == ie.shape == (0, 2) and re.shape == (0,)
    loss = ops.topk_kl(e, ve, ie, re, tau=1.0, alpha=1.0)
    loss.backward()
    assert float(loss) == 0 and e.grad.shape == (0, 10)


def test_two_calls_at_once_and_a_second_derivative():
    """two criteria on the same leaf in one graph, on two streams at once; create_graph is refused instead of answered with constants"""
    from segdistill_amd import ops
    g = torch.Generator(device='cuda').manual_seed(13)
    S = torch.randn(3, 4000, device='cuda', generator=g)
    v, i, r = _teacher(S, 6, 1.0, g, torch.float32)
    parts = []
    for rest in (r, None):
        a = S.clone().requires_grad_()
        ops.topk_kl(a, v, i, rest, tau=1.0, alpha=1.0).backward()
        parts.append(a.grad)
    both = S.clone().requires_grad_()
    (ops.topk_kl(both, v, i, r, tau=1.0, alpha=1.0) + ops.topk_kl(both, v, i, None, tau=1.0, alpha=1.0)).backward()
    assert torch.equal(both.grad, parts[0] + parts[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for k, s in enumerate(streams * 3):
        with torch.cuda.stream(s):
            a = S.clone().requires_grad_()
            loss = ops.topk_kl(a, v, i, (r, None)[k % 2], tau=1.0, alpha=1.0)
            out.append((ops.topk_logits(a.detach(), 6), torch.autograd.grad(loss, a)[0]))
    torch.cuda.synchronize()
    want = ops.topk_logits(S, 6)
    for k, (top, d) in enumerate(out):
        assert torch.equal(d, parts[k % 2]) and all(torch.equal(p, q) for p, q in zip(top, want))
    a = S.clone().requires_grad_()
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(ops.topk_kl(a, v, i, r, tau=1.0, alpha=1.0), a, create_graph=True)


def test_module_refuses_taps_of_different_classes():
    from segdistill_amd.distillation.losses import TopKLoss
    with pytest.raises(ValueError, match='classes'):
        TopKLoss(k=3)(torch.zeros(1, 19, 4, 4, device='cuda'), torch.zeros(1, 21, 4, 4, device='cuda'), torch.zeros(1, 1, 4, 4, device='cuda'), 1)


def test_module_resizes_both_taps_to_the_label_size():
    from segdistill_amd import ops
    from segdistill_amd.distillation.losses import TopKLoss
    g = torch.Generator(device='cuda').manual_seed(14)
    s = torch.randn(2, 19, 9, 9, device='cuda', generator=g).requires_grad_()
    t = torch.randn(2, 19, 9, 9, device='cuda', generator=g)
    gt = torch.randint(0, 19, (2, 1, 36, 36), device='cuda', generator=g)
    loss = TopKLoss(k=4, tau=2.0, alpha=2.0, rest=False, resize_config=dict(mode='bilinear', align_corners=False))(s, t, gt, 1)
    su, tu = (torch.nn.functional.interpolate(x, size=(36, 36), mode='bilinear', align_corners=False) for x in (s, t))
    v, i, r = ops.topk_logits(tu, 4, tau=2.0)
    want = ops.topk_kl(su, v, i, None, tau=2.0, alpha=2.0)
    assert float(loss) == pytest.approx(float(want), rel=1e-4)
    a, b = torch.autograd.grad(loss, s)[0], torch.autograd.grad(want, s)[0]
    assert float((a - b).norm() / b.norm()) < 1e-4


def test_more_rows_than_the_criterion_launches_are_named():
    from segdistill_amd import ops
    rows = 4 * 0xffffff + 1
    S = torch.zeros(rows, 2, device='cuda')
    with pytest.raises(ValueError, match=f'{rows} rows'):
        ops.topk_kl(S, S[:, :1], torch.zeros(rows, 1, device='cuda', dtype=torch.int32), tau=1.0, alpha=1.0)
    loss = ops.topk_kl(S[1:], S[1:, :1], torch.zeros(rows - 1, 1, device='cuda', dtype=torch.int32), torch.zeros(rows - 1, device='cuda'), tau=1.0, alpha=1.0)
    assert float(loss) == 0.0
