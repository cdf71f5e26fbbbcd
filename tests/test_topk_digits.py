"""The last steps of topk_kl's rows are in 64 bits: a KL of 1e-4 to 1e-1, the small difference of logarithms of size four to ten, keeps its digits.

The rows are made so that nothing else rounds.  With tau = fl(log2 e) the kernels' factor fl(log2 e / tau) is 1, every logit, value and rest is an integer, and
so every term of every softmax is a power of two: their sums have at most 24 bits and are exact in fp32, in any order.  What is left: (v - z) / tau is taken with
fl(ln 2), which is 2.8e-9 (less than 2^-28) off, and the loss is rounded once.  (The temperature the kernels answer for is 1 / ln 2; the reference takes that.)
A loss may be off by 2^-28 (sum_j p_j |v_j - z_j| + p_r |rest - m|) ln 2 + 2^-24 |loss|, here 1e-8 or less; logarithms in 32 bits are off by up to 2^-22 each."""
import math

import numpy as np
import pytest
import torch

TAU = float(np.float32(math.log2(math.e)))


def _row(V, k, seed):
    """(z [V], values [k], index [k], rest): integers.  The student differs from the teacher by one step here and there."""
    rng = np.random.default_rng(seed * 1000 + V)
    low = -int(math.ceil(math.log2(V))) - 2                                # the classes outside together: between 2^-3 and 2^-2
    z = np.full(V, low, dtype=np.int64)
    index = rng.choice(V, k, replace=False)
    values = np.concatenate([[0], -rng.integers(3, 9, k - 1)])
    z[index] = values + np.concatenate([[0], rng.integers(-1, 2, k - 1)])
    return z, values, index, -3 - int(rng.integers(0, 2))


def _exact(z, values, index, rest):
    """(loss, what it may be off by), in 64 bits, at the temperature 1 / ln 2"""
    ln2 = math.log(2.0)
    low = np.delete(z, index)
    t = np.concatenate([values, [rest]]).astype(np.float64)
    tn = np.exp2(t).sum()
    p = np.exp2(t) / tn
    q_low = np.exp2(low.astype(np.float64)).sum()
    s = q_low + np.exp2(z[index].astype(np.float64)).sum()
    gap = np.concatenate([(values - z[index]) * ln2, [rest * ln2 - math.log(q_low)]])
    loss = float((p * gap).sum() + math.log(s) - math.log(tn))
    size = float((p[:-1] * np.abs(values - z[index])).sum() + p[-1] * abs(rest - int(low.max()))) * ln2
    return loss, 2.0 ** -28 * size + 1.01 * 2.0 ** -24 * abs(loss)


def _end_in_32_bits(z, values, index, rest):
    """the same row with exact sums and every later step in 32 bits"""
    f = np.float32
    ln2 = f(math.log(2.0))
    low = np.delete(z, index)
    e = np.exp2(values.astype(np.float64)).astype(f)
    er, low_s = f(2.0 ** rest), f(np.exp2((low - low.max()).astype(np.float64)).sum())
    s, weights = f(np.exp2(z.astype(np.float64)).sum()), f(e.sum())
    ts = f(weights + er)
    terms = f((e * ((values - z[index]).astype(f) * ln2)).sum(dtype=f))
    ratio = f(np.log(s) - np.log(ts))
    kl = f(f(terms / ts) + f(f(weights / ts) * ratio))
    return float(kl + f(f(er / ts) * f(f(f(rest - int(low.max())) * ln2 - np.log(low_s)) + ratio)))


SIZES = [300, 2048, 3001, 33001, 66001]


@pytest.mark.parametrize('V', SIZES)
def test_the_bound_tells_a_32_bit_end(V):
    rows = [_row(V, 12, seed) for seed in range(12)]
    want = [_exact(*r) for r in rows]
    assert all(1e-4 < loss < 0.3 and tol < 1e-8 for loss, tol in want)
    over = [abs(_end_in_32_bits(*r) - loss) > 2 * tol for r, (loss, tol) in zip(rows, want)]
    assert sum(over) >= 6, over
    assert abs(float(np.float32(math.log(2.0))) / math.log(2.0) - 1) < 2.0 ** -28
    for z, values, index, rest in rows:                                    # sums that 24 bits hold, whatever their order
        assert np.exp2(z.astype(np.float64)).sum() * 2.0 ** -z.min() < 2 ** 24


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('layout', ['rows', 'many rows', 'planes'])
@pytest.mark.parametrize('V', SIZES)
def test_a_small_loss_keeps_its_digits(V, layout, dtype):
    """one row at a time (a mean would hide an error): by every number of waves per row, in workgroups of one and of several rows, and as class planes"""
    from segdistill_amd import ops
    if layout == 'planes' and V > 300:
        V = {2048: 21, 3001: 150, 33001: 255, 66001: 700}[V]
    for seed in range(12):
        z, values, index, rest = _row(V, 12, seed)
        loss, tol = _exact(z, values, index, rest)
        S = torch.tensor(z, device='cuda').to(dtype)
        v, i = torch.tensor(values, device='cuda').to(dtype), torch.tensor(index, device='cuda', dtype=torch.int32)
        r = torch.tensor(float(rest), device='cuda')
        if layout == 'rows':
            S, v, i, r, valid = S.view(1, V), v.view(1, 12), i.view(1, 12), r.view(1), None
        else:
            # the row among others that take no part: the last of more rows than the grid has workgroups for, or a pixel
            n = 1 + (66000 if V <= 300 else 16500 if V <= 3001 else 300) if layout == 'many rows' else 70
            shape = (n, V) if layout == 'many rows' else (1, V, 7, 10)
            valid = torch.zeros(n, dtype=torch.bool, device='cuda')
            valid[n - 1 - seed] = True
            if layout == 'many rows':
                S, v, i, r = (t.expand(n, *t.shape).contiguous() for t in (S, v, i, r))
            else:
                S, v, i = (t.view(1, -1, 1, 1).expand(1, -1, 7, 10).contiguous() for t in (S, v, i))
                r, valid = r.expand(1, 7, 10).contiguous(), valid.view(1, 7, 10)
            assert S.numel() == n * V and shape == tuple(S.shape)
        got = float(ops.topk_kl(S, v, i, r, tau=TAU, alpha=1.0, valid=valid))
        assert abs(got - loss) <= tol, (seed, got, loss, tol)
