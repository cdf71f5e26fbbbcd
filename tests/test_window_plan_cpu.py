"""The bucket plan of a Swin block's window attention (rel_bias.BucketPlan): a captured step holds the addresses of its tensors, so a checkpoint load writes
it in place.  Host logic: no GPU."""
import copy
import types
import weakref

import pytest
import torch


def _tensors(plan):
    return dict(plan.named_buffers())


def _at(plan):
    return {n: b.data_ptr() for n, b in _tensors(plan).items()}


def _same(plan, index, nb):
    from segdistill_amd.rel_bias import BucketPlan
    want = _tensors(BucketPlan(index, nb))
    return set(want) == set(_tensors(plan)) and all(torch.equal(b, want[n]) for n, b in _tensors(plan).items())


def test_a_load_writes_the_plan_where_it_is():
    from segdistill_amd.backbones.swin import WindowAttention
    att = WindowAttention(64, (7, 7), 2)
    plan, at = att.bias_plan, _at(att.bias_plan)
    sd = {n: t.clone() for n, t in att.state_dict().items()}
    for index in (sd['relative_position_index'], sd['relative_position_index'].flip(0), sd['relative_position_index'].t().contiguous()):
        sd['relative_position_index'] = index
        att.load_state_dict(sd)
        assert att.bias_plan is plan and _at(plan) == at and _same(plan, index, 169)


def test_an_update_that_does_not_fit_writes_nothing():
    from segdistill_amd.rel_bias import BucketPlan
    index = torch.arange(4000).view(40, 100) % 8
    plan = BucketPlan(index, 8)
    keep = {n: b.clone() for n, b in _tensors(plan).items()}
    for other in (torch.zeros_like(index), index.t().contiguous()):
        assert not plan.update(other)
        assert all(torch.equal(b, keep[n]) for n, b in _tensors(plan).items())
    with pytest.raises(ValueError):
        plan.update(index + 1)
    assert plan.update(index.flip(1)) and _same(plan, index.flip(1), 8)


def test_a_plan_that_is_replaced_stays_alive():
    """24 x 24 tokens, every pair in one bucket: 648 chunks more than a relative position index has"""
    from segdistill_amd.backbones.swin import WindowAttention
    att = WindowAttention(32, (24, 24), 1)
    first = att.bias_plan
    at, alive = _at(first), weakref.ref(first)
    sd = {n: t.clone() for n, t in att.state_dict().items()}
    index = sd['relative_position_index'].clone()
    sd['relative_position_index'] = torch.zeros_like(index)
    att.load_state_dict(sd)
    assert att.bias_plan is not first and _same(att.bias_plan, torch.zeros_like(index), 47 * 47)
    del first
    assert alive() is not None and _at(alive()) == at and _same(alive(), index, 47 * 47)


def _trainer(att):
    from segdistill_amd.engine import KDTrainer
    model = torch.nn.Sequential(att)
    t = KDTrainer.__new__(KDTrainer)
    t.model, t.iter = model, 0
    t.optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
    t.reducer = types.SimpleNamespace(params=list(model.parameters()))
    t._graph = object()
    return t


def test_the_trainer_keeps_its_captured_step_over_a_load_unless_a_plan_was_replaced():
    from segdistill_amd.backbones.swin import WindowAttention
    t = _trainer(WindowAttention(32, (24, 24), 1))
    assert t.model[0].bias_plan.num_chunks > 47 * 47                              # built: a captured step has used it
    graph = t._graph
    sd = {'state_dict': {n: v.clone() for n, v in t.model.state_dict().items()}, 'optimizer': t.optimizer.state_dict(), 'meta': {'iter': 3}}
    t.load_state_dict(sd)
    assert t._graph is graph and t.iter == 3
    sd['state_dict']['0.relative_position_index'] = torch.zeros_like(sd['state_dict']['0.relative_position_index'])
    with pytest.warns(UserWarning, match='relative_position_index'):
        t.load_state_dict(sd)
    assert t._graph is None


def test_a_plan_built_in_inference_mode_serves_a_backward():
    from segdistill_amd.rel_bias import BucketPlan
    with torch.inference_mode():
        index = torch.arange(12).view(3, 4) % 5
        plan = BucketPlan(index, 5)
    assert not any(b.is_inference() for b in plan.buffers()) and _same(plan, index, 5)


def test_the_plan_follows_its_buffer():
    """changed in place (the plan too, at its address), replaced, filled by hand after to_empty or on the meta device, copied with its module"""
    from segdistill_amd.backbones.swin import WindowAttention
    att = WindowAttention(64, (4, 5), 2)
    index, plan, at = att.relative_position_index, att.bias_plan, _at(att.bias_plan)
    assert att.bias_plan is plan
    index.copy_(index.flip(0).clone())
    assert att.bias_plan is plan and _at(plan) == at and _same(plan, index, 63)
    index.copy_(index.clone())                                             # (the same again)
    assert att.bias_plan is plan and att.bias_plan is plan
    other = copy.deepcopy(att)
    assert other.bias_plan is not plan and _same(other.bias_plan, index, 63)
    att.relative_position_index = index.roll(1, 0)
    assert att.bias_plan is not plan and _same(att.bias_plan, index.roll(1, 0), 63) and _same(plan, index, 63)
    keep = att.bias_plan
    att.relative_position_index = att.relative_position_index.clone()
    assert att.bias_plan is keep                                           # another tensor that says the same
    with torch.device('meta'):
        empty = WindowAttention(64, (4, 5), 2)
    assert empty.bias_plan is None
    for a in (empty, other):
        a.to_empty(device='cpu')
        a.relative_position_index.copy_(index)
        assert _same(a.bias_plan, index, 63)
    with torch.inference_mode():
        att.relative_position_index = index.clone()
    assert _same(att.bias_plan, index, 63) and _same(att.bias_plan, index, 63)


def test_a_block_that_never_trains_has_no_plan():
    from segdistill_amd.backbones.swin import WindowAttention, bias_plans
    att = WindowAttention(64, (4, 4), 2)
    att.load_state_dict(att.state_dict())
    with torch.no_grad():
        att(torch.randn(3, 16, 64))
    assert bias_plans(att) == []
    assert bias_plans(torch.nn.Sequential(att, WindowAttention(64, (4, 4), 2))) == [] and len(list(att.modules())) == 6
    assert att.bias_plan is bias_plans(att)[0]
