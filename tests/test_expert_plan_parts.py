"""An ExpertPlan put together by hand: its parts go to the kernels as plain addresses, so what they are is checked first."""
import pytest
import torch


def _parts(device):
    """offsets, order and slot of three tokens with two choices of two experts, one of them dropped."""
    return [torch.tensor(v, dtype=torch.int32, device=device) for v in ([0, 2, 5], [0, 3, 1, 4, 5, -1], [[0, 2], [-1, 1], [3, 4]])]


def _refused(parts, n_experts, error):
    import gunet_amd
    with pytest.raises(error):
        gunet_amd.ExpertPlan(*parts, n_experts)


def _refusals(device):
    offsets, order, slot = _parts(device)
    for i in range(3):
        for wrong in (torch.int64, torch.float32, torch.int16):
            parts = _parts(device)
            parts[i] = parts[i].to(wrong)
            _refused(parts, 2, TypeError)
        parts = _parts(device)
        parts[i] = parts[i].tolist()
        _refused(parts, 2, TypeError)
    _refused((offsets[:2], order, slot), 2, ValueError)                   # an expert's end is missing
    _refused((offsets, order, slot), 3, ValueError)                       # offsets of fewer experts than named
    _refused((offsets, order, slot), 1, ValueError)
    _refused((offsets[:1], order, slot), 0, ValueError)
    _refused((offsets, order[:5], slot), 2, ValueError)
    _refused((offsets, order.view(3, 2), slot), 2, ValueError)
    _refused((offsets, order, slot.view(6)), 2, ValueError)
    _refused((offsets, order, slot[:, :0]), 2, ValueError)
    _refused((offsets, order, slot.t().contiguous().t()), 2, ValueError)  # the right shape, another layout
    _refused((torch.zeros(6, dtype=torch.int32, device=device)[::2], order, slot), 2, ValueError)
    _refused((offsets, order.flip(0)[:3].repeat_interleave(4)[::2], slot), 2, ValueError)


def test_refusals_need_no_gpu():
    _refusals('cpu')
    _refused(_parts('cpu'), 2, TypeError)                                 # right in everything, but in host memory


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    _refusals('cuda')
    for i in range(3):
        parts = _parts('cuda')
        parts[i] = parts[i].cpu()
        _refused(parts, 2, (TypeError, ValueError))


@pytest.mark.gpu
def test_a_plan_from_its_parts_is_the_sorted_one():
    import gunet_amd as amd
    index = torch.tensor([[0, 1], [5, 0], [1, 1]], dtype=torch.int32, device='cuda')
    plan = amd.expert_plan(index, 2)
    made = amd.ExpertPlan(plan.offsets.clone(), plan.order.clone(), plan.slot.clone(), 2)
    assert {k: v for k, v in vars(made).items() if not torch.is_tensor(v)} == {k: v for k, v in vars(plan).items() if not torch.is_tensor(v)}
    for got, want in zip((made.offsets, made.order, made.slot), _parts('cuda')):
        assert torch.equal(got, want)
    x = torch.randn((3, 40), device='cuda')
    assert torch.equal(amd.expert_dispatch(x, made), amd.expert_dispatch(x, plan))
    empty = amd.expert_plan(index[:0], 2)
    assert amd.ExpertPlan(empty.offsets, empty.order, empty.slot, 2).n_rows == 0
