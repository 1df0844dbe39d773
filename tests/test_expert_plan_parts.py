"""An ExpertPlan put together by hand: its parts go to the kernels as plain addresses, so what they are is checked first."""
import numpy as np
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
    made = amd.ExpertPlan(plan.offsets.clone(), plan.order.clone(), plan.slot.clone(), np.int64(2))
    assert {k: v for k, v in vars(made).items() if not torch.is_tensor(v)} == {k: v for k, v in vars(plan).items() if not torch.is_tensor(v)}
    for got, want in zip((made.offsets, made.order, made.slot), _parts('cuda')):
        assert torch.equal(got, want)
    x = torch.randn((3, 40), device='cuda')
    assert torch.equal(amd.expert_dispatch(x, made), amd.expert_dispatch(x, plan))
    empty = amd.expert_plan(index[:0], 2)
    assert amd.ExpertPlan(empty.offsets, empty.order, empty.slot, 2).n_rows == 0


@pytest.mark.gpu
@pytest.mark.parametrize('experts, rows, form', [(3000, 3001, 'tile 32 x 128'), (65535, 70001, 'tile 32 x 128'), (65535, 30000, 'skinny 16 rows 2 waves'),
                                                 (65535, 9, 'raw 4 waves')])
def test_more_experts_than_the_sort_takes(experts, rows, form):
    """The experts' product takes 65535 of them, from a plan made by hand: rows that are in order already.  Exact sums of small whole numbers."""
    import gunet_amd as amd
    from mxfp4_forms import form_of
    k, n = 64, 40
    g = torch.Generator(device='cuda').manual_seed(rows)
    assert form_of(rows, k, n, experts) == form
    expert = torch.sort(torch.randint(0, experts, (rows,), generator=g, device='cuda')).values
    expert[-1] = experts - 1
    used = rows - 2                          # two rows belong to no expert
    expert[:used] = torch.sort(expert[:used]).values
    counts = torch.bincount(expert[:used], minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    row = torch.arange(rows, device='cuda', dtype=torch.int32)
    kept = torch.where(row < used, row, torch.full_like(row, -1))
    plan = amd.ExpertPlan(offsets, kept, kept.view(rows, 1), experts)
    level = torch.tensor([0., 1, -1, 2, -2, 3, 4, -4], device='cuda')
    x, w = (level[torch.randint(0, 8, shape, generator=g, device='cuda')] for shape in ((rows, k), (experts, n, k)))
    x[:, ::32], w[..., ::32] = 4, -4         # a 4 in every block: its scale is 1, and the levels stay as they are
    bias = torch.randint(-9, 10, (experts, n), generator=g, device='cuda').float()
    got = amd.mxfp4_expert_dense(x, amd.mxfp4_quantize(w), plan, bias)
    want = (x[:used, None, :] * w[expert[:used]]).sum(-1) + bias[expert[:used]]
    assert torch.equal(got[:used], want) and not got[used:].any()
    assert torch.equal(amd.mxfp4_expert_dense(x, amd.mxfp4_quantize(w), plan, bias, sorted_rows=True)[:used], want)
    assert torch.equal(amd.expert_dispatch(x, plan)[:used], x[:used])
