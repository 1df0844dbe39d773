"""Forward-mode derivatives: the calls record nothing, so a dual tensor is refused rather than stripped of its tangent."""
import pytest
import torch
from torch.autograd import forward_ad

SHAPE = (4, 64)


def _dual(device):
    return forward_ad.make_dual(torch.randn(SHAPE, device=device), torch.randn(SHAPE, device=device))


class _OnGpu(torch.Tensor):
    """A host tensor that says it is a CUDA tensor: the checks see it, no kernel does."""
    is_cuda = True


def test_checks_find_the_tangent_without_a_gpu():
    from gunet_amd.layers.expert_ops import checked
    plain = torch.randn(SHAPE).as_subclass(_OnGpu)
    assert checked(plain, 'x') is plain
    with forward_ad.dual_level():
        assert checked(plain, 'x') is plain                       # a level is open, this tensor has no part in it
        dual = forward_ad.make_dual(plain, torch.ones(SHAPE)).as_subclass(_OnGpu)
        assert not dual.requires_grad and forward_ad.unpack_dual(dual).tangent is not None
        with pytest.raises(ValueError, match='tangent'):
            checked(dual, 'x')
        with torch.no_grad(), pytest.raises(ValueError, match='tangent'):      # no_grad() keeps tangents
            checked(dual, 'x')
        with torch.inference_mode():                                           # this drops them for torch's own operations too
            checked(dual, 'x')


@pytest.mark.gpu
def test_every_call_refuses_a_dual_tensor():
    import gunet_amd as amd
    index = torch.tensor([[0, 1], [1, 0], [2, 2], [0, -1]], dtype=torch.int32, device='cuda')
    plan = amd.expert_plan(index, 3)
    w = torch.rand((4, 2), device='cuda')
    rows = torch.randn((8, 64), device='cuda')
    w4, stack = amd.mxfp4_quantize(torch.randn((8, 64), device='cuda')), amd.mxfp4_quantize(torch.randn((3, 8, 64), device='cuda'))
    with forward_ad.dual_level():
        x = _dual('cuda')
        both = forward_ad.make_dual(rows, torch.ones_like(rows))
        gate = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: amd.expert_dispatch(x, plan), lambda: amd.expert_dispatch_grad(both, plan),
                     lambda: amd.expert_combine(both, w, plan), lambda: amd.expert_combine(rows, gate, plan),
                     lambda: amd.expert_combine_grad(x, rows, w, plan), lambda: amd.expert_combine_grad(x.detach(), both, w, plan),
                     lambda: amd.mxfp4_quantize(x), lambda: amd.mxfp4_dense(x, w4), lambda: amd.mxfp4_expert_dense(x, stack, plan)):
            with pytest.raises(ValueError, match='tangent'):
                call()
        primal = forward_ad.unpack_dual(x).primal
        assert torch.equal(amd.expert_dispatch(primal, plan), amd.expert_dispatch(primal.clone(), plan))


@pytest.mark.gpu
def test_a_function_with_a_jvp_of_its_own():
    """Inside torch.autograd.Function the tangent is the function's to handle: dispatch is linear, so its tangent is dispatched too."""
    import gunet_amd as amd
    plan = amd.expert_plan(torch.tensor([[0, 1], [1, 0], [2, 2], [0, -1]], dtype=torch.int32, device='cuda'), 3)

    class Dispatch(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return amd.expert_dispatch(x, plan)

        @staticmethod
        def jvp(ctx, tangent):
            return amd.expert_dispatch(tangent, plan)

    with forward_ad.dual_level():
        x = _dual('cuda')
        out = forward_ad.unpack_dual(Dispatch.apply(x))
        primal, tangent = forward_ad.unpack_dual(x)
        assert torch.equal(out.primal, amd.expert_dispatch(primal, plan)) and torch.equal(out.tangent, amd.expert_dispatch(tangent, plan))
