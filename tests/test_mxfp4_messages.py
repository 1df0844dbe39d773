"""Refusals of the 4-bit calls name the argument that is wrong (the checks run without a GPU)."""
import pytest
import torch


class _OnGpu(torch.Tensor):
    """A host tensor that says it is a CUDA tensor: the checks see it, no kernel does."""
    is_cuda = True


def test_the_argument_that_is_wrong_is_named():
    import gunet_amd as amd
    w = amd.Mxfp4Tensor.empty((8, 64), 'cpu')
    for wrong in (torch.float64, torch.int32):
        x = torch.zeros((4, 64), dtype=wrong).as_subclass(_OnGpu)
        with pytest.raises(TypeError, match='^x must be'):
            amd.mxfp4_dense(x, w)
        with pytest.raises(TypeError, match='^x must be'):
            amd.mxfp4_dense(x, w, out_dtype=torch.float32)
    with pytest.raises(TypeError, match='^out_dtype must be'):
        amd.mxfp4_dense(torch.zeros((4, 64)).as_subclass(_OnGpu), w, out_dtype=torch.float64)
    for t in (torch.zeros((4, 64)), None):
        with pytest.raises(TypeError, match='Mxfp4Tensor'):
            amd.mxfp4_dequantize(t)
    for plan in (None, (1, 2, 3)):
        with pytest.raises(TypeError, match='ExpertPlan'):
            amd.mxfp4_expert_dense(torch.zeros((4, 64)).as_subclass(_OnGpu), w, plan)
        for call in (lambda: amd.expert_dispatch(torch.zeros((4, 64)), plan), lambda: amd.expert_dispatch_grad(torch.zeros((8, 64)), plan),
                     lambda: amd.expert_combine(torch.zeros((8, 64)), torch.zeros((4, 2)), plan),
                     lambda: amd.expert_combine_grad(torch.zeros((4, 64)), torch.zeros((8, 64)), torch.zeros((4, 2)), plan)):
            with pytest.raises(TypeError, match='ExpertPlan'):
                call()
