"""Rows sorted by expert and back, against the 64-bit restatement.  Integers are equal; a float result is a float32
sum rounded once, so it may differ from the exact value by one rounding of its type (half a step, eps / 2)
plus the float32 sum's own error, at most (terms + 1) * 2^-24 of the terms' magnitudes."""
import numpy as np
import pytest
import torch

import expert_reference as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope='module')
def amd():
    import gunet_amd
    return gunet_amd


def _index(rng, t, k, e, pattern):
    if pattern == 'even':
        return rng.integers(0, e, (t, k)).astype(np.int32)
    if pattern == 'dropped':          # every kind of value that is no expert
        bad = np.array([-1, -2 ** 31, e, e + 7, 2 ** 31 - 1], np.int64)
        keep = rng.random((t, k)) < 0.6
        return np.where(keep, rng.integers(0, e, (t, k)), bad[rng.integers(0, 5, (t, k))]).astype(np.int32)
    if pattern == 'none':
        return np.full((t, k), -1, np.int32)
    if pattern == 'one':              # all rows at the last expert, and a token naming it k times
        return np.full((t, k), e - 1, np.int32)
    return np.sort(rng.integers(0, e, (t, k)), axis=None)[::-1].reshape(t, k).astype(np.int32)


def _step(dtype):
    return torch.finfo(dtype).eps / 2


def _near(got, want, dtype, terms, size):
    """The bound above, plus one smallest step of the type where the result is subnormal in it."""
    bound = _step(dtype) * np.abs(want) + (terms + 1) * 2.0 ** -24 * size * (1 + _step(dtype)) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert (np.abs(got - want) <= bound).all(), float(np.max(np.abs(got - want) - bound))


@pytest.mark.parametrize('t, k, e', [(1, 1, 1), (1, 8, 64), (2, 3, 2), (63, 1, 5), (64, 2, 8), (65, 5, 7), (1000, 4, 128), (4096, 2, 8),
                                     (4097, 2, 1024), (8193, 1, 16), (16384, 1, 8), (3001, 3, 1000), (9000, 4, 33), (20000, 6, 64)])
@pytest.mark.parametrize('pattern', ['even', 'dropped', 'none', 'one', 'descending'])
def test_sort_is_the_stable_order(amd, t, k, e, pattern):
    index = _index(np.random.default_rng(t + k + e), t, k, e, pattern)
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    for got, want in zip((plan.offsets, plan.order, plan.slot), R.sort_by_expert(index, e)):
        assert got.dtype == torch.int32
        assert np.array_equal(got.cpu().numpy(), want)


def test_sort_walks_several_tiles_per_workgroup(amd):
    """More positions than 256 tiles of 8192 hold."""
    g = torch.Generator(device='cuda').manual_seed(1)
    index = torch.randint(-1, 37, (1100003, 2), generator=g, device='cuda', dtype=torch.int32)
    plan = amd.expert_plan(index, 37)
    flat = index.reshape(-1)
    key = torch.where(flat < 0, torch.full_like(flat, 37), flat)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key.long(), minlength=38)[:37].cpu()
    assert plan.offsets.cpu().tolist() == [0] + counts.cumsum(0).tolist()
    used = int(counts.sum())
    assert torch.equal(plan.order[:used].long(), order[:used]) and bool((plan.order[used:] == -1).all())
    slot = torch.full_like(flat, -1)
    slot[order[:used]] = torch.arange(used, device='cuda', dtype=torch.int32)
    assert torch.equal(plan.slot.reshape(-1), slot)


def test_empty_inputs(amd):
    plan = amd.expert_plan(torch.zeros((0, 2), dtype=torch.int32).cuda(), 5)
    assert plan.offsets.cpu().tolist() == [0] * 6 and plan.order.numel() == 0
    x = torch.zeros((0, 16)).cuda()
    w = torch.zeros((0, 2)).cuda()
    assert amd.expert_dispatch(x, plan).shape == (0, 16) and amd.expert_combine(x, w, plan).shape == (0, 16)
    assert amd.expert_dispatch_grad(x, plan).shape == (0, 16)
    assert [tuple(t.shape) for t in amd.expert_combine_grad(x, x, w, plan)] == [(0, 16), (0, 2)]
    # rows without columns: the dot products are empty sums
    plan = amd.expert_plan(torch.zeros((3, 2), dtype=torch.int32).cuda(), 1)
    none = torch.zeros((6, 0)).cuda()
    gr, gw = amd.expert_combine_grad(torch.zeros((3, 0)).cuda(), none, torch.ones((3, 2)).cuda(), plan)
    assert gr.shape == (6, 0) and gw.cpu().tolist() == [[0.0, 0.0]] * 3


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('t, k, e, width, pattern', [
    (1, 1, 1, 1, 'even'), (1, 8, 64, 1024, 'even'), (3, 2, 2, 7, 'dropped'), (65, 5, 7, 333, 'dropped'), (64, 4, 8, 16, 'one'),
    (17, 9, 33, 24, 'dropped'), (130, 3, 5, 512, 'none'), (257, 6, 16, 2056, 'dropped'), (1001, 2, 4, 128, 'descending'), (33, 13, 8, 8, 'even')])
def test_rows_there_and_back_with_gradients(amd, dtype, t, k, e, width, pattern):
    rng = np.random.default_rng(7 * t + k)
    index = _index(rng, t, k, e, pattern)
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    slot = plan.slot.cpu().numpy()
    x = torch.as_tensor(rng.standard_normal((t, width))).to(dtype).cuda()
    rows = torch.as_tensor(rng.standard_normal((t * k, width))).to(dtype).cuda()
    weights = torch.as_tensor(rng.random((t, k)), dtype=torch.float32).cuda()
    x64, r64, w64 = x.double().cpu().numpy(), rows.double().cpu().numpy(), weights.double().cpu().numpy()

    got = amd.expert_dispatch(x, plan)
    assert got.dtype == dtype and np.array_equal(got.double().cpu().numpy(), R.dispatch(x64, slot))
    want, size = R.combine(r64, np.ones((t, k)), slot)
    _near(amd.expert_dispatch_grad(rows, plan), want, dtype, k, size)
    want, size = R.combine(r64, w64, slot)
    out = amd.expert_combine(rows, weights, plan)
    assert out.dtype == dtype
    _near(out, want, dtype, k, size)
    want_rows, want_weights, size = R.combine_grad(x64, r64, w64, slot)
    grad_rows, grad_weights = amd.expert_combine_grad(x, rows, weights, plan)
    assert grad_rows.dtype == dtype and grad_weights.dtype == torch.float32
    _near(grad_rows, want_rows, dtype, 1, np.abs(want_rows))
    _near(grad_weights, want_weights, torch.float32, width, size)
    # the same bits again
    again = amd.expert_combine_grad(x, rows, weights, plan)
    assert torch.equal(again[0], grad_rows) and torch.equal(again[1], grad_weights)
    assert torch.equal(amd.expert_combine(rows, weights, plan), out)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('t, k, e, width, shift', [(41, 3, 5, 1001, 0), (23, 5, 4, 2050, 0), (64, 2, 3, 30, 0), (50, 4, 6, 64, 1), (19, 6, 5, 1040, 2), (70, 1, 3, 399, 0)])
def test_combine_grad_of_rows_off_16_bytes(amd, dtype, t, k, e, width, shift):
    """Rows that start on 4 or 2 bytes, by their width or because the tensor does; some, many and very many pieces."""
    rng = np.random.default_rng(width)
    plan = amd.expert_plan(torch.as_tensor(_index(rng, t, k, e, 'dropped')).cuda(), e)

    def make(n):
        v = torch.zeros(n * width + shift, dtype=dtype, device='cuda')[shift:].view(n, width)
        v.copy_(torch.as_tensor(rng.standard_normal((n, width))))
        return v

    grad, rows = make(t), make(t * k)
    weights = torch.as_tensor(rng.random((t, k)), dtype=torch.float32).cuda()
    g64, r64, w64 = (v.double().cpu().numpy() for v in (grad, rows, weights))
    want_rows, want_weights, size = R.combine_grad(g64, r64, w64, plan.slot.cpu().numpy())
    grad_rows, grad_weights = amd.expert_combine_grad(grad, rows, weights, plan)
    _near(grad_rows, want_rows, dtype, 1, np.abs(want_rows))
    _near(grad_weights, want_weights, torch.float32, width, size)
    used = int(plan.offsets[-1])
    assert used < t * k and not grad_rows[used:].any()


def test_gradients_against_differences(amd):
    """<c, combine(rows, w)> moved along a direction: central differences of a bilinear form are exact up to float32
    rounding of the sums, about 2^-23 of the terms' size over the step."""
    rng = np.random.default_rng(5)
    t, k, e, width = 37, 3, 4, 40
    plan = amd.expert_plan(torch.as_tensor(_index(rng, t, k, e, 'dropped')).cuda(), e)
    x, c = (torch.as_tensor(rng.standard_normal((t, width)), dtype=torch.float32).cuda() for _ in range(2))
    dx = torch.as_tensor(rng.standard_normal((t, width)), dtype=torch.float32).cuda()
    w, dw = (torch.as_tensor(rng.random((t, k)), dtype=torch.float32).cuda() for _ in range(2))

    def loss(x, w):
        return float((amd.expert_combine(amd.expert_dispatch(x, plan), w, plan).double() * c.double()).sum())

    rows = amd.expert_dispatch(x, plan)
    grad_rows, grad_w = amd.expert_combine_grad(c, rows, w, plan)
    grad_x = amd.expert_dispatch_grad(grad_rows, plan)
    h = 0.5
    size = float((rows.abs().sum() * c.abs().max() * 2))
    bound = size * 4 * 2.0 ** -23 / h
    assert abs((loss(x + h * dx, w) - loss(x - h * dx, w)) / (2 * h) - float((grad_x.double() * dx.double()).sum())) <= bound
    assert abs((loss(x, w + h * dw) - loss(x, w - h * dw)) / (2 * h) - float((grad_w.double() * dw.double()).sum())) <= bound


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_values_that_are_no_numbers(amd, dtype):
    """A NaN or infinity stays in the rows it belongs to; a dropped choice contributes nothing, whatever its weight holds."""
    index = torch.tensor([[0, 1], [1, -1], [-1, -1], [0, 0]], dtype=torch.int32).cuda()
    plan = amd.expert_plan(index, 2)
    rows = torch.ones((8, 16), dtype=dtype, device='cuda')
    slot = plan.slot.cpu()
    rows[slot[0, 1], 3] = float('nan')
    rows[slot[3, 0], 5] = float('inf')
    rows[5:] = float('nan')                                   # rows that no choice owns
    w = torch.tensor([[1, 2], [3, float('nan')], [float('inf'), float('nan')], [.5, .25]], device='cuda')
    out = amd.expert_combine(rows, w, plan).float().cpu()
    assert torch.isnan(out[0, 3]) and out[0, 0] == 3 and torch.equal(out[1], torch.full((16,), 3.0))
    assert torch.equal(out[2], torch.zeros(16)) and out[3, 5] == float('inf') and out[3, 0] == 0.75
    g = torch.ones((4, 16), dtype=dtype, device='cuda')
    grad_rows, grad_w = amd.expert_combine_grad(g, rows, w, plan)
    assert torch.equal(grad_rows[5:].float().cpu(), torch.zeros((3, 16))) and torch.isfinite(grad_rows.float()).all()
    grad_w = grad_w.cpu()
    assert torch.isnan(grad_w[0, 1]) and grad_w[3, 0] == float('inf')
    assert grad_w[1, 1] == 0 and grad_w[2].tolist() == [0, 0] and grad_w[0, 0] == 16 and grad_w[3, 1] == 16


def test_strided_and_unaligned_tensors(amd):
    rng = np.random.default_rng(3)
    index = torch.as_tensor(_index(rng, 21, 4, 5, 'dropped')).cuda()
    plan = amd.expert_plan(index, 5)
    wide = torch.as_tensor(rng.standard_normal((21, 64)), dtype=torch.bfloat16).cuda()
    want = amd.expert_dispatch(wide[:, ::2].contiguous(), plan)
    assert torch.equal(amd.expert_dispatch(wide[:, ::2], plan), want)
    assert torch.equal(amd.expert_dispatch(wide[:, ::2].t().contiguous().t(), plan), want)
    # packed, but not on 16 bytes: the element-wise form
    store = torch.zeros(21 * 32 + 1, dtype=torch.bfloat16, device='cuda')
    odd = store[1:].view(21, 32)
    odd.copy_(wide[:, ::2])
    assert odd.data_ptr() % 16 and torch.equal(amd.expert_dispatch(odd, plan), want)
    flipped = amd.expert_plan(index.t().contiguous().t(), 5)
    assert torch.equal(flipped.slot, plan.slot) and torch.equal(flipped.order, plan.order)


def test_rows_beyond_32_bit_offsets(amd):
    """2.3e9 elements of rows: the last rows are where they belong."""
    t, k, width = 560000, 2, 2056
    index = (torch.arange(t * k, device='cuda', dtype=torch.int32) % 3).view(t, k)
    plan = amd.expert_plan(index, 3)
    x = torch.arange(t, device='cuda', dtype=torch.float32).to(torch.bfloat16)[:, None].repeat(1, width)
    x[:, 5] = (torch.arange(t, device='cuda') % 251).to(torch.bfloat16)
    rows = amd.expert_dispatch(x, plan)
    assert rows.numel() > 2 ** 31
    pick = torch.tensor([0, 1, t * k // 2, t * k - 2, t * k - 1], device='cuda')
    assert torch.equal(rows[pick], x[(plan.order[pick] // k).long()])
    out = amd.expert_combine(rows, torch.ones((t, k), device='cuda'), plan)
    last = torch.tensor([0, t // 2, t - 1], device='cuda')
    assert torch.equal(out[last].float(), (2 * x[last].float()).to(torch.bfloat16).float())
    grad_rows, grad_w = amd.expert_combine_grad(x[:, :].contiguous(), rows, torch.ones((t, k), device='cuda'), plan)
    assert torch.equal(grad_rows[pick], x[(plan.order[pick] // k).long()])
    del rows, out, grad_rows


def test_captured_step_follows_new_inputs(amd):
    """Sort, dispatch, combine and the gradients in one graph, replayed on new routings with eager work in between."""
    rng = np.random.default_rng(11)
    t, k, e, width = 300, 3, 6, 96
    index = torch.zeros((t, k), dtype=torch.int32, device='cuda')
    x = torch.zeros((t, width), device='cuda')
    w = torch.zeros((t, k), device='cuda')

    def step():
        plan = amd.expert_plan(index, e)
        rows = amd.expert_dispatch(x, plan)
        out = amd.expert_combine(rows, w, plan)
        grad_rows, grad_w = amd.expert_combine_grad(out, rows, w, plan)
        return plan.offsets, plan.order, plan.slot, rows, out, grad_rows, grad_w, amd.expert_dispatch_grad(grad_rows, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                  # two graphs live side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for turn in range(4):
        index.copy_(torch.as_tensor(_index(rng, t, k, e, ['even', 'dropped', 'none', 'one'][turn])))
        x.copy_(torch.as_tensor(rng.standard_normal((t, width))))
        w.copy_(torch.as_tensor(rng.random((t, k))))
        for g, _ in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b), turn


def test_two_streams_at_once(amd):
    rng = np.random.default_rng(2)
    cases = []
    for s in range(2):
        index = torch.as_tensor(_index(rng, 20000, 4, 64, 'dropped')).cuda()
        x = torch.as_tensor(rng.standard_normal((20000, 64)), dtype=torch.float32).cuda()
        cases.append((index, x, torch.cuda.Stream()))
    wants = []
    for index, x, _ in cases:
        plan = amd.expert_plan(index, 64)
        wants.append(amd.expert_dispatch(x, plan))
    torch.cuda.synchronize()
    for _ in range(5):
        gots = []
        for index, x, stream in cases:
            with torch.cuda.stream(stream):
                gots.append(amd.expert_dispatch(x, amd.expert_plan(index, 64)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(gots, wants))


def test_two_host_threads_at_once(amd):
    """Each thread on a stream of its own, all entry points: no state is shared."""
    import threading
    rng = np.random.default_rng(21)
    cases = []
    for s in range(2):
        index = torch.as_tensor(_index(rng, 3000, 3, 9, 'dropped')).cuda()
        x = torch.as_tensor(rng.standard_normal((3000, 72)), dtype=torch.float32).cuda()
        w = torch.as_tensor(rng.random((3000, 3)), dtype=torch.float32).cuda()
        cases.append((index, x, w))

    def work(index, x, w):
        plan = amd.expert_plan(index, 9)
        rows = amd.expert_dispatch(x, plan)
        return (amd.expert_combine(rows, w, plan),) + amd.expert_combine_grad(x, rows, w, plan)

    wants = [work(*c) for c in cases]
    torch.cuda.synchronize()
    gots, failures = [[], []], []

    def loop(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    gots[i] = work(*cases[i])
            torch.cuda.synchronize()
        except Exception as e:          # reported by the main thread
            failures.append(e)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for got, want in zip(gots, wants):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_as_autograd_functions(amd):
    """The gradient functions inside torch's autograd, as a training step uses them, against the formula in 64 bits."""
    class Dispatch(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, plan):
            ctx.plan = plan
            return amd.expert_dispatch(x, plan)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            return amd.expert_dispatch_grad(grad, ctx.plan), None

    class Combine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows, weights, plan):
            ctx.plan = plan
            ctx.save_for_backward(rows, weights)
            return amd.expert_combine(rows, weights, plan)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            return (*amd.expert_combine_grad(grad, *ctx.saved_tensors, ctx.plan), None)

    rng = np.random.default_rng(17)
    t, k, e, width = 50, 3, 5, 24
    plan = amd.expert_plan(torch.as_tensor(_index(rng, t, k, e, 'dropped')).cuda(), e)
    x = torch.as_tensor(rng.standard_normal((t, width)), dtype=torch.float32).cuda().requires_grad_()
    w = torch.as_tensor(rng.random((t, k)), dtype=torch.float32).cuda().requires_grad_()
    Combine.apply(Dispatch.apply(x, plan) * 3, w, plan).sum().backward()      # .sum() hands back an expanded gradient
    slot = plan.slot.cpu().numpy()
    kept = slot >= 0
    x64, w64 = x.detach().double().cpu().numpy(), w.detach().double().cpu().numpy()
    want_x = np.repeat((3 * (w64 * kept).sum(1))[:, None], width, 1)
    want_w = np.where(kept, 3 * x64.sum(1)[:, None], 0)
    _near(x.grad, want_x, torch.float32, k + 2, 3 * np.abs(want_x))
    _near(w.grad, want_w, torch.float32, width + 2, np.where(kept, 3 * np.abs(x64).sum(1)[:, None], 0))


def test_refusals(amd):
    index = torch.zeros((4, 2), dtype=torch.int32).cuda()
    plan = amd.expert_plan(index, 3)
    x, w = torch.zeros((4, 8)).cuda(), torch.zeros((4, 2)).cuda()
    rows = torch.zeros((8, 8)).cuda()
    for bad in (index.long(), index.cpu(), index.float()):
        with pytest.raises(TypeError):
            amd.expert_plan(bad, 3)
    for bad in (index[0], index[:, :0]):
        with pytest.raises(ValueError):
            amd.expert_plan(bad, 3)
    for e, code in ((0, -1), (-5, -1), (1025, -4), (2 ** 31 - 1, -4)):
        with pytest.raises(amd.GunetError) as err:
            amd.expert_plan(index, e)
        assert err.value.code == code
    with pytest.raises(ValueError):
        amd.expert_dispatch(x[:3], plan)
    with pytest.raises(TypeError):
        amd.expert_dispatch(x.double(), plan)
    with pytest.raises(ValueError):
        amd.expert_combine(rows[:7], w, plan)
    with pytest.raises(TypeError):
        amd.expert_combine(rows, w.bfloat16(), plan)
    with pytest.raises(ValueError):
        amd.expert_combine(rows, w[:, :1], plan)
    with pytest.raises(TypeError):
        amd.expert_combine_grad(x.half(), rows, w, plan)
    with pytest.raises(ValueError):
        amd.expert_combine_grad(x[:, :4], rows, w, plan)
    with pytest.raises(ValueError, match='gradient'):
        amd.expert_dispatch(x.clone().requires_grad_(), plan)
    with torch.no_grad():
        assert amd.expert_dispatch(x.clone().requires_grad_(), plan).shape == (8, 8)
