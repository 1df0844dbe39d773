"""Every form of the products on 4-bit weights, at sizes that run on it: exact sums bit for bit, special values, activations.

Exact sums: the operands are multiples of 0.5 times powers of two near 1, each block with a 4 or 6 in it, so quantisation keeps them as
they are.  Every product is then a multiple of 2^-3, and where the magnitudes of an output's terms add up to less than 2^21 every partial sum, in
any order, is a float32 number: the result is the exact one and not one column can be missing from it."""
import numpy as np
import pytest
import torch

from mxfp4_forms import CASES, form_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = [f'{form}-{rows}-{k}-{n}-{e}' for form, rows, k, n, e in CASES]


@pytest.fixture(scope='module')
def amd():
    import gunet_amd
    return gunet_amd


def _operand(g, shape, spread):
    """Values that their own quantisation keeps: levels with a 4 or 6 (or their negatives) in every block, times 2^-spread .. 2^spread by block."""
    k = shape[-1]
    blocks = -(-k // 32)
    level = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device='cuda')
    x = level[torch.randint(0, 8, shape[:-1] + (blocks, 32), generator=g, device='cuda')]
    x[..., 0] = 4 + 2 * torch.randint(0, 2, x.shape[:-1], generator=g, device='cuda')
    x *= 1 - 2 * torch.randint(0, 2, x.shape, generator=g, device='cuda')
    if spread:
        x *= torch.exp2(torch.randint(-spread, spread + 1, x.shape[:-1] + (1,), generator=g, device='cuda').float())
    return x.reshape(shape[:-1] + (blocks * 32,))[..., :k].contiguous()


class _Case:
    """One product of a case: its operands, the call, and the exact value by expert."""

    def __init__(self, amd, rows, k, n, e, dtype, make, seed=0):
        self.amd, self.e = amd, e
        g = torch.Generator(device='cuda').manual_seed(rows + k + n + seed)
        if e:      # every third row asks for expert 0 (if there are two), some are dropped; the rest by chance
            top_k = 2 if rows % 2 == 0 else 1
            index = torch.randint(0, e, (rows // top_k, top_k), generator=g, device='cuda', dtype=torch.int32)
            index[::3, 0] = 0
            if index.shape[0] > 1:
                index[1, top_k - 1] = -1
            self.plan = amd.expert_plan(index, e)
            offsets = self.plan.offsets.tolist()
            self.parts = [(i, offsets[i], offsets[i + 1]) for i in range(e)]
            self.used = offsets[-1]
            order = self.plan.order[:self.used].long()
            self.x = make(g, (rows // top_k, k), 0).to(dtype)
            self.source = torch.div(order, top_k, rounding_mode='floor')       # the token of each row
            self.w = make(g, (e, n, k), 1)
            self.bias = torch.randint(-50, 51, (e, n), generator=g, device='cuda').float()
        else:
            self.x, self.w = make(g, (rows, k), 0).to(dtype), make(g, (n, k), 1)
            self.bias = torch.randint(-50, 51, (n,), generator=g, device='cuda').float()
            self.parts, self.used, self.source = [(0, 0, rows)], rows, torch.arange(rows, device='cuda')
        self.w4 = amd.mxfp4_quantize(self.w)

    def call(self, x=None, w4=None, bias=False, act=None, out=torch.float32):
        x, w4, b = self.x if x is None else x, self.w4 if w4 is None else w4, self.bias if bias else None
        if self.e:
            return self.amd.mxfp4_expert_dense(x, w4, self.plan, b, act, out)
        return self.amd.mxfp4_dense(x, w4, b, act, out)

    def exact(self):
        """float64 values of the used rows, and the largest sum of one output's terms' magnitudes."""
        out, size = [], 0.0
        w = self.w if self.e else self.w[None]
        bias = self.bias if self.e else self.bias[None]
        for i, lo, hi in self.parts:
            if lo == hi:
                continue
            x64, w64 = self.x[self.source[lo:hi]].double(), w[i].double()
            out.append(x64 @ w64.t().contiguous() + bias[i].double())
            size = max(size, float((x64.abs() @ w64.abs().t().contiguous() + bias[i].abs().double()).max()))
        return torch.cat(out), size


@pytest.mark.parametrize('form, rows, k, n, e', CASES, ids=IDS)
def test_sums_are_exact(amd, form, rows, k, n, e):
    assert form_of(rows, k, n, e) == form
    dtype = TYPES[(rows + n) % 3]
    c = _Case(amd, rows, k, n, e, dtype, _operand)
    want, size = c.exact()
    assert size < 2 ** 21
    for out in TYPES:
        got = c.call(bias=True, out=out)
        # the float32 sum is exact; a narrower type takes one rounding of it
        assert torch.equal(got[:c.used], want.float().to(out)) and not got[c.used:].any(), out
    got = c.call(bias=True, act='relu')
    assert torch.equal(got[:c.used], want.clamp(min=0).float())
    odd = torch.zeros(c.x.numel() + 1, dtype=dtype, device='cuda')[1:].view(c.x.shape)       # rows that start on no 16 bytes
    odd.copy_(c.x)
    assert torch.equal(c.call(odd, bias=True)[:c.used], want.float())


@pytest.mark.parametrize('form, rows, k, n, e', CASES, ids=IDS)
def test_special_values_stay_where_they_are(amd, form, rows, k, n, e):
    """A NaN or infinity in the first, a middle and the last row and column of each operand: its row or column of the result, nothing else."""
    assert form_of(rows, k, n, e) == form
    c = _Case(amd, rows, k, n, e, TYPES[(rows + k) % 3], _operand)
    clean = c.call()
    tokens, w = c.x.shape[0], (c.w if e else c.w[None])
    bad_tokens = sorted({0, tokens // 2, tokens - 1})[-2 if tokens > 1 else -1:]
    bad = torch.zeros_like(clean, dtype=torch.bool)
    x, w_bad = c.x.clone(), w.clone()
    for i, t in enumerate(bad_tokens):
        x[t, (0, k // 2, k - 1)[(i + rows) % 3]] = (float('nan'), float('inf'))[i % 2]
        bad[:c.used][c.source == t] = True
    for i, lo, hi in c.parts:
        for j, col in enumerate(sorted({0, n // 2, n - 1})):
            w_bad[i, col, (k - 1, k // 2, 0)[j % 3]] = (-float('inf'), float('nan'))[j % 2]
            bad[lo:hi, col] = True
    got = c.call(x, amd.mxfp4_quantize(w_bad if e else w_bad[0]))
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    assert not got[c.used:].any() and bad.any() and (tokens <= 2 or not bad.all())


ACTIVATIONS = {
    'tanh': torch.tanh, 'sigmoid': torch.sigmoid, 'elu': lambda v: torch.where(v > 0, v, torch.expm1(v)),
    'softplus': lambda v: v.clamp(min=0) + torch.log1p(torch.exp(-v.abs())),
    'selu': lambda v: 1.0507009873554805 * torch.where(v > 0, v, 1.6732632423543772 * torch.expm1(v)),
    'swish': lambda v: v * torch.sigmoid(v), 'gelu': lambda v: 0.5 * v * (1 + torch.erf(v / 2 ** 0.5)), 'softsign': lambda v: v / (1 + v.abs()),
    'exponential': torch.exp, 'hard_sigmoid': lambda v: (0.2 * v + 0.5).clamp(0, 1), 'relu': lambda v: v.clamp(min=0), 'linear': lambda v: v}


def _features(g, shape, spread):
    """Rows of differing size; the weights small enough that the sums stay near the activations' bends."""
    x = torch.randn(shape, generator=g, device='cuda')
    if spread:
        return x * (2.0 / shape[-1] ** 0.5)
    return x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device='cuda'))


FIRST = {}
for _case in CASES:       # the smallest result of each form, without experts and with
    _key = (_case[0], bool(_case[4]))
    if _key not in FIRST or _case[1] * _case[3] < FIRST[_key][1] * FIRST[_key][3]:
        FIRST[_key] = _case


@pytest.mark.parametrize('form, rows, k, n, e', list(FIRST.values()), ids=str)
def test_every_activation_in_every_form(amd, form, rows, k, n, e):
    """Both sides evaluate the activation of the same float32 sum, so only the function's own error counts: the float32 gate of the
    other layers, 1e-5 of the largest value; the exponential, whose error is relative, entry by entry, and 2^-126 below the
    smallest normal number."""
    assert form_of(rows, k, n, e) == form
    c = _Case(amd, rows, k, n, e, torch.float32, _features)
    before = c.call(bias=False).double()
    for name, f in ACTIVATIONS.items():
        got, want = c.call(act=name).double(), f(before)
        got, want = got[:c.used], want[:c.used]
        scale = want.abs() if name == 'exponential' else want.abs().max()
        assert torch.isfinite(want).all() and ((got - want).abs() <= 1e-5 * scale + 2.0 ** -126).all(), name
    assert not c.call(act='exponential')[c.used:].any()         # rows of no expert are zeros, not the activation of zero


@pytest.mark.parametrize('half', [0, 1])
def test_every_form_captured(amd, half):
    """Products of many forms in one graph, and a second graph of the same ones: replayed in turn with new inputs and eager work in between."""
    cases = sorted(FIRST.values(), key=str)[half::2]
    built = [_Case(amd, *c[1:], TYPES[i % 3], _operand) for i, c in enumerate(cases)]
    inputs = [c.x.clone() for c in built]

    def step():
        return [c.call(x, bias=True, act='relu') for c, x in zip(built, inputs)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for turn in range(4):
        for c, x in zip(built, inputs):
            x.copy_(c.x.roll(turn, 0) if turn % 2 else -c.x)
        want = step()
        for g, _ in graphs:
            g.replay()
        again = step()
        torch.cuda.synchronize()
        for i, c in enumerate(cases):
            assert torch.equal(again[i], want[i]) and all(torch.equal(outs[i], want[i]) for _, outs in graphs), (turn, c)


def test_every_form_on_two_streams(amd):
    """The same products at once on two streams, each call with a workspace of its own."""
    built = [_Case(amd, *c[1:], torch.bfloat16, _operand) for c in FIRST.values()]
    want = [c.call() for c in built]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append([c.call() for c in built])
        torch.cuda.synchronize()
        for out in got:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        del got, out
