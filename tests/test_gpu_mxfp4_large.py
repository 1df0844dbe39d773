"""4-bit matrices and products past 32-bit element and byte offsets, and the longest rows.

Rows are copies of a few base rows, in turn, so that all of a large result is compared with a small one.  The operands are values that their own
quantisation keeps and the sums are exact (as explained where they are made), so results are equal bit for bit."""
import pytest
import torch

from mxfp4_forms import form_of

pytestmark = pytest.mark.gpu

BASE = 997


@pytest.fixture(scope='module')
def amd():
    import gunet_amd
    yield gunet_amd
    torch.cuda.empty_cache()


def _values(g, shape, dtype=torch.bfloat16, density=0.5):
    """0, +-4 and +-6, one of the last two in every block: the block's scale is 1 and every product of two a multiple of 4, so that sums are exact
    in float32 while their terms' magnitudes add up to less than 2^26."""
    size = 4 + 2 * torch.randint(0, 2, shape, generator=g, device='cuda', dtype=torch.int8)
    size *= 1 - 2 * torch.randint(0, 2, shape, generator=g, device='cuda', dtype=torch.int8)
    keep = torch.rand(shape, generator=g, device='cuda') < density
    keep[..., ::32] = True
    return (size * keep).to(dtype)


def _turns(n):
    return torch.arange(n, device='cuda') % BASE


def test_quantize_past_32_bit_offsets(amd):
    """2^20 rows of 2049 (2.1e9 elements, codes of 1.1e9 bytes and rows on odd addresses), read back in both kinds of type."""
    g = torch.Generator(device='cuda').manual_seed(1)
    base = torch.randn((BASE, 2049), generator=g, device='cuda').to(torch.bfloat16)
    turn = _turns(2 ** 20 + 3)
    x = base[turn]
    assert x.numel() > 2 ** 31
    want = amd.mxfp4_quantize(base)
    got = amd.mxfp4_quantize(x)
    assert torch.equal(got.codes[0], want.codes[0][turn]) and torch.equal(got.scales[0], want.scales[0][:, turn])
    for dtype in (torch.bfloat16, torch.float32):
        assert torch.equal(amd.mxfp4_dequantize(got, dtype), amd.mxfp4_dequantize(want, dtype)[turn])


def test_a_stack_past_32_bit_offsets(amd):
    g = torch.Generator(device='cuda').manual_seed(2)
    base = torch.randn((BASE, 1000), generator=g, device='cuda').to(torch.float16)
    turn = _turns(3 * 750001)
    x = base[turn].view(3, 750001, 1000)
    assert x.numel() > 2 ** 31
    want = amd.mxfp4_quantize(base)
    got = amd.mxfp4_quantize(x)
    assert torch.equal(got.codes.view(-1, *want.codes.shape[2:]), want.codes[0][turn])
    back = amd.mxfp4_dequantize(got, torch.float16).view(-1, 1000)
    assert torch.equal(back, amd.mxfp4_dequantize(want, torch.float16)[turn])


def _expect(x, w, size=2 ** 26):
    x64, w64 = x.double(), w.double()
    assert float((x64.abs() @ w64.abs().t().contiguous()).max()) < size
    return (x64 @ w64.t().contiguous()).float()


@pytest.mark.parametrize('rows, k, n, form', [
    (2 ** 20 + 5, 64, 2056, 'tile 256 x 256'), (2 ** 20 + 5, 1100, 2051, 'tile 256 x 256'),       # results
    (40000003, 33, 61, 'rows 32'), (9000001, 300, 250, 'tile 256 x 256'),
    (2 ** 22 + 5, 2100, 48, 'tile 128 x 128')])                                                   # x, and its codes past 2^32 bytes
def test_dense_past_32_bit_offsets(amd, rows, k, n, form):
    assert form_of(rows, k, n, 0) == form and rows * max(n, k) > 2 ** 31
    g = torch.Generator(device='cuda').manual_seed(n)
    base, w = _values(g, (BASE, k)), _values(g, (n, k))
    turn = _turns(rows)
    want = _expect(base, w).to(torch.bfloat16)
    x = base[turn]
    got = amd.mxfp4_dense(x, amd.mxfp4_quantize(w))
    del x
    for first in range(0, rows, 1 << 21):
        assert torch.equal(got[first:first + (1 << 21)], want[turn[first:first + (1 << 21)]]), first


@pytest.mark.parametrize('sorted_rows', [False, True])
def test_experts_past_32_bit_offsets(amd, sorted_rows):
    t, e, k, n = 560000, 5, 96, 2051
    g = torch.Generator(device='cuda').manual_seed(5)
    index = torch.randint(-1, e, (t, 2), generator=g, device='cuda', dtype=torch.int32)
    plan = amd.expert_plan(index, e)
    base, w = _values(g, (BASE, k)), _values(g, (e, n, k))
    turn = _turns(t)
    x = base[turn]
    if sorted_rows:
        x = amd.expert_dispatch(x, plan)
    got = amd.mxfp4_expert_dense(x, amd.mxfp4_quantize(w), plan, sorted_rows=sorted_rows)
    assert got.numel() > 2 ** 31
    offsets = plan.offsets.tolist()
    token = torch.div(plan.order.long(), 2, rounding_mode='floor')
    for i in range(e):
        want = _expect(base, w[i]).to(torch.bfloat16)
        assert torch.equal(got[offsets[i]:offsets[i + 1]], want[turn[token[offsets[i]:offsets[i + 1]]]]), i
    assert offsets[e] < 2 * t and not got[offsets[e]:].any()


@pytest.mark.parametrize('rows, n, form', [(1, 70, 'skinny 16 rows 4 waves'), (17, 4100, 'skinny 32 rows 4 waves'), (40, 300, 'skinny 32 rows 8 waves'),
                                           (33, 2100, 'tile 64 x 64')])
def test_the_longest_rows(amd, rows, n, form):
    """k = 2^22, the most there is, and a column short of it; 4100 rows of it are past 2^32 bytes."""
    g = torch.Generator(device='cuda').manual_seed(rows)
    for k in (2 ** 22, 2 ** 22 - 1):
        assert form_of(rows, k, n, 0) == form
        x = _values(g, (rows, k), density=0.3)
        part = _values(g, (61, k), density=0.3)      # the columns in turn; 61 divides none of the offsets that could wrap
        want = _expect(x, part)
        part4, turn = amd.mxfp4_quantize(part), torch.arange(n, device='cuda') % 61
        w4 = amd.Mxfp4Tensor(part4.codes.index_select(1, turn), part4.scales.index_select(2, turn), (n, k))
        assert torch.equal(amd.mxfp4_dense(x, w4, None, None, torch.float32), want[:, turn])


def test_the_longest_row_there_and_back(amd):
    g = torch.Generator(device='cuda').manual_seed(9)
    x = _values(g, (5, 2 ** 22), torch.float32)
    assert torch.equal(amd.mxfp4_dequantize(amd.mxfp4_quantize(x)), x)
