"""The 4-bit microscaled format and the products on it, against 64-bit restatements.

Quantisation is equal bit for bit.  A product of two 4-bit values and their scales is exact in float32; the sum of k of them may
be off by one unit in the last place of the running sum per addition, at most k * 2^-23 of the terms'
magnitudes, the bias adds one more, and the result is rounded once to its type (half a step, eps / 2)."""
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


def _features(rng, shape, dtype):
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,)))
    return torch.as_tensor(x).to(dtype).cuda()


def _plain(t):
    """float64 values of an Mxfp4Tensor [rows, k] from its bytes."""
    return _plain3(t)[0]


def _plain3(t):
    codes, scales = t.codes.cpu().numpy(), t.scales.cpu().numpy()
    out = []
    for g in range(t.groups):
        code = np.empty(codes.shape[1:3] + (32,), np.uint8)
        code[..., 0::2], code[..., 1::2] = codes[g] & 15, codes[g] >> 4
        out.append(R.values(code, scales[g].transpose(1, 0, 2).reshape(t.rows, -1)[:, :codes.shape[2]], t.k))
    return out


def _check_product(got, x, w, bias, relu, dtype):
    want = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    k = x.shape[1]
    if bias is not None:
        want, size = want + bias, size + np.abs(bias)
    if relu:
        want = np.maximum(want, 0)
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    info = torch.finfo(dtype)
    bound = info.eps / 2 * np.abs(want) + (k + 1) * 2.0 ** -23 * size * (1 + info.eps) + info.smallest_normal * info.eps
    assert (np.abs(got - want) <= bound).all(), float(np.max((np.abs(got - want) - bound)))


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows, k', [(1, 1), (1, 32), (3, 31), (5, 33), (7, 256), (2, 257), (33, 100), (64, 1024), (17, 8200)])
def test_quantize_equals_the_definition(amd, dtype, rows, k):
    x = _features(np.random.default_rng(rows + k), (rows, k), dtype)
    t = amd.mxfp4_quantize(x)
    code, scales = R.quantize(x.double().cpu().numpy())
    blocks = code.shape[1]
    assert np.array_equal(t.codes[0].cpu().numpy(), R.pack(code))
    got = t.scales[0].cpu().numpy().transpose(1, 0, 2).reshape(rows, -1)
    assert np.array_equal(got[:, :blocks], scales) and not got[:, blocks:].any()
    back = amd.mxfp4_dequantize(t)
    assert np.array_equal(back.double().cpu().numpy(), R.values(code, scales, k))
    for low in (torch.bfloat16, torch.float16):      # rounded once from the float32 value
        assert torch.equal(amd.mxfp4_dequantize(t, low), back.to(low))


def test_quantize_ties_ends_and_special_values(amd):
    """Every middle between two levels and its neighbours at every exponent float32 has, subnormals, zeros, NaN and infinity."""
    mid = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], np.float32)
    mid = np.concatenate((mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(8))))[:47]
    rows = []
    for e in range(-149, 126):
        with np.errstate(over='ignore', under='ignore'):
            v = np.ldexp(mid, e).astype(np.float32)
        block = v[:32].copy()
        block[1::2] *= -1
        rows.append(block)
        rows.append(np.concatenate((v[15:], [v[15]] * 32))[:32])
    special = np.zeros((8, 32), np.float32)
    special[1, 4] = np.nan
    special[2, 31] = np.inf
    special[3, 0] = -np.inf
    special[4, :] = -0.0
    special[5, 7] = np.float32(3.4028235e38)
    special[6, 9] = np.float32(1e-45)
    special[7, :2] = [np.nan, np.inf]
    x = np.concatenate((np.stack(rows).astype(np.float32), special))
    t = amd.mxfp4_quantize(torch.as_tensor(x).cuda())
    code, scales = R.quantize(x)
    assert np.array_equal(t.scales[0].cpu().numpy()[0, :, :1], scales)
    assert np.array_equal(t.codes[0].cpu().numpy(), R.pack(code))
    back = amd.mxfp4_dequantize(t).double().cpu().numpy()
    want = R.values(code, scales, 32)
    assert np.array_equal(back, want, equal_nan=True) and np.isnan(back[-1]).all()
    assert np.array_equal(np.signbit(back[-4]), np.ones(32, bool))


@pytest.mark.parametrize('dtype, mantissa', [(torch.bfloat16, 7), (torch.float16, 10)], ids=str)
def test_quantize_two_byte_values_at_every_exponent(amd, dtype, mantissa):
    """Blocks with every exponent as their largest value's (subnormals too), filled with the numbers of either sign down to 2^-8 of it: every
    rounding there is, in both packed halves.  And infinities and NaN in every place of a block."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[torch.isfinite(every)]
    size = every.double().abs()
    blocks = []
    for exponent in range((1 << (15 - mantissa)) - 1):
        for rest in (0, 1, (1 << mantissa) - 1):
            top = torch.tensor([exponent << mantissa | rest], dtype=torch.int16).view(dtype)
            fill = every[(size <= top.double()) & (size >= top.double() * 2.0 ** -8)]
            fill = fill[:fill.numel() // 31 * 31].view(-1, 31)
            blocks.append(torch.cat([top.expand(fill.shape[0], 1), fill], 1))
            blocks.append(torch.cat([fill, top.expand(fill.shape[0], 1)], 1))
    x = torch.cat(blocks).contiguous()
    assert x.shape[0] > 1 << 16
    code, scales = R.quantize(x.double().numpy())
    t = amd.mxfp4_quantize(x.cuda())
    assert np.array_equal(t.codes[0].cpu().numpy(), R.pack(code))
    assert np.array_equal(t.scales[0, 0, :, 0].cpu().numpy(), scales[:, 0])
    x = torch.ones((96, 64), dtype=dtype)
    for i, bad in enumerate((float('inf'), -float('inf'), float('nan'))):
        x[32 * i + torch.arange(32), torch.arange(32)] = bad
    back = amd.mxfp4_dequantize(amd.mxfp4_quantize(x.cuda())).cpu()
    assert torch.isnan(back[:, :32]).all() and (back[:, 32:] == 1).all()


def test_quantize_stacks_strides_and_unaligned(amd):
    x = _features(np.random.default_rng(1), (3, 10, 96), torch.bfloat16)
    t = amd.mxfp4_quantize(x)
    assert t.shape == (3, 10, 96)
    for g in range(3):
        one = amd.mxfp4_quantize(x[g])
        assert torch.equal(one.codes[0], t.codes[g]) and torch.equal(one.scales[0], t.scales[g])
    flat = amd.mxfp4_quantize(x[1].t())
    assert torch.equal(flat.codes, amd.mxfp4_quantize(x[1].t().contiguous()).codes)
    store = torch.zeros(10 * 96 + 1, dtype=torch.bfloat16, device='cuda')
    odd = store[1:].view(10, 96)
    odd.copy_(x[0])
    assert torch.equal(amd.mxfp4_quantize(odd).codes[0], t.codes[0])
    assert amd.mxfp4_dequantize(amd.mxfp4_quantize(x[:, :0])).shape == (3, 0, 96)


def test_from_codes_is_the_same_tensor(amd):
    for shape in ((12, 256), (12, 100), (5, 33), (2, 7, 300)):
        x = _features(np.random.default_rng(2), shape, torch.float32)
        t = amd.mxfp4_quantize(x)
        blocks = t.codes.shape[2]
        codes = t.codes.view(shape[:-1] + (blocks * 16,)).clone()
        scales = t.scales.transpose(1, 2).reshape(t.groups, t.rows, -1)[:, :, :blocks].reshape(shape[:-1] + (blocks,))
        if shape[-1] % 32:                            # what lies behind column k in a checkpoint does not matter
            used = shape[-1] % 32
            dirty = codes.view(t.codes.shape)
            dirty[:, :, -1, (used + 1) // 2:] = 0x77
            if used % 2:
                dirty[:, :, -1, used // 2] |= 0x70
        again = amd.Mxfp4Tensor.from_codes(codes, scales, shape[-1])
        assert torch.equal(again.codes, t.codes) and torch.equal(again.scales, t.scales) and again.shape == shape


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows, k, n', [
    (1, 1, 1), (1, 32, 16), (1, 4096, 512), (2, 96, 33), (7, 1000, 130), (16, 256, 128), (17, 288, 257), (31, 513, 64), (33, 128, 96), (48, 2080, 80), (64, 8192, 48),
    (65, 104, 128), (128, 1024, 256), (129, 256, 255), (200, 640, 384), (255, 96, 512), (256, 512, 256), (257, 544, 520), (513, 33, 1027), (1030, 384, 300)])
def test_dense_against_the_exact_product(amd, dtype, rows, k, n):
    rng = np.random.default_rng(rows + k + n)
    x, w = _features(rng, (rows, k), dtype), _features(rng, (n, k), torch.float32)
    w4 = amd.mxfp4_quantize(w)
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    _check_product(amd.mxfp4_dense(x, w4), x64, w64, None, False, dtype)
    bias = rng.standard_normal(n).astype(np.float32)
    got = amd.mxfp4_dense(x, w4, torch.as_tensor(bias).cuda(), 'relu', torch.float32)
    assert got.dtype == torch.float32
    _check_product(got, x64, w64, bias.astype(np.float64), True, torch.float32)
    assert torch.equal(got, amd.mxfp4_dense(x, w4, torch.as_tensor(bias).cuda(), 'relu', torch.float32))


@pytest.mark.parametrize('dtype, rows, k, n', [
    (torch.float32, 3001, 300, 2001), (torch.bfloat16, 3000, 33, 2056), (torch.float16, 5003, 96, 1028),         # 128 x 128 tiles
    (torch.float32, 4999, 520, 4104), (torch.bfloat16, 4353, 288, 4099), (torch.float16, 4999, 32, 4112),        # 256 x 256 tiles
    (torch.bfloat16, 300, 100, 16384), (torch.float32, 20, 1000, 20000), (torch.bfloat16, 9, 2080, 16400)], ids=str)
def test_dense_in_every_tile_size(amd, dtype, rows, k, n):
    """Sizes that reach the large tiles, with ragged edges on both sides, and few rows with many columns."""
    rng = np.random.default_rng(rows)
    x, w4 = _features(rng, (rows, k), dtype), amd.mxfp4_quantize(_features(rng, (n, k), torch.float32))
    bias = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    _check_product(amd.mxfp4_dense(x, w4, bias, 'relu'), x64, w64, bias.double().cpu().numpy(), True, dtype)
    _check_product(amd.mxfp4_dense(x, w4, None, None, torch.float32), x64, w64, None, False, torch.float32)


@pytest.mark.parametrize('dtype, rows, k, n', [
    (torch.bfloat16, 4001, 520, 4090), (torch.float32, 3990, 288, 4088), (torch.float16, 4033, 33, 4096), (torch.bfloat16, 7937, 40, 4090),  # 256 x 256
    (torch.bfloat16, 3001, 300, 2008), (torch.float16, 13505, 96, 255), (torch.float32, 700, 520, 4001)], ids=str)      # 64 x 128
def test_dense_in_full_rounds_of_tiles(amd, dtype, rows, k, n):
    """Sizes whose tiles, the largest or a middling one, go over the chip at once or twice; ragged edges, an activation of its own, NaN."""
    rng = np.random.default_rng(rows)
    x, w = _features(rng, (rows, k), dtype), _features(rng, (n, k), torch.float32) * 0.05
    bias = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    w4 = amd.mxfp4_quantize(w)
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    _check_product(amd.mxfp4_dense(x, w4, bias, 'relu'), x64, w64, bias.double().cpu().numpy(), True, dtype)
    clean = amd.mxfp4_dense(x, w4, None, None, torch.float32)
    _check_product(clean, x64, w64, None, False, torch.float32)
    tanh = amd.mxfp4_dense(x, w4, None, 'tanh', torch.float32)
    assert (tanh.double() - torch.tanh(clean.double())).abs().max() <= 1e-5             # the same float32 sum on both sides
    x[rows - 1, k - 1] = float('nan')
    w[n - 1, 0] = float('inf')
    got = amd.mxfp4_dense(x, amd.mxfp4_quantize(w), None, None, torch.float32)
    assert torch.isnan(got[rows - 1]).all() and torch.isnan(got[:, n - 1]).all()
    assert torch.equal(got[:rows - 1, :n - 1], clean[:rows - 1, :n - 1])


def test_generic_activation_in_large_tiles(amd, oracle):
    rng = np.random.default_rng(8)
    w = amd.mxfp4_quantize(_features(rng, (4104, 64), torch.float32) * 0.05)
    for rows in (1500, 4500):
        x = _features(rng, (rows, 64), torch.float32)
        before = amd.mxfp4_dense(x, w).double().cpu().numpy()
        got = amd.mxfp4_dense(x, w, None, 'tanh').double().cpu().numpy()
        assert np.abs(got - np.tanh(before)).max() <= 1e-5


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows, k, n', [(1, 16384, 33), (16, 1024, 100), (16, 1024, 4100), (4, 4095, 50), (3, 4100, 4112), (15, 1090, 17), (16, 1025, 40), (16, 1, 3), (1, 4097, 1)])
def test_dense_of_a_few_rows(amd, dtype, rows, k, n):
    """Both sides of the sizes up to which x is quantised inside the product, and of those that decide how many waves share that."""
    rng = np.random.default_rng(rows + k)
    x, w4 = _features(rng, (rows, k), dtype), amd.mxfp4_quantize(_features(rng, (n, k), torch.float32))
    bias = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    _check_product(amd.mxfp4_dense(x, w4, bias, 'relu', torch.float32), x64, w64, bias.double().cpu().numpy(), True, torch.float32)
    got = amd.mxfp4_dense(x, w4, None, None, torch.float32)
    _check_product(got, x64, w64, None, False, torch.float32)
    odd = torch.zeros(rows * k + 1, dtype=dtype, device='cuda')[1:].view(rows, k)       # rows that start on no 16 bytes
    odd.copy_(x)
    assert torch.equal(amd.mxfp4_dense(odd, w4, None, None, torch.float32), got)
    tanh = amd.mxfp4_dense(x, w4, None, 'tanh', torch.float32).double().cpu().numpy()
    assert np.abs(tanh - np.tanh(got.double().cpu().numpy())).max() <= 1e-5             # the same float32 sum on both sides
    x[rows - 1, k - 1] = float('nan')
    bad = amd.mxfp4_dense(x, w4, None, None, torch.float32)
    assert torch.isnan(bad[rows - 1]).all() and torch.equal(bad[:rows - 1], got[:rows - 1])


@pytest.mark.parametrize('dtype, rows, k, n', [
    (torch.float32, 17, 1, 1), (torch.bfloat16, 24, 128, 8192), (torch.float16, 100, 33, 300), (torch.float32, 1000, 64, 1030), (torch.bfloat16, 3410, 128, 128),
    (torch.float32, 3410, 256, 256), (torch.float16, 8001, 257, 250), (torch.float32, 13505, 128, 128), (torch.bfloat16, 5001, 301, 50), (torch.float16, 2000, 2048, 100),
    (torch.float32, 4097, 1024, 64), (torch.bfloat16, 300, 512, 516), (torch.float32, 48332, 40, 7), (torch.bfloat16, 16384, 1500, 128), (torch.float16, 77, 1023, 2049)], ids=str)
def test_dense_with_small_weights(amd, dtype, rows, k, n):
    """The sizes of the network's own layers and around them: one launch that takes x as it is; every way of sharing out rows and columns."""
    rng = np.random.default_rng(rows + n)
    x, w = _features(rng, (rows, k), dtype), _features(rng, (n, k), torch.float32) * 0.05
    bias = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    w4 = amd.mxfp4_quantize(w)
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    for out in TYPES:
        _check_product(amd.mxfp4_dense(x, w4, bias, 'relu', out), x64, w64, bias.double().cpu().numpy(), True, out)
    clean = amd.mxfp4_dense(x, w4, None, None, torch.float32)
    _check_product(clean, x64, w64, None, False, torch.float32)
    assert torch.equal(clean, amd.mxfp4_dense(x, w4, None, None, torch.float32))
    odd = torch.zeros(rows * k + 1, dtype=dtype, device='cuda')[1:].view(rows, k)       # rows that start on no 16 bytes
    odd.copy_(x)
    assert torch.equal(amd.mxfp4_dense(odd, w4, None, None, torch.float32), clean)
    tanh = amd.mxfp4_dense(x, w4, None, 'tanh', torch.float32)
    assert (tanh.double() - torch.tanh(clean.double())).abs().max() <= 1e-5             # the same float32 sum on both sides
    x[rows - 1, k - 1] = float('nan')
    w[n - 1, 0] = float('inf')
    got = amd.mxfp4_dense(x, amd.mxfp4_quantize(w), None, None, torch.float32)
    assert torch.isnan(got[rows - 1]).all() and torch.isnan(got[:, n - 1]).all()
    assert torch.equal(got[:rows - 1, :n - 1], clean[:rows - 1, :n - 1])


@pytest.mark.parametrize('rows, k, n', [(300, 1100, 1000), (60, 1500, 4200), (3000, 1030, 130), (16500, 96, 255), (250, 2500, 700), (128, 1030, 8)])
def test_dense_just_past_small_weights(amd, rows, k, n):
    rng = np.random.default_rng(rows + n)
    x, w4 = _features(rng, (rows, k), torch.bfloat16), amd.mxfp4_quantize(_features(rng, (n, k), torch.float32))
    bias = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    _check_product(amd.mxfp4_dense(x, w4, bias, 'relu'), x64, w64, bias.double().cpu().numpy(), True, torch.bfloat16)
    _check_product(amd.mxfp4_dense(x, w4, None, None, torch.float32), x64, w64, None, False, torch.float32)


@pytest.mark.parametrize('rows, k, n', [(33, 8200, 2500), (64, 1000, 2048), (64, 1000, 2049), (90, 300, 1380), (512, 2080, 256), (512, 100, 260), (700, 32, 200)])
def test_dense_of_a_middling_size(amd, rows, k, n):
    """Some tens to some hundreds of rows, on both sides of the size where the form of 32 rows x 16 columns no longer has a compute unit for
    each of its workgroups; long rows, ragged edges, an activation of its own, and a row and a column of NaN."""
    rng = np.random.default_rng(rows + n)
    x, w = _features(rng, (rows, k), torch.bfloat16), _features(rng, (n, k), torch.float32) * 0.05
    bias = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    w4 = amd.mxfp4_quantize(w)
    x64, w64 = _plain(amd.mxfp4_quantize(x)), _plain(w4)
    _check_product(amd.mxfp4_dense(x, w4, bias, 'relu'), x64, w64, bias.double().cpu().numpy(), True, torch.bfloat16)
    clean = amd.mxfp4_dense(x, w4, None, None, torch.float32)
    _check_product(clean, x64, w64, None, False, torch.float32)
    # both evaluate tanh of the same float32 sum: the function's own error, as in the other layers
    tanh = amd.mxfp4_dense(x, w4, None, 'tanh', torch.float32).double().cpu().numpy()
    assert np.abs(tanh - np.tanh(clean.double().cpu().numpy())).max() <= 1e-5
    x[rows - 1, k - 1] = float('nan')
    w[n - 1, 0] = float('inf')
    got = amd.mxfp4_dense(x, amd.mxfp4_quantize(w), None, None, torch.float32)
    assert torch.isnan(got[rows - 1]).all() and torch.isnan(got[:, n - 1]).all()
    assert torch.equal(got[:rows - 1, :n - 1], clean[:rows - 1, :n - 1])


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('t, top_k, e, k, n', [(1, 1, 3, 2049, 40), (1, 2, 8, 8192, 48), (1, 16, 20, 100, 33), (4, 4, 6, 1024, 130), (4, 4, 6, 1025, 130), (2, 3, 8, 2500, 48),
                                               (16, 1, 2, 1000, 16), (17, 1, 3, 64, 16), (3, 5, 1, 33, 257)])
def test_expert_dense_of_a_few_rows(amd, dtype, t, top_k, e, k, n):
    """Both sides of the sizes up to which the tokens are quantised inside the experts' product; a dropped choice, an expert named twice."""
    rng = np.random.default_rng(t * k + top_k)
    index = rng.integers(0, e, (t, top_k)).astype(np.int32)
    if t * top_k > 2:
        index[t // 2, top_k - 1] = -1
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    x, w4 = _features(rng, (t, k), dtype), amd.mxfp4_quantize(_features(rng, (e, n, k), torch.float32))
    bias = torch.as_tensor(rng.standard_normal((e, n)), dtype=torch.float32).cuda()
    q, w64 = R.dispatch(_plain(amd.mxfp4_quantize(x)), plan.slot.cpu().numpy()), _plain3(w4)
    offsets, order = plan.offsets.cpu().numpy(), plan.order.cpu().numpy()
    got = amd.mxfp4_expert_dense(x, w4, plan, bias, 'relu', torch.float32)
    for i in range(e):
        lo, hi = offsets[i], offsets[i + 1]
        _check_product(got[lo:hi], q[lo:hi], w64[i], bias[i].double().cpu().numpy(), True, torch.float32)
    assert not got[offsets[e]:].any()
    ready = amd.expert_dispatch(x, plan)
    assert torch.equal(amd.mxfp4_expert_dense(ready, w4, plan, bias, 'relu', torch.float32, sorted_rows=True), got)
    odd = torch.zeros(t * k + 1, dtype=dtype, device='cuda')[1:].view(t, k)             # rows that start on no 16 bytes
    odd.copy_(x)
    assert torch.equal(amd.mxfp4_expert_dense(odd, w4, plan, bias, 'relu', torch.float32), got)
    x[t - 1, k - 1] = float('nan')
    bad = torch.isnan(amd.mxfp4_expert_dense(x, w4, plan)).all(1).cpu().numpy()
    assert np.array_equal(bad, (order >= 0) & (order // top_k == t - 1))


@pytest.mark.parametrize('t, top_k, e, k, n, dtype', [
    (100, 3, 40, 288, 1000, torch.bfloat16), (90, 3, 40, 520, 1001, torch.float16), (1500, 1, 64, 33, 2050, torch.float32),         # 32 x 128 tiles
    (500, 2, 64, 100, 1032, torch.float32), (3000, 1, 40, 300, 833, torch.bfloat16), (700, 3, 37, 1030, 904, torch.float16),        # 64 x 128
    (300, 1, 5, 160, 4100, torch.bfloat16), (700, 2, 5, 64, 4100, torch.float16), (1950, 2, 3, 160, 4090, torch.bfloat16)], ids=str)  # 64 x 64, 64 x 128, 256 x 256
def test_expert_dense_with_some_rows_each(amd, t, top_k, e, k, n, dtype):
    """Two to a thousand rows per expert on average, very unevenly: experts of no row, of one, of several tiles; dropped choices."""
    rng = np.random.default_rng(t + n)
    share = rng.permutation(np.arange(e) ** 2 + 0.0)
    index = np.where(rng.random((t, top_k)) < 0.05, -1, rng.choice(e, (t, top_k), p=share / share.sum())).astype(np.int32)
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    x, w4 = _features(rng, (t, k), dtype), amd.mxfp4_quantize(_features(rng, (e, n, k), torch.bfloat16))
    bias = torch.as_tensor(rng.standard_normal((e, n)), dtype=torch.float32).cuda()
    q, w64 = R.dispatch(_plain(amd.mxfp4_quantize(x)), plan.slot.cpu().numpy()), _plain3(w4)
    offsets = plan.offsets.cpu().numpy()
    assert (np.diff(offsets) == 0).any()
    got = amd.mxfp4_expert_dense(x, w4, plan, bias, 'relu')
    full = amd.mxfp4_expert_dense(x, w4, plan, None, None, torch.float32)
    tanh = amd.mxfp4_expert_dense(x, w4, plan, None, 'tanh', torch.float32)
    for i in range(e):
        lo, hi = offsets[i], offsets[i + 1]
        _check_product(got[lo:hi], q[lo:hi], w64[i], bias[i].double().cpu().numpy(), True, dtype)
        _check_product(full[lo:hi], q[lo:hi], w64[i], None, False, torch.float32)
    assert (tanh.double() - torch.tanh(full.double())).abs().max() <= 1e-5             # the same float32 sum on both sides
    assert not got[offsets[e]:].any() and not full[offsets[e]:].any() and not tanh[offsets[e]:].any()
    ready = amd.expert_dispatch(x, plan)
    assert torch.equal(amd.mxfp4_expert_dense(ready, w4, plan, bias, 'relu', sorted_rows=True), got)


@pytest.mark.parametrize('t, top_k, e, k, n', [(60, 2, 5, 1500, 208), (150, 1, 4, 2080, 130), (100, 3, 9, 33, 64)])
def test_expert_dense_of_a_middling_size(amd, t, top_k, e, k, n):
    """Ten to sixty rows per expert and few columns, one expert empty: tiles of 32 rows that end inside an expert."""
    rng = np.random.default_rng(t)
    index = rng.integers(-1, e, (t, top_k)).astype(np.int32)
    index[index == 1] = e - 1
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    x = _features(rng, (t, k), torch.float16)
    w4 = amd.mxfp4_quantize(_features(rng, (e, n, k), torch.float32))
    bias = torch.as_tensor(rng.standard_normal((e, n)), dtype=torch.float32).cuda()
    q = R.dispatch(_plain(amd.mxfp4_quantize(x)), plan.slot.cpu().numpy())
    offsets = plan.offsets.cpu().numpy()
    got = amd.mxfp4_expert_dense(x, w4, plan, bias, 'relu')
    for i in range(e):
        lo, hi = offsets[i], offsets[i + 1]
        if lo < hi:
            _check_product(got[lo:hi], q[lo:hi], _plain3(w4)[i], bias[i].double().cpu().numpy(), True, torch.float16)
    assert not got[offsets[e]:].any()


@pytest.mark.parametrize('t, top_k, e, k, n', [(3000, 2, 3, 160, 3000), (1700, 1, 6, 40, 8200), (700, 3, 40, 64, 4104)])
def test_expert_dense_in_every_tile_size(amd, t, top_k, e, k, n):
    """Uneven experts, one of them empty and one of a single row, in tiles of 256, 128 and 64 rows."""
    rng = np.random.default_rng(t)
    index = rng.integers(-1, e, (t, top_k)).astype(np.int32)
    index[index == 1] = 0
    index[5, 0] = 1
    if e > 4:
        index[index == 4] = 2
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    x = _features(rng, (t, k), torch.bfloat16)
    w4 = amd.mxfp4_quantize(_features(rng, (e, n, k), torch.bfloat16))
    bias = torch.as_tensor(rng.standard_normal((e, n)), dtype=torch.float32).cuda()
    q = R.dispatch(_plain(amd.mxfp4_quantize(x)), plan.slot.cpu().numpy())
    offsets = plan.offsets.cpu().numpy()
    got = amd.mxfp4_expert_dense(x, w4, plan, bias)
    w64 = _plain3(w4)
    for i in range(e):
        a, b = offsets[i], offsets[i + 1]
        _check_product(got[a:b], q[a:b], w64[i], bias[i].double().cpu().numpy(), False, torch.bfloat16)
    assert not got[offsets[-1]:].any() and offsets[-1] < t * top_k


@pytest.mark.parametrize('rows', [3, 40, 300])
def test_every_activation(amd, oracle, rows):
    """Both sides evaluate the activation of the same float32 sum, so only the function's own error counts: the float32 gate of the
    other layers.  The sums reach 123 here, whose exponential is no float32 number: above the type's largest value the
    result is infinity, and since the function's error is relative (2 units in the last place = 2.4e-7), the exponential is held to the gate
    entry by entry rather than against its largest value; exp(-87.4) and less lies below the smallest normal number,
    2^-126, where a result may be rounded to any subnormal or zero: off by at most 2^-126."""
    rng = np.random.default_rng(4)
    x, w = _features(rng, (rows, 160), torch.float32), amd.mxfp4_quantize(_features(rng, (40, 160), torch.float32) * 0.05)
    before = amd.mxfp4_dense(x, w).double().cpu().numpy()
    for name in ('tanh', 'sigmoid', 'elu', 'softplus', 'selu', 'swish', 'gelu', 'softsign', 'exponential', 'hard_sigmoid', 'relu', 'linear'):
        got = amd.mxfp4_dense(x, w, None, name).double().cpu().numpy()
        want = np.asarray(oracle.ACTIVATIONS[name](before), np.float64)
        over = np.abs(want) > torch.finfo(torch.float32).max
        assert (got[over] == np.inf).all(), name
        scale = np.abs(want[~over]) if name == 'exponential' else np.abs(want).max()
        off = np.abs(got[~over] - want[~over])
        assert (off <= 1e-5 * scale + 2.0 ** -126).all(), (name, before[~over][off > 1e-5 * scale + 2.0 ** -126][:5])


@pytest.mark.parametrize('rows', [1, 40, 300])
def test_special_values_stay_in_their_rows(amd, rows):
    rng = np.random.default_rng(6)
    x = _features(rng, (rows, 320), torch.float32)
    w = _features(rng, (70, 320), torch.float32)
    clean = amd.mxfp4_dense(x, amd.mxfp4_quantize(w))
    x[rows // 2, 300] = float('nan')
    w[33, 2] = float('inf')
    w4 = amd.mxfp4_quantize(w)
    got = amd.mxfp4_dense(x, w4)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[rows // 2] = True
    bad[:, 33] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    assert (amd.mxfp4_dense(x, w4, None, 'relu')[bad] == 0).all()          # as the float32 layers have it


def test_scales_at_the_ends_of_the_range(amd):
    """Products far below and above float32's range: zeros and infinities, no NaN, neighbours unharmed."""
    x = torch.ones((2, 64), device='cuda')
    x[0] *= 2.0 ** -120
    x[1] *= 2.0 ** 120
    w = torch.ones((3, 64), device='cuda')
    w[0] *= 2.0 ** -120
    w[1] *= 2.0 ** 120
    got = amd.mxfp4_dense(x, amd.mxfp4_quantize(w)).cpu()
    assert got[0, 0] == 0 and got[1, 1] == float('inf')
    assert got[0, 1] == 64 and got[1, 0] == 64 and got[0, 2] == 64 * 2.0 ** -120 and got[1, 2] == 64 * 2.0 ** 120


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('t, top_k, e, k, n, pattern', [
    (1, 1, 1, 32, 16, 'even'), (1, 2, 8, 256, 128, 'even'), (5, 3, 70, 100, 33, 'dropped'), (32, 4, 32, 512, 96, 'even'), (100, 2, 3, 288, 130, 'dropped'),
    (300, 2, 4, 128, 256, 'one'), (40, 2, 5, 64, 48, 'none'), (700, 2, 5, 160, 300, 'dropped'), (900, 3, 200, 96, 64, 'even')])
def test_expert_dense_against_the_exact_products(amd, dtype, t, top_k, e, k, n, pattern):
    rng = np.random.default_rng(t + k)
    index = {'even': lambda: rng.integers(0, e, (t, top_k)), 'dropped': lambda: rng.integers(-1, e, (t, top_k)),
             'one': lambda: np.full((t, top_k), e - 1), 'none': lambda: np.full((t, top_k), -1)}[pattern]().astype(np.int32)
    plan = amd.expert_plan(torch.as_tensor(index).cuda(), e)
    x = _features(rng, (t, k), dtype)
    w4 = amd.mxfp4_quantize(_features(rng, (e, n, k), torch.bfloat16))
    bias = torch.as_tensor(rng.standard_normal((e, n)), dtype=torch.float32).cuda()
    q = R.dispatch(_plain(amd.mxfp4_quantize(x)), plan.slot.cpu().numpy())
    offsets = plan.offsets.cpu().numpy()
    got = amd.mxfp4_expert_dense(x, w4, plan, bias, 'relu')
    ready = amd.mxfp4_expert_dense(amd.expert_dispatch(x, plan), w4, plan, bias, 'relu', sorted_rows=True)
    assert got.dtype == dtype and torch.equal(got, ready)
    w64 = _plain3(w4)
    for i in range(e):
        a, b = offsets[i], offsets[i + 1]
        _check_product(got[a:b], q[a:b], w64[i], bias[i].double().cpu().numpy(), True, dtype)
    assert not got[offsets[-1]:].any()


def test_a_whole_expert_layer(amd):
    """route -> dispatch on 4-bit rows -> two products per expert -> weighted sum, each stage against the exact value of its own input."""
    rng = np.random.default_rng(9)
    t, top_k, e, c, hidden = 150, 2, 6, 128, 256
    plan = amd.expert_plan(torch.as_tensor(rng.integers(-1, e, (t, top_k)).astype(np.int32)).cuda(), e)
    slot, offsets = plan.slot.cpu().numpy(), plan.offsets.cpu().numpy()
    x = _features(rng, (t, c), torch.bfloat16)
    w1 = amd.mxfp4_quantize(_features(rng, (e, hidden, c), torch.bfloat16))
    w2 = amd.mxfp4_quantize(_features(rng, (e, c, hidden), torch.bfloat16))
    gate = torch.as_tensor(rng.random((t, top_k)), dtype=torch.float32).cuda()
    h = amd.mxfp4_expert_dense(x, w1, plan, None, 'relu')
    y = amd.mxfp4_expert_dense(h, w2, plan, None, None, sorted_rows=True)
    out = amd.expert_combine(y, gate, plan)
    q = R.dispatch(_plain(amd.mxfp4_quantize(x)), slot)
    qh = _plain(amd.mxfp4_quantize(h))
    for i in range(e):
        a, b = offsets[i], offsets[i + 1]
        _check_product(h[a:b], q[a:b], _plain3(w1)[i], None, True, torch.bfloat16)
        _check_product(y[a:b], qh[a:b], _plain3(w2)[i], None, False, torch.bfloat16)
    want, size = R.combine(y.double().cpu().numpy(), gate.double().cpu().numpy(), slot)
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) + 3 * 2.0 ** -24 * 1.01 * size).all()


def test_dense_layer_in_four_bits(amd):
    rng = np.random.default_rng(12)
    dense = amd.hybrid_gnn.Dense(48, 'relu')
    dense.load_weights({'d/kernel': rng.standard_normal((104, 48)).astype(np.float32), 'd/bias': rng.standard_normal(48).astype(np.float32)}, 'd', 'cuda')
    layer = amd.Mxfp4Dense.from_dense(dense)
    x = _features(rng, (2, 30, 104), torch.float32)
    got = layer(x)
    assert got.shape == (2, 30, 48)
    xq = _plain(amd.mxfp4_quantize(x.view(60, 104)))
    wq = _plain(amd.mxfp4_quantize(dense.kernel.t()))
    _check_product(got.view(60, 48), xq, wq, dense.bias.double().cpu().numpy(), True, torch.float32)
    _check_product(layer(x, None).view(60, 48), xq, wq, dense.bias.double().cpu().numpy(), False, torch.float32)


def test_every_form_in_one_graph(amd):
    """One product of each form side by side in one graph, replayed with new inputs and eager work between the replays."""
    rng = np.random.default_rng(14)
    sizes = [(1, 1024, 48), (5, 4000, 64), (3410, 128, 128), (100, 33, 300), (64, 2080, 80), (20, 1100, 9000), (40, 1500, 9000), (700, 1030, 4001), (3000, 33, 2056),
             (3990, 64, 4088)]
    xs = [torch.zeros((rows, k), dtype=torch.bfloat16, device='cuda') for rows, k, _ in sizes]
    ws = [amd.mxfp4_quantize(_features(rng, (n, k), torch.float32)) for _, k, n in sizes]
    shapes = [(2, 2, 8, 256, 64), (96, 2, 64, 64, 520), (900, 2, 64, 64, 520), (700, 2, 5, 64, 4100)]
    ws += [amd.mxfp4_quantize(_features(rng, (e, n, k), torch.float32)) for _, _, e, k, n in shapes]
    index = [torch.zeros((t, top_k), dtype=torch.int32, device='cuda') for t, top_k, *_ in shapes]
    xs += [torch.zeros((t, k), dtype=torch.bfloat16, device='cuda') for t, _, _, k, _ in shapes]

    def step():
        out = [amd.mxfp4_dense(x, w) for x, w in zip(xs[:len(sizes)], ws)]
        plans = [amd.expert_plan(i, shape[2]) for i, shape in zip(index, shapes)]
        return out + [amd.mxfp4_expert_dense(x, w, p) for x, w, p in zip(xs[len(sizes):], ws[len(sizes):], plans)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for turn in range(4):
        for x in xs:
            x.copy_(torch.as_tensor(rng.standard_normal(tuple(x.shape))))
        for i, shape in zip(index, shapes):
            i.copy_(torch.as_tensor(rng.integers(-1, shape[2], tuple(i.shape)).astype(np.int32)))
        g.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn
        assert all(a.float().abs().max() > 0 for a in out)


def test_captured_layer_follows_new_inputs(amd):
    """Small and large products in two graphs that live together, replayed with eager work and new inputs in between."""
    rng = np.random.default_rng(13)
    e, c, n = 4, 160, 96
    w1, w2 = amd.mxfp4_quantize(_features(rng, (e, n, c), torch.float32)), amd.mxfp4_quantize(_features(rng, (80, n), torch.float32))
    graphs = []
    for t in (3, 400):
        index = torch.zeros((t, 2), dtype=torch.int32, device='cuda')
        x = torch.zeros((t, c), device='cuda')

        def step(index=index, x=x):
            plan = amd.expert_plan(index, e)
            h = amd.mxfp4_expert_dense(x, w1, plan, None, 'relu')
            return amd.mxfp4_dense(amd.expert_combine(h, torch.ones_like(index, dtype=torch.float32), plan), w2)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, index, x, step, out))
    for turn in range(4):
        for g, index, x, step, out in graphs:
            index.copy_(torch.as_tensor(rng.integers(-1, e, tuple(index.shape)).astype(np.int32)))
            x.copy_(torch.as_tensor(rng.standard_normal(tuple(x.shape))))
        for g, *_ in graphs:
            g.replay()
        for g, index, x, step, out in graphs:
            want = step()
            torch.cuda.synchronize()
            assert torch.equal(out, want), turn


def test_two_streams_at_once(amd):
    rng = np.random.default_rng(14)
    w = amd.mxfp4_quantize(_features(rng, (512, 1024), torch.bfloat16))
    xs = [_features(rng, (rows, 1024), torch.bfloat16) for rows in (700, 5)]
    want = [amd.mxfp4_dense(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(amd.mxfp4_dense(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(amd):
    x = torch.zeros((4, 64)).cuda()
    w = amd.mxfp4_quantize(torch.zeros((8, 64)).cuda())
    for bad in (x.cpu(), x.double(), x.int()):
        with pytest.raises(TypeError):
            amd.mxfp4_quantize(bad)
        with pytest.raises(TypeError):
            amd.mxfp4_dense(bad, w)
    for bad in (x[0], x[:, :0], x.view(1, 1, 4, 64)):
        with pytest.raises(ValueError):
            amd.mxfp4_quantize(bad)
    with pytest.raises(ValueError):
        amd.mxfp4_dense(x[:, :32], w)
    with pytest.raises(TypeError):
        amd.mxfp4_dense(x, torch.zeros((8, 64)).cuda())
    with pytest.raises(ValueError):
        amd.mxfp4_dense(x, w, torch.zeros(7).cuda())
    with pytest.raises(TypeError):
        amd.mxfp4_dense(x, w, torch.zeros(8).cuda().half())
    with pytest.raises(NotImplementedError):
        amd.mxfp4_dense(x, w, None, 'maxout')
    with pytest.raises(TypeError):
        amd.mxfp4_dense(x, w, None, None, torch.float64)
    with pytest.raises(TypeError):
        amd.mxfp4_dequantize(w, torch.int8)
    with pytest.raises(ValueError, match='gradient'):
        amd.mxfp4_dense(x.clone().requires_grad_(), w)
    stack = amd.mxfp4_quantize(torch.zeros((3, 8, 64)).cuda())
    with pytest.raises(ValueError):
        amd.mxfp4_dense(x, stack)
    plan = amd.expert_plan(torch.zeros((4, 2), dtype=torch.int32).cuda(), 3)
    with pytest.raises(ValueError):
        amd.mxfp4_expert_dense(x, w, plan)
    with pytest.raises(ValueError):
        amd.mxfp4_expert_dense(x[:3], stack, plan)
    with pytest.raises(ValueError):
        amd.mxfp4_expert_dense(x, stack, plan, sorted_rows=True)
    with pytest.raises(ValueError):
        amd.mxfp4_expert_dense(x, stack, plan, torch.zeros(8).cuda())
    with pytest.raises(ValueError):
        amd.Mxfp4Tensor.from_codes(torch.zeros((8, 30), dtype=torch.uint8).cuda(), torch.zeros((8, 2), dtype=torch.uint8).cuda(), 64)
    with pytest.raises(ValueError):
        amd.Mxfp4Dense.from_dense(amd.hybrid_gnn.Dense(8))
    for codes, scales in ((w.codes[:, :7], w.scales), (w.codes, w.scales[:, :, :7]), (w.codes.transpose(1, 2), w.scales)):
        with pytest.raises(ValueError):
            amd.Mxfp4Tensor(codes, scales, (8, 64))
    with pytest.raises(TypeError):
        amd.Mxfp4Tensor(w.codes.int(), w.scales, (8, 64))
