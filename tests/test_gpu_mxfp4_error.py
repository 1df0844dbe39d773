"""How far a Dense layer in 4 bits may be from the unquantised one."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _off(v):
    """How far quantising may move each value of v [rows, k]: a quarter of itself, or a sixteenth of its block's largest.
    In units of the block's scale the largest lies in [4, 8).  Below 2 a value is off by half a step at most, 1/4 <= 4 / 16; in [2, 4) by 1/2 <= v / 4;
    in [4, 6] by 1 <= v / 4; above 6, where it saturates, by v - 6 <= v / 4."""
    rows, k = v.shape
    padded = np.zeros((rows, -(-k // 32) * 32))
    padded[:, :k] = np.abs(v)
    largest = np.repeat(padded.reshape(rows, -1, 32).max(-1), 32, 1)[:, :k]
    return np.maximum(np.abs(v) / 4, largest / 16)


@pytest.mark.parametrize('rows, k, n, act', [(60, 104, 128, None), (500, 128, 96, 'relu'), (40, 1024, 300, None), (3, 2000, 70, 'relu')])
def test_distance_from_the_unquantised_layer(rows, k, n, act):
    """|q(x) q(w) - x w| <= |x| dw + dx |w| + dx dw with the bounds of _off, plus both float32 sums' rounding, k + 1 additions of at most
    2^-23 of the terms' magnitudes each; a ReLU moves no two values further apart.  And it is coarse: 0.16 of the results' size on normal data."""
    import gunet_amd as amd
    rng = np.random.default_rng(k)
    dense = amd.hybrid_gnn.Dense(n, act)
    kernel = (rng.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)
    dense.load_weights({'d/kernel': kernel, 'd/bias': rng.standard_normal(n).astype(np.float32)}, 'd', 'cuda')
    x = torch.as_tensor(rng.standard_normal((rows, k)), dtype=torch.float32).cuda()
    plain, four = dense(x).double().cpu().numpy(), amd.Mxfp4Dense.from_dense(dense)(x).double().cpu().numpy()
    x64, w64 = x.double().cpu().numpy(), kernel.astype(np.float64).T
    dx, dw = _off(x64), _off(w64)
    moved = np.abs(x64) @ dw.T + dx @ np.abs(w64).T + dx @ dw.T
    size = (np.abs(x64) + dx) @ (np.abs(w64) + dw).T + np.abs(dense.bias.double().cpu().numpy())
    assert (np.abs(four - plain) <= moved + 2 * (k + 1) * 2.0 ** -23 * size).all()
    assert not np.array_equal(four, plain)
