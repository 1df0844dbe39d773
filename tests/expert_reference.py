"""Plain 64-bit numpy restatements of the expert-row operators and of the 4-bit microscaled format, from their
definitions (test infrastructure; nothing here is imported by the package)."""
import numpy as np

LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
# middles between neighbouring levels; the level above wins a tie where its number is even
MIDDLES = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5])


def sort_by_expert(index, n_experts):
    """(offsets, order, slot) of index [T, k]."""
    t, k = index.shape
    flat = index.reshape(-1)
    rows = [[] for _ in range(n_experts)]
    for f, e in enumerate(flat.tolist()):
        if 0 <= e < n_experts:
            rows[e].append(f)
    offsets = np.concatenate(([0], np.cumsum([len(r) for r in rows]))).astype(np.int32)
    order = np.full(t * k, -1, np.int32)
    slot = np.full(t * k, -1, np.int32)
    members = [f for r in rows for f in r]
    order[:len(members)] = members
    slot[members] = np.arange(len(members))
    return offsets, order, slot.reshape(t, k)


def dispatch(x, slot):
    rows = np.zeros((slot.size, x.shape[1]))
    t, j = np.nonzero(slot >= 0)
    rows[slot[t, j]] = x[t]
    return rows


def combine(rows, weights, slot):
    """(out, sum of the terms' magnitudes)."""
    got = np.where((slot >= 0)[..., None], rows[np.maximum(slot, 0)], 0.0) if slot.size else np.zeros(slot.shape + (rows.shape[1],))
    terms = got * weights[..., None]
    return terms.sum(1), np.abs(terms).sum(1)


def combine_grad(grad, rows, weights, slot):
    """(grad_rows, grad_weights, sum of the magnitudes behind each grad_weights entry)."""
    grad_rows = np.zeros_like(rows)
    grad_weights = np.zeros(slot.shape)
    size = np.zeros(slot.shape)
    for t, j in zip(*np.nonzero(slot >= 0)):
        r = slot[t, j]
        grad_rows[r] = weights[t, j] * grad[t]
        grad_weights[t, j] = grad[t] @ rows[r]
        size[t, j] = np.abs(grad[t]) @ np.abs(rows[r])
    return grad_rows, grad_weights, size


def quantize(x):
    """x [rows, k] (exact in float64) -> (level numbers with sign bit [rows, blocks, 32], scale bytes [rows, blocks])."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    blocks = -(-k // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :k] = x
    v = v.reshape(rows, blocks, 32)
    with np.errstate(invalid='ignore'):
        top = np.abs(v).max(-1)
    bad = ~np.isfinite(top)
    safe = np.where(bad | (top == 0), 1.0, top)
    e = np.frexp(safe)[1] - 1 - 2
    e = np.where(top == 0, -127, np.maximum(e, -127))
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    a = np.abs(np.where(bad[..., None], 0.0, v)) * np.exp2(-e.astype(np.float64))[..., None]
    code = np.zeros(a.shape, np.uint8)
    for i, m in enumerate(MIDDLES):
        code = np.where((a > m) | ((a == m) & (i % 2 == 1)), i + 1, code)
    code = (code | np.where(np.signbit(v), 8, 0)).astype(np.uint8)
    code[bad] = 0
    return code, scales


def values(code, scales, k):
    """float64 [rows, k] of level numbers and scale bytes."""
    sign = np.where(code & 8, -1.0, 1.0)
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (sign * LEVELS[code & 7] * scale[..., None]).reshape(code.shape[0], -1)[:, :k]


def pack(code):
    """[rows, blocks, 32] level numbers -> bytes [rows, blocks, 16], the even column in the low four bits."""
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)
