"""The largest products on 4-bit weights: one launch holds 2^32 - 1 threads, and a call that needs more is refused before anything reaches a
GPU (the addresses are never read)."""
import ctypes as C

import pytest

from mxfp4_forms import form_of

INVALID = -1
P = C.c_void_p(1 << 20)

# (rows, k, n_out, experts): the last size that fits, and the next one.  Threads a workgroup and the results it computes follow from the form.
EDGES = [
    ((2 ** 30 - 1024, 64, 64, 0), (2 ** 30 - 1023, 64, 64, 0)),         # 128 x 128 tiles of 512 threads, in eights
    ((2 ** 30 - 1024, 4096, 128, 0), (2 ** 30, 4096, 128, 0)),
    ((1, 32, 2 ** 27 - 16, 0), (1, 32, 2 ** 27 - 15, 0)),               # one row: 512 threads for 16 results
    ((60000, 32, 8944, 60000), (60000, 32, 8945, 60000)),               # a row an expert: 128 threads for 16 results
]


@pytest.fixture(scope='module')
def lib():
    import gunet_amd
    return gunet_amd._lib.lib


def _call(lib, rows, k, n, e):
    if e:
        return lib.gunet_mxfp4_expert_dense_forward(P, 1, P, None, rows, 1, e, k, P, P, None, n, 0, P, 1, P, 1 << 62, None)
    return lib.gunet_mxfp4_dense_forward(P, 1, rows, k, P, P, None, n, 0, P, 1, P, 1 << 62, None)


def test_what_one_launch_cannot_hold_is_refused(lib):
    for fits, beyond in EDGES:
        assert form_of(*fits), fits
        assert form_of(*beyond) == '', beyond
        assert _call(lib, *beyond) == INVALID and b'launch' in lib.gunet_last_error(), beyond
    for rows, k, n in ((2 ** 31 - 1, 1, 1), (2 ** 31 - 1, 64, 128), (2 ** 30 + 1, 4096, 64), (2 ** 29, 32, 2 ** 10), (4, 32, 2 ** 31 - 1)):
        assert form_of(rows, k, n, 0) == '' and _call(lib, rows, k, n, 0) == INVALID and b'launch' in lib.gunet_last_error(), (rows, k, n)
    assert form_of(2 ** 31 - 1, 4096, 256, 4) == '' and _call(lib, 2 ** 31 - 1, 4096, 256, 4) == INVALID and b'launch' in lib.gunet_last_error()


def test_what_is_refused_is_what_exceeds_the_threads():
    """The rule from the forms' names: sizes of a spread, each side of the border."""
    import random
    rng = random.Random(3)
    seen = [0, 0]
    for _ in range(4000):
        rows, n, k = (int(2 ** rng.uniform(0, top)) for top in (31, 31, 14))
        small = rows <= 16 and rows * k <= 16384
        form = form_of(rows, k, n, 0)
        if small:
            waves = 16 if rows * k > 4096 and -(-n // 16) <= 256 else 8
            threads = -(-n // 16) * 64 * waves
        elif form.startswith('tile'):
            m, c = (int(v) for v in form[5:].split(' x '))
            threads = -(-(-(-rows // m) * -(-n // c)) // 8) * 8 * {(64, 64): 256, (64, 128): 256, (128, 128): 512, (256, 256): 512}[m, c]
        else:
            continue
        assert bool(form) == (threads < 2 ** 32), (rows, k, n, form)
        seen[bool(form)] += 1
    assert min(seen) > 20
