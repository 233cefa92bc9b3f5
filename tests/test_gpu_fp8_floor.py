"""The scale byte at its floor: 0 up to 448 * 2^-127 = 1.75 * 2^-119, then one
more at every doubling; and the values that such blocks hold."""
import numpy as np
import pytest

import fp8_util as F
from gpu_util import bf16_round, dev_bf16, host, torch
from test_gpu_fp8 import u8

pytestmark = pytest.mark.gpu
EDGE = 1.75 * 2.0 ** -119
STEP = 2.0 ** -126          # bf16 steps by 2^-7 of 2^-119 around the edge
AMAX = [0.0, 2.0 ** -133, 2.0 ** -126, EDGE - STEP, EDGE, EDGE + STEP, 2.0 ** -118, 2 * EDGE,
        2 * EDGE + 2 * STEP, 4 * EDGE, 4 * EDGE + 4 * STEP]
BYTES = [0, 0, 0, 0, 0, 1, 1, 1, 2, 2, 3]


def blocks():
    """Row r: its largest magnitude AMAX[r], ties and small values beside it."""
    x = np.zeros((len(AMAX), 128), np.float64)
    for r, a in enumerate(AMAX):
        x[r] = a * np.linspace(-1, 1, 128)
        x[r, 0] = -a
    b = bf16_round(x.astype(np.float32))
    assert np.array_equal(np.abs(b).max(1), np.float32(AMAX))
    return b


def test_rows():
    import u15b200
    ops, x = u15b200.CudaOps(0), blocks()
    n = len(AMAX)
    q, s, y = u8(n * 128), u8(F.scale_bytes(n, 128)), torch.empty(n, 128, dtype=torch.bfloat16,
                                                                   device="cuda")
    ops.quant_rows_fp8(dev_bf16(x), q, s, n, 128)
    ops.dequant_fp8(q, s, y, n, 128)
    assert F.unpack(host(s), n, 128)[:, 0].tolist() == BYTES
    wq, ws = F.quantise(x.astype(np.float64))
    assert ws[:, 0].tolist() == BYTES
    assert np.array_equal(host(q).reshape(n, 128), wq)
    # what they stand for, a rounding to bf16 behind it (steps of 2^-133 at the least)
    v = F.values(wq, ws)
    assert np.array_equal(host(y), bf16_round(v.astype(np.float32)))


def test_weights():
    import u15b200
    ops, x = u15b200.CudaOps(0), blocks()
    n = len(AMAX)
    q, s = u8(n * 128), u8(n * F.scale_bytes(1, 128))
    ops.quant_weight_fp8(dev_bf16(x), q, s, n, 1, 128)        # an expert of one row each
    got = host(s).reshape(n, -1)
    assert [F.unpack(g, 1, 128)[0, 0] for g in got] == BYTES
    assert np.array_equal(host(q).reshape(n, 128), F.quantise(x.astype(np.float64))[0])
