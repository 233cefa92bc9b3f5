"""The quantising norm on rows whose sum of squares is not a finite f32: a row
that holds an Inf, and a finite row whose squares overflow, have a mean of Inf
and a reciprocal root of 0, so every finite value of theirs becomes 0 and the
Inf itself NaN, whatever the width."""
import numpy as np
import pytest

import fp8_util as F
from gpu_util import bf16_round, dev_bf16, host, randn, torch
from test_gpu_fp8 import activations, check_normed, u8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import u15b200
    return u15b200.CudaOps(0)


# 1 / dim in f32 is exact, above and below the true value; the last two are
# wider than the rows that the kernel holds in registers
@pytest.mark.parametrize("dim", [16, 256, 4096, 272, 1040, 12288, 1552, 4112, 16384, 16400, 20000])
@pytest.mark.parametrize("add", [False, True])
def test_norm_of_sums_past_f32(ops, dim, add):
    rows = 7
    x = activations(rows, dim, 5)
    at = [dim // 3, dim - 1]
    x[3] = 1e25                       # 1e50 is past f32's largest
    x[4, at[0]] = -2e19               # one square, 4e38, is enough
    x[5, at[0]] = 1e18                # 1e36: a finite sum, as any row
    x = bf16_round(x)
    x[1, at] = np.inf
    x[2, at] = -np.inf
    d = activations(rows, dim, 6)
    if add:
        d[3:6] = 0                    # the values above stay what they are
    w = bf16_round(randn((1, dim), 7, 0.2, 1.0))
    q, s = u8(rows * dim), u8(F.scale_bytes(rows, dim))
    out = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
    ops.mot_add_rms_norm_quant_fp8(dev_bf16(x), dev_bf16(d) if add else None, dev_bf16(w), None, out,
                                   q, s, rows, dim, 1e-6)
    ops.sync()
    got, sb = host(q).reshape(rows, dim) & 0x7F, F.unpack(host(s), rows, dim)
    for r in (1, 2):
        inf = np.zeros(dim, bool)
        inf[at] = True
        assert (got[r][inf] == 0x7F).all() and (got[r][~inf] == 0).all(), r
        clear = np.ones(sb.shape[1], bool)
        clear[[a // 128 for a in at]] = False
        assert (sb[r][clear] == 0).all()
    assert (got[3:5] == 0).all() and (sb[3:5] == 0).all()
    fin = [0, 5, 6]
    t = (bf16_round(x[fin] + d[fin]) if add else x[fin]).astype(np.float64)
    assert np.array_equal(host(out)[fin], t)
    y = t / np.sqrt((t * t).mean(1, keepdims=True) + np.float32(1e-6)) * w[0]
    check_normed(host(q).reshape(rows, dim)[fin], F.pack(sb[fin], dim), y, len(fin), dim)


@pytest.mark.parametrize("dim", [256, 272, 1552, 16400])
def test_norm_of_a_nan_is_nan(ops, dim):
    x = activations(3, dim, 8)
    x[1, dim // 2] = np.nan
    q, s = u8(3 * dim), u8(F.scale_bytes(3, dim))
    w = np.ones((1, dim), np.float32)
    ops.mot_add_rms_norm_quant_fp8(dev_bf16(x), None, dev_bf16(w), None, None, q, s, 3, dim, 1e-6)
    nan = (host(q).reshape(3, dim) & 0x7F) == 0x7F
    assert nan[1].all() and not nan[[0, 2]].any()
