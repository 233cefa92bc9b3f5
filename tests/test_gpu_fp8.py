"""GPU checks of the 8-bit floating point operators against the format
restated in numpy float64 (fp8_util.py).

Codes and scales of the quantisers must be equal bit for bit: their inputs are
bf16, the scaling by a power of two exact, the rounding IEEE. The norm's
output may be off by half an e4m3 step plus the f32 error before rounding.
Products may be off by the f32 sum's error (fp8_util.sum_error) plus half a
step of the output's type: 2^-8 of the value for bf16, 2^-24 for f32.
"""
import numpy as np
import pytest

import fp8_util as F
from gpu_util import bf16_round, dev_bf16, host, randn, torch

pytestmark = pytest.mark.gpu
STORE, RESID, SWIGLU, F32 = 0, 1, 2, 3
# f32 arithmetic ahead of a rounding (a mean over a row, a root, a division,
# two products): under 2^-18 of the value at every size tested here
PRE = 2.0 ** -18


@pytest.fixture(scope="module")
def ops():
    import u15b200
    return u15b200.CudaOps(0)


def u8(n, fill=0xAA):
    return torch.full((n,), fill, dtype=torch.uint8, device="cuda")


def dev_u8(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.uint8)).cuda()


def activations(rows, cols, seed):
    r = np.random.default_rng(seed)
    gain = np.exp(0.5 * r.normal(size=cols))
    gain[r.integers(0, cols, max(1, cols // 512))] *= 12
    return bf16_round(r.normal(size=(rows, cols)) * gain)


def quantised(rows, cols, seed, std=None, tall=1):
    v = activations(rows, cols, seed) if std is None else bf16_round(randn((rows, cols), seed, std))
    return F.quantise(v.astype(np.float64), tall)


def weights(E, N, K, seed):
    """E experts' (codes, scale bytes), and the stacked device tensors."""
    parts = [quantised(N, K, seed + e, 0.02, 128) for e in range(E)]
    q = dev_u8(np.stack([p[0] for p in parts]))
    s = dev_u8(np.concatenate([F.pack(p[1], K) for p in parts]))
    return parts, q, s


def by_expert(segs, rows, fn):
    """fn(rows' slice, expert) of every segment, joined."""
    out = [fn(slice(a, b), e) for a, b, e in (segs or [(0, rows, 0)]) if b > a]
    return [np.concatenate(p) for p in zip(*out)]


# ------------------------------------------------------------------ quantisers
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 128), (130, 144), (33, 1040), (257, 4096),
                                       (5, 12288), (2, 20000)])
def test_quant_rows_bit_exact(ops, rows, cols):
    x = activations(rows, cols, rows)
    x[rows // 2] = 0
    q, s = u8(rows * cols + 64), u8(F.scale_bytes(rows, cols) + 64)
    ops.quant_rows_fp8(dev_bf16(x), q, s, rows, cols)
    y = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    ops.dequant_fp8(q, s, y, rows, cols)
    wq, ws = F.quantise(x.astype(np.float64))
    got, gs = host(q), host(s)
    assert np.array_equal(F.unpack(gs, rows, cols), ws)
    assert np.array_equal(got[:rows * cols].reshape(rows, cols), wq)
    assert np.array_equal(host(y), F.values(wq, ws).astype(np.float32))
    # bytes that stand for nothing keep what they held
    free = np.ones(gs.size, bool)
    free[F.places(rows, cols)] = False
    assert (gs[free] == 0xAA).all() and (got[rows * cols:] == 0xAA).all()


def test_quant_ties_extremes_and_not_finite(ops):
    x = np.zeros((8, 256), np.float32)
    x[0, :128] = 448 * np.arange(128) / 128                     # ties of bf16 against e4m3
    x[0, 0] = 448
    x[1, :4] = [2.0 ** -133, -2.0 ** -130, 2.0 ** -126, 0]      # the scale byte's floor
    x[2, :3] = [3.3e38, -1.0, 1e30]
    x[3, 128:] = -0.0
    x[4, :128] = 449.0                                          # bf16 448 or 450: just past 448
    x[5, 7] = np.nan
    x[5, 8:16] = 2.5
    x[6, 130] = np.inf
    x[7, 200] = -np.inf
    x = bf16_round(x)
    x[5, 7], x[6, 130], x[7, 200] = np.nan, np.inf, -np.inf
    xd = dev_bf16(x)
    q, s = u8(8 * 256), u8(F.scale_bytes(8, 256))
    ops.quant_rows_fp8(xd, q, s, 8, 256)
    got = host(q).reshape(8, 256)
    fin = np.where(np.isfinite(x), x, 0).astype(np.float64)
    wq, ws = F.quantise(fin)
    assert np.array_equal(F.unpack(host(s), 8, 256)[:6], ws[:6])
    keep = np.isfinite(x)
    assert np.array_equal(got[:6][keep[:6]], wq[:6][keep[:6]])
    assert ((got & 0x7F) == 0x7F)[~keep].all() and ((got & 0x7F) != 0x7F)[keep].all()


@pytest.mark.parametrize("E,N,K", [(1, 1, 16), (2, 130, 144), (2, 256, 4096), (3, 40, 528)])
def test_quant_weight_bit_exact(ops, E, N, K):
    w = bf16_round(randn((E, N, K), 7, 0.02))
    q, s = u8(E * N * K), u8(E * F.scale_bytes(N, K))
    ops.quant_weight_fp8(dev_bf16(w), q, s, E, N, K)
    y = torch.empty(E, N, K, dtype=torch.bfloat16, device="cuda")
    ops.dequant_fp8(q, s, y, N, K, n_experts=E)
    for e in range(E):
        wq, ws = F.quantise(w[e].astype(np.float64), 128)
        per = host(s)[e * F.scale_bytes(N, K):][:F.scale_bytes(N, K)]
        assert np.array_equal(F.unpack(per, N, K), ws)
        assert np.array_equal(host(q).reshape(E, N, K)[e], wq)
        assert np.array_equal(host(y)[e], F.values(wq, ws).astype(np.float32))


def test_calls_side_by_side(ops):
    """Several products at once on streams of their own give what they give alone."""
    cases = [(3, 2048, 1024), (100, 1024, 768), (300, 512, 2048), (512, 2048, 4096)]
    streams = [torch.cuda.Stream() for _ in cases]
    made, want = [], []
    for M, K, N in cases:
        xq, xs, _ = random_quantised(ops, M, K, M, 1.0)
        wq, ws, _ = random_quantised(ops, N, K, N, 0.05)
        made.append((xq, xs, wq.view(1, N, K), ws))
        y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        ops.mot_linear_fp8(*made[-1], None, y, M, K, N)
        want.append(y)
    torch.cuda.synchronize()
    out = [torch.empty_like(y) for y in want]
    for _ in range(10):
        for st, a, y, (M, K, N) in zip(streams, made, out, cases):
            with torch.cuda.stream(st):
                ops.mot_linear_fp8(*a, None, y, M, K, N)
    torch.cuda.synchronize()
    ops.sync()
    for y, t in zip(out, want):
        assert torch.equal(y, t)


def test_scale_buffers_are_sized(ops):
    assert ops.fp8_scale(129, 528, n_experts=2).numel() == 2 * F.scale_bytes(129, 528)


# ------------------------------------------------------------------ the norm
def check_normed(q, s, y, rows, dim):
    """Codes and packed scales of the exact normed rows y."""
    sb = F.unpack(s, rows, dim)
    a = F.block_amax(y)
    assert (a * (1 - PRE) <= 448 * 2.0 ** (sb - 127)).all()
    assert ((a * (1 + PRE) > 448 * 2.0 ** (sb - 128.0)) | (sb == 0)).all()
    v = F.values(q.reshape(rows, dim), sb)
    assert (np.abs(v - y) <= F.half_step(y, sb) + PRE * np.abs(y)).all()


@pytest.mark.parametrize("rows,dim", [(1, 16), (1, 4096), (7, 128), (130, 1040), (33, 4096),
                                      (65, 4112), (9, 12288), (3, 16400), (5000, 272),
                                      (1200, 4096)])
@pytest.mark.parametrize("form", ["plain", "add", "add_in_place", "add_unstored", "copy"])
def test_norm(ops, rows, dim, form):
    x = activations(rows, dim, 1)
    d = activations(rows, dim, 2) if form.startswith("add") else None
    w = bf16_round(randn((2, dim), 3, 0.2, 1.0))
    segs = [(0, rows // 2, 1), (rows // 2, rows, 0)]
    xd, dd = dev_bf16(x), None if d is None else dev_bf16(d)
    out = {"plain": None, "add": torch.empty_like(xd), "add_in_place": xd, "add_unstored": None,
           "copy": torch.empty_like(xd)}[form]
    q, s = u8(rows * dim), u8(F.scale_bytes(rows, dim))
    ops.mot_add_rms_norm_quant_fp8(xd, dd, dev_bf16(w), segs, out, q, s, rows, dim, 1e-6)
    t = x if d is None else bf16_round(x + d)
    if out is not None:
        assert np.array_equal(host(out), t)
    t = t.astype(np.float64)
    n = t / np.sqrt((t * t).mean(1, keepdims=True) + np.float32(1e-6))
    y, = by_expert(segs, rows, lambda r, e: (n[r] * w[e],))
    check_normed(host(q), host(s), y, rows, dim)
    if form == "add_in_place":
        assert np.array_equal(host(dd), d)


def test_norm_of_zeros_and_not_finite(ops):
    x = activations(4, 256, 5)
    x[1] = 0
    x[2, 3] = np.nan
    x[3, 5] = np.inf
    w = np.ones((1, 256), np.float32)
    q, s = u8(4 * 256), u8(F.scale_bytes(4, 256))
    ops.mot_add_rms_norm_quant_fp8(dev_bf16(x), None, dev_bf16(w), None, None, q, s, 4, 256, 1e-6)
    got = host(q).reshape(4, 256)
    assert (got[1] == 0).all() and (F.unpack(host(s), 4, 256)[1] == 0).all()
    assert ((got[2] & 0x7F) == 0x7F).all() and (got[3, 5] & 0x7F) == 0x7F
    assert ((got[0] & 0x7F) != 0x7F).all()


# ------------------------------------------------------------------ the product
SHAPES = [(1, 16, 1), (1, 4096, 256), (2, 128, 40), (7, 528, 129), (16, 512, 128), (17, 4096, 320),
          (33, 1040, 1000), (64, 640, 768), (65, 256, 256), (100, 12288, 136), (128, 1152, 512),
          (129, 512, 264), (200, 1552, 513), (256, 2048, 1024), (300, 144, 77), (385, 4096, 640),
          (700, 384, 2048)]


def segments_of(M, kind):
    return {"one": None, "two": [(0, M // 3, 1), (M // 3, M, 0)],
            "many": [(0, M // 5, 0), (M // 5, M // 5, 1), (M // 5, M // 2, 1), (M // 2, M, 0)]}[kind]


def run_linear(ops, M, K, N, segs, epi, seed=11, bias=False):
    E = 2
    xq, xs = quantised(M, K, seed)
    W, wq, ws = weights(E, N, K, seed + 1)
    r = bf16_round(randn((M, N), seed + 5))
    b = bf16_round(randn((E, N), seed + 6, 0.5)) if bias else None
    extra = 3 * N
    y = torch.full((M * N + extra,), 77.0, device="cuda",
                   dtype=torch.float32 if epi == F32 else torch.bfloat16)
    ops.mot_linear_fp8(dev_u8(xq), dev_u8(F.pack(xs, K)), wq, ws, segs, y, M, K, N, epilogue=epi,
                       resid=dev_bf16(r) if epi == RESID else None,
                       bias=dev_bf16(b) if bias else None)
    ops.sync()
    got = host(y)
    assert (got[M * N:] == 77).all()          # rows behind the last keep what they held

    def want(rows, e):
        return F.product(xq[rows], xs[rows], *W[e]) + (
            np.broadcast_to(b[e] if bias else np.zeros(N), (rows.stop - rows.start, N)),)
    p, S, bb = by_expert(segs, M, want)
    t = p + bb + (r if epi == RESID else 0)
    tol = F.sum_error(S, K) + 2.0 ** -23 * (np.abs(t) + np.abs(p))
    tol += np.abs(t) * (2.0 ** -24 if epi == F32 else 2.0 ** -8)
    err = np.abs(got[:M * N].reshape(M, N) - t)
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()
    return err, S


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("segs", ["one", "two", "many"])
def test_linear(ops, M, K, N, segs):
    run_linear(ops, M, K, N, segments_of(M, segs), STORE)


def test_linear_empty_and_single_row_segments(ops):
    """Segments of no rows at either end and in the middle, and of one row."""
    for M in (3, 70, 150, 600):
        run_linear(ops, M, 272, 384, [(0, 0, 1), (0, 1, 0), (1, 1, 1), (1, M - 1, 1),
                                      (M - 1, M, 0), (M, M, 1)], RESID)


def test_linear_unaligned_outputs(ops):
    """y, residual and bias off every 16-byte boundary."""
    for M, N in [(5, 256), (70, 512), (300, 512), (2100, 512)]:
        K, E = 256, 1
        xq, xs = quantised(M, K, 15)
        W, wq, ws = weights(E, N, K, 16)
        r, b = dev_bf16(randn(M * N + 1, 17))[1:], dev_bf16(randn(N + 1, 18))[1:]
        args = (dev_u8(xq), dev_u8(F.pack(xs, K)), wq, ws, None)
        for kw in (dict(epilogue=RESID, resid=r), dict(bias=b)):
            y = torch.zeros(M * N + 1, dtype=torch.bfloat16, device="cuda")
            ops.mot_linear_fp8(*args, y[1:], M, K, N, **kw)
            kw = {k: v.clone() if torch.is_tensor(v) else v for k, v in kw.items()}
            want = torch.empty(M * N, dtype=torch.bfloat16, device="cuda")
            ops.mot_linear_fp8(*args, want, M, K, N, **kw)
            assert torch.equal(y[1:], want) and y[0] == 0


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_residual(ops, M, K, N):
    run_linear(ops, M, K, N, segments_of(M, "two"), RESID)


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_f32(ops, M, K, N):
    run_linear(ops, M, K, N, segments_of(M, "two"), F32, bias=True)


@pytest.mark.parametrize("M", [5, 300])
def test_linear_bias(ops, M):
    run_linear(ops, M, 256, 200, segments_of(M, "two"), STORE, bias=True)


def test_linear_scales_apply_per_block(ops):
    """Scales of very different sizes in neighbouring blocks and rows (2^-40 to
    2^40): each block's product is scaled by its own pair."""
    M, K, N = 200, 1152, 384
    r = np.random.default_rng(3)
    xq, wq = r.integers(0, 0x7F, (M, K)).astype(np.uint8), r.integers(0, 0x7F, (N, K)).astype(np.uint8)
    xs = r.integers(87, 168, (M, 9))
    ws = np.repeat(r.integers(87, 168, (N // 128, 9)), 128, 0)
    for m in (3, 100, 200):
        y = torch.empty(m, N, dtype=torch.float32, device="cuda")
        ops.mot_linear_fp8(dev_u8(xq[:m]), dev_u8(F.pack(xs[:m], K)), dev_u8(wq[None]),
                           dev_u8(F.pack(ws, K)), None, y, m, K, N, epilogue=F32)
        p, S = F.product(xq[:m], xs[:m], wq, ws)
        assert (np.abs(host(y) - p) <= F.sum_error(S, K) + 2.0 ** -24 * np.abs(p)).all()


def test_linear_scales_per_weight_row(ops):
    """The products read a scale for every weight row: rows need not share it."""
    K, N = 512, 256
    r = np.random.default_rng(4)
    wq = r.integers(0, 0x7F, (N, K)).astype(np.uint8)
    ws = r.integers(110, 130, (N, 4))
    for M in (9, 260):
        xq, xs = quantised(M, K, 21)
        y = torch.empty(M, N, dtype=torch.float32, device="cuda")
        ops.mot_linear_fp8(dev_u8(xq), dev_u8(F.pack(xs, K)), dev_u8(wq[None]),
                           dev_u8(F.pack(ws, K)), None, y, M, K, N, epilogue=F32)
        p, S = F.product(xq, xs, wq, ws)
        assert (np.abs(host(y) - p) <= F.sum_error(S, K) + 2.0 ** -24 * np.abs(p)).all()


def test_linear_residual_in_place(ops):
    for M in (19, 300):
        K, N = 512, 384
        xq, xs = quantised(M, K, 31)
        W, wq, ws = weights(2, N, K, 32)
        rd = dev_bf16(randn((M, N), 33))
        y = torch.empty_like(rd)
        args = (dev_u8(xq), dev_u8(F.pack(xs, K)), wq, ws, segments_of(M, "two"))
        ops.mot_linear_fp8(*args, y, M, K, N, epilogue=RESID, resid=rd)
        ops.mot_linear_fp8(*args, rd, M, K, N, epilogue=RESID, resid=rd)
        assert torch.equal(y, rd)


def test_nan_row_stays_in_its_row(ops):
    for M in (6, 140, 300):
        K, N = 384, 256
        xq, xs = quantised(M, K, 41)
        xq[M - 2, 200] = 0x7F
        W, wq, ws = weights(1, N, K, 42)
        y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        ops.mot_linear_fp8(dev_u8(xq), dev_u8(F.pack(xs, K)), wq, ws, None, y, M, K, N)
        bad = np.isnan(host(y))
        assert bad[M - 2].all() and bad.sum() == N


def test_repeats_bit_identical(ops):
    for M, K, N in [(3, 4096, 512), (70, 2048, 1024), (300, 1024, 768)]:
        xq, xs = quantised(M, K, 51)
        W, wq, ws = weights(2, N, K, 52)
        outs = []
        for _ in range(3):
            y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
            ops.mot_linear_fp8(dev_u8(xq), dev_u8(F.pack(xs, K)), wq, ws, segments_of(M, "two"), y,
                               M, K, N)
            outs.append(y)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def torch_values(q, s, rows, cols):
    """A quantised tensor's values in float64 on the device."""
    at = torch.from_numpy(F.places(rows, cols)).cuda()
    f = torch.exp2(s[at].double() - 127).repeat_interleave(128, 1)[:, :cols]
    return q.view(torch.float8_e4m3fn).reshape(rows, cols).double() * f


def random_quantised(ops, rows, cols, seed, std):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (std * torch.randn(rows, cols, generator=g, device="cuda")).bfloat16()
    q, s = u8(rows * cols), ops.fp8_scale(rows, cols)
    ops.quant_rows_fp8(x, q, s, rows, cols)
    return q, s, torch_values(q, s, rows, cols)


@pytest.mark.parametrize("M,K,N,segs", [
    (2100, 640, 4096, [(0, 2100, 0)]),                         # a part-empty last round: half-width tiles
    (1800, 512, 6144, [(0, 77, 0), (77, 1800, 1)]),            # several rounds, an odd boundary
    (3000, 384, 2176, [(0, 250, 1), (250, 251, 0), (251, 1600, 1), (1600, 3000, 0)]),
    (1030, 272, 8192, [(0, 320, 0), (320, 1030, 1)]),
    # fewer tiles than pairs: two, three and four pairs a tile
    (512, 2064, 4096, [(0, 512, 0)]), (300, 12288, 2048, [(0, 300, 1)]),
    (400, 8192, 1536, [(0, 100, 0), (100, 400, 1)]), (450, 2304, 4000, [(0, 130, 1), (130, 450, 0)]),
    (1100, 12288, 1024, [(0, 1100, 0)]), (1030, 2320, 1500, [(0, 70, 1), (70, 1030, 0)]),
    (1300, 4096, 520, [(0, 700, 1), (700, 700, 0), (700, 1300, 0)]),
    (2100, 4096, 512, [(0, 2100, 1)]), (2200, 2320, 700, [(0, 70, 1), (70, 2200, 0)]),
    (2500, 1168, 256, [(0, 700, 1), (700, 700, 0), (700, 2500, 0)])])
@pytest.mark.parametrize("epi", [STORE, RESID, SWIGLU])
def test_many_tiles(ops, M, K, N, segs, epi):
    """More tiles than CTA pairs: the accumulators' shared columns, the scale
    sets' turns over tiles of odd group counts, and the last round."""
    if epi == SWIGLU:
        N -= N % 256                                            # whole gate and up blocks
    xq, xs, x = random_quantised(ops, M, K, 1, 1.0)
    W = [random_quantised(ops, N, K, 2 + e, 0.05) for e in range(2)]
    wq, ws = torch.cat([w[0] for w in W]).view(2, N, K), torch.cat([w[1] for w in W])
    cols = N // 2 if epi == SWIGLU else N
    r = torch.randn(M, N, device="cuda").bfloat16() if epi == RESID else None
    y = torch.empty(M, cols, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(xq, xs, wq, ws, segs, y, M, K, N, epilogue=epi, resid=r)
    ops.sync()
    t = torch.cat([x[a:b] @ W[e][2].T for a, b, e in segs])
    S = torch.cat([x[a:b].abs() @ W[e][2].abs().T for a, b, e in segs])
    err = F.sum_error(S, K) + 2.0 ** -23 * t.abs()
    if epi == SWIGLU:
        g, u = t.view(M, -1, 2, 128).unbind(2)
        eg, eu = err.view(M, -1, 2, 128).unbind(2)
        silu = g / (1 + torch.exp(-g))
        t = (silu * u).flatten(1)
        err = (1.1 * eg * (u.abs() + eu) + silu.abs() * eu).flatten(1) + 2.0 ** -20 * t.abs()
    if epi == RESID:
        t = t + r.double()
        err = err + 2.0 ** -23 * t.abs()
    assert ((y.double() - t).abs() <= err + 2.0 ** -8 * t.abs()).all()


# Units of some hundred rows: their first rows rounded down to 64, their heights
# to 32, so boundaries lie beside both; the last CTA past the columns; a last k-block alone
# in its stage; the k-blocks of a tile split over up to four pairs
EIGHT = [(0, 63, 0), (63, 64, 1), (64, 65, 0), (65, 161, 1), (161, 257, 0), (257, 257, 1),
         (257, 450, 1), (450, 1024, 0)]


@pytest.mark.parametrize("M,K,N,segs", [
    (65, 16, 128, None), (90, 656, 100, None), (130, 784, 128, [(0, 1, 0), (1, 130, 1)]),
    (66, 272, 129, [(0, 65, 1), (65, 66, 0)]),
    (96, 400, 384, [(0, 32, 0), (32, 96, 1)]), (97, 1168, 640, [(0, 31, 1), (31, 97, 0)]),
    (160, 640, 136, [(0, 64, 0), (64, 160, 1)]), (193, 4240, 256, [(0, 127, 1), (127, 193, 0)]),
    (257, 8208, 392, None), (320, 2176, 260, [(0, 1, 1), (1, 320, 0)]),
    (1000, 528, 768, [(0, 77, 0), (77, 1000, 1)]), (1024, 272, 1160, EIGHT), (1024, 1296, 513, None),
    (1025, 1296, 513, None),
    # more rows, of columns that leave them off 32 bytes or end inside a run of 32
    (1100, 144, 1000, [(0, 300, 1), (300, 1100, 0)]), (1301, 272, 777, [(0, 33, 0), (33, 1301, 1)]),
    (1200, 144, 272, None), (2100, 144, 1000, [(0, 300, 1), (300, 2100, 0)]),
    (2201, 272, 777, [(0, 33, 0), (33, 2201, 1)]), (2048, 144, 272, None), (2049, 16, 272, None)])
@pytest.mark.parametrize("epi", [STORE, RESID, F32])
def test_linear_units(ops, M, K, N, segs, epi):
    run_linear(ops, M, K, N, segs, epi, bias=epi != RESID)


# ------------------------------------------------------------------ SwiGLU
def swiglu_ref(xq, xs, W, M, K, segs):
    """silu(gate) * up of every row, and what f32 sums may be off by there."""
    p, S = by_expert(segs, M, lambda r, e: F.product(xq[r], xs[r], *W[e]))
    p, S = (a.reshape(M, -1, 2, 128).transpose(2, 0, 1, 3).reshape(2, M, -1) for a in (p, S))
    g, u = p
    eg, eu = F.sum_error(S, K) + 2.0 ** -23 * np.abs(p)
    silu = g / (1 + np.exp(-g))
    # |silu'| <= 1.1; the exponential, its sum, the division and the product
    # are each within a few units of 2^-23 (2^-20 together)
    err = 1.1 * eg * (np.abs(u) + eu) + np.abs(silu) * eu + 2.0 ** -20 * np.abs(silu * u)
    return silu * u, err


@pytest.mark.parametrize("M,K,I", [(1, 4096, 128), (1, 16, 256), (9, 640, 384), (33, 1040, 128),
                                   (65, 512, 640), (128, 256, 256), (130, 144, 256), (300, 1024, 640),
                                   (70, 4240, 128), (190, 400, 384), (333, 1168, 896),
                                   (1024, 272, 384)])
@pytest.mark.parametrize("segs", ["one", "many"])
def test_swiglu(ops, M, K, I, segs):
    segs = segments_of(M, segs)
    xq, xs = quantised(M, K, 61)
    W, wq, ws = weights(2, 2 * I, K, 62)
    xd, sd = dev_u8(xq), dev_u8(F.pack(xs, K))
    y = torch.full((M * I + I,), 55.0, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(xd, sd, wq, ws, segs, y, M, K, 2 * I, epilogue=SWIGLU)
    yq, sy = u8(M * I + I), u8(F.scale_bytes(M, I))
    ops.mot_swiglu_fp8(xd, sd, wq, ws, segs, yq, sy, M, K, 2 * I)
    ops.sync()
    want, err = swiglu_ref(xq, xs, W, M, K, segs)
    got = host(y)
    assert (got[M * I:] == 55).all()
    assert (np.abs(got[:M * I].reshape(M, I) - want) <= err + 2.0 ** -8 * np.abs(want)).all()
    q, s = host(yq), host(sy)
    assert (q[M * I:] == 0xAA).all()
    free = np.ones(s.size, bool)
    free[F.places(M, I)] = False
    assert (s[free] == 0xAA).all()
    sb = F.unpack(s, M, I)
    a, ea = F.block_amax(want), F.block_amax(err)
    assert (a - ea <= 448 * 2.0 ** (sb - 127)).all()
    assert ((a + ea > 448 * 2.0 ** (sb - 128.0)) | (sb == 0)).all()
    # the error before rounding also moves the step: half a step at |want| + err
    v = F.values(q[:M * I].reshape(M, I), sb)
    assert (np.abs(v - want) <= F.half_step(np.abs(want) + err, sb) + err).all()


@pytest.mark.parametrize("M", [20, 200, 2100])
def test_swiglu_unaligned_output(ops, M):
    K, I = 256, 384
    xq, xs = quantised(M, K, 71)
    W, wq, ws = weights(1, 2 * I, K, 72)
    args = (dev_u8(xq), dev_u8(F.pack(xs, K)), wq, ws, None)
    want = torch.empty(M * I, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(*args, want, M, K, 2 * I, epilogue=SWIGLU)
    y = torch.full((M * I + 2,), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(*args, y[1:], M, K, 2 * I, epilogue=SWIGLU)
    assert torch.equal(y[1:-1], want) and y[0] == 5 and y[-1] == 5


# ------------------------------------------------------------------ together
def ffn_inputs(rows, h, i, seed):
    W, gu, gs = weights(2, 2 * i, h, seed)
    D, dn, ds = weights(2, h, i, seed + 10)
    return dict(x=dev_bf16(activations(rows, h, seed + 20)), d=dev_bf16(activations(rows, h, seed + 21)),
                w=dev_bf16(randn((2, h), seed + 22, 0.1, 1.0)), gu=gu, gs=gs, dn=dn, ds=ds)


def ffn_steps(ops, t, segs, rows, h, i, add):
    s = torch.empty_like(t["x"])
    q, sc = u8(rows * h), u8(F.scale_bytes(rows, h))
    ops.mot_add_rms_norm_quant_fp8(t["x"], t["d"] if add else None, t["w"], segs, s, q, sc, rows, h,
                                   1e-6)
    hq, hs = u8(rows * i), u8(F.scale_bytes(rows, i))
    ops.mot_swiglu_fp8(q, sc, t["gu"], t["gs"], segs, hq, hs, rows, h, 2 * i)
    y = torch.empty_like(s)
    ops.mot_linear_fp8(hq, hs, t["dn"], t["ds"], segs, y, rows, i, h, epilogue=RESID, resid=s)
    return y


@pytest.mark.parametrize("rows,h,i", [(1, 4096, 512), (5, 272, 128), (64, 1024, 384),
                                      (333, 528, 640)])
@pytest.mark.parametrize("add", [True, False])
def test_ffn_is_its_steps(ops, rows, h, i, add):
    """The feed-forward block equals its three operators run one by one, out of
    place and in place."""
    t = ffn_inputs(rows, h, i, 71)
    segs = segments_of(rows, "two")
    want = ffn_steps(ops, t, segs, rows, h, i, add)
    ws = ops.ffn_fp8_workspace(rows, h, i)
    y = torch.empty_like(t["x"])
    x0 = t["x"].clone()
    rest = (t["w"], t["gu"], t["gs"], t["dn"], t["ds"], segs)
    ops.mot_ffn_fp8(t["x"], t["d"] if add else None, *rest, y, ws, rows, h, i, 1e-6)
    assert torch.equal(t["x"], x0)
    if add:                                           # over the residual's addend
        d = t["d"].clone()
        ops.mot_ffn_fp8(t["x"], d, *rest, d, ws, rows, h, i, 1e-6)
        assert torch.equal(d, want)
    ops.mot_ffn_fp8(t["x"], t["d"] if add else None, *rest, t["x"], ws, rows, h, i, 1e-6)
    ops.sync()
    assert torch.equal(y, want) and torch.equal(t["x"], want)
    assert torch.isfinite(y).all()


def test_ffn_close_to_unquantised(ops):
    """Against float64 without any rounding to 8 bits. Every factor of a
    product is off by at most 2^-4 of itself (its block's smallest values by
    less than 2^-10 of a step, far below), independently, so a product's
    relative error in the 2-norm stays under 2^-4 * sqrt(2) for one layer of
    products and under twice that through two and the activation."""
    rows, h, i = 150, 512, 256
    rng = np.random.default_rng(5)
    x, d = bf16_round(rng.normal(size=(rows, h))), bf16_round(rng.normal(size=(rows, h)))
    g, dn = bf16_round(0.05 * rng.normal(size=(2 * i, h))), bf16_round(0.05 * rng.normal(size=(h, i)))
    gq, gs, dq, ds = u8(g.size), ops.fp8_scale(2 * i, h), u8(dn.size), ops.fp8_scale(h, i)
    ops.quant_weight_fp8(dev_bf16(g), gq, gs, 1, 2 * i, h)
    ops.quant_weight_fp8(dev_bf16(dn), dq, ds, 1, h, i)
    y = torch.empty(rows, h, dtype=torch.bfloat16, device="cuda")
    w = np.ones((1, h), np.float32)
    ops.mot_ffn_fp8(dev_bf16(x), dev_bf16(d), dev_bf16(w), gq[None], gs, dq[None], ds, None, y,
                    ops.ffn_fp8_workspace(rows, h, i), rows, h, i, 1e-6)
    s = bf16_round(x + d).astype(np.float64)
    n = s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-6)
    p = (n @ g.T).reshape(rows, -1, 2, 128)
    gate, up = p[:, :, 0].reshape(rows, i), p[:, :, 1].reshape(rows, i)
    u = (gate / (1 + np.exp(-gate)) * up) @ dn.T
    got = host(y) - s
    assert np.linalg.norm(got - u) / np.linalg.norm(u) < 2 * np.sqrt(2) * 2.0 ** -4


def test_other_stream_and_graph(ops):
    """On a side stream, and captured into a graph and replayed on new inputs;
    two graphs with workspaces of their own, replayed in turn."""
    for rows in (3, 300, 1500, 2100):
        h, i = 512, 256
        segs = segments_of(rows, "two")
        t = ffn_inputs(rows, h, i, 81)
        rest = (t["w"], t["gu"], t["gs"], t["dn"], t["ds"], segs)
        new = [dev_bf16(activations(rows, h, 90 + k)) for k in range(2)]
        wss = [ops.ffn_fp8_workspace(rows, h, i) for _ in range(2)]
        want = []
        for x in new:
            y = torch.empty_like(x)
            ops.mot_ffn_fp8(x, t["d"], *rest, y, wss[0], rows, h, i, 1e-6)
            want.append(y)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        y = torch.empty_like(t["x"])
        with torch.cuda.stream(side):
            ops.mot_ffn_fp8(new[0], t["d"], *rest, y, wss[0], rows, h, i, 1e-6)
        side.synchronize()
        assert torch.equal(y, want[0])
        graphs, outs = [], []
        for k in range(2):
            out = torch.empty_like(t["x"])
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                ops.mot_ffn_fp8(t["x"], t["d"], *rest, out, wss[k], rows, h, i, 1e-6)
            graphs.append(g)
            outs.append(out)
        for k in (0, 1, 0):
            t["x"].copy_(new[k])
            graphs[k].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[k], want[k])


def test_refusals_in_python(ops):
    from u15b200 import U15Error
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    q, s = u8(512), u8(512)
    for bad in [lambda: ops.quant_rows_fp8(x.float(), q, s, 4, 128),
                lambda: ops.quant_rows_fp8(x, q, s[:100], 4, 128),
                lambda: ops.quant_rows_fp8(x, q[:511], s, 4, 128),
                lambda: ops.quant_rows_fp8(x.t(), q, s, 4, 128),
                lambda: ops.quant_rows_fp8(x.cpu(), q, s, 4, 128),
                lambda: ops.quant_rows_fp8(x[:, 8:].contiguous(), q, s, 4, 120),
                lambda: ops.dequant_fp8(q, s, x, 5, 128)]:
        with pytest.raises(U15Error):
            bad()
    empty = torch.empty(0, 128, dtype=torch.bfloat16, device="cuda")
    ops.quant_rows_fp8(empty, q, s, 0, 128)          # no rows: nothing to do
    assert (host(q) == 0xAA).all()
