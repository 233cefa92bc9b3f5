"""The products' forms for more than 2048 rows, CTA pairs of their own and
several pairs a tile, against the format restated in float64: the quantised
SwiGLU rows, residuals in place, NaN, scales of every row, f32 outputs, and the
feed-forward block and the layer that run them.

Sizes: 256 x 256 tiles on at most 74 pairs. PERSISTENT holds more tiles than
that, so that pairs take a second and a later one; SPLIT so few, over a long K,
that two, three or four pairs share a tile.
"""
import numpy as np
import pytest

import fp8_util as F
from gpu_util import bf16_round, dev_bf16, host, randn, torch
from test_gpu_fp8 import (F32, RESID, STORE, SWIGLU, activations, by_expert, check_normed, dev_u8,
                          ffn_inputs, ffn_steps, quantised, random_quantised, run_linear,
                          torch_values, u8)

pytestmark = pytest.mark.gpu
PERSISTENT = [(2100, 640, 4096, [(0, 2100, 1)]),
              (2305, 272, 8192, [(0, 77, 0), (77, 2305, 1)]),
              (2816, 1168, 2304, [(0, 250, 1), (250, 251, 0), (251, 251, 1), (251, 2816, 0)]),
              (4096, 16, 4096, [(0, 512, 0), (512, 4096, 1)])]
SPLIT = [(2100, 4096, 512, [(0, 2100, 1)]),                                    # four
         (2200, 2320, 512, [(0, 70, 1), (70, 2200, 0)]),                       # three
         (2500, 4096, 256, [(0, 700, 1), (700, 700, 0), (700, 2500, 0)]),      # four
         (2300, 12288, 768, [(0, 1, 0), (1, 2300, 1)])]                        # two


@pytest.fixture(scope="module")
def ops():
    import u15b200
    return u15b200.CudaOps(0)


def inputs(ops, M, K, N, seed=1):
    """xq, xs, x in float64, stacked weights and scales, each expert's values."""
    x = random_quantised(ops, M, K, seed, 1.0)
    W = [random_quantised(ops, N, K, seed + 1 + e, 0.05) for e in range(2)]
    wq, ws = torch.cat([w[0] for w in W]).view(2, N, K), torch.cat([w[1] for w in W])
    return *x, wq, ws, [w[2] for w in W]


def products(x, W, segs):
    """The exact products and the sums of their terms' magnitudes."""
    return (torch.cat([x[a:b] @ W[e].T for a, b, e in segs]),
            torch.cat([x[a:b].abs() @ W[e].abs().T for a, b, e in segs]))


def check_swiglu(yq, sy, x, W, segs, K):
    """Codes and scale bytes of the quantised SwiGLU rows, by the bounds that
    test_gpu_fp8.test_swiglu derives."""
    M = x.shape[0]
    p, S = (t.view(M, -1, 2, 128) for t in products(x, W, segs))
    (g, u), (eg, eu) = p.unbind(2), (F.sum_error(S, K) + 2.0 ** -23 * p.abs()).unbind(2)
    silu = g / (1 + torch.exp(-g))
    want = silu * u
    err = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu + 2.0 ** -20 * want.abs()
    want, err = (t.flatten(1).cpu().numpy() for t in (want, err))
    sb = F.unpack(host(sy), M, want.shape[1])
    a, ea = F.block_amax(want), F.block_amax(err)
    assert (a - ea <= 448 * 2.0 ** (sb - 127)).all()
    assert ((a + ea > 448 * 2.0 ** (sb - 128.0)) | (sb == 0)).all()
    v = F.values(host(yq)[:want.size].reshape(want.shape), sb)
    assert (np.abs(v - want) <= F.half_step(np.abs(want) + err, sb) + err).all()


@pytest.mark.parametrize("M,K,N,segs", PERSISTENT + SPLIT)
def test_swiglu_quantised(ops, M, K, N, segs):
    xq, xs, x, wq, ws, W = inputs(ops, M, K, N)
    n = N // 2
    yq, sy = u8(M * n + n), u8(F.scale_bytes(M, n))
    ops.mot_swiglu_fp8(xq, xs, wq, ws, segs, yq, sy, M, K, N)
    ops.sync()
    check_swiglu(yq, sy, x, W, segs, K)
    q, s = host(yq), host(sy)
    assert (q[M * n:] == 0xAA).all()
    free = np.ones(s.size, bool)
    free[F.places(M, n)] = False
    assert (s[free] == 0xAA).all()


@pytest.mark.parametrize("M,K,N,segs", [PERSISTENT[1], SPLIT[0]])
def test_swiglu_quantised_off_32_bytes(ops, M, K, N, segs):
    """Rows that begin on 16 bytes, not on 32."""
    xq, xs, _, wq, ws, _ = inputs(ops, M, K, N)
    out = []
    for off in (0, 16):
        yq, sy = u8(M * N // 2 + 32), u8(F.scale_bytes(M, N // 2))
        ops.mot_swiglu_fp8(xq, xs, wq, ws, segs, yq[off:], sy, M, K, N)
        assert (yq[:off] == 0xAA).all() and (yq[off + M * N // 2:] == 0xAA).all()
        out.append((yq[off:off + M * N // 2], sy))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


@pytest.mark.parametrize("M,K,N,segs", [(2100, 272, 4100, [(0, 77, 0), (77, 2100, 1)]),
                                        (2200, 2320, 700, [(0, 70, 1), (70, 2200, 0)]),
                                        (2100, 4096, 512, [(0, 2100, 1)]),
                                        (2500, 4096, 256, [(0, 700, 1), (700, 2500, 0)])])
@pytest.mark.parametrize("epi", [STORE, F32])
def test_linear_bias_and_f32(ops, M, K, N, segs, epi):
    run_linear(ops, M, K, N, segs, epi, bias=True)


@pytest.mark.parametrize("M,K,N,segs", [PERSISTENT[0], PERSISTENT[1], SPLIT[0], SPLIT[1],
                                        (2201, 272, 777, [(0, 33, 0), (33, 2201, 1)]),
                                        (2200, 2320, 700, [(0, 70, 1), (70, 2200, 0)])])
def test_residual_in_place(ops, M, K, N, segs):
    xq, xs, x, wq, ws, W = inputs(ops, M, K, N)
    r = dev_bf16(randn((M, N), 33))
    y = r.clone()
    ops.mot_linear_fp8(xq, xs, wq, ws, segs, y, M, K, N, epilogue=RESID, resid=y)
    ops.sync()
    p, S = products(x, W, segs)
    t = p + r.double()
    tol = F.sum_error(S, K) + 2.0 ** -23 * (t.abs() + p.abs()) + 2.0 ** -8 * t.abs()
    assert ((y.double() - t).abs() <= tol).all()


@pytest.mark.parametrize("M,K,N,segs", [PERSISTENT[1], SPLIT[0]])
def test_nan_stays_in_its_row_and_column(ops, M, K, N, segs):
    xq, xs, _, wq, ws, _ = inputs(ops, M, K, N)
    xq, wq = xq.clone().view(M, K), wq.clone()
    for row in (0, M - 2):
        xq[row, K // 2] = 0x7F
    wq[1, 5, K - 1] = 0xFF
    y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(xq, xs, wq, ws, segs, y, M, K, N)
    want = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    want[[0, M - 2]] = True
    for a, b, e in segs:
        if e == 1:
            want[a:b, 5] = True
    assert torch.equal(torch.isnan(y), want)


@pytest.mark.parametrize("M,K,N", [(2100, 1040, 4096), (2100, 4096, 512)])
def test_scales_of_every_row_and_block(ops, M, K, N):
    """Weight rows need not share a scale, and neighbouring blocks' differ by up to 2^80."""
    r = np.random.default_rng(3)
    nb = -(-K // 128)
    q = [dev_u8(r.integers(0, 0x7F, (n, K))) for n in (M, N)]
    s = [dev_u8(F.pack(r.integers(87, 168, (n, nb)), K)) for n in (M, N)]
    x, w = (torch_values(a.flatten(), b, n, K) for a, b, n in zip(q, s, (M, N)))
    y = torch.empty(M, N, dtype=torch.float32, device="cuda")
    ops.mot_linear_fp8(q[0], s[0], q[1][None], s[1], None, y, M, K, N, epilogue=F32)
    p, S = products(x, [w], [(0, M, 0)])
    assert ((y.double() - p).abs() <= F.sum_error(S, K) + 2.0 ** -24 * p.abs()).all()


def test_repeats_and_calls_side_by_side(ops):
    """The same bits again, alone and beside calls of the other forms on other streams."""
    cases = [PERSISTENT[0], SPLIT[0], (3, 2048, 1024, [(0, 3, 0)]), (300, 1024, 768, [(0, 300, 1)]),
             SPLIT[3]]
    streams = [torch.cuda.Stream() for _ in cases]
    made, want = [], []
    for M, K, N, segs in cases:
        xq, xs, _, wq, ws, _ = inputs(ops, M, K, N, seed=M)
        made.append((xq, xs, wq, ws, segs))
        y, yq, sy = (torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), u8(M * N // 2),
                     u8(F.scale_bytes(M, N // 2)))
        ops.mot_linear_fp8(*made[-1], y, M, K, N)
        ops.mot_swiglu_fp8(*made[-1], yq, sy, M, K, N)
        want.append((y, yq, sy))
    torch.cuda.synchronize()
    out = [[torch.empty_like(y), torch.empty_like(q), torch.full_like(s, 0xAA)] for y, q, s in want]
    for _ in range(10):
        for st, a, (y, yq, sy), (M, K, N, _) in zip(streams, made, out, cases):
            with torch.cuda.stream(st):
                ops.mot_linear_fp8(*a, y, M, K, N)
                ops.mot_swiglu_fp8(*a, yq, sy, M, K, N)
    torch.cuda.synchronize()
    ops.sync()
    for a, b in zip(out, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("rows,h,i", [(2305, 512, 2048), (2100, 2320, 256)])
def test_feed_forward_step_by_step(ops, rows, h, i):
    """Each operator of the block against float64 on the codes that it was
    given, and the block equal to them, again and in place."""
    t = ffn_inputs(rows, h, i, 71)
    segs = [(0, 333, 1), (333, rows, 0)]
    s = torch.empty_like(t["x"])
    q, sc = u8(rows * h), u8(F.scale_bytes(rows, h))
    ops.mot_add_rms_norm_quant_fp8(t["x"], t["d"], t["w"], segs, s, q, sc, rows, h, 1e-6)
    assert torch.equal(s, (t["x"].float() + t["d"].float()).bfloat16())
    v = host(s).astype(np.float64)
    n = v / np.sqrt((v * v).mean(1, keepdims=True) + np.float32(1e-6))
    w = host(t["w"]).astype(np.float64)
    y, = by_expert(segs, rows, lambda r, e: (n[r] * w[e],))
    check_normed(host(q), host(sc), y, rows, h)
    hq, hs = u8(rows * i), u8(F.scale_bytes(rows, i))
    ops.mot_swiglu_fp8(q, sc, t["gu"], t["gs"], segs, hq, hs, rows, h, 2 * i)

    def experts(q_, s_, n_, k_):
        return [torch_values(a.flatten(), b, n_, k_) for a, b in zip(q_, s_.view(2, -1))]
    check_swiglu(hq, hs, torch_values(q, sc, rows, h), experts(t["gu"], t["gs"], 2 * i, h), segs, h)
    p, S = products(torch_values(hq, hs, rows, i), experts(t["dn"], t["ds"], h, i), segs)
    want = ffn_steps(ops, t, segs, rows, h, i, True)
    r = p + s.double()
    tol = F.sum_error(S, i) + 2.0 ** -23 * (r.abs() + p.abs()) + 2.0 ** -8 * r.abs()
    assert ((want.double() - r).abs() <= tol).all()
    ws = ops.ffn_fp8_workspace(rows, h, i)
    rest = (t["w"], t["gu"], t["gs"], t["dn"], t["ds"], segs)
    for _ in range(3):
        out = torch.empty_like(s)
        ops.mot_ffn_fp8(t["x"], t["d"], *rest, out, ws, rows, h, i, 1e-6)
        assert torch.equal(out, want)
    ops.mot_ffn_fp8(t["x"], t["d"], *rest, t["x"], ws, rows, h, i, 1e-6)
    ops.sync()
    assert torch.equal(t["x"], want)


class Layer:
    """A layer whose passes of T rows run the persistent form: 2048 inner columns."""
    H, NH, KV, I, T = 512, 4, 1, 2048, 2305
    SEGS = [(0, 333, 1), (333, 2305, 0)]

    def __init__(self, zero=()):
        import u15b200
        r = np.random.default_rng(7)
        H, NH, KV, I = self.H, self.NH, self.KV, self.I
        shapes = {"q_proj": (NH * 128, H), "k_proj": (KV * 128, H), "v_proj": (KV * 128, H),
                  "o_proj": (H, NH * 128), "gate_proj": (I, H), "up_proj": (I, H),
                  "down_proj": (H, I)}
        self.W = []
        self.m = u15b200.Model(n_layers=1, hidden=H, heads=NH, kv_heads=KV, head_dim=128, inter=I,
                               n_experts=2, fp8=True)
        for e in range(2):
            w = {n: bf16_round(r.normal(0, 0.0 if n in zero else 0.05, s)) for n, s in shapes.items()}
            for n, k in [("input_layernorm", H), ("post_attention_layernorm", H), ("q_norm", 64),
                         ("k_norm", 64), ("q_norm_hw", 64), ("k_norm_hw", 64)]:
                w[n] = bf16_round(r.normal(1, 0.1, k))
            self.m.bind_expert_layer(0, e, w)
            self.W.append(w)
        self.m.finalize()
        self.x0 = dev_bf16(activations(self.T, H, 3))
        t = torch.arange(self.T, dtype=torch.int32, device="cuda")
        self.pos = [t, torch.zeros_like(t), torch.zeros_like(t)]

    def run(self, **kw):
        x, kv = self.x0.clone(), self.m.make_cache(self.T)
        self.m.layer_forward(0, x, kv, 0, self.T, *self.pos, segments=self.SEGS, **kw)
        return x, kv


def test_layer_is_the_operators(ops):
    a = Layer(zero=("o_proj",))
    x, kv = a.run(fp8=True)
    H, I, T = a.H, a.I, a.T

    def twin(parts):
        w = np.stack(parts)
        q, s = u8(w.size).view(w.shape), ops.fp8_scale(w.shape[1], w.shape[2], 2)
        ops.quant_weight_fp8(dev_bf16(w), q, s, *w.shape)
        return q, s
    gu = twin([np.stack([w["gate_proj"].reshape(-1, 128, H), w["up_proj"].reshape(-1, 128, H)], 1)
               .reshape(2 * I, H) for w in a.W])
    down = twin([w["down_proj"] for w in a.W])
    qkv = twin([np.concatenate([w["q_proj"], w["k_proj"], w["v_proj"]]) for w in a.W])
    ln, post = (dev_bf16(np.stack([w[n] for w in a.W])) for n in ("input_layernorm",
                                                                   "post_attention_layernorm"))
    y = torch.empty_like(x)
    ops.mot_ffn_fp8(a.x0, None, post, *gu, *down, a.SEGS, y, ops.ffn_fp8_workspace(T, H, I), T, H, I,
                    1e-6)
    assert torch.equal(x, y)
    q, s, n = u8(T * H), ops.fp8_scale(T, H), (a.NH + 2 * a.KV) * 128
    ops.mot_add_rms_norm_quant_fp8(a.x0, None, ln, a.SEGS, None, q, s, T, H, 1e-6)
    out = torch.empty(T, n, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(q, s, *qkv, a.SEGS, out, T, H, n)
    v = kv.read(0, True, T)
    assert torch.equal(v, out[:, (a.NH + a.KV) * 128:].reshape(T, a.KV, 128).transpose(0, 1))


@pytest.mark.parametrize("zero", [("down_proj",), ("o_proj",), ()])
def test_layer_near_the_bf16_layer(zero):
    """By the bound that test_gpu_fp8_layer.test_near_the_bf16_layer derives."""
    a = Layer(zero)
    d = [a.run(fp8=f)[0].double() - a.x0.double() for f in (False, True)]
    off = ((d[1] - d[0]).norm() / d[0].norm()).item()
    assert 0 < off < 2 * np.sqrt(2) * 2.0 ** -4


def test_layer_repeats(ops):
    a = Layer()
    x, _ = a.run(fp8=True)
    assert torch.isfinite(x).all()
    for _ in range(3):
        assert torch.equal(a.run(fp8=True)[0], x)
