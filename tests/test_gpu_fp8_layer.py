"""The layer with fp8 projections (U15C_MODEL_FP8, U15C_FWD_FP8): its halves
equal the public operators run one by one on the same weights, every way of
running a pass agrees, and it stays near the bf16 layer."""
import numpy as np
import pytest

from gpu_util import bf16_round, dev_bf16, torch

pytestmark = pytest.mark.gpu
H, NH, KV, I = 512, 4, 1, 640
QKV = (NH + 2 * KV) * 128
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    import u15b200
    return u15b200.CudaOps(0)


def weights(seed, zero=()):
    r = np.random.default_rng(seed)
    w = {}
    for n, shape in [("q_proj", (NH * 128, H)), ("k_proj", (KV * 128, H)), ("v_proj", (KV * 128, H)),
                     ("o_proj", (H, NH * 128)), ("gate_proj", (I, H)), ("up_proj", (I, H)),
                     ("down_proj", (H, I))]:
        w[n] = bf16_round(r.normal(0, 0.0 if n in zero else 0.05, shape))
    for n, k in [("input_layernorm", H), ("post_attention_layernorm", H), ("q_norm", 64),
                 ("k_norm", 64), ("q_norm_hw", 64), ("k_norm_hw", 64)]:
        w[n] = bf16_round(r.normal(1, 0.1, k))
    return w


def model(zero=(), n_layers=1, **kw):
    import u15b200
    m = u15b200.Model(n_layers=n_layers, hidden=H, heads=NH, kv_heads=KV, head_dim=128, inter=I,
                      n_experts=2, **kw)
    W = []
    for e in range(2):
        W.append(weights(7 + e, zero))
        for li in range(n_layers):
            m.bind_expert_layer(li, e, W[-1])
    m.finalize()
    return m, W


def positions(T):
    return [torch.arange(T, dtype=torch.int32, device="cuda"),
            *(torch.zeros(T, dtype=torch.int32, device="cuda") for _ in range(2))]


def rows(T, seed=3):
    return dev_bf16(np.random.default_rng(seed).normal(size=(T, H)))


def stacked(W, name):
    """A projection of both experts in the bound layout."""
    if name == "qkv":
        s = [np.concatenate([w["q_proj"], w["k_proj"], w["v_proj"]]) for w in W]
    elif name == "gu":
        s = [np.stack([w["gate_proj"].reshape(-1, 128, H), w["up_proj"].reshape(-1, 128, H)], 1)
             .reshape(2 * I, H) for w in W]
    else:
        s = [w[name] for w in W]
    return np.stack(s)


def quantised(ops, a):
    E, N, K = a.shape
    q, s = torch.empty(E, N, K, dtype=torch.uint8, device="cuda"), ops.fp8_scale(N, K, E)
    ops.quant_weight_fp8(dev_bf16(a), q, s, E, N, K)
    return q, s


@pytest.mark.parametrize("T,split", [(1, 0), (70, 33), (300, 41)])
def test_values_and_feed_forward_are_the_operators(ops, T, split):
    """With o_proj zero the layer is the feed-forward block of its input; the V it
    caches is the quantised norm's projection."""
    m, W = model(zero=("o_proj",), fp8=True)
    x0 = rows(T)
    segs = [(0, split, 1), (split, T, 0)]
    x, kv = x0.clone(), m.make_cache(T)
    m.layer_forward(0, x, kv, 0, T, *positions(T), segments=segs, fp8=True)
    # the feed-forward half
    gq, gs = quantised(ops, stacked(W, "gu"))
    dq, ds = quantised(ops, stacked(W, "down_proj"))
    y = torch.empty_like(x0)
    post = dev_bf16(np.stack([w["post_attention_layernorm"] for w in W]))
    ops.mot_ffn_fp8(x0, None, post, gq, gs, dq, ds, segs, y, ops.ffn_fp8_workspace(T, H, I), T, H, I,
                    EPS)
    assert torch.equal(x, y)
    # the norm and the projection
    wq, ws = quantised(ops, stacked(W, "qkv"))
    ln = dev_bf16(np.stack([w["input_layernorm"] for w in W]))
    q, s = torch.empty(T, H, dtype=torch.uint8, device="cuda"), ops.fp8_scale(T, H)
    ops.mot_add_rms_norm_quant_fp8(x0, None, ln, segs, None, q, s, T, H, EPS)
    qkv = torch.empty(T, QKV, dtype=torch.bfloat16, device="cuda")
    ops.mot_linear_fp8(q, s, wq, ws, segs, qkv, T, H, QKV)
    v = kv.read(0, True, T)
    assert torch.equal(v, qkv[:, (NH + KV) * 128:].reshape(T, KV, 128).transpose(0, 1))


@pytest.mark.parametrize("zero", [("down_proj",), ("o_proj",), ()])
def test_near_the_bf16_layer(zero):
    """The update of each half, and of both, against the bf16 layer's. A half
    holds two products in a row; each factor of a product carries a relative
    error of at most 2^-4 per value, so a product's 2-norm is off by at most
    sqrt(2) 2^-4 of its own and two in a row by twice that. Scores are off by the
    same share of their own small size, which the softmax passes on weaker."""
    m, _ = model(zero=zero, fp8=True)
    T = 200
    out = {}
    for fp8 in (False, True):
        x, kv = rows(T), m.make_cache(T)
        m.layer_forward(0, x, kv, 0, T, *positions(T), segments=[(0, 60, 0), (60, T, 1)], fp8=fp8)
        out[fp8] = x.double() - rows(T).double()
    off = ((out[True] - out[False]).norm() / out[False].norm()).item()
    assert 0 < off < 2 * np.sqrt(2) * 2.0 ** -4


def test_ways_of_a_pass_agree():
    """layer by layer, a whole pass, two branches together, and through host memory."""
    m, _ = model(n_layers=2, fp8=True)
    T = 96
    pos = positions(T)
    want, kv = rows(T), m.make_cache(T)
    for li in range(2):
        m.layer_forward(li, want, kv, 0, T, *pos, segments=[(0, T, 1)], fp8=True)
    x, kv = rows(T), m.make_cache(T)
    m.forward(x, kv, 0, T, *pos, segments=[(0, T, 1)], fp8=True)
    assert torch.equal(x, want)
    both = torch.cat([rows(T), rows(T, 4)])
    slots = [{"kv": m.make_cache(T), "kv_off": 0, "kv_len": T, "pos": pos} for _ in range(2)]
    m.forward_many(both, T, slots, expert=1, fp8=True)
    # more rows may run another form of the product, whose f32 sums round apart;
    # outputs then differ by a bf16 step here and there, and quantised values by one of theirs
    off = ((both[:T].double() - want.double()).norm() / want.double().norm()).item()
    assert off < 2.0 ** -8
    xh, out = rows(T).cpu().pin_memory(), torch.empty(T, H, dtype=torch.bfloat16).pin_memory()
    m.layer_forward_host(0, xh, out, m.make_cache(T), 0, T, *pos, segments=[(0, T, 1)], fp8=True)
    one = rows(T)
    m.layer_forward(0, one, m.make_cache(T), 0, T, *pos, segments=[(0, T, 1)], fp8=True)
    off = ((out.double() - one.cpu().double()).norm() / one.cpu().double().norm()).item()
    assert off < 2.0 ** -8


def test_refusals_and_sizes():
    import u15b200
    from u15b200 import U15Error
    m, _ = model(int8=True, fp8=True)
    plain, _ = model()
    T = 8
    for mm, kw, word in [(plain, dict(fp8=True), "e4m3"), (m, dict(fp8=True, int8=True), "not both")]:
        with pytest.raises(U15Error, match=word):
            mm.layer_forward(0, rows(T), mm.make_cache(T), 0, T, *positions(T), **kw)
    with pytest.raises(U15Error, match="one device"):
        u15b200.Model(n_layers=1, hidden=H, heads=4, kv_heads=2, head_dim=128, inter=512,
                      n_experts=2, fp8=True, tp_size=2)
    for kw in (dict(int8=True), dict(fp8=True)):
        x = rows(T)
        m.layer_forward(0, x, m.make_cache(T), 0, T, *positions(T), **kw)
        assert torch.isfinite(x).all()
    assert m.weight_bytes() > plain.weight_bytes() and m.scratch_bytes(T) > plain.scratch_bytes(T)
