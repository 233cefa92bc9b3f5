"""An fp8 pass needs e4m3 twins of the weights that are bound now: it is
refused before finalize and after any projection is bound again."""
import pytest

from gpu_util import dev_bf16, torch
from test_gpu_fp8_layer import H, I, KV, NH, model, positions, rows, weights

pytestmark = pytest.mark.gpu
T = 8
PROJECTIONS = ["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"]


def run(m, **kw):
    x = rows(T)
    m.layer_forward(0, x, m.make_cache(T), 0, T, *positions(T), **kw)
    return x


def refused(m):
    from u15b200 import U15Error
    with pytest.raises(U15Error, match="finalize"):
        run(m, fp8=True)
    x, kv = rows(T), m.make_cache(T)
    with pytest.raises(U15Error, match="finalize"):
        m.forward(x, kv, 0, T, *positions(T), fp8=True)
    slot = {"kv": kv, "kv_off": 0, "kv_len": T, "pos": positions(T)}
    with pytest.raises(U15Error, match="finalize"):
        m.forward_many(x, T, [slot], expert=1, fp8=True)
    host = rows(T).cpu().pin_memory()
    out = torch.zeros_like(host).pin_memory()
    with pytest.raises(U15Error, match="finalize"):
        m.layer_forward_host(0, host, out, kv, 0, T, *positions(T), fp8=True)
    with pytest.raises(U15Error, match="finalize"):
        m.layer_forward_host_async(0, host, out, kv, 0, T, *positions(T), fp8=True)
    m.host_drain()
    torch.cuda.synchronize()


def test_not_finalized():
    import u15b200
    m = u15b200.Model(n_layers=1, hidden=H, heads=NH, kv_heads=KV, head_dim=128, inter=I, n_experts=2,
                      fp8=True)
    for e in range(2):
        m.bind_expert_layer(0, e, weights(7 + e))
    refused(m)
    run(m)                                     # the bf16 pass needs no twins
    m.finalize()
    assert torch.equal(run(m, fp8=True), run(model(fp8=True)[0], fp8=True))


@pytest.mark.parametrize("name", PROJECTIONS)
def test_bound_again(name):
    m, W = model(fp8=True)
    m.bind_expert_layer(0, 1, {name: weights(9)[name]})
    refused(m)
    run(m)
    m.finalize()
    want, _ = model(fp8=True)
    want.bind_expert_layer(0, 1, {name: weights(9)[name]})
    want.finalize()
    assert torch.equal(run(m, fp8=True), run(want, fp8=True))


def test_random_weights():
    m, _ = model(fp8=True)
    m.bind_random(seed=1, std=0.05, norm_mean=1.0, norm_std=0.1)
    refused(m)
    m.finalize()
    assert torch.isfinite(run(m, fp8=True)).all()


def test_norms_have_no_twins():
    """The norms' gains are read as they are bound."""
    m, _ = model(fp8=True)
    before = run(m, fp8=True)
    new = weights(9)
    m.bind_expert_layer(0, 0, {n: new[n] for n in new if n not in PROJECTIONS})
    after = run(m, fp8=True)
    assert torch.isfinite(after).all() and not torch.equal(before, after)


def test_a_refused_bind_changes_nothing():
    from u15b200 import U15Error
    m, W = model(fp8=True)
    with pytest.raises(U15Error):
        m.bind_expert_layer(0, 5, {"q_proj": W[0]["q_proj"]})
    assert torch.isfinite(run(m, fp8=True)).all()


def test_int8_passes_are_as_they_were():
    """The int8 tier does not follow the rule: a pass keeps the twins of the last finalize."""
    m, _ = model(int8=True, fp8=True)
    before = run(m, int8=True)
    m.bind_expert_layer(0, 0, {"q_proj": weights(9)["q_proj"]})
    assert torch.equal(run(m, int8=True), before)
    refused(m)
