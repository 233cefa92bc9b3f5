"""A tensor that an fp8 entry point needs and is not given is refused with the
library's error. No kernel runs: the check comes before the call."""
import pytest
import torch

from u15b200 import CudaOps, U15Error, ops
from u15b200 import _lib as L

ROWS, K, N, E = 4, 256, 256, 2


class NoCalls:
    def __getattr__(self, name):
        if name == "u15c_ffn_fp8_workspace_bytes":       # host arithmetic
            return getattr(L.lib(), name)
        return lambda *a: pytest.fail(name + " was called")


@pytest.fixture
def args(monkeypatch):
    """Tensors in host memory, with the host in the place of the current device."""
    monkeypatch.setattr(ops, "_device", lambda: -1)
    monkeypatch.setattr(ops, "_raw_stream", lambda d: 0)
    monkeypatch.setattr(ops, "lib", NoCalls)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    return dict(x=bf(ROWS, K), q=u8(ROWS, K), s=u8(512), w=bf(E, K), wq=u8(E, N, K), ws=u8(E * 1024),
                y=bf(ROWS, N))


CALLS = {
    "quant_rows_fp8": (lambda o, t: o.quant_rows_fp8(t["x"], t["q"], t["s"], ROWS, K), "xqs"),
    "quant_weight_fp8": (lambda o, t: o.quant_weight_fp8(t["x"], t["q"], t["s"], 1, ROWS, K), "xqs"),
    "dequant_fp8": (lambda o, t: o.dequant_fp8(t["q"], t["s"], t["y"], ROWS, K), "qsy"),
    "norm": (lambda o, t: o.mot_add_rms_norm_quant_fp8(t["x"], None, t["w"], None, None, t["q"],
                                                       t["s"], ROWS, K, 1e-6), "xqsw"),
    "linear": (lambda o, t: o.mot_linear_fp8(t["q"], t["s"], t["wq"], t["ws"], None, t["y"], ROWS, K,
                                             N), ["q", "s", "wq", "ws", "y"]),
    "swiglu": (lambda o, t: o.mot_swiglu_fp8(t["q"], t["s"], t["wq"], t["ws"], None, t["y"], t["s"],
                                             ROWS, K, N), ["q", "s", "wq", "ws", "y"]),
    "ffn": (lambda o, t: o.mot_ffn_fp8(t["x"], None, t["w"], t["wq"], t["ws"], t["wq"], t["ws"], None,
                                       t["y"], t["s"], ROWS, K, 128, 1e-6), ["x", "w", "wq", "ws", "y", "s"]),
}


@pytest.mark.parametrize("name", CALLS)
def test_absent_tensors(args, name):
    call, names = CALLS[name]
    o = object.__new__(CudaOps)
    for n in names:
        with pytest.raises(U15Error):
            call(o, {**args, n: None})
