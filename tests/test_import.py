"""The package imports on a PyTorch that was built without CUDA, which has no
CUDA bindings in torch._C."""
import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "vpipe-sensenova-u1.5_b200")
CODE = """
import sys
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
sys.path.insert(0, sys.argv[1])
import u15b200
print(u15b200.CudaOps.__name__)
"""


def test_imports_without_cuda_bindings():
    p = subprocess.run([sys.executable, "-c", CODE, PKG], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stderr
    assert p.stdout.strip() == "CudaOps"


@pytest.mark.gpu
def test_stream_without_the_binding():
    """The public way to the current stream gives the binding's."""
    import torch
    from u15b200 import ops
    side = torch.cuda.Stream()
    assert ops._public_stream(ops._device()) == ops._raw_stream(ops._device())
    with torch.cuda.stream(side):
        assert ops._public_stream(0) == ops._raw_stream(0) == side.cuda_stream == ops._stream()
