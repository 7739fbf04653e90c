"""Calls of the dense operators at the edges of what their documentation allows (CPU only)."""
import subprocess
import sys

import pytest

from conftest import PKG

torch = pytest.importorskip("torch")


def test_import_without_torch_cuda_bindings():
    """A torch built without CUDA imports the package, and its tensors are refused by name."""
    code = """
import sys, torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
sys.path.insert(0, %r)
import glmx
for call in (lambda: glmx.quantize_rows(torch.zeros(2, 8)), lambda: glmx.sample(torch.zeros(2, 8), torch.zeros(2)),
             lambda: glmx.GatedFFN(*(torch.zeros(s, dtype=torch.bfloat16) for s in ((8, 8),) * 3)),
             lambda: glmx.gated_ffn(*(torch.zeros(s, dtype=torch.bfloat16) for s in ((2, 8),) + ((8, 8),) * 3)),
             lambda: glmx.Int8Linear(torch.zeros(8, 8, dtype=torch.int8), torch.zeros(8))):
    try:
        call()
    except ValueError as e:
        assert "CUDA" in str(e), e
    else:
        raise AssertionError("a CPU tensor was taken")
print("imported")
""" % PKG
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr[-2000:]
