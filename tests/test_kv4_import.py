"""CPU: the package on a torch build without CUDA."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import torch
for name in [n for n in vars(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import madi_b200
from madi_b200 import kv4
c = kv4.Cache.empty(1, 1, 64, device="cpu")
x = torch.zeros((1, 1, 64))
for call in (lambda: kv4.store(c, x, x), lambda: kv4.load(c, 1, k_out=x, v_out=x.clone()), lambda: kv4.attn(x, c, 1)):
    try:
        call()
    except ValueError as e:
        assert "host memory" in str(e)
    else:
        raise AssertionError("a cache in host memory was taken")
"""


def test_import_without_cuda_in_torch():
    """A torch build without CUDA has none of torch._C's _cuda_ names: the package is imported all the
    same, as before it held the 4-bit cache, and its calls refuse host memory."""
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
