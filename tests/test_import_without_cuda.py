"""The package on a build of torch without CUDA, which lacks the names that only a CUDA build defines: it imports, and
its operators refuse CPU tensors as they do elsewhere."""
import subprocess
import sys

from conftest import PKG

PROGRAM = r"""
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_getCurrent")]:
    delattr(torch._C, name)
from lcgemm import layer, model, ops
x = torch.zeros((4, 128), dtype=torch.bfloat16)
q, s, ids = x.to(torch.float8_e4m3fn), torch.zeros((4, 1)), torch.zeros(4, dtype=torch.int64)
for call in (lambda: ops.quantize_fp8(x), lambda: ops.swiglu_fp8(x), lambda: ops.add_rmsnorm_fp8(x, x, x[0], 1e-6),
             lambda: ops.gemm_fp8(q, s, q, s[:1]), lambda: ops.token_logprobs(x, ids)):
    try:
        call()
    except RuntimeError as e:
        assert "no CPU implementation" in str(e), e
    else:
        raise AssertionError("not refused")
print("refused")
"""


def test_the_package_imports_and_refuses_cpu_tensors():
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=PKG, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]
    assert done.stdout.split() == ["refused"]
