"""The compiled Python calls on tensors that have no memory of their own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
import rustorch_b200 as rb
x = torch.zeros((3, 4, 256), device="cuda")
q, s = rb.fp8_quantize(x)
m = torch.zeros((3, 4), device="cuda")
torch.cuda.synchronize()
for call in (lambda X, Q, S, M: rb.layer_norm_fwd(X),
             lambda X, Q, S, M: rb.layer_norm_backward(X, M, M, X),
             lambda X, Q, S, M: rb.layer_norm_backward(Q, M, M, X, x_scale=S),
             lambda X, Q, S, M: rb.fp8_quantize(X),
             lambda X, Q, S, M: rb.fp8_dequantize(Q, S),
             lambda X, Q, S, M: rb.fp8_matmul(Q, S, Q.t(), S.t()),
             lambda X, Q, S, M: rb.matmul_backward_fp8(Q, S, None, X, need_a=False)):
    try:
        torch.vmap(call)(x, q, s, m)
    except RuntimeError as e:
        print("refused:", str(e).splitlines()[0])
    else:
        raise AssertionError("not refused")
    assert torch.equal(rb.fp8_dequantize(*rb.fp8_quantize(x)), x)  # the next call is as usual
print("fine")
"""


def test_a_transforms_tensors(gpu):
    """torch.vmap's tensors have no data pointer: asking for it throws in the
    middle of a call, which ends as an exception and does not end the process."""
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True,
                       timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, (r.returncode, r.stdout, r.stderr[-2000:])
