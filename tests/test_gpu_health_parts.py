"""The health word's part for products and orthogonal updates, in processes of their own: nothing of it before the first of them, one word for all."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
from flash_sinkhorn_b200 import _lib, experts as ex
lib = _lib.load()
x, w = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(2, 64, 64, dtype=torch.bfloat16, device="cuda")
off = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
calls = {"mm": lambda: ex.grouped_mm(x, w, off), "mm8": lambda: ex.grouped_mm8(x, w, off), "ortho": lambda: ex.orthogonalize(w)}
order = ORDER
assert lib.fs_device_error() == 0 and lib.fs_clear_device_error() == 0
if CAPTURED:  # the first call of all is captured, without one before it
    outs = []
    for name in order:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = calls[name]()
        graph.replay()
        outs.append((graph, out))
    torch.cuda.synchronize()
    for name, (graph, out) in zip(order, outs):
        assert torch.equal(out, calls[name]()) and bool(torch.isfinite(out).all())
usual = lib.fs_set_product_limit(0)
outs = [calls[name]() for name in order]
lib.fs_set_product_limit(usual)
assert lib.fs_device_error() == 1 and all(bool(torch.isnan(out).all()) for out in outs)
assert lib.fs_clear_device_error() == 0 and lib.fs_device_error() == 0
for name in order:
    assert bool(torch.isfinite(calls[name]()).all()) and lib.fs_device_error() == 0
"""


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("order", [["ortho"], ["mm8"], ["mm", "mm8", "ortho"]])
def test_one_word_for_products_and_updates(order, captured):
    script = SCRIPT.replace("ORDER", repr(order)).replace("CAPTURED", repr(captured))
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr[-2000:]
