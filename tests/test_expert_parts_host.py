"""Layer norm, 8-bit products and orthogonal updates without a GPU: names, scratch sizes, refusals."""
import os

import pytest
import torch

from flash_sinkhorn_b200 import _lib


@pytest.fixture(scope="module")
def ex():
    if not os.path.exists(_lib.library_path()):
        import __graft_entry__
        __graft_entry__.build()
    from flash_sinkhorn_b200 import experts
    return experts


def test_names(ex):
    assert ex.Blocks8._fields == ("codes", "scales")
    assert {"layer_norm", "to_blocks8", "Blocks8", "grouped_mm8", "orthogonalize"} <= set(ex.__all__)
    assert {"fs_layer_norm", "fs_grouped_mm8", "fs_weights8", "fs_orthogonalize"} <= set(_lib.torch_binding().entries())


def test_scratch():
    lib = _lib.load()
    assert lib.fs_grouped_mm8_bytes(1, 2048, 0) == 0 and lib.fs_grouped_mm8_bytes(0, 8, 0) == 0  # single tokens need none
    assert lib.fs_grouped_mm8_bytes(300, 130, 0) == -(-300 * 144 // 256) * 256 + 300 * 2 * 4
    assert lib.fs_grouped_mm8_bytes(2**31 - 512, 8192, 1) > 2**31 * 8191  # no wrap at 2^32
    assert lib.fs_layer_norm_grad_bytes(10**6, 2048) == lib.fs_layer_norm_grad_bytes(10**5, 2048) > 0 == lib.fs_layer_norm_grad_bytes(0, 8)
    assert lib.fs_orthogonalize_bytes(4, 65536, 65536) > 4 * 65536**2 * 2 * 5 and lib.fs_orthogonalize_bytes(0, 4, 4) == 0


@pytest.mark.parametrize("r", [2**31 - 1, 2**31 - 511])
def test_products_of_too_many_rows_are_refused(r):
    lib = _lib.load()
    at = 256  # never read
    assert lib.fs_grouped_mm8(at, 2, 16, 8, None, r, at, 256, 16, at, 2, 8, 16, 0, at, at, 2, 8, at, 1 << 62, None) == 1
    assert b"2^31 - 512" in lib.fs_last_error()


def test_refusals_on_the_host(ex):
    x, w = torch.zeros(6, 16, dtype=torch.bfloat16), torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    q = ex.Blocks8(torch.zeros(2, 8, 16, dtype=torch.float8_e4m3fn), torch.zeros(2, 1, 1))
    off = torch.zeros(3, dtype=torch.int32)
    r = ex.Routing(torch.zeros(3, 2), *[torch.zeros(3, 2, dtype=torch.int32)] * 5)
    calls = [
        lambda: ex.layer_norm(x), lambda: ex.layer_norm(x.double()), lambda: ex.layer_norm(x[:, :0]), lambda: ex.layer_norm(x, eps=-1.0),
        lambda: ex.to_blocks8(w), lambda: ex.to_blocks8(w[0]), lambda: ex.to_blocks8(w.float()), lambda: ex.to_blocks8(w[:0]),
        lambda: ex.grouped_mm8(x, q, off), lambda: ex.grouped_mm8(x, w, off), lambda: ex.grouped_mm8(x, w.half(), off),
        lambda: ex.grouped_mm8(x, ex.Blocks8(w, q.scales), off), lambda: ex.grouped_mm8(x, ex.Blocks8(q.codes, q.scales[:1]), off),
        lambda: ex.grouped_mm8(x, q, off, gather=True), lambda: ex.expert_mlp(x, q, w, r), lambda: ex.expert_mlp(x, q, q, r),
        lambda: ex.orthogonalize(x), lambda: ex.orthogonalize(x[0]), lambda: ex.orthogonalize(x, dtype=torch.float32),
        lambda: ex.orthogonalize(x, coefficients=(1.0, 2.0)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
