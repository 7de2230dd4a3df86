"""8-bit products and orthogonal updates whose waits give up, in every kernel that has some: what is left is NaN, the health word says so, and the
next call is as before. What gives up are the warps that read results, at once (a limit of no clocks), or the meetings of a chain of products at
their first look that finds a CTA missing (one clock): loads and products of theirs are in flight then.
"""
import ctypes

import pytest
import torch

from test_gpu_experts import BF16, FP32, gen, normal
from test_gpu_mm8 import offsets_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    from flash_sinkhorn_b200 import experts
    return experts


@pytest.fixture(scope="module")
def lib():
    from flash_sinkhorn_b200 import _lib
    return _lib.load()


def given_up(lib, call, clocks=0):
    """The result and the health word of a call under the limit; the word is cleared."""
    before = lib.fs_set_product_limit(clocks)
    try:
        out = call()
        word = lib.fs_device_error()
    finally:
        lib.fs_set_product_limit(before)
        torch.cuda.synchronize()
        assert lib.fs_clear_device_error() == 0
    assert lib.fs_device_error() == 0
    return out, word


def product(lib, x, codes, scales, off, transposed, dtype):
    """The product by itself, on this thread (a backward pass has its own thread, and limits hold for threads)."""
    e, n, k = codes.shape
    n, k = (k, n) if transposed else (n, k)
    out = torch.empty(x.shape[0], n, device="cuda", dtype=dtype)
    size = lib.fs_grouped_mm8_bytes(x.shape[0], k, int(transposed))
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    assert lib.fs_grouped_mm8(p(x), 2, x.stride(0), x.shape[0], None, x.shape[0], p(codes), codes.stride(0), codes.stride(1), p(scales), e, n, k,
                              int(transposed), p(off), p(out), 0 if dtype == FP32 else 2, n, p(ws), size,
                              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    return out


# short tiles; tiles of 128 x 128; pairs; transposed: tiles of 128 x 128, pairs. Many stages to a tile, and more tiles than CTAs
@pytest.mark.parametrize("counts,n,k,transposed", [
    ([30] * 64, 1000, 640, False), ([100, 41, 90], 200, 1500, False), ([100] * 40, 900, 256, False), ([900, 800, 2000, 3000, 10, 700], 2048, 384, False),
    ([5, 9, 0, 100], 200, 256, True), ([300, 20], 1300, 100, True), ([900, 800, 2000, 3000, 10, 700], 520, 2048, True), ([200] * 60, 384, 520, True)])
def test_8_bit_products(ex, lib, counts, n, k, transposed):
    g = gen(sum(counts) + n)
    q = ex.to_blocks8(normal(g, len(counts), n, k, dtype=BF16))
    spare = 3
    x, off = normal(g, sum(counts) + spare, n if transposed else k, dtype=BF16), offsets_of(counts)
    for dtype in (BF16, FP32):
        call = lambda: product(lib, x, q.codes, q.scales, off, transposed, dtype)
        want = call()
        for _ in range(3):
            out, word = given_up(lib, call)
            assert word == 1 and torch.isnan(out[:-spare]).all() and not out[-spare:].any()
            assert torch.equal(call(), want)


# chains of 1, 32, 96 and 295 tiles; tiles of 128 x 64, 128 x 128 and pairs; tall and wide
@pytest.mark.parametrize("batch,n,k", [(1, 60, 70), (1, 512, 512), (3, 500, 400), (5, 640, 200), (1, 1024, 2360), (1, 1024, 2432), (2, 3000, 900), (20, 512, 600),
                                       (4, 1024, 2048)])
def test_orthogonal_updates(ex, lib, batch, n, k):
    m = normal(gen(n), batch, n, k)
    want = ex.orthogonalize(m)
    for _ in range(3):
        out, word = given_up(lib, lambda: ex.orthogonalize(m))
        assert word == 1 and torch.isnan(out).all()
        assert torch.equal(ex.orthogonalize(m), want)


@pytest.mark.parametrize("batch,n,k", [(1, 60, 70), (1, 512, 512), (3, 500, 400), (1, 1024, 2360)])
def test_meetings(ex, lib, batch, n, k):
    """A CTA that does not wait for the others leaves NaN where it had still to write, and the others, which miss it then, too."""
    m = normal(gen(k), batch, n, k)
    want = ex.orthogonalize(m)
    words = []
    for _ in range(5):
        out, word = given_up(lib, lambda: ex.orthogonalize(m), clocks=1)
        assert torch.isnan(out).any() if word else torch.equal(out, want)
        assert torch.equal(out[~torch.isnan(out)], want[~torch.isnan(out)])
        words.append(word)
        assert torch.equal(ex.orthogonalize(m), want)
    assert any(words) or batch * n * k < 128 * 64  # one CTA meets nobody
