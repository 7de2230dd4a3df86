"""Layer norm, 8-bit products and orthogonal updates where offsets pass 32 bits, and on both sides of their choices between kernels."""
import pytest
import torch

from test_gpu_experts import BF16, FP16, FP32, ULP, gen, normal
from test_gpu_layer_norm import check as check_norm
from test_gpu_mm8 import blocks8, close, grouped, offsets_of, rows8, wide
from test_gpu_orthogonalize import check as check_ortho, plain as plain_ortho

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    from flash_sinkhorn_b200 import experts
    return experts


def test_layer_norm_past_32_bits(ex):
    rows, f = 270_000, 8192  # 2.2e9 values
    x = torch.empty(rows, f, device="cuda", dtype=BF16)
    x[:64] = normal(gen(1), 64, f, dtype=BF16)
    x[64:] = 1.0
    x[-70:] = normal(gen(2), 70, f, dtype=BF16)
    w, b = 1 + 0.2 * normal(gen(3), f), normal(gen(4), f)
    y = ex.layer_norm(x, w, b)
    assert torch.equal(y[-70:], ex.layer_norm(x[-70:].clone(), w, b)) and torch.equal(y[:64], ex.layer_norm(x[:64].clone(), w, b))
    del y
    dy = torch.zeros_like(x)
    dy[-70:] = normal(gen(5), 70, f, dtype=BF16)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    dx, dw = torch.autograd.grad(ex.layer_norm(x, w, b), leaves, dy)
    part = [x[-70:].detach().clone().requires_grad_(), w.detach().clone().requires_grad_()]
    px, pw = torch.autograd.grad(ex.layer_norm(*part, b), part, dy[-70:].clone())
    assert torch.equal(dx[-70:], px) and not dx[:-70].any()
    assert ((dw - pw).abs() <= 2.0**-17 * (1 + pw.abs())).all()  # the same 70 terms in another order


@pytest.mark.parametrize("f,dtype", [(32, BF16), (256, BF16), (264, FP16), (4096, BF16), (4104, BF16), (8192, FP32), (8196, FP32), (16384, BF16), (32768, FP16),
                                     (32776, BF16), (2047, BF16), (2049, FP16), (4097, FP32), (8193, BF16)])
@pytest.mark.parametrize("rows", [3, 700])
def test_layer_norm_at_the_edges_of_its_plans(ex, f, dtype, rows):
    g = gen(f)
    check_norm(ex.layer_norm, normal(g, rows, f, dtype=dtype), 1 + 0.2 * normal(g, f), normal(g, f), normal(g, rows, f, dtype=dtype))


def test_weights_past_32_bits(ex):
    e, n, k = 9, 16384, 32768 - 128  # 4.8e9 codes
    g = gen(6)
    codes = torch.zeros(e, n, k, device="cuda", dtype=torch.float8_e4m3fn)
    codes[-1, -300:] = normal(g, 300, k).clamp(-4, 4).to(torch.float8_e4m3fn)
    scales = torch.ones(e, n // 128, k // 128, device="cuda")
    scales[-1] = torch.rand(n // 128, k // 128, generator=g, device="cuda") + 0.5
    q = ex.Blocks8(codes, scales)
    for rows in (1, 20, 300):
        x = normal(g, rows, k, dtype=BF16)
        off = offsets_of([0] * (e - 1) + [rows])
        y = ex.grouped_mm8(x, q, off)
        last = codes[-1, -300:].double() * scales[-1].double().repeat_interleave(128, 0)[-300:].repeat_interleave(128, 1)
        want, size = rows8(x) @ last.T, rows8(x).abs() @ last.abs().T
        # 255 blocks are added in fp32: 2^-24 each besides the bound of one
        bound = ULP[BF16] * want.abs() + (2.0**-15 + 256 * 2.0**-24) * size + 1e-30
        assert ((y[:, -300:].double() - want).abs() <= bound).all()
        assert not y[:, :-300].any()


@pytest.mark.parametrize("mean", [2, 39, 41, 100, 159, 161, 400])
@pytest.mark.parametrize("e,n,k", [(6, 640, 260), (24, 512, 512)])
def test_tiles_by_the_rows_of_a_mean_group(ex, mean, e, n, k):
    """All kernels, and the transposed ones, give the same sums to within their roundings, whatever the sizes of the groups."""
    g = gen(mean)
    counts = torch.randint(0, 2 * mean + 1, (e,), generator=g, device="cuda").tolist()
    counts[0] = mean * e - sum(counts[1:]) if mean * e > sum(counts[1:]) else 0
    x = normal(g, sum(counts) + 5, k, dtype=BF16).requires_grad_()
    w = normal(g, e, n, k, scale=k**-0.5, dtype=BF16)
    off = offsets_of(counts)
    codes, scales = blocks8(w)
    v = codes * wide(scales, n, k)
    y = ex.grouped_mm8(x, w, off)
    close(y, *grouped(rows8(x), v, off[1:].tolist()), BF16)
    dy = normal(g, *y.shape, dtype=BF16)
    close(torch.autograd.grad(y, x, dy)[0], *grouped(rows8(dy), v, off[1:].tolist(), transposed=True), BF16)


def test_orthogonalize_matrices_past_32_bits_apart(ex):
    store = torch.zeros((1 << 31) + 64 * 96, device="cuda", dtype=FP16)
    g = store.as_strided((2, 64, 80), (1 << 31, 96, 1))
    g.copy_(normal(gen(7), 2, 64, 80, dtype=FP16))
    assert torch.equal(ex.orthogonalize(g), ex.orthogonalize(g.clone()))


@pytest.mark.parametrize("batch,n,k", [(1, 1024, 2304), (1, 1024, 2432), (2, 768, 1536), (5, 1100, 520), (140, 128, 136), (300, 64, 72), (18, 256, 1024)])
def test_orthogonalize_in_one_launch_and_in_many(ex, batch, n, k):
    g = normal(gen(batch), batch, n, k, dtype=BF16)
    check_ortho(ex.orthogonalize(g), plain_ortho(g))


def test_orthogonalize_of_a_large_stack(ex):
    g = normal(gen(8), 40, 1024, 1152, dtype=BF16)
    y = ex.orthogonalize(g)
    check_ortho(y[[0, 17, 39]], plain_ortho(g[[0, 17, 39]]))
