"""Routed experts without a GPU: the binding loads, names are where the documentation says, refusals are ValueErrors."""
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


def test_binding_knows_the_entry_points(ex):
    names = _lib.torch_binding().entries()
    assert names and set(names) <= set(_lib.SIGNATURES)
    assert ex.Routing._fields == ("gates", "experts", "offsets", "pairs", "rows", "position")


def test_scratch_of_a_routing():
    lib = _lib.load()
    assert lib.fs_route_bytes(32, 64, 4) == 0  # one block counts and numbers its own pairs
    assert 0 < lib.fs_route_bytes(65536, 128, 8) <= 128 * 4 * 296
    assert lib.fs_route_bytes(1 << 28, 1024, 4) <= 1024 * 4 * 296
    assert lib.fs_route_bytes(10, 1025, 2) == 0


@pytest.mark.parametrize("t", [(1 << 31) - 1, (1 << 31) - 200, (1 << 31) - 14_000_000])
def test_scratch_of_the_longest_batches(t):
    """Up to 2^31 - 1 pairs, as the arguments are checked: one count for each expert and block, at most 148 blocks."""
    assert _lib.load().fs_route_bytes(t, 4, 1) == 4 * 4 * 148


@pytest.mark.parametrize("r", [(1 << 31) - 1, (1 << 31) - 511])
def test_products_of_too_many_rows_are_refused(r):
    """Before anything else is looked at: a tile of the last rows would reach past 2^31."""
    lib = _lib.load()
    at = 256  # never read
    for call in (lambda: lib.fs_grouped_mm(at, 8, 8, at, r, at, 64, 8, 1, 2, 8, 8, at, at, 2, 8, 2, None),
                 lambda: lib.fs_grouped_mm_wgrad(at, 8, at, 8, r, 2, 8, 8, at, at, 2, None)):
        assert call() == 1 and b"2^31 - 512" in lib.fs_last_error()  # FS_ERR_BAD_ARG


def test_refusals_on_the_host(ex):
    x, w = torch.zeros(6, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16)
    r = ex.Routing(torch.zeros(3, 2), *[torch.zeros(3, 2, dtype=torch.int32)] * 5)
    calls = [
        lambda: ex.route_tokens(torch.zeros(4, 8), 2), lambda: ex.route_tokens(torch.zeros(4), 2),
        lambda: ex.route_tokens(torch.zeros(4, 8, dtype=torch.float64), 2), lambda: ex.route_tokens(torch.zeros(4, 8), 2, normalize="no"),
        lambda: ex.grouped_mm(x, w, r), lambda: ex.grouped_mm(x, w[0], r), lambda: ex.grouped_mm(x.float(), w.float(), r),
        lambda: ex.grouped_mm(x, w.half(), r), lambda: ex.grouped_mm(x, w, torch.zeros(3, dtype=torch.int32), gather=True),
        lambda: ex.gated_act(x), lambda: ex.gated_act(x[0]), lambda: ex.gated_act(x[:, :3]), lambda: ex.gated_act(x, (1, 2)),
        lambda: ex.combine_rows(x, r), lambda: ex.combine_rows(x[0], r), lambda: ex.combine_rows(x, None),
        lambda: ex.expert_mlp(x, w, w, r), lambda: ex.expert_mlp(x[0], w, w, r), lambda: ex.expert_mlp(x, w.half(), w, r),
        lambda: ex.expert_mlp(x, w, w, None), lambda: ex.transport_bias(x, w), lambda: ex.transport_bias(x, x[:, :4]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(TypeError):
        ex.route_tokens("logits", 2)


def test_missing_binding_fails_loudly(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(_lib, "_LIB_PATH", str(tmp_path / "none.so"))
    with pytest.raises(ImportError):
        _lib.torch_binding()
