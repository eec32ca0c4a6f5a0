"""Workspace sizes and the checks of tensors that the token-path operators make
before any CUDA call; they run without a GPU."""
import pytest

import ttfoil


@pytest.mark.parametrize("T,D,gate_rows", [(4, 16385, 0), (4, 1 << 20, 0), (1, (1 << 32) - 1, 1), ((1 << 31) + 1, 64, 0),
                                           ((1 << 32) - 1, 64, 0), ((1 << 32) - 1, 1, 7), ((1 << 32) - 1, 16384, 1 << 30)])
def test_block_norm_workspace_is_zero_out_of_range(T, D, gate_rows):
    assert ttfoil.block_norm_grad_ws_bytes(T, D, gate_rows) == 0


@pytest.mark.parametrize("T,V,D", [((1 << 24) + 1, 10, 64), (10, (1 << 24) + 1, 64), (10, 10, (1 << 20) + 1),
                                   ((1 << 32) - 1, 10, 64), ((1 << 32) - 1, (1 << 32) - 1, (1 << 32) - 1)])
def test_embed_rows_workspace_is_zero_out_of_range(T, V, D):
    assert ttfoil.embed_rows_grad_ws_bytes(T, V, D) == 0


def test_workspaces_at_the_ends_of_the_ranges():
    for gate_rows in (0, 1, 2, 1000, 1 << 31, (1 << 32) - 1):
        for T in (1, 2, 1 << 31):
            for D in (1, 2, 64, 4096, 16384):
                assert ttfoil.block_norm_grad_ws_bytes(T, D, gate_rows) > 0
    assert ttfoil.block_norm_grad_ws_bytes(0, 64, 0) == 0 and ttfoil.block_norm_grad_ws_bytes(4, 0, 0) == 0
    for T in (1, 33, 1 << 24):
        for V in (1, 1 << 24):
            for D in (1, 1 << 20):
                assert ttfoil.embed_rows_grad_ws_bytes(T, V, D) >= 16 * T
    assert ttfoil.embed_rows_grad_ws_bytes(0, 4, 4) == 0 and ttfoil.embed_rows_grad_ws_bytes(4, 0, 4) == 0
