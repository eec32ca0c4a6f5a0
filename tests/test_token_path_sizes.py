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


@pytest.mark.parametrize("D", [8, 64, 250, 264, 2050, 4096, 8200, 16384])
@pytest.mark.parametrize("gate_rows", [0, 1, 2, 37, 1000, 1 << 30])
def test_block_norm_workspace_grows_with_the_tokens(D, gate_rows):
    need = [ttfoil.block_norm_grad_ws_bytes(T, D, gate_rows) for T in range(1, 3000)]
    assert all(a <= b for a, b in zip(need, need[1:]))
    for T in (149, 297, 5000, 18945, 70001):
        top = ttfoil.block_norm_grad_ws_bytes(T, D, gate_rows)
        for t in (n for n in (1, 2, 3, 36, 37, 148, 296, T // 3, T // 2, T - 1) if n < T):
            assert ttfoil.block_norm_grad_ws_bytes(t, D, gate_rows) <= top
            if gate_rows > 1:  # one vector for all tokens: gate_rows follows T
                assert ttfoil.block_norm_grad_ws_bytes(t, D, t) <= top


@pytest.mark.parametrize("D", [1, 64, 2048, 2049, 4096, 10000, 1 << 18, 1 << 20])
def test_embed_rows_workspace_grows_with_the_tokens(D):
    need = [ttfoil.embed_rows_grad_ws_bytes(T, 65536, D) for T in range(1, 18000)]
    assert all(a <= b for a, b in zip(need, need[1:]))
    assert need[-1] <= ttfoil.embed_rows_grad_ws_bytes(1 << 24, 65536, D)
