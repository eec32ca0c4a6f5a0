"""Workspace sizes and the checks of tensors that the token-path operators make
before any CUDA call; they run without a GPU."""
import pytest

import ttfoil


@pytest.mark.parametrize("T,D,gate_rows", [(4, 16385, 0), (4, 1 << 20, 0), (1, (1 << 32) - 1, 1),
                                           ((1 << 31) + 1, 64, 0), ((1 << 32) - 1, 64, 0), ((1 << 32) - 1, 1, 7),
                                           ((1 << 32) - 1, 16384, 1 << 30)])
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


# ------------------------------------------------ tensors the calls refuse ---

@pytest.fixture
def host(monkeypatch):
    """The Python calls with tensors of the host (device -1) and a library that only
    counts: what is wrong has to be found before it is called."""
    import torch
    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, args)) or 0

    monkeypatch.setattr(ttfoil, "_place", lambda stream: (-1, 0))
    monkeypatch.setattr(ttfoil, "_lib", Library())

    def zeros(*shape, dtype="bfloat16"):
        return torch.zeros(*shape, dtype=getattr(torch, dtype))

    return calls, zeros


def each_refused(calls, call, args, wrong):
    """`call` runs with `args` and not with any one of the `wrong` ones in place."""
    call(**args)
    assert len(calls) == 1
    for name, values in wrong.items():
        for v in values:
            with pytest.raises(ttfoil.FoilError):
                call(**{**args, name: v})
            assert len(calls) == 1, (name, v.dtype, v.shape)


def test_w4_calls_refuse_tensors_of_another_type_or_too_short(host):
    calls, z = host
    K, N, M, group = 100, 40, 3, 32
    packed = z(3 * (1024 + 4 * 48), dtype="uint8")
    each_refused(calls, lambda **a: ttfoil.w4_matvec(M=M, K=K, N=N, group=group, zeros=True, **a),
                 dict(x=z(M, K), packed=packed, y=z(M, N), bias=z(N)),
                 dict(x=[z(M, K, dtype="float16"), z(M, K, dtype="float32"), z(M - 1, K), z(M, K - 1), z(M * K - 1),
                         z(1, M, 2 * K), z(M, K + 1, dtype="float64")[:, :K]],
                      packed=[packed[:-1], z(5000, dtype="int32"), z(5000)],
                      y=[z(M, N, dtype="float32"), z(M - 1, N), z(M, N - 1), z(4, N + 3)[:2, :N]],
                      bias=[z(N - 1), z(N, dtype="float32"), z(N, dtype="float16")]))
    for ld, ok in ((101, True), (102, False)):  # a row stride of the caller's
        x = z(2 * 101 + K)
        if ok:
            ttfoil.w4_matvec(x, packed, z(M, N), M, K, N, group, zeros=True, ld_x=ld)
        else:
            with pytest.raises(ttfoil.FoilError):
                ttfoil.w4_matvec(x, packed, z(M, N), M, K, N, group, zeros=True, ld_x=ld)


def test_w4_conversions_refuse_tensors_of_another_type_or_too_short(host):
    calls, z = host
    K, N, group = 64, 32, 64
    packed = z(2 * (1024 + 64), dtype="uint8")
    each_refused(calls, lambda **a: ttfoil.w4_pack(K=K, N=N, group=group, **a),
                 dict(codes=z(N, K, dtype="uint8"), scales=z(N, 1), packed=packed),
                 dict(codes=[z(N, K - 1, dtype="uint8"), z(N, K, dtype="int32")],
                      scales=[z(N - 1, 1), z(N, 1, dtype="float32")], packed=[packed[1:], z(2000)],
                      zero_points=[z(N - 1, 1, dtype="uint8"), z(N, 1)]))
    for call, own in ((lambda **a: ttfoil.w4_quantize_tiles(Kt=2, Nt=1, group=group, **a), z(2048)),
                      (lambda **a: ttfoil.w4_dequantize_tiles(K=K, N=N, group=group, **a), z(2048)),
                      (lambda **a: ttfoil.w4_dequantize_tiles(K=33, N=N, group=group, transpose=True, **a), z(2048))):
        calls.clear()
        each_refused(calls, call, dict(tiles=own, packed=packed),
                     dict(tiles=[own[:-1], z(2048, dtype="float32")], packed=[packed[1:], z(2176)]))


def test_block_norm_refuses_tensors_of_another_type_or_too_short(host):
    calls, z = host
    T, D = 5, 24
    short = dict(u=[z(T - 1, D), z(T, D, dtype="float32"), z(T, D, dtype="float16")],
                 w_post=[z(D - 1), z(D, dtype="float32")], w_pre=[z(D - 1), z(D, dtype="float16")],
                 gate=[z(2, D), z(3, D, dtype="float32")], rstd_post=[z(T), z(T - 1, dtype="float32")],
                 rstd_pre=[z(T), z(T - 1, dtype="float32")], h=[z(T, D, dtype="float32"), z(T, D - 8)])
    same = dict(u=z(T, D), w_post=z(D), w_pre=z(D), gate=z(3, D), rstd_post=z(T, dtype="float32"),
                rstd_pre=z(T, dtype="float32"), h=z(T, D))
    kw = dict(T=T, D=D, post=True, gate_rows=2)
    each_refused(calls, lambda **a: ttfoil.block_norm(**kw, **a), dict(same, resid=z(T, D), y=z(T, D)),
                 dict(short, resid=[z(T - 1, D), z(T, D, dtype="float16"), z(T, D, dtype="float64")],
                      y=[z(T, D, dtype="float32"), z(T - 1, D)]))
    calls.clear()
    f = dict(dtype="float32")
    each_refused(calls, lambda **a: ttfoil.block_norm_grad(**kw, **a),
                 dict(same, dh=z(T, D), dy=z(T, D), dresid=z(T, D), du=z(T, D), dgate=z(3, D), dw_post=z(D, **f),
                      dw_pre=z(D, **f), ws=z(1000, dtype="uint8")),
                 dict(short, dh=[z(T - 1, D), z(T, D, **f)], dy=[z(T, D, **f)], dresid=[z(T, D, **f), z(2, D)],
                      du=[z(T, D, **f), z(T - 1, D)], dgate=[z(2, D), z(3, D, **f)], dw_post=[z(D), z(D - 1, **f)],
                      dw_pre=[z(D), z(D - 1, **f)]))
    with pytest.raises(ttfoil.FoilError):
        ttfoil._ws_bytes(z(10, dtype="uint8"), 11)


def test_embed_rows_refuses_tensors_of_another_type_or_too_short(host):
    calls, z = host
    T, V, D = 5, 7, 24
    ids = z(T, dtype="int64")
    bad_ids = [ids[1:], z(T), z(T, dtype="float32"), z(T, dtype="complex64"), z(T, dtype="bool"), z(T, dtype="int16")]
    each_refused(calls, lambda **a: ttfoil.embed_rows(T=T, V=V, D=D, **a), dict(ids=ids, table=z(V, D), out=z(T, D)),
                 dict(ids=bad_ids, table=[z(V - 1, D), z(V, D, dtype="float32"), z(V, D, dtype="float16")],
                      out=[z(T - 1, D), z(T, D, dtype="float16"), z(T, D, dtype="float64")]))
    calls.clear()
    f = dict(dtype="float32")
    each_refused(calls, lambda **a: ttfoil.embed_rows_grad(T=T, V=V, D=D, **a),
                 dict(ids=ids, dout=z(T, D), dtable=z(V, D, **f), ws=z(1000, dtype="uint8")),
                 dict(ids=bad_ids, dout=[z(T - 1, D), z(T, D, dtype="float16")],
                      dtable=[z(V, D), z(V - 1, D, **f), z(V, D, dtype="float64")]))


def test_calls_accept_larger_tensors_and_bits(host):
    """More rows, wider rows, dense vectors, bf16 as 16-bit integers."""
    calls, z = host
    packed = z(1024 + 64, dtype="uint8")
    for x in (z(9, 64), z(4, 100), z(4, 100)[:, 3:67], z(4 * 64), z(2, 2, 64), z(4, 64, dtype="int16")):
        ttfoil.w4_matvec(x, packed, z(4, 16), 4, 64, 16, 64)
    assert [c[1][1] for c in calls] == [0, 100, 100, 0, 0, 0]
