"""Refusals and size queries of the token-path operators (w4_*, block_norm*,
embed_rows*): every check precedes any CUDA call, so they run without a GPU on
addresses that are never dereferenced."""
import ctypes

import pytest

BASE = 1 << 40


def at(i):
    """The i-th of a set of addresses far from one another."""
    return BASE + (i << 36)


@pytest.fixture(scope="module")
def L():
    import ttfoil
    return ttfoil.lib()


def refused(L, rc, text):
    assert rc == 1, rc
    assert text in L.foil_last_error().decode(), L.foil_last_error()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [0, 1])
def test_w4_packed_bytes(L, group, zeros):
    block = 1024 + 128 // group * 16 * (3 if zeros else 2)
    assert L.foil_w4_packed_bytes(1, 1, group, zeros) == block
    assert L.foil_w4_packed_bytes(128, 16, group, zeros) == block
    assert L.foil_w4_packed_bytes(129, 17, group, zeros) == 4 * block
    assert L.foil_w4_packed_bytes(1 << 24, 1 << 24, group, zeros) == (1 << 17) * (1 << 20) * block
    assert L.foil_w4_packed_bytes(0, 16, group, zeros) == 0
    assert L.foil_w4_packed_bytes(16, 0, group, zeros) == 0
    assert L.foil_w4_packed_bytes((1 << 24) + 1, 16, group, zeros) == 0
    assert L.foil_w4_packed_bytes(128, 16, 16, zeros) == 0


def test_w4_refusals(L):
    x, w, y, b = at(0), at(1), at(2), at(3)

    def mv(x=x, ld_x=0, w=w, bias=None, y=y, ld_y=0, M=2, K=256, N=64, group=64, zeros=0):
        return L.foil_w4_matvec_dev(x, ld_x, w, bias, y, ld_y, M, K, N, group, zeros, 0, None)

    refused(L, mv(group=48), "group must be")
    refused(L, mv(K=0), "from 1 to 2^24")
    refused(L, mv(K=32769), "at most 32768")
    refused(L, mv(M=65), "at most 64 rows")
    refused(L, mv(x=None), "null")
    refused(L, mv(w=w + 8), "misaligned")
    refused(L, mv(x=x + 1), "misaligned")
    refused(L, mv(bias=b + 1), "misaligned")
    refused(L, mv(ld_x=255), "row stride")
    refused(L, mv(ld_y=63), "row stride")
    refused(L, mv(ld_y=1 << 46), "too large")
    refused(L, mv(y=x), "overlaps an input")
    refused(L, mv(y=w + 1024), "overlaps an input")
    refused(L, mv(bias=y), "overlaps an input")
    # x and y as neighbouring column slices of one buffer, but one column in common
    refused(L, mv(x=x, ld_x=400, y=x + 2 * 255, ld_y=400), "overlaps an input")
    assert mv(M=0) == 0 and mv(N=0) == 0

    refused(L, L.foil_w4_pack_dev(None, b, None, w, 64, 64, 64, None), "null")
    refused(L, L.foil_w4_pack_dev(x, b + 1, None, w, 64, 64, 64, None), "misaligned")
    refused(L, L.foil_w4_pack_dev(x, b, None, w, 0, 64, 64, None), "from 1 to 2^24")
    refused(L, L.foil_w4_pack_dev(w + 100, b, None, w, 64, 64, 64, None), "overlaps")
    refused(L, L.foil_w4_quantize_tiles_dev(x, w, 70000, 1, 64, 0, None), "tile counts")
    refused(L, L.foil_w4_quantize_tiles_dev(x, w, 1, 1, 65, 0, None), "group must be")
    refused(L, L.foil_w4_quantize_tiles_dev(x + 8, w, 1, 1, 64, 0, None), "misaligned")
    refused(L, L.foil_w4_quantize_tiles_dev(w, w, 1, 1, 64, 0, None), "overlaps")
    refused(L, L.foil_w4_dequantize_tiles_dev(w, x, 64, 64, 100, 0, 0, None), "group must be")
    refused(L, L.foil_w4_dequantize_tiles_dev(w, None, 64, 64, 64, 0, 0, None), "null")
    refused(L, L.foil_w4_dequantize_tiles_dev(w, w, 64, 64, 64, 0, 0, None), "overlaps")
    refused(L, L.foil_w4_dequantize_tiles_dev(w, x, 1 << 22, 64, 64, 0, 0, None), "tile counts")
    assert L.foil_w4_quantize_tiles_dev(None, None, 0, 4, 64, 0, None) == 0
    assert L.foil_w4_dequantize_tiles_dev(None, None, 0, 4, 64, 0, 0, None) == 0


def forward_args(**kw):
    a = dict(resid=at(0), ld_resid=0, u=at(1), ld_u=0, post=1, w_post=at(2), gate=at(3), ld_gate=0, gate_rows=1,
             gate_act=0, w_pre=at(4), h=at(5), ld_h=0, y=at(6), ld_y=0, rstd_post=at(7), rstd_pre=at(8), T=4, D=64,
             fp32=0, scale=1.0, eps=1e-5)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values()) + [None]


def test_block_norm_refusals(L):
    def call(**kw):
        return L.foil_block_norm_dev(*forward_args(**kw))

    refused(L, call(D=16385), "at most 16384")
    refused(L, call(resid=None), "null")
    refused(L, call(h=None, y=None, w_pre=None, rstd_pre=None), "null")
    refused(L, call(u=None), "without the block's output")
    refused(L, call(post=0), "without the post norm")
    refused(L, call(y=None), "without y")
    refused(L, call(gate_rows=0), "gate_rows")
    refused(L, call(gate_act=2), "activation")
    refused(L, call(eps=-1.0), "eps")
    refused(L, call(eps=float("nan")), "eps")
    refused(L, call(eps=float("inf")), "eps")
    refused(L, call(w_pre=at(4) + 1), "misaligned")
    refused(L, call(rstd_pre=at(8) + 2), "misaligned")
    refused(L, call(resid=at(0) + 2, fp32=1), "misaligned")
    refused(L, call(ld_u=63), "row stride")
    refused(L, call(y=at(5)), "two outputs overlap")
    refused(L, call(h=at(1)), "overlaps an input")
    refused(L, call(y=at(0)), "overlaps an input")
    refused(L, call(h=at(0) + 2), "overlaps an input")           # shifted, not in place
    refused(L, call(h=at(0), ld_h=65), "overlaps an input")      # another stride
    refused(L, call(y=at(3)), "overlaps an input")
    refused(L, call(rstd_pre=at(0)), "overlaps an input")
    refused(L, call(rstd_pre=at(7)), "two outputs overlap")
    assert call(T=0) == 0 and call(D=0) == 0


def backward_args(**kw):
    a = dict(dh=at(0), ld_dh=0, dy=at(1), ld_dy=0, h=at(2), ld_h=0, rstd_pre=at(3), w_pre=at(4), u=at(5), ld_u=0,
             post=1, rstd_post=at(6), w_post=at(7), gate=at(8), ld_gate=0, gate_rows=1, gate_act=0, dresid=at(9),
             ld_dresid=0, du=at(10), ld_du=0, dgate=at(11), ld_dgate=0, dw_post=at(12), dw_pre=at(13), ws=at(14),
             ws_bytes=1 << 30, T=4, D=64, fp32=0, scale=1.0)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values()) + [None]


def test_block_norm_grad_refusals(L):
    def call(**kw):
        return L.foil_block_norm_grad_dev(*backward_args(**kw))

    refused(L, call(D=16385), "at most 16384")
    refused(L, call(dresid=None, du=None, dgate=None, dw_post=None, dw_pre=None), "no output")
    refused(L, call(dh=None, dy=None), "both null")
    refused(L, call(h=None), "needs h and rstd_pre")
    refused(L, call(rstd_pre=None), "needs h and rstd_pre")
    refused(L, call(dy=None), "without dy")
    refused(L, call(u=None), "need the block's output")
    refused(L, call(rstd_post=None), "rstd_post")
    refused(L, call(post=0), "without the post norm")
    refused(L, call(gate=None), "without a gate")
    refused(L, call(gate_rows=0), "gate_rows")
    refused(L, call(gate_act=7), "activation")
    refused(L, call(dw_pre=at(13) + 1), "misaligned")
    refused(L, call(ld_dy=10), "row stride")
    refused(L, call(dresid=at(0)), "overlaps an input")
    refused(L, call(du=at(5)), "overlaps an input")
    refused(L, call(du=at(9)), "two outputs overlap")
    refused(L, call(ws=at(2)), "overlaps an input")
    need = L.foil_block_norm_grad_ws_bytes(4, 64, 1)
    refused(L, call(ws_bytes=need - 1), "workspace")
    refused(L, call(ws=None), "workspace")
    refused(L, call(ws=at(14) + 8), "workspace")
    assert call(D=0) == 0


def test_embed_rows_refusals(L):
    ids, table, out, ws = at(0), at(1), at(2), at(3)

    def look(ids=ids, idb=4, table=table, ld_t=0, out=out, ld_o=0, T=8, V=100, D=64, fp32=0):
        return L.foil_embed_rows_dev(ids, idb, table, ld_t, out, ld_o, T, V, D, fp32, 1.0, -1, None)

    def grad(ids=ids, idb=4, dout=out, ld_o=0, dtable=table, ld_t=0, T=8, V=100, D=64, fp32=0, ws=ws, n=1 << 30):
        return L.foil_embed_rows_grad_dev(ids, idb, dout, ld_o, dtable, ld_t, T, V, D, fp32, 1.0, -1, 0, ws, n, None)

    for call in (look, grad):
        refused(L, call(idb=2), "id_bytes")
        refused(L, call(T=(1 << 24) + 1), "2^24")
        refused(L, call(V=(1 << 24) + 1), "2^24")
        refused(L, call(ids=None), "null")
        refused(L, call(ids=ids + 4, idb=8), "misaligned")
        refused(L, call(ld_t=63), "row stride")
        refused(L, call(ld_o=63), "row stride")
    refused(L, look(table=None), "null")
    refused(L, look(out=None), "null")
    refused(L, look(out=out + 2, fp32=1), "misaligned")
    refused(L, look(out=table), "overlaps")
    refused(L, look(out=ids), "overlaps")
    assert look(T=0) == 0 and look(D=0) == 0
    refused(L, grad(dout=None), "null")
    refused(L, grad(dtable=None), "null")
    refused(L, grad(dtable=table + 2), "misaligned")
    refused(L, grad(dtable=out), "overlaps")
    need = L.foil_embed_rows_grad_ws_bytes(8, 100, 64)
    if need:
        refused(L, grad(n=need - 1), "workspace")
        refused(L, grad(ws=None), "workspace")
        refused(L, grad(ws=ids), "overlap")
    assert grad(V=0) == 0 and grad(D=0) == 0


def test_counts_that_32_bits_could_not_hold(L):
    many = (1 << 31) + 1
    refused(L, L.foil_block_norm_dev(*forward_args(T=many)), "2^31")
    refused(L, L.foil_block_norm_grad_dev(*backward_args(T=many)), "2^31")
    wide = (1 << 20) + 1
    refused(L, L.foil_embed_rows_dev(at(0), 4, at(1), 0, at(2), 0, 1, 1, wide, 0, 1.0, -1, None), "2^20")
    refused(L, L.foil_embed_rows_grad_dev(at(0), 4, at(2), 0, at(1), 0, 1, 1, wide, 0, 1.0, -1, 0, at(3), 1 << 40,
                                          None), "2^20")
    far = 1 << 32
    refused(L, L.foil_block_norm_dev(*forward_args(ld_u=far)), "too large")
    refused(L, L.foil_embed_rows_dev(at(0), 4, at(1), far, at(2), 0, 1, 1, 64, 0, 1.0, -1, None), "too large")


def test_binding_refuses_tensors_it_cannot_describe():
    import torch
    import ttfoil
    host = torch.zeros(4, 64, dtype=torch.int16)
    with pytest.raises(Exception):  # no CUDA device here, or not a CUDA tensor
        ttfoil.embed_rows(torch.zeros(4, dtype=torch.int32), host, host, 4, 4, 64)
    for bad in (host.t(), host[0].expand(4, 64), host[:, :48].unsqueeze(0)):
        with pytest.raises(ttfoil.FoilError):
            ttfoil._mat(bad, 0, -1)
    with pytest.raises(ttfoil.FoilError):
        ttfoil._mat(host, 0, 0)  # on another device
    with pytest.raises(ttfoil.FoilError):
        ttfoil._vec(host, 0)
    with pytest.raises(ttfoil.FoilError):
        ttfoil._vec(host[:, :3], -1)
    assert ttfoil._mat(host[:, :48], 0, -1)[1] == 64 and ttfoil._mat(host.view(-1), 0, -1)[1] == 0
    assert ttfoil._mat(host[:1, :48], 0, -1)[1] == 0 and ttfoil._mat(None, 5, -1) == (None, 5)
    with pytest.raises(ttfoil.FoilError):
        ttfoil._is_fp32(None, host, torch.zeros(1))
    with pytest.raises(ttfoil.FoilError):
        ttfoil._gate_act("tanh")
    with pytest.raises(ttfoil.FoilError):
        ttfoil._id_bytes(torch.zeros(3), 4)
    assert ctypes.sizeof(ctypes.c_void_p) == 8
