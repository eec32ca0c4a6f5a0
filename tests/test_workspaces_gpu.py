"""One workspace, made for the largest batch, serves the smaller ones: no call
touches what lies behind the size for its own tokens."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import ttfoil as tf  # noqa: E402
from test_token_path_gpu import (BF, F32, Norm, check_backward, close, embed_grad, embed_ref, gen,  # noqa: E402
                                 make_ids, randn, run_backward, run_forward)


@pytest.fixture(autouse=True, scope="module")
def device():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    tf.device_error()


@pytest.mark.parametrize("D,gate_rows", [(264, 0), (264, 1), (264, 37), (264, 1 << 30), (2050, 2), (4104, 50), (64, 3)])
def test_block_norm_gradient_of_fewer_tokens(D, gate_rows):
    most = 400
    ws = torch.full((tf.block_norm_grad_ws_bytes(most, D, gate_rows),), 255, dtype=torch.uint8, device="cuda")
    for T in (most, 297, 296, 149, 148, 75, 37, 5, 1):
        need = tf.block_norm_grad_ws_bytes(T, D, gate_rows)
        assert need <= ws.numel()
        ws.fill_(255)
        p = Norm(T, D, False, True, gate_rows, "sigmoid" if gate_rows else "none")
        saved = run_forward(p)
        check_backward(p, saved, run_backward(p, saved, ws=ws))
        assert (ws[need:] == 255).all(), T


@pytest.mark.parametrize("D", [40, 2050])
def test_embed_rows_gradient_of_fewer_tokens(D):
    V, most = 500, 17000
    ws = torch.empty(tf.embed_rows_grad_ws_bytes(most, V, D), dtype=torch.uint8, device="cuda")
    for T in (most, 16385, 16383, 8192, 8191, 4095, 4096, 40, 33, 32, 1):
        need = tf.embed_rows_grad_ws_bytes(T, V, D)
        assert need <= ws.numel()
        ws.fill_(255)
        g = gen(T)
        ids = make_ids(g, T, V, "frequent")
        dout = randn(g, T, D, dtype=BF)
        got = embed_grad(ids.cuda(), dout.cuda(), V, 1.3, ws=ws)
        ref, slack = embed_ref(ids, dout, V, 1.3)
        close(got, ref, slack, F32)
        assert (ws[need:] == 255).all(), T
