"""Block norms where they can go wrong: gates far from zero, infinities and NaN
in rows whose last channels several threads see, teams of CTAs that take many
rows.  Against 64-bit formulas; tolerances as in test_token_path_gpu.py."""
import math

import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import ttfoil as tf  # noqa: E402
from test_token_path_gpu import (BF, F32, F64, Norm, check_backward, check_forward, gen, grad64, randn,  # noqa: E402
                                 run_backward, run_forward)


@pytest.fixture(autouse=True, scope="module")
def device():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    tf.device_error()


# --------------------------------------------------------------- sigmoid gate ---

def far_gates():
    """bf16 gates from -88 to 88, every one at 1/64 of its binade or finer."""
    g = torch.cat([torch.arange(-88, 89, dtype=F64), torch.linspace(-30, 30, 1871, dtype=F64)])
    return g.to(BF)


def test_forward_gate_is_a_logistic_function_to_the_last_bits():
    """h = scale * act(g) * u with u = 2^30.  exp2 is within 2^-22, the reciprocal
    within 2^-23, at most six operations round (2^-24 each) and the exponent's rest
    is taken to first order (2^-23): below 2^-20.  A value below 2^-126 may be 0."""
    gate = far_gates()
    D = 2048
    assert gate.numel() == D
    u = torch.full((1, D), 2.0 ** 30, dtype=BF)
    h = torch.empty(1, D, dtype=F32, device="cuda")
    tf.block_norm(torch.zeros(1, D, device="cuda"), u.cuda(), h, None, 1, D, gate=gate.cuda().view(1, D),
                  gate_act="sigmoid", scale=1.0)
    ref = 2.0 ** 30 / (1 + torch.exp(-gate.to(F64)))
    err = (h.cpu().to(F64)[0] - ref).abs()
    worst = (err / ref).argmax().item()
    lim = 2.0 ** -20 * ref + 2.0 ** (30 - 126)
    assert (err <= lim).all(), (gate[worst].item(), (err / ref)[worst].item() * 2.0 ** 24)


@pytest.mark.parametrize("gate_rows", [1, 3])
def test_gradient_of_gates_far_from_zero(gate_rows):
    """dgate = act'(g) sum of scale dh u; act' = act(g) act(-g) has no cancellation,
    so nothing but roundings of 32 bits (2^-19 in all) precede the one to bf16.  act'
    below 2^-126 may be 0, which is off by at most 2^-126 scale sum |dh u|."""
    gate = far_gates()
    T, D, n = 6, 2048, 6 // gate_rows
    g = gen(gate_rows)
    dh = randn(g, T, D, dtype=F32).abs() + 0.5
    u = randn(g, T, D).abs() + 0.5
    gates = gate.view(1, D).expand(n, D).contiguous()
    dgate = torch.empty(n, D, dtype=BF, device="cuda")
    ws = torch.empty(tf.block_norm_grad_ws_bytes(T, D, gate_rows) + 16, dtype=torch.uint8, device="cuda")
    tf.block_norm_grad(dh.cuda(), None, None, u.cuda(), None, None, T, D, ws, gate=gates.cuda(), dgate=dgate,
                       gate_rows=gate_rows, gate_act="sigmoid", scale=0.5)
    a = gate.to(F64)
    slope = 1 / ((1 + torch.exp(-a)) * (1 + torch.exp(a)))
    total = 0.5 * (dh.to(F64) * u.to(F64)).view(n, gate_rows, D).sum(1)
    ref = slope * total
    err = (dgate.cpu().to(F64) - ref).abs()
    lim = 2.0 ** -8 * (1 + 2.0 ** -7) * ref + 2.0 ** -19 * ref + 2.0 ** -126 * total
    worst = (err / lim).max(0).values.argmax().item()
    assert (err <= lim).all(), (gate[worst].item(), (err / lim)[:, worst])


def test_gates_without_end():
    """Infinite gates open and close, a NaN stays in its channel."""
    D = 264
    gate = randn(gen(1), 2, D)
    gate[0, 3], gate[0, 100], gate[1, 263], gate[1, 5] = math.inf, -math.inf, math.nan, 3.0e38
    u = randn(gen(2), 2, D)
    h = torch.empty(2, D, dtype=F32, device="cuda")
    tf.block_norm(torch.ones(2, D, device="cuda"), u.cuda(), h, None, 2, D, gate=gate.cuda(), gate_act="sigmoid")
    h = h.cpu()
    assert h[0, 3] == 1 + u[0, 3].float() and h[0, 100] == 1 and h[1, 5] == 1 + u[1, 5].float()
    assert torch.isnan(h[1, 263]) and torch.isnan(h).sum() == 1
    dgate, du = (torch.empty(2, D, dtype=BF, device="cuda") for _ in range(2))
    ws = torch.empty(tf.block_norm_grad_ws_bytes(2, D, 1) + 16, dtype=torch.uint8, device="cuda")
    tf.block_norm_grad(torch.ones(2, D, device="cuda"), None, None, u.cuda(), None, du, 2, D, ws, gate=gate.cuda(),
                       dgate=dgate, gate_act="sigmoid")
    dgate, du = dgate.cpu(), du.cpu()
    assert dgate[0, 3] == 0 and dgate[0, 100] == 0 and dgate[1, 5] == 0
    assert du[0, 3] == 1 and du[0, 100] == 0 and du[1, 5] == 1
    assert torch.isnan(du[1, 263]) and torch.isnan(du).sum() == 1
    assert torch.isnan(dgate[1, 263]) and torch.isnan(dgate).sum() == 1
