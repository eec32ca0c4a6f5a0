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


@pytest.mark.parametrize("D", [2048, 2046, 2047])  # vectors of 8, 2 and 1
def test_forward_gate_is_a_logistic_function_to_the_last_bits(D):
    """h = scale * act(g) * u with u = 2^30.  exp2 is within 2^-22, the reciprocal
    within 2^-23, at most six operations round (2^-24 each) and the exponent's rest
    is taken to first order (2^-23): below 2^-20.  A value below 2^-126 may be 0."""
    gate = far_gates()[-D:]
    u = torch.full((1, D), 2.0 ** 30, dtype=BF)
    h = torch.empty(1, D, dtype=F32, device="cuda")
    tf.block_norm(torch.zeros(1, D, device="cuda"), u.cuda(), h, None, 1, D, gate=gate.cuda().view(1, D),
                  gate_act="sigmoid", scale=1.0)
    ref = 2.0 ** 30 / (1 + torch.exp(-gate.to(F64)))
    err = (h.cpu().to(F64)[0] - ref).abs()
    worst = (err / ref).argmax().item()
    lim = 2.0 ** -20 * ref + 2.0 ** (30 - 126)
    assert (err <= lim).all(), (gate[worst].item(), (err / ref)[worst].item() * 2.0 ** 24)


@pytest.mark.parametrize("D", [2048, 2046, 2047])
@pytest.mark.parametrize("gate_rows", [1, 3])
def test_gradient_of_gates_far_from_zero(gate_rows, D):
    """dgate = act'(g) sum of scale dh u; act' = act(g) act(-g) has no cancellation,
    so nothing but roundings of 32 bits (2^-19 in all) precede the one to bf16.  act'
    below 2^-126 may be 0, which is off by at most 2^-126 scale sum |dh u|."""
    gate = far_gates()[:D]
    T, n = 6, 6 // gate_rows
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


@pytest.mark.parametrize("D", [264, 266, 267])
def test_gates_without_end(D):
    """Infinite gates open and close, a NaN stays in its channel."""
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


# ------------------------------------------------------------ non-finite rows ---

def kinds(t):
    """0 for a number, 1 and 2 for an infinity by its sign, 3 for NaN."""
    t = t.cpu().to(F64)
    return torch.isnan(t) * 3 + torch.isposinf(t) * 1 + torch.isneginf(t) * 2


# Threads past D: none, in a warp's teams, in a CTA, in a cluster; vectors of 8, 2, 1.
ODD = [(24, False), (24, True), (34, False), (50, False), (258, False), (51, True), (200, False), (1000, True),
       (2050, False), (2049, False), (4104, True), (4104, False), (8200, False), (5001, True)]


@pytest.mark.parametrize("D,fp32", ODD)
@pytest.mark.parametrize("where,gate_rows", [("dy", 0), ("dy", 1), ("h", 0), ("h", 2), ("dh", 0), ("dh", 1)])
def test_gradient_of_an_infinity_in_the_last_channel(D, fp32, where, gate_rows):
    """It makes infinities and NaN where the formula does, in its row only."""
    T, row = 5, 2
    p = Norm(T, D, fp32, True, gate_rows, "sigmoid" if gate_rows else "none", seed=3)
    saved = run_forward(p)
    base = run_backward(p, saved)
    if where == "h":
        saved["h"][row, D - 1] = math.inf
    else:
        getattr(p, where)[row, D - 1] = math.inf
    out = run_backward(p, saved)
    ref = grad64(p, saved["h"].cpu(), saved["rstd_pre"].cpu(), saved["rstd_post"].cpu())
    assert torch.equal(kinds(out["dresid"]), kinds(ref["dresid"][0]))
    if where == "dh":
        assert torch.equal(kinds(out["du"]), kinds(ref["du"][0]))
    keep = [t for t in range(T) if t != row]
    for k in ("dresid", "du"):
        assert torch.equal(out[k][keep], base[k][keep]), k


@pytest.mark.parametrize("D,fp32", ODD)
@pytest.mark.parametrize("gate_rows", [0, 1, 2])
def test_gradient_without_post_norm_does_not_look_at_the_output(D, fp32, gate_rows):
    """du = scale act dh' where there is no post norm, whatever u holds."""
    T = 5
    p = Norm(T, D, fp32, False, gate_rows, "none", seed=5)
    saved = run_forward(p)
    base = run_backward(p, saved, want=("dresid", "du"))
    p.u[2, D - 1], p.u[3, 0], p.u[4] = math.inf, math.nan, -math.inf
    out = run_backward(p, saved, want=("dresid", "du"))
    for k in ("dresid", "du"):
        assert torch.isfinite(base[k]).all() and torch.equal(out[k], base[k]), k


# --------------------------------------------------- many rows of one CTA's team ---

@pytest.mark.parametrize("T,D", [(900, 2049), (1100, 2048), (700, 5120), (400, 8200), (330, 16384), (700, 3000)])
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("gate_rows", [1, 7])
def test_forward_of_more_rows_than_teams(T, D, fp32, gate_rows):
    """Teams of a CTA and of a cluster go on to other rows: sums in turn, rows asked
    for ahead."""
    p = Norm(T, D, fp32, True, gate_rows, "sigmoid")
    check_forward(p, run_forward(p))


@pytest.mark.parametrize("T,D", [(700, 2050), (500, 4096), (400, 4104), (300, 8200), (120, 16384), (250, 4097)])
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("gate_rows", [0, 1, 50])
def test_gradient_of_more_rows_than_teams(T, D, fp32, gate_rows):
    p = Norm(T, D, fp32, True, gate_rows, "sigmoid" if gate_rows == 1 else "none")
    saved = run_forward(p)
    check_backward(p, saved, run_backward(p, saved))
