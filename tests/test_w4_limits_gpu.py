"""4-bit weights at the limits of their range: subnormal and overflowing groups,
rows of x near the largest and the smallest bf16 numbers, in every size of batch.
Against 64-bit formulas; tolerances as in test_token_path_gpu.py."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import ttfoil as tf  # noqa: E402
from test_token_path_gpu import (BF, F64, close, gen, make_weights, matvec_slack, pack, quantized, randn,  # noqa: E402
                                 real_weights, tile, untile)


@pytest.fixture(autouse=True, scope="module")
def device():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    tf.device_error()


def quantize(w, group, zeros):
    K, N = w.shape
    packed = torch.empty(tf.w4_packed_bytes(K, N, group, zeros), dtype=torch.uint8, device="cuda")
    tf.w4_quantize_tiles(tile(w).cuda(), packed, K // 32, N // 32, group, zeros=zeros)
    return packed


def dequantize(packed, K, N, group, zeros):
    out = torch.empty(K * N, dtype=BF, device="cuda")
    tf.w4_dequantize_tiles(packed, out, K, N, group, zeros=zeros)
    return untile(out.cpu(), K, N)[0]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_groups_of_subnormal_weights(group, zeros):
    """Every largest magnitude m 2^-133, m = 1 to 256, of both signs: the scale has
    few bits there, so w / s reaches 10 and the clamp counts."""
    g = gen(group)
    K, N = 128, 512
    m = torch.arange(1, N // 2 + 1, dtype=F64).repeat_interleave(2)
    part = torch.randint(-1000, 1001, (K, N), generator=g).to(F64) / 1000
    units = torch.trunc(part * m)
    sign = torch.tensor([1.0, -1.0], dtype=F64).repeat(N // 2)
    for k0 in range(0, K, group):
        units[k0 + 5] = m * sign
    w = (units * 2.0 ** -133).to(BF)
    assert torch.equal(w.to(F64), units * 2.0 ** -133)  # whole multiples, up to 8 bits
    got = dequantize(quantize(w, group, zeros), K, N, group, zeros)
    assert torch.equal(got, quantized(w, group, zeros).to(BF))
