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


def test_quantize_groups_whose_range_overflows_stand_for_nan():
    """lo and hi of one group are numbers, hi - lo is not: NaN as weights and in
    products of few and of many rows; the other columns are as without it."""
    g = gen(8)
    K, group = 256, 64
    w = randn(g, K, 64, std=0.05)
    w[70, 3], w[100, 3] = 3.0e38, -3.0e38
    packed = quantize(w, group, True)
    got = dequantize(packed, K, 64, group, True)
    bad = torch.zeros(K, 64, dtype=torch.bool)
    bad[64:128, 3] = True
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
    for M in (1, 5, 16, 17, 64):
        y = torch.empty(M, 64, dtype=BF, device="cuda")
        x = randn(g, M, K) * 2.0 ** torch.randint(-30, 31, (M, K), generator=g)  # sums that are not exact
        tf.w4_matvec(x.to(BF).cuda(), packed, y, M, K, 64, group, zeros=True)
        assert torch.isnan(y[:, 3]).all(), M
        y[:, 3] = 0
        assert torch.isfinite(y).all(), M


@pytest.mark.parametrize("M", [7, 16, 17, 33, 48, 64])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_matvec_rows_near_both_ends_of_the_range(M, group, zeros):
    """Rows scaled by 2^-118 to 2^120, the ordinary ones among them with the bits
    they have in ordinary company: a batch of any size holds what a row alone holds."""
    g = gen(M + group)
    K, N = 1320, 70
    codes, scales, zp = make_weights(g, K, N, group, zeros)
    w = real_weights(codes, scales, zp, group)
    x = randn(g, M, K).clamp(-8, 8)
    packed = pack(codes, scales, zp, group)
    plain = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(x.cuda(), packed, plain, M, K, N, group, zeros=zeros)
    powers = ([0, 60, -80, 119, -118, 0, 23, 110, -100, 100] * 7)[:M]
    scale = torch.tensor([2.0 ** p for p in powers], dtype=F64)[:, None]
    xs = (x.to(F64) * scale).to(BF)
    y = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(xs.cuda(), packed, y, M, K, N, group, zeros=zeros)
    close(y.cpu().to(F64) / scale, (xs.to(F64) / scale) @ w.t(),
          matvec_slack(xs.to(F64) / scale, codes, scales, zp, group, w), BF)
    for m in range(M):
        if powers[m] == 0:
            assert torch.equal(y[m].view(torch.int16), plain[m].view(torch.int16)), m


@pytest.mark.parametrize("M", [1, 12, 17, 40, 64])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_matvec_of_the_largest_numbers(M, group):
    """The largest bf16 number in every place against the largest codes: sums of a
    group reach 15 group 2^128, the scales bring them back."""
    K, N = 2 * group, 16
    big = torch.finfo(BF).max
    codes = torch.full((N, K), 15, dtype=torch.uint8)
    scales = torch.full((N, 2), 2.0 ** -20, dtype=BF)
    zp = torch.zeros(N, 2, dtype=torch.uint8)
    x = torch.full((M, K), big, dtype=BF)
    x[M // 2] *= -1
    y = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(x.cuda(), pack(codes, scales, zp, group), y, M, K, N, group, zeros=True)
    w = real_weights(codes, scales, zp, group)
    ref = x.to(F64) @ w.t()
    close(y, ref, matvec_slack(x, codes, scales, zp, group, w), BF)


@pytest.mark.parametrize("M", [6, 16, 40, 64])
def test_matvec_rows_do_not_depend_on_their_company(M):
    """Another row's values change nothing of a row's bits in a batch of one size;
    a row of a batch and the row by itself agree within both calls' bounds."""
    g = gen(M)
    K, N, group = 4104, 330, 32
    codes, scales, zp = make_weights(g, K, N, group, True)
    w = real_weights(codes, scales, zp, group)
    packed = pack(codes, scales, zp, group)
    x = randn(g, M, K)
    a, b, one = (torch.empty(m, N, dtype=BF, device="cuda") for m in (M, M, 1))
    tf.w4_matvec(x.cuda(), packed, a, M, K, N, group, zeros=True)
    other = randn(g, M, K)
    other[3] = x[3]
    tf.w4_matvec(other.cuda(), packed, b, M, K, N, group, zeros=True)
    assert torch.equal(a[3].view(torch.int16), b[3].view(torch.int16))
    tf.w4_matvec(x[3:4].cuda(), packed, one, 1, K, N, group, zeros=True)
    ref, slack = x[3:4].to(F64) @ w.t(), matvec_slack(x[3:4], codes, scales, zp, group, w)
    close(one, ref, slack, BF)
    close(a[3:4], ref, slack, BF)
