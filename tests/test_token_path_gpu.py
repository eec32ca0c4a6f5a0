"""Parity of the token-path operators (4-bit weights, block norms, embedding
rows and their gradients) with plain 64-bit implementations on the CPU.

Tolerances count roundings: an output of b significant bits is off by at most
half a step, HALF[dtype] relative to its value; fp32 sums and products add the
error bounds written at each comparison (2^-24 relative for an operation).
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import ttfoil as tf  # noqa: E402

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}
TINY = 2.0 ** -120


@pytest.fixture(autouse=True, scope="module")
def device():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    tf.device_error()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def close(got, ref, slack, dtype, what=""):
    """|got - ref| within half a step of the output's type plus `slack`."""
    got = got.detach().cpu().to(F64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(ref).all() and torch.isfinite(got).all(), what
    err = (got - ref).abs()
    lim = HALF[dtype] * ref.abs() * (1 + 2.0 ** -7) + slack + TINY
    worst = (err / lim).max().item() if err.numel() else 0.0
    assert worst <= 1.0, (what, worst)


# ------------------------------------------------------------ 4-bit weights ---

def make_weights(g, K, N, group, zeros):
    groups = -(-K // group)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(N, groups, generator=g) + 0.5) * 0.1).to(BF)
    zp = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, zp


def real_weights(codes, scales, zp, group):
    """(N, K) in 64 bits."""
    K = codes.shape[1]
    s = scales.to(F64).repeat_interleave(group, 1)[:, :K]
    z = zp.to(F64).repeat_interleave(group, 1)[:, :K] if zp is not None else 8.0
    return (codes.to(F64) - z) * s


def pack(codes, scales, zp, group, fill=0):
    N, K = codes.shape
    packed = torch.full((tf.w4_packed_bytes(K, N, group, zp is not None),), fill, dtype=torch.uint8, device="cuda")
    tf.w4_pack(codes.cuda(), scales.cuda(), packed, K, N, group, zero_points=zp.cuda() if zp is not None else None)
    return packed


def matvec_slack(x, codes, scales, zp, group, w):
    """Error bound of the sums.  A group's partial sum of (16 + q) x and its
    correction (16 + z) sum(x) are each at most 31 sum|x|; the matrix pipe adds
    in steps of 16 with at most 2^-23 relative error of the partial sum each.
    The groups' sums are then added in fp32: at most K / group + 16 additions of
    2^-24 relative to sum |w x|."""
    K = codes.shape[1]
    xa = x.to(F64).abs()
    sa = scales.to(F64).repeat_interleave(group, 1)[:, :K]
    per_group = (group / 16 + 2) * 62 * 2.0 ** -23 * (xa @ sa.t())
    return per_group + (K / group + 18) * 2.0 ** -24 * (xa @ w.abs().t())


def check_matvec(M, K, N, group, zeros, bias, relu, seed=0, ld_x=0, x_off=0, ld_y=0, y_off=0):
    g = gen(seed)
    codes, scales, zp = make_weights(g, K, N, group, zeros)
    w = real_weights(codes, scales, zp, group)
    x = randn(g, M, K)
    b = randn(g, N, std=0.5) if bias else None
    packed = pack(codes, scales, zp, group)
    lx, ly = ld_x or K, ld_y or N
    xb = torch.full((x_off + M * lx,), float("nan"), dtype=BF, device="cuda")
    xv = xb[x_off:].view(M, lx)[:, :K]
    xv.copy_(x)
    yb = torch.full((y_off + M * ly,), 77.0, dtype=BF, device="cuda")
    yv = yb[y_off:].view(M, ly)[:, :N]
    tf.w4_matvec(xv, packed, yv, M, K, N, group, zeros=zeros, bias=b.cuda() if bias else None, relu=relu, ld_x=ld_x,
                 ld_y=ld_y)
    ref = x.to(F64) @ w.t()
    if bias:
        ref = ref + b.to(F64)
    if relu:
        ref = ref.clamp(min=0)
    close(yv, ref, matvec_slack(x, codes, scales, zp, group, w), BF, "matvec")
    rest = yb.clone()
    rest[y_off:].view(M, ly)[:, :N] = 77.0
    assert (rest == 77.0).all(), "wrote outside its rows"
    return packed


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 31, 15), (1, 128, 16), (2, 129, 17), (3, 256, 100), (7, 300, 40),
                                   (8, 1000, 129), (9, 512, 64), (16, 2050, 33), (17, 640, 48), (33, 200, 31),
                                   (64, 384, 272)])
def test_matvec_shapes(M, K, N, group, zeros):
    check_matvec(M, K, N, group, zeros, bias=N % 2 == 1, relu=K % 2 == 1, seed=M + K + N)


@pytest.mark.parametrize("M,K,N,group,zeros", [(1, 4096, 4096, 128, False), (1, 8192, 1000, 64, True),
                                               (4, 4096, 11000, 32, True), (5, 14344, 520, 128, True),
                                               (16, 8192, 2048, 64, False), (1, 32768, 160, 128, False),
                                               (16, 32768, 96, 32, True), (8, 32767, 50, 64, True),
                                               (64, 4096, 1024, 128, False), (2, 96, 70000, 64, False)])
def test_matvec_large(M, K, N, group, zeros):
    check_matvec(M, K, N, group, zeros, bias=True, relu=False, seed=K)


@pytest.mark.parametrize("x_off,ld_x,y_off,ld_y", [(1, 0, 0, 0), (0, 517, 3, 0), (8, 520, 0, 130), (0, 0, 1, 201),
                                                   (3, 519, 5, 133)])
@pytest.mark.parametrize("M", [1, 6, 20])
def test_matvec_strides(M, x_off, ld_x, y_off, ld_y):
    check_matvec(M, 515, 129, 64, True, bias=True, relu=False, x_off=x_off, ld_x=ld_x, y_off=y_off, ld_y=ld_y)


@pytest.mark.parametrize("M,K,N,group,zeros", [(3, 200, 37, 64, True), (16, 1300, 70, 32, False)])
def test_matvec_ignores_what_lies_past_the_weights(M, K, N, group, zeros):
    """Any finite codes, scales and zero points past K and N: the same bits."""
    g = gen(5)
    codes, scales, zp = make_weights(g, K, N, group, zeros)
    x = randn(g, M, K).cuda()
    Kp, Np = -(-K // 128) * 128, -(-N // 16) * 16
    full_c = torch.randint(0, 16, (Np, Kp), generator=g, dtype=torch.uint8)
    full_s = randn(g, Np, Kp // group, std=3.0)
    full_z = torch.randint(0, 16, (Np, Kp // group), generator=g, dtype=torch.uint8) if zeros else None
    full_c[:N, :K] = codes
    full_s[:N, :scales.shape[1]] = scales
    if zeros:
        full_z[:N, :scales.shape[1]] = zp
    out = []
    for c, s, z in ((codes, scales, zp), (full_c, full_s, full_z)):
        y = torch.empty(M, N, dtype=BF, device="cuda")
        tf.w4_matvec(x, pack(c, s, z, group), y, M, K, N, group, zeros=zeros)
        out.append(y)
    assert torch.equal(out[0].view(torch.int16), out[1].view(torch.int16))


def test_matvec_non_finite_rows_stay_apart():
    """An infinity or NaN in one row of x leaves the other rows as they are."""
    g = gen(6)
    K, N, group = 1000, 100, 64
    codes, scales, zp = make_weights(g, K, N, group, True)
    packed = pack(codes, scales, zp, group)
    x = randn(g, 4, K)
    y0, y1 = (torch.empty(4, N, dtype=BF, device="cuda") for _ in range(2))
    tf.w4_matvec(x.cuda(), packed, y0, 4, K, N, group, zeros=True)
    x[1, 999] = float("nan")
    x[3, 0] = float("inf")
    tf.w4_matvec(x.cuda(), packed, y1, 4, K, N, group, zeros=True)
    assert torch.equal(y0[[0, 2]].view(torch.int16), y1[[0, 2]].view(torch.int16))
    assert torch.isnan(y1[1]).all() and not torch.isfinite(y1[3]).any()


# More than 16 rows, x in whole 16-byte pieces: one block of k and many, its
# second half without values, columns past the last tile, splits of K.
@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("M,K,N", [(17, 8, 1), (64, 64, 16), (31, 72, 127), (33, 128, 128), (48, 136, 129), (32, 1024, 300),
                                   (63, 1928, 40), (64, 4104, 1000), (18, 8192, 260), (50, 16384, 130)])
def test_matvec_batches(M, K, N, group, zeros):
    check_matvec(M, K, N, group, zeros, bias=N % 2 == 1, relu=K % 16 == 8, seed=M + K + N)


@pytest.mark.parametrize("M,K,N", [(40, 32768, 520), (64, 2048, 40000), (64, 256, 100000), (33, 4096, 4096)])
def test_matvec_large_batches(M, K, N):
    check_matvec(M, K, N, 64, True, bias=True, relu=False, seed=K)


@pytest.mark.parametrize("x_off,ld_x,y_off,ld_y", [(8, 520, 3, 0), (16, 528, 0, 131), (0, 536, 5, 133)])
@pytest.mark.parametrize("M", [20, 64])
def test_matvec_batch_strides(M, x_off, ld_x, y_off, ld_y):
    check_matvec(M, 515, 129, 64, True, bias=True, relu=False, x_off=x_off, ld_x=ld_x, y_off=y_off, ld_y=ld_y)


def test_matvec_batch_rows_stand_alone_and_repeat():
    """An infinity or a NaN stays in its row; the others' bits, and those of a
    replayed graph, are the same; nor do weights past K and N matter."""
    g = gen(11)
    M, K, N, group = 50, 1000, 200, 64
    codes, scales, zp = make_weights(g, K, N, group, True)
    x = randn(g, M, K)
    packed = pack(codes, scales, zp, group)
    y = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(x.cuda(), packed, y, M, K, N, group, zeros=True)
    bad = x.clone()
    bad[3, 17], bad[40, 999] = float("nan"), float("inf")
    xs, yb = bad.cuda(), torch.empty_like(y)
    tf.w4_matvec(xs, packed, yb, M, K, N, group, zeros=True)
    keep = [i for i in range(M) if i not in (3, 40)]
    assert torch.equal(y[keep].view(torch.int16), yb[keep].view(torch.int16))
    assert torch.isnan(yb[3]).all() and not torch.isfinite(yb[40]).any()
    graph = torch.cuda.CUDAGraph()
    again = torch.empty_like(y)
    with torch.cuda.graph(graph):
        for _ in range(3):
            tf.w4_matvec(xs, packed, again, M, K, N, group, zeros=True)
    xs.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.view(torch.int16), again.view(torch.int16))
    Kp, Np = 1024, 208
    full_c = torch.randint(0, 16, (Np, Kp), generator=g, dtype=torch.uint8)
    full_s = randn(g, Np, Kp // group, std=3.0)
    full_z = torch.randint(0, 16, (Np, Kp // group), generator=g, dtype=torch.uint8)
    full_c[:N, :K], full_s[:N, :scales.shape[1]], full_z[:N, :zp.shape[1]] = codes, scales, zp
    tf.w4_matvec(x.cuda(), pack(full_c, full_s, full_z, group), again, M, K, N, group, zeros=True)
    assert torch.equal(y.view(torch.int16), again.view(torch.int16))
    assert tf.device_error() == 0


def test_matvec_batches_at_once_and_between_other_products():
    """Calls on two streams at once, and in line with the tile product, which
    holds tensor memory too: the bits of a call by itself."""
    g = gen(23)
    M, K, N, group = 64, 2048, 4096, 128
    codes, scales, _ = make_weights(g, K, N, group, False)
    packed = pack(codes, scales, None, group)
    x = randn(g, M, K).cuda()
    alone = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(x, packed, alone, M, K, N, group)
    a, b = tile(randn(g, 256, 512)).cuda(), tile(randn(g, 512, 256)).cuda()
    ref = torch.empty(256 * 256, dtype=BF, device="cuda")
    tf.matmul_tiles(a, b, ref, 8, 16, 8)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ys = [[torch.empty_like(alone) for _ in range(8)] for _ in streams]
    cs = [torch.empty_like(ref) for _ in streams]
    for i in range(8):
        for s, y, c in zip(streams, ys, cs):
            with torch.cuda.stream(s):
                tf.w4_matvec(x, packed, y[i], M, K, N, group)
                tf.matmul_tiles(a, b, c, 8, 16, 8)
    torch.cuda.synchronize()
    for y, c in zip(ys, cs):
        assert all(torch.equal(v.view(torch.int16), alone.view(torch.int16)) for v in y)
        assert torch.equal(c.view(torch.int16), ref.view(torch.int16))
    assert tf.device_error() == 0


@pytest.mark.parametrize("M,K,group,zeros", [(8, 300, 64, True), (13, 4200, 128, False), (16, 20000, 32, True)])
def test_matvec_rows_of_very_different_size(M, K, group, zeros):
    """Rows scaled by powers of two from 2^-118 to 2^100: each within its own bound,
    and the ordinary rows' bits do not depend on their neighbours."""
    g = gen(K)
    N = 70
    codes, scales, zp = make_weights(g, K, N, group, zeros)
    w = real_weights(codes, scales, zp, group)
    x = randn(g, M, K)
    packed = pack(codes, scales, zp, group)
    plain = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(x.cuda(), packed, plain, M, K, N, group, zeros=zeros)
    powers = [0, 40, -80, 100, -118, 0, 23, -66] * 2
    scale = torch.tensor([2.0 ** p for p in powers[:M]], dtype=F64)[:, None]
    xs = (x.to(F64) * scale).to(BF)
    xs[5] = 0
    y = torch.empty(M, N, dtype=BF, device="cuda")
    tf.w4_matvec(xs.cuda(), packed, y, M, K, N, group, zeros=zeros)
    # a power of two changes nothing but exponents: the rows' errors scale with them
    close((y.cpu().to(F64) / scale), (xs.to(F64) / scale) @ w.t(),
          matvec_slack(xs.to(F64) / scale, codes, scales, zp, group, w), BF)
    assert torch.equal(y[0].view(torch.int16), plain[0].view(torch.int16)) and (y[5] == 0).all()


def test_matvec_repeats_bit_for_bit_and_rows_do_not_depend_on_their_company():
    g = gen(7)
    K, N, group = 4100, 1030, 32
    codes, scales, zp = make_weights(g, K, N, group, True)
    packed = pack(codes, scales, zp, group)
    x = randn(g, 64, K).cuda()
    first = torch.empty(64, N, dtype=BF, device="cuda")
    tf.w4_matvec(x, packed, first, 64, K, N, group, zeros=True)
    again = torch.empty_like(first)
    tf.w4_matvec(x, packed, again, 64, K, N, group, zeros=True)
    assert torch.equal(first.view(torch.int16), again.view(torch.int16))


def untile(t, rows, cols):
    rt, ct = -(-rows // 32), -(-cols // 32)
    m = t.view(rt, ct, 2, 2, 16, 16).permute(0, 2, 4, 1, 3, 5).reshape(rt * 32, ct * 32)
    return m[:rows, :cols], m


@pytest.mark.parametrize("K,N", [(1, 1), (32, 32), (33, 65), (128, 16), (130, 100), (1000, 257), (4096, 640)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("transpose", [False, True])
def test_dequantize_tiles_exact(K, N, group, zeros, transpose):
    """s * (q - z) is exact in fp32, so one rounding: equal bits; zeros in the padding."""
    g = gen(K + N)
    codes, scales, zp = make_weights(g, K, N, group, zeros)
    packed = pack(codes, scales, zp, group, fill=255)
    tiles = torch.full((-(-K // 32) * -(-N // 32) * 1024,), 5.0, dtype=BF, device="cuda")
    tf.w4_dequantize_tiles(packed, tiles, K, N, group, zeros=zeros, transpose=transpose)
    ref = real_weights(codes, scales, zp, group).to(F32).to(BF)
    ref = ref if transpose else ref.t()
    got, whole = untile(tiles.cpu(), *ref.shape)
    assert torch.equal(got, ref)
    assert (whole[ref.shape[0]:] == 0).all() and (whole[:, ref.shape[1]:] == 0).all()


def tile(m):
    rt, ct = m.shape[0] // 32, m.shape[1] // 32
    return m.reshape(rt, 2, 16, ct, 2, 16).permute(0, 3, 1, 4, 2, 5).reshape(-1).contiguous()


def quantized(w, group, zeros):
    """Values (K, N) the definition gives for bf16 weights w (K, N), in 64 bits."""
    out = torch.empty(w.shape, dtype=F64)
    for k0 in range(0, w.shape[0], group):
        p = w[k0:k0 + group].to(F64)
        if zeros:
            lo, hi = p.amin(0).clamp(max=0), p.amax(0).clamp(min=0)
            s = ((hi - lo) / 15).to(BF).to(F64)
            d = torch.where(s > 0, s, 1.0)
            z = torch.round(-lo / d).clamp(0, 15)
            out[k0:k0 + group] = ((torch.round(p / d) + z).clamp(0, 15) - z) * s
        else:
            s = (p.abs().amax(0) / 7).to(BF).to(F64)
            out[k0:k0 + group] = torch.round(p / torch.where(s > 0, s, 1.0)).clamp(-8, 7) * s
    return out


@pytest.mark.parametrize("Kt,Nt", [(1, 1), (3, 2), (4, 5), (9, 3), (40, 11)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_tiles_exact(Kt, Nt, group, zeros):
    g = gen(Kt * 100 + Nt)
    w = randn(g, 32 * Kt, 32 * Nt, std=0.05)
    w[:, 3] = 0                                     # groups of zeros
    w[:32, 5] = w[:32, 5].abs() + 0.01              # one sign
    w[:32, 6] = -w[:32, 6].abs() - 0.01
    w[0, 7] = 30.0                                  # one large value
    w[:, 8] = w[:, 8] * 1e-30                       # tiny
    packed = torch.empty(tf.w4_packed_bytes(32 * Kt, 32 * Nt, group, zeros), dtype=torch.uint8, device="cuda")
    out = torch.empty(w.numel(), dtype=BF, device="cuda")
    tf.w4_quantize_tiles(tile(w).cuda(), packed, Kt, Nt, group, zeros=zeros)
    tf.w4_dequantize_tiles(packed, out, 32 * Kt, 32 * Nt, group, zeros=zeros)
    got, _ = untile(out.cpu(), 32 * Kt, 32 * Nt)
    assert torch.equal(got, quantized(w, group, zeros).to(BF))


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_non_finite_groups_stand_for_nan(zeros):
    g = gen(3)
    w = randn(g, 128, 64, std=0.05)
    w[5, 2], w[40, 9], w[70, 11] = float("inf"), float("nan"), -float("inf")
    packed = torch.empty(tf.w4_packed_bytes(128, 64, 32, zeros), dtype=torch.uint8, device="cuda")
    out = torch.empty(w.numel(), dtype=BF, device="cuda")
    tf.w4_quantize_tiles(tile(w).cuda(), packed, 4, 2, 32, zeros=zeros)
    tf.w4_dequantize_tiles(packed, out, 128, 64, 32, zeros=zeros)
    got, _ = untile(out.cpu(), 128, 64)
    bad = torch.zeros(128, 64, dtype=torch.bool)
    bad[0:32, 2] = bad[32:64, 9] = bad[64:96, 11] = True
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()


# --------------------------------------------------------------- block norm ---

class Norm:
    """Inputs, 64-bit results and error bounds of one block_norm problem."""

    def __init__(self, T, D, fp32=False, post=True, gate_rows=1, act="none", w_pre=True, w_post=True, seed=0,
                 scale=0.7, eps=1e-5):
        g = gen(seed + T * 7 + D)
        self.T, self.D, self.rt = T, D, (F32 if fp32 else BF)
        self.post, self.act, self.scale, self.eps = post, act, scale, eps
        self.resid = randn(g, T, D, dtype=self.rt)
        self.u = randn(g, T, D, std=0.8)
        self.w_post = randn(g, D, std=0.3).add_(1) if post and w_post else None
        self.w_pre = randn(g, D, std=0.3).add_(1) if w_pre else None
        self.rows = gate_rows
        self.n = -(-T // gate_rows) if gate_rows else 0
        self.gate = randn(g, self.n, D) if gate_rows else None
        self.dh = randn(g, T, D, dtype=self.rt)
        self.dy = randn(g, T, D)

    def gate64(self):
        """act(gate) and its derivative for each token."""
        if self.gate is None:
            return torch.ones(self.T, self.D, dtype=F64), torch.zeros(self.T, self.D, dtype=F64)
        a = self.gate.to(F64)[torch.arange(self.T) // self.rows]
        if self.act == "sigmoid":
            s = torch.sigmoid(a)
            return s, s * (1 - s)
        return a, torch.ones_like(a)

    def forward64(self, resid=None, u=None, w_post=None, w_pre=None, gate=None):
        resid = self.resid.to(F64) if resid is None else resid
        u = self.u.to(F64) if u is None else u
        ones = torch.ones(self.D, dtype=F64)
        w_post = (self.w_post.to(F64) if self.w_post is not None else ones) if w_post is None else w_post
        w_pre = (self.w_pre.to(F64) if self.w_pre is not None else ones) if w_pre is None else w_pre
        a = self.gate64()[0] if gate is None else gate
        rp = (u.square().mean(1) + self.eps).rsqrt() if self.post else None
        b = u * rp[:, None] * w_post if self.post else u
        b = self.scale * a * b
        h = resid + b
        r = (h.square().mean(1) + self.eps).rsqrt()
        return {"h": h, "y": h * r[:, None] * w_pre, "rp": rp, "r": r, "b": b}

    def cuda(self, *names):
        return [None if getattr(self, n) is None else getattr(self, n).cuda() for n in names]


# Sums of at most 16384 squares of equal sign, at most 74 additions deep, and the
# root: 2^-18 relative; with the products around it, 2^-17 of the terms' magnitude.
REL = 2.0 ** -17


def check_forward(p, out):
    ref = p.forward64()
    mag = p.resid.to(F64).abs() + ref["b"].abs()
    wp = p.w_pre.to(F64).abs() if p.w_pre is not None else torch.ones(p.D, dtype=F64)
    close(out["h"], ref["h"], REL * mag, p.rt, "h")
    close(out["y"], ref["y"], REL * mag * ref["r"][:, None] * wp, BF, "y")
    if out.get("rstd_pre") is not None:
        close(out["rstd_pre"], ref["r"], 2.0 ** -16 * ref["r"], F32, "rstd_pre")
    if out.get("rstd_post") is not None:
        close(out["rstd_post"], ref["rp"], 2.0 ** -17 * ref["rp"], F32, "rstd_post")


def run_forward(p, stream=None, stats=True):
    out = {"h": torch.empty(p.T, p.D, dtype=p.rt, device="cuda"), "y": torch.empty(p.T, p.D, dtype=BF, device="cuda")}
    if stats:
        out["rstd_pre"] = torch.empty(p.T, device="cuda")
        out["rstd_post"] = torch.empty(p.T, device="cuda") if p.post else None
    resid, u, w_post, w_pre, gate = p.cuda("resid", "u", "w_post", "w_pre", "gate")
    tf.block_norm(resid, u, out["h"], out["y"], p.T, p.D, w_pre=w_pre, post=p.post, w_post=w_post, gate=gate,
                  gate_rows=p.rows or 1, gate_act=p.act, scale=p.scale, eps=p.eps, rstd_post=out.get("rstd_post"),
                  rstd_pre=out.get("rstd_pre"), stream=stream)
    return out


SHAPES = [(1, 1), (2, 7), (1, 8), (5, 16), (3, 100), (17, 129), (1, 1024), (33, 1000), (4, 1023), (9, 2048), (2, 4096),
          (3, 5120), (300, 640), (2, 8200), (1, 16383), (2, 16384), (1030, 72)]


@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("post,gate_rows,act", [(True, 1, "sigmoid"), (True, 0, "none"), (False, 1, "none"),
                                                (True, 2, "none"), (False, 1 << 30, "sigmoid"), (False, 0, "none")])
def test_block_norm_forward(T, D, fp32, post, gate_rows, act):
    p = Norm(T, D, fp32, post, gate_rows, act, w_pre=D % 3 != 0, w_post=D % 2 == 0)
    check_forward(p, run_forward(p, stats=T % 2 == 1))


def grad64(p, h, rstd_pre, rstd_post, dh=True, dy=True):
    """Gradients and error bounds from the formulas, on the saved h and factors."""
    T, D = p.T, p.D
    one = torch.ones(D, dtype=F64)
    wpre = p.w_pre.to(F64) if p.w_pre is not None else one
    wpost = p.w_post.to(F64) if p.w_post is not None else one
    d0 = p.dh.to(F64) if dh else torch.zeros(T, D, dtype=F64)
    r = rstd_pre.to(F64)[:, None]
    hh = h.to(F64) * r
    y = p.dy.to(F64) if dy else torch.zeros(T, D, dtype=F64)
    a = y * wpre
    dres = d0 + r * (a - hh * (a * hh).mean(1, keepdim=True))
    mag = d0.abs() + r * (a.abs() + hh.abs() * (a * hh).abs().mean(1, keepdim=True))
    act, dact = p.gate64()
    u = p.u.to(F64)
    rp = rstd_post.to(F64)[:, None] if p.post else torch.ones(T, 1, dtype=F64)
    uh = u * rp
    pv = uh * wpost
    dp = p.scale * dres * act
    mdp = abs(p.scale) * mag * act.abs()
    if p.post:
        b, mb = dp * wpost, mdp * wpost.abs()
        du = rp * (b - uh * (b * uh).mean(1, keepdim=True))
        mdu = rp * (mb + uh.abs() * (mb * uh.abs()).mean(1, keepdim=True))
    else:
        du, mdu = dp, mdp
    out = {"dresid": (dres, 2.0 ** -16 * mag), "du": (du, 2.0 ** -15 * mdu)}
    # sums over tokens: at most 2048 additions in a row
    out["dw_pre"] = ((y * hh).sum(0), 2.0 ** -13 * (y * hh).abs().sum(0))
    out["dw_post"] = ((dp * uh).sum(0), 2.0 ** -13 * (mdp * uh.abs()).sum(0))
    if p.gate is not None:
        seg = torch.arange(T) // p.rows
        z = torch.zeros(p.n, D, dtype=F64)
        out["dgate"] = (z.index_add(0, seg, p.scale * dres * pv * dact),
                        2.0 ** -13 * z.index_add(0, seg, abs(p.scale) * mag * pv.abs() * dact))
    return out


def run_backward(p, saved, want=("dresid", "du", "dgate", "dw_post", "dw_pre"), dh=True, dy=True, stream=None, ws=None):
    out = {}
    shapes = {"dresid": (p.T, p.D), "du": (p.T, p.D), "dgate": (p.n, p.D), "dw_post": (p.D,), "dw_pre": (p.D,)}
    types = {"dresid": p.rt, "du": BF, "dgate": BF, "dw_post": F32, "dw_pre": F32}
    for k in shapes:
        ok = k in want and (k != "dgate" or p.gate is not None) and (k != "dw_post" or p.post) and (k != "dw_pre" or dy)
        out[k] = torch.full(shapes[k], 9.0, dtype=types[k], device="cuda") if ok else None
    u, w_post, w_pre, gate, gdh, gdy = p.cuda("u", "w_post", "w_pre", "gate", "dh", "dy")
    n = tf.block_norm_grad_ws_bytes(p.T, p.D, p.rows)
    ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda") if ws is None else ws
    tf.block_norm_grad(gdh if dh else None, gdy if dy else None, saved["h"], u, out["dresid"], out["du"], p.T, p.D, ws,
                       rstd_pre=saved["rstd_pre"], w_pre=w_pre if dy else None, dw_pre=out["dw_pre"], post=p.post,
                       rstd_post=saved["rstd_post"], w_post=w_post, dw_post=out["dw_post"], gate=gate,
                       dgate=out["dgate"], gate_rows=p.rows or 1, gate_act=p.act, scale=p.scale, stream=stream)
    return out


def check_backward(p, saved, out, dh=True, dy=True):
    ref = grad64(p, saved["h"].cpu(), saved["rstd_pre"].cpu(),
                 saved["rstd_post"].cpu() if p.post else None, dh, dy)
    for k, t in out.items():
        if t is not None:
            close(t, ref[k][0], ref[k][1], t.dtype, k)


@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("post,gate_rows,act", [(True, 1, "sigmoid"), (True, 0, "none"), (False, 1, "none"),
                                                (True, 2, "none"), (True, 1 << 30, "sigmoid"), (False, 0, "none")])
def test_block_norm_gradient(T, D, fp32, post, gate_rows, act):
    p = Norm(T, D, fp32, post, gate_rows, act, w_pre=D % 3 != 0, w_post=D % 2 == 0)
    saved = run_forward(p)
    check_backward(p, saved, run_backward(p, saved))


@pytest.mark.parametrize("gate_rows", [3, 37, 128, 500, 1999, 2000])
def test_block_norm_gradient_of_shared_gates(gate_rows):
    p = Norm(2000, 264, False, True, gate_rows, "sigmoid")
    saved = run_forward(p)
    check_backward(p, saved, run_backward(p, saved))


@pytest.mark.parametrize("T,D,gate_rows", [(2500, 1, 0), (77, 2, 1), (3, 8, 2), (19003, 24, 1), (700, 17, 700),
                                           (3001, 40, 7), (2500, 64, 1000), (20001, 96, 0), (1999, 129, 1),
                                           (1205, 250, 60), (2000, 256, 1)])
def test_block_norm_of_narrow_rows(T, D, gate_rows):
    """Several rows share a warp; the last CTA's teams are without tokens."""
    p = Norm(T, D, D % 3 == 0, True, gate_rows, "sigmoid" if T % 2 else "none")
    saved = run_forward(p)
    check_forward(p, saved)
    check_backward(p, saved, run_backward(p, saved))


@pytest.mark.parametrize("want", [("dresid",), ("du",), ("dgate",), ("dw_post",), ("dw_pre",), ("du", "dw_pre")])
@pytest.mark.parametrize("dh,dy", [(True, True), (True, False), (False, True)])
def test_block_norm_gradient_parts(want, dh, dy):
    if not dy and want == ("dw_pre",):
        return
    p = Norm(50, 200, True, True, 8, "none")
    saved = run_forward(p)
    check_backward(p, saved, run_backward(p, saved, want=want, dh=dh, dy=dy), dh, dy)


def test_block_norm_gradient_against_differences():
    """Along a random direction of all inputs, the loss <dh, h> + <dy, y> rises
    as the gradient says.  Each of the gradient's terms is off by half a step of
    its type (2^-8) at most, and the difference quotient in 64 bits by far less."""
    p = Norm(6, 48, True, True, 2, "sigmoid", seed=4)
    saved = run_forward(p)
    out = {k: v.cpu().to(F64) for k, v in run_backward(p, saved).items()}
    g = gen(11)
    names = {"resid": "dresid", "u": "du", "w_post": "dw_post", "w_pre": "dw_pre"}
    step = {n: torch.randn(getattr(p, n).shape, generator=g, dtype=F64) for n in names}
    gstep = torch.randn(p.gate.shape, generator=g, dtype=F64)

    def loss(e):
        kw = {n: getattr(p, n).to(F64) + e * step[n] for n in names}
        kw["gate"] = torch.sigmoid(p.gate.to(F64) + e * gstep)[torch.arange(p.T) // p.rows]
        f = p.forward64(**kw)
        return (f["h"] * p.dh.to(F64)).sum() + (f["y"] * p.dy.to(F64)).sum()

    e = 1e-5
    slope = (loss(e) - loss(-e)).item() / (2 * e)
    terms = torch.cat([(out[d] * step[n]).reshape(-1) for n, d in names.items()] + [(out["dgate"] * gstep).reshape(-1)])
    assert abs(terms.sum().item() - slope) <= 2.0 ** -8 * terms.abs().sum().item() + 1e-6 * abs(slope)


def test_block_norm_no_tokens():
    """T = 0: sums over tokens are zeros, nothing else is touched."""
    p = Norm(3, 40)
    dw = torch.full((2, 40), 3.0, device="cuda")
    tf.block_norm_grad(None, None, None, None, None, None, 0, 40, None, dw_pre=dw[0], post=True, dw_post=dw[1])
    assert (dw == 0).all()
    h = torch.full((3, 40), 3.0, dtype=BF, device="cuda")
    tf.block_norm(p.resid.cuda(), p.u.cuda(), h, None, 0, 40)
    assert (h == 3).all()


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("D", [64, 129])
def test_block_norm_parts_and_in_place(fp32, D):
    p = Norm(11, D, fp32, True, 1, "none")
    full = run_forward(p)
    resid, u, w_post, w_pre, gate = p.cuda("resid", "u", "w_post", "w_pre", "gate")
    kw = dict(post=True, w_post=w_post, gate=gate, scale=p.scale, eps=p.eps)
    h = torch.empty_like(full["h"])
    tf.block_norm(resid, u, h, None, 11, D, **kw)
    assert torch.equal(h, full["h"])
    y = torch.empty_like(full["y"])
    tf.block_norm(resid, u, None, y, 11, D, w_pre=w_pre, **kw)
    assert torch.equal(y, full["y"])
    # no branch: the plain norm of the stream
    h2, y2 = torch.empty_like(h), torch.empty_like(y)
    tf.block_norm(resid, None, h2, y2, 11, D, w_pre=w_pre, eps=p.eps)
    assert torch.equal(h2, resid)
    x = p.resid.to(F64)
    ref = x * (x.square().mean(1, keepdim=True) + p.eps).rsqrt() * p.w_pre.to(F64)
    close(y2, ref, REL * ref.abs(), BF)
    # in place
    tf.block_norm(resid, u, resid, u, 11, D, w_pre=w_pre, **kw)
    assert torch.equal(resid, full["h"]) and torch.equal(u, full["y"])


@pytest.mark.parametrize("D,pad,off", [(64, 8, 0), (64, 3, 0), (64, 8, 1), (200, 56, 4), (129, 1, 0)])
@pytest.mark.parametrize("fp32", [False, True])
def test_block_norm_strides(D, pad, off, fp32):
    """Rows with gaps and unaligned starts; the gaps stay as they are."""
    T = 9
    p = Norm(T, D, fp32, True, 3, "sigmoid")

    def view(rows, dtype, src=None):
        buf = torch.full((off + rows * (D + pad),), 123.0, dtype=dtype, device="cuda")
        v = buf[off:].view(rows, D + pad)[:, :D]
        if src is not None:
            v.copy_(src)
        return buf, v

    def gaps(buf, rows):
        b = buf.clone()
        b[off:].view(rows, D + pad)[:, :D] = 123.0
        return bool((b == 123.0).all())

    resid, u, gate = (view(t.shape[0], t.dtype, t)[1] for t in (p.resid, p.u, p.gate))
    (hb, h), (yb, y) = view(T, p.rt), view(T, BF)
    w_post, w_pre = p.cuda("w_post", "w_pre")
    saved = {"rstd_pre": torch.empty(T, device="cuda"), "rstd_post": torch.empty(T, device="cuda"), "h": h, "y": y}
    tf.block_norm(resid, u, h, y, T, D, w_pre=w_pre, post=True, w_post=w_post, gate=gate, gate_rows=3,
                  gate_act="sigmoid", scale=p.scale, eps=p.eps, rstd_post=saved["rstd_post"],
                  rstd_pre=saved["rstd_pre"])
    check_forward(p, saved)
    assert gaps(hb, T) and gaps(yb, T)
    dh, dy = view(T, p.rt, p.dh)[1], view(T, BF, p.dy)[1]
    (rb, dresid), (ub, du), (gb, dgate) = view(T, p.rt), view(T, BF), view(p.n, BF)
    dw = torch.empty(2, D, device="cuda")
    ws = torch.empty(max(16, tf.block_norm_grad_ws_bytes(T, D, 3)), dtype=torch.uint8, device="cuda")
    tf.block_norm_grad(dh, dy, h, u, dresid, du, T, D, ws, rstd_pre=saved["rstd_pre"], w_pre=w_pre, dw_pre=dw[0],
                       post=True, rstd_post=saved["rstd_post"], w_post=w_post, dw_post=dw[1], gate=gate, dgate=dgate,
                       gate_rows=3, gate_act="sigmoid", scale=p.scale)
    check_backward(p, saved, {"dresid": dresid, "du": du, "dgate": dgate, "dw_pre": dw[0], "dw_post": dw[1]})
    assert gaps(rb, T) and gaps(ub, T) and gaps(gb, p.n)


def test_block_norm_zero_and_non_finite_rows():
    """A row of zeros gives zeros; a NaN or infinity stays in its row."""
    p = Norm(6, 512, False, True, 0)
    p.resid[1] = 0
    p.u[1] = 0
    base = run_forward(p)
    assert (base["y"][1] == 0).all() and (base["h"][1] == 0).all()
    p.resid[3, 7] = float("nan")
    p.u[5, 9] = float("inf")
    out = run_forward(p)
    keep = [0, 1, 2, 4]
    assert torch.equal(out["y"][keep], base["y"][keep]) and torch.equal(out["h"][keep], base["h"][keep])
    assert torch.isnan(out["y"][3]).all() and not torch.isfinite(out["y"][5]).all()


def test_block_norm_gradient_repeats_bit_for_bit():
    p = Norm(3000, 520, False, True, 100, "sigmoid")
    saved = run_forward(p)
    a, b = run_backward(p, saved), run_backward(p, saved)
    for k in a:
        assert torch.equal(a[k], b[k]), k


# ------------------------------------------------------------ embedding rows ---

def make_ids(g, T, V, kind):
    if kind == "one":
        return torch.full((T,), V // 2)
    if kind == "frequent":  # falls as 1 / rank
        return (torch.rand(T, generator=g, dtype=F64) * math.log(V)).exp().long().clamp(1, V) - 1
    if kind == "sorted":
        return torch.sort(torch.randint(0, V, (T,), generator=g))[0]
    return torch.randint(0, V, (T,), generator=g)


IDS = [(1, 1, 1, "any"), (1, 10, 64, "any"), (7, 3, 33, "any"), (64, 5, 128, "any"), (100, 1000, 1000, "any"),
       (1000, 70, 256, "frequent"), (3000, 50000, 64, "frequent"), (513, 17, 4096, "frequent"), (2000, 9, 96, "one"),
       (5000, 300, 24, "sorted"), (40, 262145, 16, "any"), (20000, 131, 40, "frequent"), (33, 40, 5001, "any"),
       (70000, 257, 8, "any")]


@pytest.mark.parametrize("T,V,D,kind", IDS)
@pytest.mark.parametrize("fp32,long_ids", [(False, True), (True, False)])
def test_embed_rows(T, V, D, kind, fp32, long_ids):
    g = gen(T + V)
    ids = make_ids(g, T, V, kind).to(torch.int64 if long_ids else torch.int32)
    table = randn(g, V, D)
    out = torch.empty(T, D, dtype=F32 if fp32 else BF, device="cuda")
    tf.embed_rows(ids.cuda(), table.cuda(), out, T, V, D, scale=1.7)
    ref = table.to(F64)[ids.long()] * float(np.float32(1.7))
    close(out, ref, 2.0 ** -24 * ref.abs(), out.dtype)
    assert tf.device_error() == 0


def embed_grad(ids, dout, V, scale, ws=None, stream=None, dtable=None, **kw):
    T, D = dout.shape
    dtable = torch.full((V, D), 5.0, device="cuda") if dtable is None else dtable
    n = tf.embed_rows_grad_ws_bytes(T, V, D)
    ws = torch.full((max(16, n),), 255, dtype=torch.uint8, device="cuda") if ws is None else ws
    tf.embed_rows_grad(ids, dout, dtable, T, V, D, ws, scale=scale, stream=stream, **kw)
    return dtable


def embed_ref(ids, dout, V, scale):
    """Sums in 64 bits and their error bound: n additions of 2^-24 and the scale."""
    z = torch.zeros(V, dout.shape[1], dtype=F64)
    n = torch.zeros(V, 1, dtype=F64).index_add(0, ids, torch.ones(len(ids), 1, dtype=F64))
    s = float(np.float32(scale))
    return (z.index_add(0, ids, dout.to(F64)) * s,
            (n + 2) * 2.0 ** -24 * s * z.index_add(0, ids, dout.to(F64).abs()))


@pytest.mark.parametrize("T,V,D,kind", IDS)
@pytest.mark.parametrize("fp32,long_ids", [(False, True), (True, False)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_rows_gradient(T, V, D, kind, fp32, long_ids, accumulate):
    g = gen(T + V + 1)
    ids = make_ids(g, T, V, kind).to(torch.int64 if long_ids else torch.int32)
    dout = randn(g, T, D, dtype=F32 if fp32 else BF)
    got = embed_grad(ids.cuda(), dout.cuda(), V, 1.7, accumulate=accumulate)
    ref, slack = embed_ref(ids.long(), dout, V, 1.7)
    if accumulate:
        untouched = torch.ones(V, dtype=torch.bool)
        untouched[ids.long()] = False
        assert (got.cpu()[untouched] == 5.0).all()
        ref, slack = ref + 5.0, slack + 2.0 ** -24 * ref.abs()
    close(got, ref, slack, F32)
    again = embed_grad(ids.cuda(), dout.cuda(), V, 1.7, accumulate=accumulate)
    assert torch.equal(got, again)
    assert tf.device_error() == 0


@pytest.mark.parametrize("T", [60, 9000])
def test_embed_rows_padding_and_bad_ids(T):
    V, D, pad = 50, 72, 7
    g = gen(2)
    ids = torch.randint(0, V, (T,), generator=g)
    ids[::3] = pad
    table, dout = randn(g, V, D).cuda(), randn(g, T, D)
    dout[::3] = float("nan")           # what stands in padded rows is not read into the sums
    out = torch.empty(T, D, dtype=BF, device="cuda")

    def check(ids_dev, alive):
        tf.embed_rows(ids_dev, table, out, T, V, D, pad_id=pad)
        assert (out.cpu()[~alive] == 0).all()
        assert torch.equal(out.cpu()[alive], table.cpu()[ids[alive]])
        got = embed_grad(ids_dev, dout.cuda(), V, 1.0, pad_id=pad)
        ref, slack = embed_ref(ids[alive], dout[alive], V, 1.0)
        close(got, ref, slack, F32)
        assert (got[pad] == 0).all()

    check(ids.cuda(), ids != pad)
    assert tf.device_error() == 0
    alive = ids != pad
    bad = ids.clone()
    for i, v in ((1, V), (4, -1), (5, 2 ** 40), (10, -(2 ** 40)), (T - 1, V + 1)):
        bad[i], alive[i] = v, False
        dout[i] = float("nan")
    check(bad.cuda(), alive)
    assert tf.device_error() == tf.DEVERR_BAD_INDEX
    assert tf.device_error() == 0
    # a padding id outside the table is not an error
    ids[alive.logical_not()] = -100
    out2 = torch.empty_like(out)
    tf.embed_rows(ids.cuda(), table, out2, T, V, D, pad_id=-100)
    assert torch.equal(out, out2) and tf.device_error() == 0


def test_embed_rows_all_padding_and_no_tokens():
    ids = torch.full((300,), 3, device="cuda")
    dout = torch.full((300, 40), 2.0, dtype=BF, device="cuda")
    assert (embed_grad(ids, dout, 20, 1.0, pad_id=3) == 0).all()
    assert (embed_grad(ids, dout, 20, 1.0, pad_id=3, accumulate=True) == 5.0).all()
    assert (embed_grad(ids[:0], dout[:0], 20, 1.0) == 0).all()
    assert (embed_grad(ids[:0], dout[:0], 20, 1.0, accumulate=True) == 5.0).all()
    out = torch.empty(300, 40, dtype=BF, device="cuda")
    empty = torch.empty(0, 40, dtype=BF, device="cuda")
    tf.embed_rows(ids, empty, out, 300, 0, 40, pad_id=3)
    assert (out == 0).all() and tf.device_error() == 0


@pytest.mark.parametrize("D,pad,off", [(64, 8, 0), (63, 2, 1), (64, 5, 0), (256, 64, 4)])
def test_embed_rows_strides(D, pad, off):
    T, V = 500, 37
    g = gen(9)
    ids = make_ids(g, T, V, "frequent").cuda()

    def view(rows, dtype, fill=123.0):
        buf = torch.full((off + rows * (D + pad),), fill, dtype=dtype, device="cuda")
        return buf, buf[off:].view(rows, D + pad)[:, :D]

    def gaps(buf, rows):
        b = buf.clone()
        b[off:].view(rows, D + pad)[:, :D] = 123.0
        return bool((b == 123.0).all())

    table = view(V, BF)[1]
    table.copy_(randn(g, V, D))
    ob, out = view(T, F32)
    tf.embed_rows(ids, table, out, T, V, D, scale=2.0)
    assert torch.equal(out, table[ids].float() * 2) and gaps(ob, T)
    dout = view(T, BF)[1]
    dout.copy_(randn(g, T, D))
    db, dtable = view(V, F32)
    embed_grad(ids, dout, V, 2.0, dtable=dtable)
    ref, slack = embed_ref(ids.cpu(), dout.cpu(), V, 2.0)
    close(dtable, ref, slack, F32)
    assert gaps(db, V)


def test_embed_rows_far_offsets():
    """Rows whose element offsets pass 2^32."""
    V, D = 70000, 65536
    if torch.cuda.mem_get_info()[0] < 3 * V * D * 4:
        pytest.skip("not enough memory")
    table = torch.zeros(V, D, dtype=BF, device="cuda")
    ids = torch.tensor([V - 1, 3, 65537, V - 1], device="cuda")
    table[ids] = randn(gen(1), 4, D).cuda()
    out = torch.empty(4, D, dtype=BF, device="cuda")
    tf.embed_rows(ids, table, out, 4, V, D)
    assert torch.equal(out, table[ids])
    del table
    dtable = embed_grad(ids, out, V, 1.0)
    assert torch.equal(dtable[3], out[1].float()) and torch.equal(dtable[65537], out[2].float())
    assert torch.equal(dtable[V - 1], out[0].float() + out[3].float())
    assert dtable[V - 2].abs().max() == 0 and dtable[0].abs().max() == 0
    assert dtable.count_nonzero(1).gt(0).sum() == 3


# -------------------------------------------------------- together, streams ---

def test_streams_and_captured_graphs():
    """The operators on a side stream and replayed from a graph give the bits of
    an ordinary call; two graphs with workspaces of their own do not disturb
    each other."""
    g = gen(21)
    K, N, M, V, T = 1024, 512, 4, 300, 700
    codes, scales, zp = make_weights(g, K, N, 64, True)
    packed = pack(codes, scales, zp, 64)
    x = randn(g, M, K).cuda()
    ids = make_ids(g, T, V, "frequent").cuda()
    dout = randn(g, T, K).cuda()
    p = Norm(T, K, False, True, 50, "sigmoid")
    saved = run_forward(p)
    resid, u, w_post, w_pre, gate, dh, dy = p.cuda("resid", "u", "w_post", "w_pre", "gate", "dh", "dy")

    def outputs():
        e = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        return {"mv": e(M, N), "h": e(T, K), "y": e(T, K), "dresid": e(T, K), "du": e(T, K), "dgate": e(p.n, K),
                "dw_pre": e(K, dtype=F32), "dw_post": e(K, dtype=F32), "dtable": e(V, K, dtype=F32),
                "ws1": e(tf.block_norm_grad_ws_bytes(T, K, 50) + 16, dtype=torch.uint8),
                "ws2": e(tf.embed_rows_grad_ws_bytes(T, V, K) + 16, dtype=torch.uint8)}

    def work(o):
        tf.w4_matvec(x, packed, o["mv"], M, K, N, 64, zeros=True)
        tf.block_norm(resid, u, o["h"], o["y"], T, K, w_pre=w_pre, post=True, w_post=w_post, gate=gate, gate_rows=50,
                      gate_act="sigmoid", scale=p.scale, eps=p.eps)
        tf.block_norm_grad(dh, dy, saved["h"], u, o["dresid"], o["du"], T, K, o["ws1"], rstd_pre=saved["rstd_pre"],
                           w_pre=w_pre, dw_pre=o["dw_pre"], post=True, rstd_post=saved["rstd_post"], w_post=w_post,
                           dw_post=o["dw_post"], gate=gate, dgate=o["dgate"], gate_rows=50, gate_act="sigmoid",
                           scale=p.scale)
        tf.embed_rows_grad(ids, dout, o["dtable"], T, V, K, o["ws2"])

    def same(a, b):
        for k in a:
            if not k.startswith("ws"):
                assert torch.equal(a[k], b[k]), k

    plain = outputs()
    work(plain)
    torch.cuda.synchronize()
    side, on_side = torch.cuda.Stream(), outputs()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(on_side)
    side.synchronize()
    same(plain, on_side)

    graphs = []
    for _ in range(2):
        o = outputs()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            work(o)
        graphs.append((gr, o, torch.cuda.Stream()))
    for _ in range(3):
        for gr, o, s in graphs:
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for gr, o, _ in graphs:
        same(plain, o)
    x.mul_(2)  # the replay reads the tensors anew
    work(plain)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    same(plain, graphs[0][1])
    assert tf.device_error() == 0


def test_decode_step_through_the_operators():
    """ids -> embedding rows -> norm -> 4-bit product with relu -> 4-bit product ->
    norm, gate and residual -> 4-bit logits, for a few tokens, against 64 bits
    (each stage from the stage before it as the GPU left it)."""
    g = gen(31)
    M, V, D, F, group = 5, 700, 512, 1344, 64
    table = randn(g, V, D)
    ids = torch.tensor([3, 699, 3, 0, 41])
    ws = {}
    for name, (k, n) in {"up": (D, F), "down": (F, D), "head": (D, V)}.items():
        c, s, z = make_weights(g, k, n, group, True)
        s = (s.float() / math.sqrt(k)).to(BF)
        ws[name] = (pack(c, s, z, group), real_weights(c, s, z, group), (c, s, z))
    w1, w2, w3 = (randn(g, D, std=0.2).add_(1) for _ in range(3))
    gate = randn(g, M, D)
    e = lambda n, dtype=BF: torch.empty(M, n, dtype=dtype, device="cuda")  # noqa: E731
    h0, x1, f, o, h1, x2, logits = e(D, F32), e(D), e(F), e(D), e(D, F32), e(D), e(V)
    tf.embed_rows(ids.cuda(), table.cuda(), h0, M, V, D, scale=math.sqrt(D))
    tf.block_norm(h0, None, None, x1, M, D, w_pre=w1.cuda())
    tf.w4_matvec(x1, ws["up"][0], f, M, D, F, group, zeros=True, relu=True)
    tf.w4_matvec(f, ws["down"][0], o, M, F, D, group, zeros=True)
    tf.block_norm(h0, o, h1, x2, M, D, w_pre=w3.cuda(), post=True, w_post=w2.cuda(), gate=gate.cuda(),
                  gate_act="sigmoid", scale=0.5)
    tf.w4_matvec(x2, ws["head"][0], logits, M, D, V, group, zeros=True)
    torch.cuda.synchronize()
    assert tf.device_error() == 0

    def n64(v):
        return v * (v.square().mean(1, keepdim=True) + 1e-5).rsqrt()

    c64 = lambda t: t.cpu().to(F64)  # noqa: E731
    ref = table.to(F64)[ids] * float(np.float32(math.sqrt(D)))
    close(h0, ref, 2.0 ** -24 * ref.abs(), F32, "embed")
    ref = n64(c64(h0)) * w1.to(F64)
    close(x1, ref, REL * ref.abs(), BF, "norm")
    for x, y, name, relu in ((x1, f, "up", True), (f, o, "down", False), (x2, logits, "head", False)):
        ref = c64(x) @ ws[name][1].t()
        c, s, z = ws[name][2]
        close(y, ref.clamp(min=0) if relu else ref, matvec_slack(x.cpu(), c, s, z, group, ws[name][1]), BF, name)
    branch = 0.5 * torch.sigmoid(gate.to(F64)) * n64(c64(o)) * w2.to(F64)
    ref = c64(h0) + branch
    mag = c64(h0).abs() + branch.abs()
    close(h1, ref, REL * mag, F32, "residual")
    rr = (ref.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    close(x2, ref * rr * w3.to(F64), REL * mag * rr * w3.to(F64).abs(), BF, "norm 2")


def test_training_step_through_the_operators():
    """Forward and backward of embedding -> norm -> frozen 4-bit product (as tile
    streams through the GEMM, and its transpose for the input gradient) ->
    norm, residual: the table's gradient against automatic differentiation in
    64 bits.  Every intermediate is rounded to bf16 (2^-8), a handful of them on
    each path, so the gradient's norm-wise error stays within 2^-8 times the
    square root of the number of roundings (under 16): 2^-6."""
    g = gen(41)
    T, V, D, group = 96, 50, 128, 32
    table = randn(g, V, D)
    ids = torch.randint(0, V, (T,), generator=g)
    codes, scales, zp = make_weights(g, D, D, group, True)
    packed = pack(codes, scales, zp, group)
    w1, w2, w3 = (randn(g, D, std=0.2).add_(1) for _ in range(3))
    d1, d2, d3 = w1.cuda(), w2.cuda(), w3.cuda()
    dh, dy = randn(g, T, D), randn(g, T, D)
    e = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731

    def product(x, transpose):
        wt, xt, yt, y = e(D * D), e(T * D), e(T * D), e(T, D)
        tf.w4_dequantize_tiles(packed, wt, D, D, group, zeros=True, transpose=transpose)
        tf.tilize(x, xt, T, D)
        tf.matmul_tiles(xt, wt, yt, T // 32, D // 32, D // 32)
        tf.untilize(yt, y, T, D)
        return y

    h0, x1, r1 = e(T, D, dtype=F32), e(T, D), e(T, dtype=F32)
    tf.embed_rows(ids.cuda(), table.cuda(), h0, T, V, D)
    tf.block_norm(h0, None, None, x1, T, D, w_pre=d1, rstd_pre=r1)
    u = product(x1, False)
    h1, y, rp, r2 = e(T, D, dtype=F32), e(T, D), e(T, dtype=F32), e(T, dtype=F32)
    tf.block_norm(h0, u, h1, y, T, D, w_pre=d3, post=True, w_post=d2, scale=0.5, rstd_post=rp, rstd_pre=r2)
    dres, du, dw2, dw3 = e(T, D, dtype=F32), e(T, D), e(D, dtype=F32), e(D, dtype=F32)
    ws = e(max(16, tf.block_norm_grad_ws_bytes(T, D, 0)), dtype=torch.uint8)
    tf.block_norm_grad(dh.float().cuda(), dy.cuda(), h1, u, dres, du, T, D, ws, rstd_pre=r2, w_pre=d3, dw_pre=dw3,
                       post=True, rstd_post=rp, w_post=d2, dw_post=dw2, scale=0.5)
    dx1 = product(du, True)
    dh0, dw1 = e(T, D, dtype=F32), e(D, dtype=F32)
    tf.block_norm_grad(dres, dx1, h0, None, dh0, None, T, D, ws, rstd_pre=r1, w_pre=d1, dw_pre=dw1)
    dtable = embed_grad(ids.cuda(), dh0, V, 1.0)

    leaves = [t.to(F64).requires_grad_() for t in (table, w1, w2, w3)]
    tb, a1, a2, a3 = leaves

    def n64(v):
        return v * (v.square().mean(1, keepdim=True) + 1e-5).rsqrt()

    s0 = tb[ids]
    uu = (n64(s0) * a1) @ real_weights(codes, scales, zp, group).t()
    s1 = s0 + 0.5 * n64(uu) * a2
    (s1 * dh.to(F64)).sum().add((n64(s1) * a3 * dy.to(F64)).sum()).backward()
    for got, leaf in ((dtable, tb), (dw1, a1), (dw2, a2), (dw3, a3)):
        err = (got.cpu().to(F64) - leaf.grad).norm() / leaf.grad.norm()
        assert err <= 2.0 ** -6, err.item()
