"""Cases, plain forms and exact results of the token-path operators.

The operators: products of a few rows with 4-bit weights (``w4_matvec`` and the
conversions between tile streams and 4-bit storage), the norms around a
residual block with gate and residual scale (``block_norm``, its gradient) and
the scaled row lookup with its gradient (``embed_rows``).  ``run`` computes
them with elementary torch operations, or, where ``own`` is true, through the
framework's entry points; ``exact`` gives the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_GROUPS = (32, 64, 128)
_LIB = None


def _tf():
    global _LIB
    if _LIB is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-foil_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import ttfoil
        _LIB = ttfoil
    return _LIB


# ------------------------------------------------------------------ cases ---

def _matvec(M, K, N, group, zeros, bias, relu):
    return {"op": "w4_matvec", "M": M, "K": K, "N": N, "group": group, "zeros": zeros, "bias": bias, "relu": relu}


def _norm(op, T, D, fp32, post, gate_rows, act):
    """gate_rows: tokens that share one gate row, 0 = no gate."""
    return {"op": op, "T": T, "D": D, "fp32": fp32, "post": post, "gate_rows": gate_rows, "act": act}


def _embed(op, T, V, D, fp32, long_ids, pad):
    return {"op": op, "T": T, "V": V, "D": D, "fp32": fp32, "long_ids": long_ids, "pad": pad}


def listed():
    cases = [
        # one decoded token through a small projection: launch latency counts
        ("matvec_token_small", _matvec(1, 2048, 2048, 64, False, True, False)),
        # one decoded token through a wide projection
        ("matvec_token_wide", _matvec(1, 4096, 16384, 128, False, False, False)),
        # five rows (a short draft), ragged sizes, small groups, zero points, bias and relu
        ("matvec_draft_ragged", _matvec(5, 4100, 10250, 32, True, True, True)),
        # a batch of sixteen sequences through the largest projection
        ("matvec_batch_large", _matvec(16, 8192, 24576, 128, True, False, False)),
        # weights quantised and laid out again, as when a checkpoint is converted and its error is looked at
        ("quantize_weights", {"op": "w4_quantize", "K": 4096, "N": 8192, "group": 64, "zeros": False}),
        # weights laid out for the input gradient's product (transposed operand)
        ("dequantize_transposed", {"op": "w4_dequantize", "K": 8192, "N": 8192, "group": 128, "zeros": True,
                                   "transpose": True}),
        # the norms of one decoded token
        ("norm_token", _norm("block_norm", 1, 4096, False, True, 1, "none")),
        # a prompt with the residual stream in 32 bits and a gate for each token
        ("norm_prompt", _norm("block_norm", 8192, 5120, True, True, 1, "sigmoid")),
        # gradients of a ragged batch whose sequences share a gate row each
        ("norm_grad_shared", _norm("block_norm_grad", 4099, 2050, False, True, 512, "none")),
        # gradients of a long batch, one gate vector for all tokens
        ("norm_grad_long", _norm("block_norm_grad", 16384, 4096, False, True, 16384, "none")),
        # lookup of a prompt batch into a 32-bit residual stream
        ("embed_prompt", _embed("embed_rows", 8191, 65536, 4096, True, False, False)),
        # the table's gradient of a training batch: many rows of a few frequent tokens
        ("embed_grad", _embed("embed_rows_grad", 16384, 65536, 2048, False, True, True)),
    ]
    return [dict(case, name=name) for name, case in cases]


def _spread(rng, lo, hi):
    """A size from [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("w4_matvec", "w4_matvec", "w4_quantize", "w4_dequantize", "block_norm", "block_norm",
                     "block_norm_grad", "block_norm_grad", "embed_rows", "embed_rows_grad"))
    if op == "w4_matvec":
        K = _spread(rng, 32, 16384)
        return _matvec(_spread(rng, 1, 64), K, _spread(rng, 1, min(32768, (8192 * 24576) // K)), rng.choice(_GROUPS),
                       rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.3)
    if op in ("w4_quantize", "w4_dequantize"):
        Kt = _spread(rng, 1, 256)
        Nt = _spread(rng, 1, min(512, 65536 // Kt))
        case = {"op": op, "K": 32 * Kt, "N": 32 * Nt, "group": rng.choice(_GROUPS), "zeros": rng.random() < 0.5}
        if op == "w4_dequantize":
            case["K"] -= rng.randrange(32)
            case["N"] -= rng.randrange(32)
            case["transpose"] = rng.random() < 0.5
        return case
    if op in ("block_norm", "block_norm_grad"):
        D = _spread(rng, 16, 16384)
        D = D if rng.random() < 0.4 else (D + 7) // 8 * 8
        T = _spread(rng, 1, min(32768, (16384 * 2560) // D))
        gate = rng.choice((0, 1, 1, T, max(1, T // 3)))
        return _norm(op, T, D, rng.random() < 0.5, rng.random() < 0.7, gate, rng.choice(("none", "sigmoid")))
    D = _spread(rng, 16, 8192)
    D = D if rng.random() < 0.4 else (D + 7) // 8 * 8
    V = _spread(rng, 50, min(200000, (65536 * 2048) // D))
    T = _spread(rng, 1, min(65536, (16384 * 2048) // D))
    return _embed(op, T, V, D, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)


# ------------------------------------------------------------------ inputs ---

_EPS = 1e-5


def _dims(case):
    groups = -(-case["K"] // case["group"])
    return -(-case["N"] // 16), -(-case["K"] // 128), groups


def _block_bytes(case):
    per = 128 // case["group"] * 16
    return 1024 + per * (3 if case["zeros"] else 2)


def _pack(codes, scales, zeros, case):
    """The 4-bit storage of codes (N, K), scales and zeros (N, groups): blocks of
    16 columns n by 128 k.  A block holds 1024 bytes of codes, [half 2][row 8]
    [t 4][b 4] words for n = 8 half + row, k = 32 b + 8 t + 0..7, nibbles in the
    order k 0 2 4 6 1 3 5 7; then its scales [group][n] (bf16) and, if there are
    any, zero points [group][n] (one byte each)."""
    nt, kb, _ = _dims(case)
    ng = 128 // case["group"]
    dev = codes.device
    full = torch.zeros(nt * 16, kb * 128, dtype=torch.uint8, device=dev)
    full[:case["N"], :case["K"]] = codes
    # nt half row kb b t p nib o   (k in 8 = 4 p + 2 nib + o; byte = 2 o + p)
    c = full.view(nt, 2, 8, kb, 4, 4, 2, 2, 2).permute(0, 3, 1, 2, 5, 4, 8, 6, 7)
    c = (c[..., 0] | (c[..., 1] << 4)).reshape(nt, kb, 1024)
    s = torch.zeros(nt * 16, kb * ng, dtype=torch.bfloat16, device=dev)
    s[:case["N"], :scales.shape[1]] = scales
    parts = [c, s.view(nt, 16, kb, ng).permute(0, 2, 3, 1).reshape(nt, kb, ng * 16).contiguous().view(torch.uint8)]
    if zeros is not None:
        z = torch.zeros(nt * 16, kb * ng, dtype=torch.uint8, device=dev)
        z[:case["N"], :zeros.shape[1]] = zeros
        parts.append(z.view(nt, 16, kb, ng).permute(0, 2, 3, 1).reshape(nt, kb, ng * 16))
    return torch.cat(parts, dim=2).reshape(-1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    bf = torch.bfloat16

    def randn(*shape, std=1.0, dtype=bf):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    st = {"case": case}
    op = case["op"]
    if op in ("w4_matvec", "w4_dequantize"):
        K, N = case["K"], case["N"]
        groups = _dims(case)[2]
        codes = torch.randint(0, 16, (N, K), generator=g, device=dev, dtype=torch.uint8)
        scales = (torch.rand(N, groups, generator=g, device=dev) * 0.8 + 0.6).mul_(0.2 / math.sqrt(K)).to(bf)
        zeros = torch.randint(4, 12, (N, groups), generator=g, device=dev, dtype=torch.uint8) if case["zeros"] else None
        st["packed"] = _pack(codes, scales, zeros, case)
        if op == "w4_matvec":
            st["x"] = randn(case["M"], K)
            st["bias"] = randn(N, std=0.1) if case["bias"] else None
            st["y"] = torch.empty(case["M"], N, dtype=bf, device=dev)
        else:
            st["tiles"] = torch.empty(-(-K // 32) * -(-N // 32) * 1024, dtype=bf, device=dev)
    elif op == "w4_quantize":
        # weights of a trained layer: near normal, a few columns several times larger
        w = torch.randn(case["K"] * case["N"], generator=g, device=dev) * 0.02
        w *= 1 + 4 * (torch.rand(w.shape, generator=g, device=dev) < 0.001)
        st["b"] = w.to(bf)
        nt, kb, _ = _dims(case)
        st["packed"] = torch.empty(nt * kb * _block_bytes(case), dtype=torch.uint8, device=dev)
        st["tiles"] = torch.empty_like(st["b"])
    elif op in ("block_norm", "block_norm_grad"):
        T, D = case["T"], case["D"]
        rt = torch.float32 if case["fp32"] else bf
        # a few large channels, as residual streams have
        chan = 1 + 6 * (torch.rand(D, generator=g, device=dev) < 0.01)
        st["u"] = (torch.randn(T, D, generator=g, device=dev) * 0.7).to(bf)
        st["w_post"] = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(bf) if case["post"] else None
        st["w_pre"] = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(bf)
        rows = -(-T // case["gate_rows"]) if case["gate_rows"] else 0
        st["gate"] = randn(rows, D, std=0.5) if rows else None
        st["scale"] = 0.5
        if op == "block_norm":
            st["resid"] = (torch.randn(T, D, generator=g, device=dev) * chan).to(rt)
            st["h"] = torch.empty(T, D, dtype=rt, device=dev)
            st["y"] = torch.empty(T, D, dtype=bf, device=dev)
            st["rstd_post"] = torch.empty(T, device=dev) if case["post"] else None
            st["rstd_pre"] = torch.empty(T, device=dev)
        else:
            st["h"] = (torch.randn(T, D, generator=g, device=dev) * chan).to(rt)
            st["rstd_post"] = (st["u"].float().square().mean(1) + _EPS).rsqrt() if case["post"] else None
            st["rstd_pre"] = (st["h"].float().square().mean(1) + _EPS).rsqrt()
            st["dh"] = (torch.randn(T, D, generator=g, device=dev) * 0.1).to(rt)
            st["dy"] = randn(T, D, std=0.1)
            st["dresid"] = torch.empty(T, D, dtype=rt, device=dev)
            st["du"] = torch.empty(T, D, dtype=bf, device=dev)
            st["dgate"] = torch.empty(rows, D, dtype=bf, device=dev) if rows else None
            st["dw_post"] = torch.empty(D, device=dev) if case["post"] else None
            st["dw_pre"] = torch.empty(D, device=dev)
            if own:
                n = _tf().block_norm_grad_ws_bytes(T, D, case["gate_rows"])
                st["ws"] = torch.empty(max(16, n), dtype=torch.uint8, device=dev)
    else:
        T, V, D = case["T"], case["V"], case["D"]
        # token frequencies fall about as 1 / rank; ranks scattered over the vocabulary
        rank = torch.exp(torch.rand(T, generator=g, device=dev, dtype=torch.float64) * math.log(V)).long() - 1
        st["ids"] = torch.randperm(V, generator=g, device=dev)[rank.clamp_(0, V - 1)]
        st["pad_id"] = int(V // 2) if case["pad"] else -1
        if case["pad"]:
            st["ids"][torch.rand(T, generator=g, device=dev) < 0.1] = st["pad_id"]
        if not case["long_ids"]:
            st["ids"] = st["ids"].to(torch.int32)
        st["scale"] = math.sqrt(D)
        ft = torch.float32 if case["fp32"] else bf
        if op == "embed_rows":
            st["table"] = randn(V, D, std=0.02)
            st["out"] = torch.empty(T, D, dtype=ft, device=dev)
        else:
            st["dout"] = randn(T, D, std=0.1, dtype=ft)
            st["dtable"] = torch.empty(V, D, device=dev)
            if own:
                n = _tf().embed_rows_grad_ws_bytes(T, V, D)
                st["ws"] = torch.empty(max(16, n), dtype=torch.uint8, device=dev)
    return st


# -------------------------------------------------------------------- run ---

def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    tf, case = _tf(), st["case"]
    op = case["op"]
    if op == "w4_matvec":
        tf.w4_matvec(st["x"], st["packed"], st["y"], case["M"], case["K"], case["N"], case["group"],
                     zeros=case["zeros"], bias=st["bias"], relu=case["relu"])
        return st["y"]
    if op == "w4_quantize":
        tf.w4_quantize_tiles(st["b"], st["packed"], case["K"] // 32, case["N"] // 32, case["group"],
                             zeros=case["zeros"])
        tf.w4_dequantize_tiles(st["packed"], st["tiles"], case["K"], case["N"], case["group"], zeros=case["zeros"])
        return st["tiles"]
    if op == "w4_dequantize":
        tf.w4_dequantize_tiles(st["packed"], st["tiles"], case["K"], case["N"], case["group"], zeros=case["zeros"],
                               transpose=case["transpose"])
        return st["tiles"]
    if op == "block_norm":
        tf.block_norm(st["resid"], st["u"], st["h"], st["y"], case["T"], case["D"], w_pre=st["w_pre"],
                      post=case["post"], w_post=st["w_post"], gate=st["gate"], gate_rows=case["gate_rows"],
                      gate_act=case["act"], scale=st["scale"], eps=_EPS, rstd_post=st["rstd_post"],
                      rstd_pre=st["rstd_pre"])
        return [st[k] for k in ("h", "y", "rstd_pre", "rstd_post") if st[k] is not None]
    if op == "block_norm_grad":
        tf.block_norm_grad(st["dh"], st["dy"], st["h"], st["u"], st["dresid"], st["du"], case["T"], case["D"],
                           st["ws"], rstd_pre=st["rstd_pre"], w_pre=st["w_pre"], dw_pre=st["dw_pre"],
                           post=case["post"], rstd_post=st["rstd_post"], w_post=st["w_post"], dw_post=st["dw_post"],
                           gate=st["gate"], dgate=st["dgate"], gate_rows=case["gate_rows"], gate_act=case["act"],
                           scale=st["scale"])
        return [st[k] for k in ("dresid", "du", "dw_pre", "dw_post", "dgate") if st[k] is not None]
    if op == "embed_rows":
        tf.embed_rows(st["ids"], st["table"], st["out"], case["T"], case["V"], case["D"], scale=st["scale"],
                      pad_id=st["pad_id"])
        return st["out"]
    tf.embed_rows_grad(st["ids"], st["dout"], st["dtable"], case["T"], case["V"], case["D"], st["ws"],
                       scale=st["scale"], pad_id=st["pad_id"])
    return st["dtable"]


def _unpack(packed, case, dtype):
    """Weights (N, K) of the 4-bit storage (see _pack)."""
    nt, kb, _ = _dims(case)
    ng = 128 // case["group"]
    blk = packed.view(nt, kb, _block_bytes(case))
    c = blk[:, :, :1024]
    q = torch.stack((c & 15, c >> 4), dim=-1).view(nt, kb, 2, 8, 4, 4, 2, 2, 2)  # nt kb half row t b o p nib
    q = q.permute(0, 2, 3, 1, 5, 4, 7, 8, 6).reshape(nt * 16, kb * ng, case["group"]).to(dtype)
    s = blk[:, :, 1024:1024 + 32 * ng].contiguous().view(torch.bfloat16).view(nt, kb, ng, 16)
    s = s.permute(0, 3, 1, 2).reshape(nt * 16, kb * ng, 1).to(dtype)
    if case["zeros"]:
        z = blk[:, :, 1024 + 32 * ng:].reshape(nt, kb, ng, 16).permute(0, 3, 1, 2).reshape(nt * 16, kb * ng, 1)
        q = q - z.to(dtype)
    else:
        q = q - 8
    return (q * s).view(nt * 16, kb * 128)[:case["N"], :case["K"]]


def _tilize(m):
    """Row-major (R, C) -> tile stream, zero-padded to whole 32 x 32 tiles of 16 x 16 faces."""
    rt, ct = -(-m.shape[0] // 32), -(-m.shape[1] // 32)
    m = torch.nn.functional.pad(m, (0, ct * 32 - m.shape[1], 0, rt * 32 - m.shape[0]))
    return m.reshape(rt, 2, 16, ct, 2, 16).permute(0, 3, 1, 4, 2, 5).reshape(-1)


def _untilize(t, rows, cols):
    return t.view(rows // 32, cols // 32, 2, 2, 16, 16).permute(0, 2, 4, 1, 3, 5).reshape(rows, cols)


def _fake_quantize(w, group, zeros):
    """4-bit values of w (N, K), groups along K (the last one may be short)."""
    N, K = w.shape
    groups = -(-K // group)
    w = torch.nn.functional.pad(w, (0, groups * group - K)).view(N, groups, group)
    if zeros:
        lo, hi = w.amin(2, keepdim=True).clamp(max=0), w.amax(2, keepdim=True).clamp(min=0)
        s = ((hi - lo) / 15).to(torch.bfloat16).to(w.dtype)
        ok = s > 0
        d = torch.where(ok, s, torch.ones_like(s))
        z = torch.where(ok, torch.round(-lo / d).clamp(0, 15), torch.full_like(s, 8))
        q = torch.where(ok, (torch.round(w / d) + z).clamp(0, 15), z)
        q = q - z
    else:
        s = (w.abs().amax(2, keepdim=True) / 7).to(torch.bfloat16).to(w.dtype)
        ok = s > 0
        q = torch.where(ok, torch.round(w / torch.where(ok, s, torch.ones_like(s))).clamp(-8, 7), torch.zeros_like(w))
    return (s * q).view(N, -1)[:, :K]


def _act(gate, act):
    return torch.sigmoid(gate) if act == "sigmoid" else gate


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    bf = torch.bfloat16
    if op == "w4_matvec":
        y = st["x"].float() @ _unpack(st["packed"], case, torch.float32).t()
        if st["bias"] is not None:
            y = y + st["bias"].float()
        if case["relu"]:
            y = torch.where(y > 0, y, torch.zeros_like(y))
        return y.to(bf)
    if op == "w4_quantize":
        w = _untilize(st["b"], case["K"], case["N"]).t().float()
        return _tilize(_fake_quantize(w, case["group"], case["zeros"]).t()).to(bf)
    if op == "w4_dequantize":
        w = _unpack(st["packed"], case, torch.float32)
        return _tilize(w if case["transpose"] else w.t()).to(bf)
    if op == "block_norm":
        p = st["u"].float()
        out = []
        if case["post"]:
            rp = (p.square().mean(1) + _EPS).rsqrt()
            out = [rp]
            p = p * rp[:, None] * st["w_post"].float()
        if st["gate"] is not None:
            gate = _act(st["gate"].float(), case["act"])
            p = p * gate.repeat_interleave(case["gate_rows"], 0)[:case["T"]]
        h = st["resid"].float() + st["scale"] * p
        r = (h.square().mean(1) + _EPS).rsqrt()
        y = h * r[:, None] * st["w_pre"].float()
        return [h.to(st["h"].dtype), y.to(bf), r] + out
    if op == "block_norm_grad":
        return _grad(st, torch.float32)
    keep = (st["ids"] != st["pad_id"])[:, None]
    if op == "embed_rows":
        rows = st["table"][st["ids"].long()].float() * st["scale"]
        return torch.where(keep, rows, torch.zeros_like(rows)).to(st["out"].dtype)
    rows = st["dout"].float()
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    return torch.zeros_like(st["dtable"]).index_add_(0, st["ids"].long(), rows) * st["scale"]


def _grad(st, dt):
    case = st["case"]
    T, D = case["T"], case["D"]
    hh = st["h"].to(dt) * st["rstd_pre"].to(dt)[:, None]
    dy = st["dy"].to(dt)
    a = dy * st["w_pre"].to(dt)
    dh = st["dh"].to(dt) + st["rstd_pre"].to(dt)[:, None] * (a - hh * (a * hh).mean(1, keepdim=True))
    out = [dh.to(st["dresid"].dtype), None, (dy * hh).sum(0).float()]
    dz = st["scale"] * dh
    p = uh = st["u"].to(dt)
    if case["post"]:
        uh = uh * st["rstd_post"].to(dt)[:, None]
        p = uh * st["w_post"].to(dt)
    dgate = None
    if st["gate"] is not None:
        rows = case["gate_rows"]
        gate = st["gate"].to(dt)
        act = _act(gate, case["act"])
        d = dz * p
        n = gate.shape[0]
        d = torch.nn.functional.pad(d, (0, 0, 0, n * rows - T)).view(n, rows, D).sum(1)
        if case["act"] == "sigmoid":
            d = d * act * (1 - act)
        dgate = d.to(torch.bfloat16)
        dz = dz * act.repeat_interleave(rows, 0)[:T]
    if case["post"]:
        out.append((dz * uh).sum(0).float())
        b = dz * st["w_post"].to(dt)
        dz = st["rstd_post"].to(dt)[:, None] * (b - uh * (b * uh).mean(1, keepdim=True))
    out[1] = dz.to(torch.bfloat16)
    return out + ([dgate] if dgate is not None else [])


# ------------------------------------------------------------------- work ---

def work(case):
    op = case["op"]
    if op.startswith("w4"):
        K, N = case["K"], case["N"]
        groups = -(-K // case["group"])
        packed = N * K / 2 + N * groups * (3 if case["zeros"] else 2)
        if op == "w4_matvec":
            M = case["M"]
            return {"bytes": packed + 2 * M * (K + N) + (2 * N if case["bias"] else 0), "flops": 2 * M * K * N}
        if op == "w4_dequantize":
            return {"bytes": packed + 2 * K * N, "flops": 2 * K * N}
        return {"bytes": 2 * packed + 4 * K * N, "flops": 6 * K * N}
    if op.startswith("block_norm"):
        T, D = case["T"], case["D"]
        rb = 4 if case["fp32"] else 2
        gate = 2 * D * -(-T // case["gate_rows"]) if case["gate_rows"] else 0
        if op == "block_norm":
            return {"bytes": T * D * (2 * rb + 4) + gate + 8 * T + 4 * D, "flops": 10 * T * D}
        return {"bytes": T * D * (3 * rb + 6) + 2 * gate + 8 * T + 12 * D, "flops": 25 * T * D}
    T, V, D = case["T"], case["V"], case["D"]
    row = D * (4 if case["fp32"] else 2)
    ids = T * (8 if case["long_ids"] else 4)
    if op == "embed_rows":
        return {"bytes": T * (2 * D + row) + ids, "flops": T * D}
    return {"bytes": T * row + ids + 4 * V * D, "flops": T * D + V * D}


# ------------------------------------------------------------------ exact ---

def _exact_codes(st, case):
    """(codes minus zero points, scales) in 64 bits, read word by word from the storage."""
    nt, kb, _ = _dims(case)
    group, ng = case["group"], 128 // case["group"]
    N, K = case["N"], case["K"]
    raw = st["packed"].view(nt * kb, _block_bytes(case))
    dev = raw.device
    n = torch.arange(N, device=dev)[:, None]
    out = torch.empty(N, K, dtype=torch.float64, device=dev)
    step = max(1, (1 << 25) // N)
    for k0 in range(0, K, step):
        k = torch.arange(k0, min(K, k0 + step), device=dev)[None, :]
        block = (n // 16) * kb + k // 128
        word = (n % 16) * 16 + (k % 32 // 8) * 4 + k % 128 // 32
        nib = (k % 8) // 2 + 4 * (k % 2)
        byte = raw[block, word * 4 + nib // 2].to(torch.int64)
        code = (byte >> (4 * (nib % 2))) & 15
        slot = (k % 128 // group) * 16 + n % 16
        lo = raw[block, 1024 + 2 * slot].to(torch.int32)
        hi = raw[block, 1025 + 2 * slot].to(torch.int32)
        scale = ((hi << 24) | (lo << 16)).view(torch.float32).to(torch.float64)
        zero = raw[block, 1024 + 32 * ng + slot].to(torch.int64) if case["zeros"] else 8
        out[:, k0:k0 + k.shape[1]] = (code - zero).to(torch.float64) * scale
    return out


def _exact_tiles(m):
    """Tile stream of a row-major matrix by the address of each element."""
    R, C = m.shape
    rt, ct = -(-R // 32), -(-C // 32)
    out = torch.zeros(rt * ct * 1024, dtype=m.dtype, device=m.device)
    r = torch.arange(R, device=m.device)[:, None]
    c = torch.arange(C, device=m.device)[None, :]
    addr = ((r // 32) * ct + c // 32) * 1024 + ((r % 32 // 16) * 2 + c % 32 // 16) * 256 + (r % 16) * 16 + c % 16
    out[addr.reshape(-1)] = m.reshape(-1)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "w4_matvec":
        y = torch.einsum("mk,nk->mn", st["x"].to(f64), _exact_codes(st, case))
        y = y + st["bias"].to(f64) if case["bias"] else y
        return y.clamp(min=0) if case["relu"] else y
    if op == "w4_dequantize":
        w = _exact_codes(st, case)
        return _exact_tiles(w if case["transpose"] else w.t().contiguous())
    if op == "w4_quantize":
        K, N, group = case["K"], case["N"], case["group"]
        r = torch.arange(K, device="cuda")[:, None]
        c = torch.arange(N, device="cuda")[None, :]
        addr = ((r // 32) * (N // 32) + c // 32) * 1024 + ((r % 32 // 16) * 2 + c % 32 // 16) * 256 \
            + (r % 16) * 16 + c % 16
        w = st["b"][addr].to(f64)
        res = torch.empty_like(w)
        for k0 in range(0, K, group):
            part = w[k0:k0 + group]
            if case["zeros"]:
                lo, hi = part.min(0).values.clamp(max=0), part.max(0).values.clamp(min=0)
                s = ((hi - lo) / 15).to(torch.bfloat16).to(f64)
                div = torch.where(s > 0, s, 1.0)
                z = torch.round(-lo / div).clamp(0, 15)
                res[k0:k0 + group] = ((torch.round(part / div) + z).clamp(0, 15) - z) * s
            else:
                s = (part.abs().max(0).values / 7).to(torch.bfloat16).to(f64)
                res[k0:k0 + group] = torch.round(part / torch.where(s > 0, s, 1.0)).clamp(-8, 7) * s
        return _exact_tiles(res)
    if op == "block_norm":
        T, D = case["T"], case["D"]
        z = st["u"].to(f64)
        tail = []
        if case["post"]:
            rp = 1 / torch.sqrt((z * z).sum(1) / D + _EPS)
            tail = [rp]
            z = torch.einsum("td,t,d->td", z, rp, st["w_post"].to(f64))
        if st["gate"] is not None:
            ga = st["gate"].to(f64)
            ga = 1 / (1 + torch.exp(-ga)) if case["act"] == "sigmoid" else ga
            z = z * ga[torch.arange(T, device="cuda") // case["gate_rows"]]
        h = st["resid"].to(f64) + z * st["scale"]
        r = 1 / torch.sqrt((h * h).sum(1) / D + _EPS)
        return [h, torch.einsum("td,t,d->td", h, r, st["w_pre"].to(f64)), r] + tail
    if op == "block_norm_grad":
        return _exact_grad(st)
    ids = st["ids"].long()
    if op == "embed_rows":
        out = st["table"].to(f64)[ids] * st["scale"]
        out[ids == st["pad_id"]] = 0
        return out
    live = ids != st["pad_id"]
    out = torch.zeros(case["V"], case["D"], dtype=f64, device="cuda")
    return out.index_put_((ids[live],), st["dout"][live].to(f64), accumulate=True) * st["scale"]


def _exact_grad(st):
    """The gradients by automatic differentiation of the forward's definition in
    64 bits, the two root-mean-square factors taken from their saved values."""
    case = st["case"]
    T, D = case["T"], case["D"]
    f64 = torch.float64

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v, r):
            ctx.save_for_backward(v, r)
            return v * r[:, None]

        @staticmethod
        def backward(ctx, d):
            # r = (mean v^2 + eps)^(-1/2):  dr/dv_j = -r^3 v_j / D
            v, r = ctx.saved_tensors
            return r[:, None] * d - (r ** 3 / D * (d * v).sum(1))[:, None] * v, None

    def leaf(t):
        return None if t is None else t.to(f64).requires_grad_()

    u, w_post, w_pre, gate = leaf(st["u"]), leaf(st["w_post"]), leaf(st["w_pre"]), leaf(st["gate"])
    resid = torch.zeros(T, D, dtype=f64, device="cuda", requires_grad=True)
    z = u
    if case["post"]:
        z = Norm.apply(z, st["rstd_post"].to(f64)) * w_post
    if gate is not None:
        a = 1 / (1 + torch.exp(-gate)) if case["act"] == "sigmoid" else gate
        z = z * a[torch.arange(T, device="cuda") // case["gate_rows"]]
    branch = resid + z * st["scale"]
    h = branch + (st["h"].to(f64) - branch.detach())  # the saved h, with the branch's derivative
    y = Norm.apply(h, st["rstd_pre"].to(f64)) * w_pre
    ((y * st["dy"].to(f64)).sum() + (h * st["dh"].to(f64)).sum()).backward()
    return [t.grad for t in (resid, u, w_pre, w_post, gate) if t is not None]
