// C-ABI of the token-path operators (include/foil_c.h): argument checks, then
// the launchers of kernels/w4.cu, kernels/w4_batch.cu, kernels/block_norm.cu
// and kernels/embed_rows.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "entry.hpp"
#include "kernels/block_norm.cuh"
#include "kernels/embed_rows.cuh"
#include "kernels/w4.cuh"

namespace {

using foil::aligned16;
using foil::FoilError;
using foil::guarded;

[[noreturn]] void invalid(const char* what, const char* msg) {
    throw FoilError(FOIL_ERR_INVALID, std::string(what) + ": " + msg);
}

void launched(const char* what, cudaError_t e) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        throw FoilError(FOIL_ERR_CUDA, std::string(what) + ": CUDA launch failed: " + cudaGetErrorString(e));
    }
}

// The memory of one argument, for the overlap rules: [begin, end), in rows of
// `row` bytes `pitch` bytes apart if pitch is not 0.
struct Span {
    uintptr_t begin = 0, end = 0;
    uint64_t pitch = 0, row = 0;
    Span(const void* p, uint64_t bytes) : begin((uintptr_t)p), end((uintptr_t)p + (p ? bytes : 0)) {}
};
// Two matrices of one pitch may interleave (column slices of one buffer).
bool overlap(const Span& a, const Span& b) {
    if (a.begin >= b.end || b.begin >= a.end) return false;
    if (a.pitch == 0 || a.pitch != b.pitch) return true;
    const uint64_t d = b.begin >= a.begin ? (b.begin - a.begin) % a.pitch
                                          : (a.pitch - (a.begin - b.begin) % a.pitch) % a.pitch;
    return d < a.row || a.pitch - d < b.row;
}

// rows x cols elements with a row stride; `ld` 0 becomes the dense stride.
Span matrix(const char* what, const void* p, uint64_t& ld, uint64_t rows, uint64_t cols, uint64_t elem) {
    if (ld == 0) ld = cols;
    if (!p) return Span(nullptr, 0);
    if (ld < cols) invalid(what, "a row stride is shorter than a row");
    if ((uintptr_t)p % elem) invalid(what, "misaligned pointer");
    if (ld >= (1ull << 32) || (rows && ld > (1ull << 46) / rows)) invalid(what, "tensor too large");
    Span s(p, rows ? ((rows - 1) * ld + cols) * elem : 0);
    s.pitch = ld * elem, s.row = cols * elem;
    return s;
}

// No output may overlap an input or another output.
void disjoint(const char* what, std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
    for (const Span* o = outs.begin(); o != outs.end(); ++o) {
        for (const Span& in : ins)
            if (overlap(*o, in)) invalid(what, "an output overlaps an input");
        for (const Span* q = outs.begin(); q != o; ++q)
            if (overlap(*o, *q)) invalid(what, "two outputs overlap");
    }
}

bool weights_ok(uint32_t K, uint32_t N, uint32_t group) {
    return K >= 1 && N >= 1 && K <= (1u << 24) && N <= (1u << 24) && (group == 32 || group == 64 || group == 128);
}

foil::w4::Weights weights(const char* what, uint32_t K, uint32_t N, uint32_t group, int32_t zeros) {
    if (group != 32 && group != 64 && group != 128) invalid(what, "group must be 32, 64 or 128");
    if (!weights_ok(K, N, group)) invalid(what, "K and N must be from 1 to 2^24");
    return foil::w4::Weights{K, N, group, zeros ? 1u : 0u};
}

}  // namespace

// ---------------------------------------------------------- 4-bit weights ---
extern "C" uint64_t foil_w4_packed_bytes(uint32_t K, uint32_t N, uint32_t group, int32_t zeros) {
    return weights_ok(K, N, group) ? foil::w4::packed_bytes(foil::w4::Weights{K, N, group, zeros ? 1u : 0u}) : 0;
}

extern "C" int foil_w4_pack_dev(const uint8_t* codes, const uint16_t* scales, const uint8_t* zero_points,
                                void* packed, uint32_t K, uint32_t N, uint32_t group, void* stream) {
    const char* what = "foil_w4_pack_dev";
    return guarded([&] {
        const foil::w4::Weights w = weights(what, K, N, group, zero_points != nullptr);
        if (!codes || !scales || !packed || !aligned16(packed) || (uintptr_t)scales % 2)
            invalid(what, "null or misaligned pointer");
        const uint64_t groups = (uint64_t)N * ((K + group - 1) / group);
        disjoint(what, {Span(packed, foil::w4::packed_bytes(w))},
                 {Span(codes, (uint64_t)N * K), Span(scales, 2 * groups), Span(zero_points, groups)});
        launched(what, foil::w4::pack(codes, scales, zero_points, (uint8_t*)packed, w, (cudaStream_t)stream));
    });
}

extern "C" int foil_w4_quantize_tiles_dev(const uint16_t* tiles, void* packed, uint32_t Kt, uint32_t Nt,
                                          uint32_t group, int32_t zeros, void* stream) {
    const char* what = "foil_w4_quantize_tiles_dev";
    return guarded([&] {
        if (Kt == 0 || Nt == 0) return;
        if (Kt > 65535 || Nt > 65535) invalid(what, "tile counts must be <= 65535");
        const foil::w4::Weights w = weights(what, 32 * Kt, 32 * Nt, group, zeros);
        if (!tiles || !packed || !aligned16(tiles) || !aligned16(packed)) invalid(what, "null or misaligned pointer");
        disjoint(what, {Span(packed, foil::w4::packed_bytes(w))}, {Span(tiles, (uint64_t)Kt * Nt * 2048)});
        launched(what, foil::w4::quantize_tiles(tiles, (uint8_t*)packed, w, (cudaStream_t)stream));
    });
}

extern "C" int foil_w4_dequantize_tiles_dev(const void* packed, uint16_t* tiles, uint32_t K, uint32_t N,
                                            uint32_t group, int32_t zeros, int32_t transpose, void* stream) {
    const char* what = "foil_w4_dequantize_tiles_dev";
    return guarded([&] {
        if (K == 0 || N == 0) return;
        const foil::w4::Weights w = weights(what, K, N, group, zeros);
        if (K > 32u * 65535u || N > 32u * 65535u) invalid(what, "tile counts must be <= 65535");
        if (!tiles || !packed || !aligned16(tiles) || !aligned16(packed)) invalid(what, "null or misaligned pointer");
        const uint64_t out = (uint64_t)((K + 31) / 32) * ((N + 31) / 32) * 2048;
        disjoint(what, {Span(tiles, out)}, {Span(packed, foil::w4::packed_bytes(w))});
        launched(what, foil::w4::dequantize_tiles((const uint8_t*)packed, tiles, w, transpose != 0,
                                                  (cudaStream_t)stream));
    });
}

extern "C" int foil_w4_matvec_dev(const uint16_t* x, uint64_t ld_x, const void* packed, const uint16_t* bias,
                                  uint16_t* y, uint64_t ld_y, uint32_t M, uint32_t K, uint32_t N, uint32_t group,
                                  int32_t zeros, int32_t relu, void* stream) {
    const char* what = "foil_w4_matvec_dev";
    return guarded([&] {
        if (M == 0 || N == 0) return;
        const foil::w4::Weights w = weights(what, K, N, group, zeros);
        if (M > foil::w4::kMaxRows)
            invalid(what, "at most 64 rows (for more, dequantise and use foil_matmul_tiles_dev)");
        if (K > foil::w4::kMaxK) invalid(what, "K must be at most 32768");
        if (!x || !packed || !y || !aligned16(packed) || (uintptr_t)bias % 2)
            invalid(what, "null or misaligned pointer");
        const Span sx = matrix(what, x, ld_x, M, K, 2), sy = matrix(what, y, ld_y, M, N, 2);
        disjoint(what, {sy}, {sx, Span(packed, foil::w4::packed_bytes(w)), Span(bias, 2ull * N)});
        launched(what, foil::w4::matvec(x, ld_x, (const uint8_t*)packed, bias, y, ld_y, M, w, relu != 0,
                                        M > foil::w4::kWarpRows ? foil_error_word() : nullptr, (cudaStream_t)stream));
    });
}

// ------------------------------------------------------------ block norms ---
extern "C" int foil_block_norm_dev(const void* resid, uint64_t ld_resid, const uint16_t* u, uint64_t ld_u,
                                   int32_t post, const uint16_t* w_post, const uint16_t* gate, uint64_t ld_gate,
                                   uint32_t gate_rows, int32_t gate_act, const uint16_t* w_pre, void* h,
                                   uint64_t ld_h, uint16_t* y, uint64_t ld_y, float* rstd_post, float* rstd_pre,
                                   uint32_t T, uint32_t D, int32_t fp32, float scale, float eps, void* stream) {
    const char* what = "foil_block_norm_dev";
    return guarded([&] {
        if (T == 0 || D == 0) return;
        if (D > foil::norm::kMaxD) invalid(what, "D must be at most 16384");
        if (T > foil::norm::kMaxT) invalid(what, "T must be at most 2^31");
        if (!resid || (!h && !y)) invalid(what, "null pointer");
        if (!u && (post || w_post || gate || rstd_post)) invalid(what, "post norm or gate without the block's output");
        if (!post && (w_post || rstd_post)) invalid(what, "w_post or rstd_post without the post norm");
        if (!y && (w_pre || rstd_pre)) invalid(what, "w_pre or rstd_pre without y");
        if (gate && gate_rows == 0) invalid(what, "gate_rows must be positive");
        if (gate_act != FOIL_GATE_NONE && gate_act != FOIL_GATE_SIGMOID) invalid(what, "unknown gate activation");
        if (!(eps >= 0.0f) || std::isinf(eps)) invalid(what, "eps must be finite and not negative");
        if ((uintptr_t)w_post % 2 || (uintptr_t)w_pre % 2 || (uintptr_t)rstd_post % 4 || (uintptr_t)rstd_pre % 4)
            invalid(what, "misaligned pointer");
        const uint64_t re = fp32 ? 4 : 2, grows = gate ? (T - 1) / gate_rows + 1 : 0;
        const Span sr = matrix(what, resid, ld_resid, T, D, re), su = matrix(what, u, ld_u, T, D, 2),
                   sg = matrix(what, gate, ld_gate, grows, D, 2), sh = matrix(what, h, ld_h, T, D, re),
                   sy = matrix(what, y, ld_y, T, D, 2), spo(rstd_post, 4ull * T), spr(rstd_pre, 4ull * T),
                   wpo(w_post, 2ull * D), wpr(w_pre, 2ull * D);
        // In place: every thread reads its elements of a row before it writes them.
        const bool h_on_resid = h && h == resid && ld_h == ld_resid, y_on_u = y && y == u && ld_y == ld_u;
        disjoint(what, {sh, sy, spo, spr}, {sg, wpo, wpr});
        disjoint(what, {sy, spo, spr}, {sr});
        disjoint(what, {sh, spo, spr}, {su});
        if (!h_on_resid) disjoint(what, {sh}, {sr});
        if (!y_on_u) disjoint(what, {sy}, {su});
        foil::norm::Forward p{};
        p.resid = resid, p.u = u, p.w_post = w_post, p.gate = gate, p.w_pre = w_pre, p.h = h, p.y = y;
        p.rstd_post = rstd_post, p.rstd_pre = rstd_pre;
        p.ld_resid = ld_resid, p.ld_u = ld_u, p.ld_gate = ld_gate, p.ld_h = ld_h, p.ld_y = ld_y;
        p.gate_rows = gate ? gate_rows : 1, p.gate_act = (uint32_t)gate_act, p.post = post ? 1 : 0, p.T = T, p.D = D;
        p.scale = scale, p.eps = eps;
        launched(what, foil::norm::forward(p, fp32 != 0, (cudaStream_t)stream));
    });
}

extern "C" uint64_t foil_block_norm_grad_ws_bytes(uint32_t T, uint32_t D, uint32_t gate_rows) {
    if (T > foil::norm::kMaxT || D > foil::norm::kMaxD) return 0;
    return foil::norm::backward_ws_bytes(T, D, gate_rows);
}

extern "C" int foil_block_norm_grad_dev(const void* dh, uint64_t ld_dh, const uint16_t* dy, uint64_t ld_dy,
                                        const void* h, uint64_t ld_h, const float* rstd_pre, const uint16_t* w_pre,
                                        const uint16_t* u, uint64_t ld_u, int32_t post, const float* rstd_post,
                                        const uint16_t* w_post, const uint16_t* gate, uint64_t ld_gate,
                                        uint32_t gate_rows, int32_t gate_act, void* dresid, uint64_t ld_dresid,
                                        uint16_t* du, uint64_t ld_du, uint16_t* dgate, uint64_t ld_dgate,
                                        float* dw_post, float* dw_pre, void* ws, uint64_t ws_bytes, uint32_t T,
                                        uint32_t D, int32_t fp32, float scale, void* stream) {
    const char* what = "foil_block_norm_grad_dev";
    return guarded([&] {
        if (D == 0) return;
        if (D > foil::norm::kMaxD) invalid(what, "D must be at most 16384");
        if (T > foil::norm::kMaxT) invalid(what, "T must be at most 2^31");
        if (!dresid && !du && !dgate && !dw_post && !dw_pre) invalid(what, "no output is wanted");
        if (!dh && !dy && T) invalid(what, "dh and dy are both null");
        if (dy && T && (!h || !rstd_pre)) invalid(what, "dy needs h and rstd_pre");
        if (!dy && T && (w_pre || dw_pre)) invalid(what, "w_pre or dw_pre without dy");
        if (T && (du || dgate || dw_post) && !u) invalid(what, "du, dgate and dw_post need the block's output");
        if (T && u && post && !rstd_post) invalid(what, "the post norm needs rstd_post");
        if (!post && (w_post || dw_post || rstd_post)) invalid(what, "w_post, dw_post or rstd_post without the post norm");
        if (dgate && !gate && T) invalid(what, "dgate without a gate");
        if (gate && gate_rows == 0) invalid(what, "gate_rows must be positive");
        if (gate_act != FOIL_GATE_NONE && gate_act != FOIL_GATE_SIGMOID) invalid(what, "unknown gate activation");
        if ((uintptr_t)w_post % 2 || (uintptr_t)w_pre % 2 || (uintptr_t)rstd_post % 4 || (uintptr_t)rstd_pre % 4 ||
            (uintptr_t)dw_post % 4 || (uintptr_t)dw_pre % 4)
            invalid(what, "misaligned pointer");
        const uint64_t need = foil::norm::backward_ws_bytes(T, D, gate ? gate_rows : 0);
        if (ws_bytes < need || (need && !ws) || !aligned16(ws)) invalid(what, "workspace too small or misaligned");
        const uint64_t re = fp32 ? 4 : 2, grows = gate && T ? (T - 1) / gate_rows + 1 : 0;
        const Span sdh = matrix(what, dh, ld_dh, T, D, re), sdy = matrix(what, dy, ld_dy, T, D, 2),
                   sh = matrix(what, h, ld_h, T, D, re), su = matrix(what, u, ld_u, T, D, 2),
                   sg = matrix(what, gate, ld_gate, grows, D, 2), sdr = matrix(what, dresid, ld_dresid, T, D, re),
                   sdu = matrix(what, du, ld_du, T, D, 2), sdg = matrix(what, dgate, ld_dgate, grows, D, 2);
        disjoint(what, {sdr, sdu, sdg, Span(dw_post, 4ull * D), Span(dw_pre, 4ull * D), Span(ws, need)},
                 {sdh, sdy, sh, su, sg, Span(w_post, 2ull * D), Span(w_pre, 2ull * D), Span(rstd_post, 4ull * T),
                  Span(rstd_pre, 4ull * T)});
        foil::norm::Backward p{};
        p.dh = dh, p.h = h, p.dy = dy, p.w_pre = w_pre, p.u = u, p.w_post = w_post, p.gate = gate;
        p.rstd_pre = rstd_pre, p.rstd_post = rstd_post, p.dresid = dresid, p.du = du, p.dgate = dgate;
        p.dw_post = dw_post, p.dw_pre = dw_pre, p.ws = (float*)ws;
        p.ld_dh = ld_dh, p.ld_dy = ld_dy, p.ld_h = ld_h, p.ld_u = ld_u, p.ld_gate = ld_gate;
        p.ld_dresid = ld_dresid, p.ld_du = ld_du, p.ld_dgate = ld_dgate;
        p.gate_rows = gate ? gate_rows : 0, p.gate_act = (uint32_t)gate_act, p.post = post ? 1 : 0, p.T = T, p.D = D;
        p.scale = scale;
        launched(what, foil::norm::backward(p, fp32 != 0, (cudaStream_t)stream));
    });
}

// --------------------------------------------------------- embedding rows ---
namespace {
void check_ids(const char* what, const void* ids, int32_t id_bytes, uint32_t T, uint32_t V, uint32_t D) {
    if (id_bytes != 4 && id_bytes != 8) invalid(what, "id_bytes must be 4 or 8");
    if (T > foil::embed::kMaxRows || V > foil::embed::kMaxRows) invalid(what, "T and V must be at most 2^24");
    if (D > foil::embed::kMaxD) invalid(what, "D must be at most 2^20");
    if (T && !ids) invalid(what, "null pointer");
    if ((uintptr_t)ids % (uint32_t)id_bytes) invalid(what, "misaligned pointer");
}
}  // namespace

extern "C" int foil_embed_rows_dev(const void* ids, int32_t id_bytes, const uint16_t* table, uint64_t ld_table,
                                   void* out, uint64_t ld_out, uint32_t T, uint32_t V, uint32_t D, int32_t fp32,
                                   float scale, int64_t pad_id, void* stream) {
    const char* what = "foil_embed_rows_dev";
    return guarded([&] {
        if (T == 0 || D == 0) return;
        check_ids(what, ids, id_bytes, T, V, D);
        if (!out || (V && !table)) invalid(what, "null pointer");
        const Span st = matrix(what, table, ld_table, V, D, 2), so = matrix(what, out, ld_out, T, D, fp32 ? 4 : 2);
        disjoint(what, {so}, {st, Span(ids, (uint64_t)T * id_bytes)});
        foil::embed::Lookup p{};
        p.ids = ids, p.table = table, p.out = out, p.ld_table = ld_table, p.ld_out = ld_out;
        p.T = T, p.V = V, p.D = D, p.id_bytes = id_bytes, p.scale = scale, p.pad_id = pad_id;
        p.err = foil_error_word();
        launched(what, foil::embed::lookup(p, fp32 != 0, (cudaStream_t)stream));
    });
}

extern "C" uint64_t foil_embed_rows_grad_ws_bytes(uint32_t T, uint32_t V, uint32_t D) {
    if (T > foil::embed::kMaxRows || V > foil::embed::kMaxRows || D > foil::embed::kMaxD) return 0;
    return foil::embed::gradient_ws_bytes(T, V, D);
}

extern "C" int foil_embed_rows_grad_dev(const void* ids, int32_t id_bytes, const void* dout, uint64_t ld_dout,
                                        float* dtable, uint64_t ld_dtable, uint32_t T, uint32_t V, uint32_t D,
                                        int32_t fp32, float scale, int64_t pad_id, int32_t accumulate, void* ws,
                                        uint64_t ws_bytes, void* stream) {
    const char* what = "foil_embed_rows_grad_dev";
    return guarded([&] {
        if (V == 0 || D == 0) return;
        check_ids(what, ids, id_bytes, T, V, D);
        if (!dtable || (T && !dout)) invalid(what, "null pointer");
        const uint64_t need = foil::embed::gradient_ws_bytes(T, V, D);
        if (ws_bytes < need || (need && !ws) || !aligned16(ws)) invalid(what, "workspace too small or misaligned");
        const Span sd = matrix(what, dout, ld_dout, T, D, fp32 ? 4 : 2), st = matrix(what, dtable, ld_dtable, V, D, 4);
        disjoint(what, {st, Span(ws, need)}, {sd, Span(ids, (uint64_t)T * id_bytes)});
        foil::embed::Gradient p{};
        p.ids = ids, p.dout = dout, p.dtable = dtable, p.ws = ws, p.ld_dout = ld_dout, p.ld_dtable = ld_dtable;
        p.T = T, p.V = V, p.D = D, p.id_bytes = id_bytes, p.scale = scale, p.pad_id = pad_id;
        p.accumulate = accumulate ? 1 : 0;
        p.err = foil_error_word();
        launched(what, foil::embed::gradient(p, fp32 != 0, (cudaStream_t)stream));
    });
}
