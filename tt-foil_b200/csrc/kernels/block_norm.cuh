// Launchers of the block norm kernels (block_norm.cu).  Arguments are checked
// by the caller; each returns a cudaError_t.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace foil {
namespace norm {

constexpr uint32_t kMaxD = 16384;
constexpr uint32_t kMaxT = 1u << 31;  // tokens are counted in 32 bits

struct Forward {
    const void* resid;
    const uint16_t *u, *w_post, *gate, *w_pre;
    void* h;
    uint16_t* y;
    float *rstd_post, *rstd_pre;
    uint64_t ld_resid, ld_u, ld_gate, ld_h, ld_y;
    uint32_t gate_rows, gate_act, post, T, D;
    float scale, eps;
};

struct Backward {
    const void *dh, *h;
    const uint16_t *dy, *w_pre, *u, *w_post, *gate;
    const float *rstd_pre, *rstd_post;
    void* dresid;
    uint16_t *du, *dgate;
    float *dw_post, *dw_pre, *ws;
    uint64_t ld_dh, ld_dy, ld_h, ld_u, ld_gate, ld_dresid, ld_du, ld_dgate;
    uint32_t gate_rows, gate_act, post, T, D;
    float scale;
};

uint64_t backward_ws_bytes(uint32_t T, uint32_t D, uint32_t gate_rows);
cudaError_t forward(const Forward& p, bool fp32, cudaStream_t s);
cudaError_t backward(const Backward& p, bool fp32, cudaStream_t s);

}  // namespace norm
}  // namespace foil
