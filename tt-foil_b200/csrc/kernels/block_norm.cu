// The norms after a residual block and before the next one, fused with the
// block's gate, its scale and the residual addition; and their gradients.
// The formulas stand at foil_block_norm_dev in include/foil_c.h.
#include "block_norm.cuh"

#include "common.cuh"

namespace foil {
namespace norm {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load(const uint16_t* p, uint64_t i) { return bf16_bits_to_f32(p[i]); }
__device__ __forceinline__ float load(const float* p, uint64_t i) { return p[i]; }
__device__ __forceinline__ void store(uint16_t* p, uint64_t i, float v) { p[i] = (uint16_t)(cvt_bf16x2(v, 0.0f) & 0xffffu); }
__device__ __forceinline__ void store(float* p, uint64_t i, float v) { p[i] = v; }

__device__ __forceinline__ float act(float g, uint32_t kind) { return kind ? 1.0f / (1.0f + expf(-g)) : g; }

// Sum over the CTA, the same value in every thread.
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[kThreads / 32];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < kThreads / 32; ++i) s += part[i];
    return s;
}

// One CTA for each token.
template <class R>
__global__ void __launch_bounds__(kThreads) forward_kernel(Forward p) {
    const uint64_t t = blockIdx.x;
    const R* resid = static_cast<const R*>(p.resid) + t * p.ld_resid;
    const uint16_t* u = p.u ? p.u + t * p.ld_u : nullptr;
    const uint16_t* gate = p.gate ? p.gate + t / p.gate_rows * p.ld_gate : nullptr;
    float rp = 1.0f;
    if (u && p.post) {
        float s = 0.0f;
        for (uint32_t i = threadIdx.x; i < p.D; i += kThreads) s += load(u, i) * load(u, i);
        rp = 1.0f / sqrtf(block_sum(s) / (float)p.D + p.eps);
        if (p.rstd_post && threadIdx.x == 0) p.rstd_post[t] = rp;
    }
    auto branch = [&](uint32_t i) {
        float v = load(resid, i);
        if (u) {
            float b = load(u, i);
            if (p.post) b *= rp;
            if (p.w_post) b *= load(p.w_post, i);
            if (gate) b *= act(load(gate, i), p.gate_act);
            v += p.scale * b;
        }
        return v;
    };
    float r = 0.0f;
    if (p.y) {
        float s = 0.0f;
        for (uint32_t i = threadIdx.x; i < p.D; i += kThreads) s += branch(i) * branch(i);
        r = 1.0f / sqrtf(block_sum(s) / (float)p.D + p.eps);
        if (p.rstd_pre && threadIdx.x == 0) p.rstd_pre[t] = r;
    }
    for (uint32_t i = threadIdx.x; i < p.D; i += kThreads) {
        const float v = branch(i);
        if (p.h) store(static_cast<R*>(p.h) + t * p.ld_h, i, v);
        if (p.y) store(p.y + t * p.ld_y, i, v * r * (p.w_pre ? load(p.w_pre, i) : 1.0f));
    }
}

// The row sums of a token's gradients: c1 = mean(a hhat), c2 = mean(b uhat).
template <class R>
struct RowGrad {
    const Backward& p;
    uint64_t t;
    float rh, ru, c1;
    __device__ float hhat(uint32_t i) const { return load(static_cast<const R*>(p.h) + t * p.ld_h, i) * rh; }
    __device__ float a(uint32_t i) const { return load(p.dy + t * p.ld_dy, i) * (p.w_pre ? load(p.w_pre, i) : 1.0f); }
    __device__ float dh(uint32_t i) const {
        float v = p.dh ? load(static_cast<const R*>(p.dh) + t * p.ld_dh, i) : 0.0f;
        if (p.dy) v += rh * (a(i) - hhat(i) * c1);
        return v;
    }
    __device__ float uhat(uint32_t i) const { return load(p.u + t * p.ld_u, i) * ru; }
    __device__ float gate(uint32_t i) const { return load(p.gate + t / p.gate_rows * p.ld_gate, i); }
    __device__ float pv(uint32_t i) const { return uhat(i) * (p.w_post ? load(p.w_post, i) : 1.0f); }
    __device__ float dp(uint32_t i) const {
        return p.scale * dh(i) * (p.gate ? act(gate(i), p.gate_act) : 1.0f);
    }
};

template <class R>
__device__ RowGrad<R> row_grad(const Backward& p, uint64_t t) {
    RowGrad<R> g{p, t, 0.0f, 1.0f, 0.0f};
    if (p.dy) g.rh = p.rstd_pre[t], g.c1 = p.ws[t];
    if (p.post && p.u) g.ru = p.rstd_post[t];
    return g;
}

template <class R>
__global__ void __launch_bounds__(kThreads) backward_rows(Backward p) {
    const uint64_t t = blockIdx.x;
    RowGrad<R> g{p, t, p.dy ? p.rstd_pre[t] : 0.0f, p.post && p.u ? p.rstd_post[t] : 1.0f, 0.0f};
    if (p.dy) {
        float s = 0.0f;
        for (uint32_t i = threadIdx.x; i < p.D; i += kThreads) s += g.a(i) * g.hhat(i);
        g.c1 = block_sum(s) / (float)p.D;
        if (threadIdx.x == 0) p.ws[t] = g.c1;
    }
    float c2 = 0.0f;
    if (p.du && p.post) {
        float s = 0.0f;
        for (uint32_t i = threadIdx.x; i < p.D; i += kThreads) s += g.dp(i) * g.pv(i);
        c2 = block_sum(s) / (float)p.D;
    }
    for (uint32_t i = threadIdx.x; i < p.D; i += kThreads) {
        if (p.dresid) store(static_cast<R*>(p.dresid) + t * p.ld_dresid, i, g.dh(i));
        if (p.du) {
            float v = g.dp(i);
            if (p.post) v = g.ru * (v * (p.w_post ? load(p.w_post, i) : 1.0f) - g.uhat(i) * c2);
            store(p.du + t * p.ld_du, i, v);
        }
    }
}

// One thread for each column: the sums over tokens.
template <class R>
__global__ void __launch_bounds__(kThreads) backward_columns(Backward p) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= p.D) return;
    float dw_pre = 0.0f, dw_post = 0.0f, dgate = 0.0f;
    for (uint32_t t = 0; t < p.T; ++t) {
        const RowGrad<R> g = row_grad<R>(p, t);
        if (p.dw_pre) dw_pre += load(p.dy + t * p.ld_dy, i) * g.hhat(i);
        if (p.dw_post) dw_post += g.dp(i) * g.uhat(i);
        if (p.dgate) {
            dgate += p.scale * g.dh(i) * g.pv(i);
            if (t % p.gate_rows == p.gate_rows - 1 || t == p.T - 1) {
                if (p.gate_act) {
                    const float s = act(g.gate(i), p.gate_act);
                    dgate *= s * (1.0f - s);
                }
                store(p.dgate + t / p.gate_rows * p.ld_dgate, i, dgate);
                dgate = 0.0f;
            }
        }
    }
    if (p.dw_pre) p.dw_pre[i] = dw_pre;
    if (p.dw_post) p.dw_post[i] = dw_post;
}

cudaError_t count(cudaError_t e) {
    if (e == cudaSuccess) foil_count_launch();
    return e;
}

}  // namespace

uint64_t backward_ws_bytes(uint32_t T, uint32_t D, uint32_t gate_rows) {
    (void)D, (void)gate_rows;
    return 4ull * T;
}

cudaError_t forward(const Forward& p, bool fp32, cudaStream_t s) {
    if (fp32)
        forward_kernel<float><<<p.T, kThreads, 0, s>>>(p);
    else
        forward_kernel<uint16_t><<<p.T, kThreads, 0, s>>>(p);
    return count(cudaGetLastError());
}

template <class R>
static cudaError_t backward_typed(const Backward& p, cudaStream_t s) {
    if (p.T) {
        backward_rows<R><<<p.T, kThreads, 0, s>>>(p);
        const cudaError_t e = count(cudaGetLastError());
        if (e != cudaSuccess) return e;
    }
    if (!p.dw_pre && !p.dw_post && !p.dgate) return cudaSuccess;
    backward_columns<R><<<(p.D + kThreads - 1) / kThreads, kThreads, 0, s>>>(p);
    return count(cudaGetLastError());
}

cudaError_t backward(const Backward& p, bool fp32, cudaStream_t s) {
    return fp32 ? backward_typed<float>(p, s) : backward_typed<uint16_t>(p, s);
}

}  // namespace norm
}  // namespace foil
