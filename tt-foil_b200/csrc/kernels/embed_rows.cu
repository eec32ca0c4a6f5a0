// Embedding rows: scaled lookup and the table's gradient.
#include "embed_rows.cuh"

#include "common.cuh"

namespace foil {
namespace embed {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t load_id(const void* ids, int32_t id_bytes, uint64_t t) {
    return id_bytes == 8 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
}
__device__ __forceinline__ float load(const uint16_t* p, uint64_t i) { return bf16_bits_to_f32(p[i]); }
__device__ __forceinline__ float load(const float* p, uint64_t i) { return p[i]; }
__device__ __forceinline__ void store(uint16_t* p, uint64_t i, float v) { p[i] = (uint16_t)(cvt_bf16x2(v, 0.0f) & 0xffffu); }
__device__ __forceinline__ void store(float* p, uint64_t i, float v) { p[i] = v; }

// One CTA for each token.
template <class O>
__global__ void __launch_bounds__(kThreads) lookup_kernel(Lookup p) {
    const uint64_t t = blockIdx.x;
    const int64_t id = load_id(p.ids, p.id_bytes, t);
    const bool ok = id != p.pad_id && id >= 0 && id < (int64_t)p.V;
    if (!ok && id != p.pad_id && threadIdx.x == 0) atomicOr(p.err, kErrBadIndex);
    O* out = static_cast<O*>(p.out) + t * p.ld_out;
    for (uint32_t i = threadIdx.x; i < p.D; i += kThreads)
        store(out, i, ok ? p.scale * load(p.table, (uint64_t)id * p.ld_table + i) : 0.0f);
}

// One CTA for each table row: looks through all ids.
template <class I>
__global__ void __launch_bounds__(kThreads) gradient_kernel(Gradient p) {
    const uint64_t v = blockIdx.x;
    float* row = p.dtable + v * p.ld_dtable;
    __shared__ uint32_t hit;
    for (uint32_t i0 = 0; i0 < p.D; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        float s = 0.0f;
        bool any = false;
        for (uint32_t t0 = 0; t0 < p.T; t0 += kThreads) {
            const uint32_t t = t0 + threadIdx.x;
            const int64_t id = t < p.T ? load_id(p.ids, p.id_bytes, t) : -1;
            const bool bad = t < p.T && id != p.pad_id && (id < 0 || id >= (int64_t)p.V);
            if (bad && v == 0) atomicOr(p.err, kErrBadIndex);
            if (!__syncthreads_or(t < p.T && id == (int64_t)v && id != p.pad_id)) continue;
            for (uint32_t j = 0; j < kThreads && t0 + j < p.T; ++j) {
                if (threadIdx.x == j) hit = id == (int64_t)v && id != p.pad_id;
                __syncthreads();
                if (hit && i < p.D) s += load(static_cast<const I*>(p.dout) + (uint64_t)(t0 + j) * p.ld_dout, i);
                any |= hit != 0;
                __syncthreads();
            }
        }
        if (i < p.D && (any || !p.accumulate)) row[i] = (p.accumulate ? row[i] : 0.0f) + p.scale * s;
    }
}

cudaError_t count(cudaError_t e) {
    if (e == cudaSuccess) foil_count_launch();
    return e;
}

}  // namespace

uint64_t gradient_ws_bytes(uint32_t T, uint32_t V, uint32_t D) {
    (void)T, (void)V, (void)D;
    return 0;
}

cudaError_t lookup(const Lookup& p, bool fp32, cudaStream_t s) {
    if (fp32)
        lookup_kernel<float><<<p.T, kThreads, 0, s>>>(p);
    else
        lookup_kernel<uint16_t><<<p.T, kThreads, 0, s>>>(p);
    return count(cudaGetLastError());
}

cudaError_t gradient(const Gradient& p, bool fp32, cudaStream_t s) {
    if (fp32)
        gradient_kernel<float><<<p.V, kThreads, 0, s>>>(p);
    else
        gradient_kernel<uint16_t><<<p.V, kThreads, 0, s>>>(p);
    return count(cudaGetLastError());
}

}  // namespace embed
}  // namespace foil
