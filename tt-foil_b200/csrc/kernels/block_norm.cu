// The norms after a residual block and before the next one, fused with the
// block's gate, its scale and the residual addition; and their gradients.
// The formulas stand at foil_block_norm_dev in include/foil_c.h.
//
// HBM-bound: every tensor is read and written once.  A row lives in the
// registers of one warp (up to 32 E channels) or one CTA, E channels a thread,
// and a warp or CTA goes over many rows, the weights in its registers.
// Channels are moved in vectors of 16 bytes where D, the strides and the
// pointers allow, else of 4 bytes (even D), else one by one.
#include "block_norm.cuh"

#include <cstring>

#include "common.cuh"

namespace foil {
namespace norm {
namespace {

// V values of type T (uint16_t: bf16 bits) as loaded.
template <class T, int V>
struct Raw {
    static constexpr int kWords = (sizeof(T) * V + 3) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (sizeof(T) * V >= 16) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if constexpr (sizeof(T) * V == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (sizeof(T) * V == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        return i % 2 ? __uint_as_float(w[i / 2] & 0xffff0000u) : bf16_bits_to_f32(w[i / 2] & 0xffffu);
    }
};

template <int V>
__device__ __forceinline__ void put(uint16_t* p, const float* v) {
    if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3]),
                                                  cvt_bf16x2(v[4], v[5]), cvt_bf16x2(v[6], v[7]));
    } else if constexpr (V == 2) {
        *reinterpret_cast<uint32_t*>(p) = cvt_bf16x2(v[0], v[1]);
    } else {
        *p = (uint16_t)(cvt_bf16x2(v[0], 0.0f) & 0xffffu);
    }
}
template <int V>
__device__ __forceinline__ void put(float* p, const float* v) {
    if constexpr (V == 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (V == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
        *p = v[0];
    }
}

__device__ __forceinline__ float act(float g, uint32_t kind) { return kind ? 1.0f / (1.0f + expf(-g)) : g; }

// The threads that hold one row: a warp, or the whole CTA.
struct Team {
    uint32_t size, rank;   // threads, this thread
    uint32_t index, count; // this team, teams of the grid
    float* shared;         // 2 x N x 32 floats, CTA teams only
    uint32_t flip;

    // Sums of N values over the team, the same bits in every thread.
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
        if (size == 32u) return;
        float* part = shared + flip * (N * 32);
        flip ^= 1u;  // two sets in turn: one barrier a sum
        if (rank % 32u == 0u)
#pragma unroll
            for (int n = 0; n < N; ++n) part[n * 32 + rank / 32u] = v[n];
        __syncthreads();
        const uint32_t warps = size / 32u;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float s = rank % 32u < warps ? part[n * 32 + rank % 32u] : 0.0f;
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            v[n] = s;
        }
    }
};

__device__ __forceinline__ Team team_of(uint32_t size, float* shared) {
    if (size == 32u) {
        const uint32_t per = blockDim.x / 32u;
        return Team{32u, threadIdx.x % 32u, blockIdx.x * per + threadIdx.x / 32u, gridDim.x * per, shared, 0u};
    }
    return Team{size, threadIdx.x, blockIdx.x, gridDim.x, shared, 0u};
}

template <class T, int V, int NV>
__device__ __forceinline__ void load_row(Raw<T, V> (&r)[NV], const T* p, const Team& t, uint32_t D) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t i = (j * t.size + t.rank) * V;
        if (p && i < D)
            r[j].load(p + i);
        else
            r[j].zero();
    }
}

template <class R, int V, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) forward_kernel(const Forward p, uint32_t team_size) {
    __shared__ float shared[64];
    Team team = team_of(team_size, shared);
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    Raw<uint16_t, V> w_post[NV], w_pre[NV];
    load_row(w_post, p.w_post, team, p.D);
    load_row(w_pre, p.w_pre, team, p.D);
    const float inv_d = 1.0f / (float)p.D;
    for (uint64_t t = team.index; t < p.T; t += team.count) {
        Raw<R, V> resid[NV];
        Raw<uint16_t, V> u[NV], gate[NV];
        load_row(u, p.u ? p.u + t * p.ld_u : nullptr, team, p.D);
        load_row(resid, static_cast<const R*>(p.resid) + t * p.ld_resid, team, p.D);
        load_row(gate, p.gate ? p.gate + (uint32_t)t / p.gate_rows * p.ld_gate : nullptr, team, p.D);
        float k = p.scale;
        if (p.post) {
            float s[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) s[0] = fmaf(u[j].get(i), u[j].get(i), s[0]);
            team.sum(s);
            const float rp = 1.0f / sqrtf(s[0] * inv_d + p.eps);
            if (p.rstd_post && team.rank == 0) p.rstd_post[t] = rp;
            k *= rp;
        }
        float h[NV][V], s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float b = u[j].get(i) * k;
                if (p.w_post) b *= w_post[j].get(i);
                if (p.gate) b *= act(gate[j].get(i), p.gate_act);
                h[j][i] = p.u ? resid[j].get(i) + b : resid[j].get(i);
                s[0] = fmaf(h[j][i], h[j][i], s[0]);
            }
        if (p.h)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const uint32_t i = (j * team.size + team.rank) * V;
                if (i < p.D) put<V>(static_cast<R*>(p.h) + t * p.ld_h + i, h[j]);
            }
        if (!p.y) continue;
        team.sum(s);
        const float r = 1.0f / sqrtf(s[0] * inv_d + p.eps);
        if (p.rstd_pre && team.rank == 0) p.rstd_pre[t] = r;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t i = (j * team.size + team.rank) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[j][e] *= r;
                if (p.w_pre) h[j][e] *= w_pre[j].get(e);
            }
            if (i < p.D) put<V>(p.y + t * p.ld_y + i, h[j]);
        }
    }
}

// Backward.  A team takes a chunk of consecutive tokens and sums dw_pre,
// dw_post and, for a gate row that several tokens share, dgate in its
// registers.  Chunks do not cross the tokens of a gate row unless they hold
// all of them, so a gate row's gradient is either complete in a chunk or a
// run of chunks.  The chunks' sums go to the workspace and sum_chunks adds
// them in order.
struct Chunks {
    uint32_t rows, count;     // tokens of a chunk, chunks
    uint32_t per_gate;        // chunks of a gate row, 0: a chunk holds whole gate rows
    uint32_t gates;           // gate rows
};
Chunks plan_chunks(uint32_t T, uint32_t D, uint32_t gate_rows, uint32_t sms) {
    // Enough teams to fill the GPU, at least 8 tokens each: a chunk writes and
    // reads 3 x 4 bytes a channel beside the 12 and more of each token.
    const uint32_t teams = sms * (D > 256 ? 2 : 16);
    uint32_t rows = (T + teams - 1) / teams;
    rows = rows < 8 ? 8 : rows;
    Chunks c{};
    if (gate_rows > T) gate_rows = T;
    c.gates = gate_rows ? (T + gate_rows - 1) / gate_rows : 0;
    if (gate_rows > rows) {
        c.per_gate = (gate_rows + rows - 1) / rows;
        c.rows = (gate_rows + c.per_gate - 1) / c.per_gate;
        c.per_gate = (gate_rows + c.rows - 1) / c.rows;
        c.count = c.per_gate * c.gates;
    } else {
        c.rows = gate_rows ? rows / gate_rows * gate_rows : rows;
        c.count = (T + c.rows - 1) / c.rows;
    }
    return c;
}

template <class R, int V, int NV>
struct Loaded {
    Raw<R, V> dh[NV], h[NV];
    Raw<uint16_t, V> dy[NV], u[NV], gate[NV];
    float rh, ru;
    __device__ __forceinline__ void load(const Backward& p, const Team& team, uint64_t t) {
        load_row(dy, p.dy ? p.dy + t * p.ld_dy : nullptr, team, p.D);
        load_row(h, p.dy ? static_cast<const R*>(p.h) + t * p.ld_h : nullptr, team, p.D);
        load_row(u, p.u ? p.u + t * p.ld_u : nullptr, team, p.D);
        load_row(dh, p.dh ? static_cast<const R*>(p.dh) + t * p.ld_dh : nullptr, team, p.D);
        load_row(gate, p.gate ? p.gate + (uint32_t)t / p.gate_rows * p.ld_gate : nullptr, team, p.D);
        rh = p.dy ? p.rstd_pre[t] : 0.0f;
        ru = p.post && p.u ? p.rstd_post[t] : 1.0f;
    }
};

template <class R, int V, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS)
backward_kernel(const Backward p, const Chunks c, uint32_t team_size) {
    __shared__ float shared[192];
    Team team = team_of(team_size, shared);
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    if (team.index >= c.count) return;  // whole warps, or nobody
    // Tokens [t0, t1).
    uint64_t t0, t1;
    if (c.per_gate) {
        const uint64_t gate0 = (uint64_t)(team.index / c.per_gate) * p.gate_rows;
        const uint64_t end = min((uint64_t)p.T, gate0 + p.gate_rows);
        t0 = min(end, gate0 + (uint64_t)(team.index % c.per_gate) * c.rows);
        t1 = min(end, t0 + c.rows);
    } else {
        t0 = (uint64_t)team.index * c.rows;
        t1 = min((uint64_t)p.T, t0 + c.rows);
    }
    Raw<uint16_t, V> w_post[NV], w_pre[NV];
    load_row(w_post, p.w_post, team, p.D);
    load_row(w_pre, p.w_pre, team, p.D);
    float dw_post[NV][V] = {}, dw_pre[NV][V] = {}, dgate[NV][V] = {};
    const float inv_d = 1.0f / (float)p.D;
    for (uint64_t t = t0; t < t1; ++t) {
        Loaded<R, V, NV> x;
        x.load(p, team, t);
        // c1 = mean(a hhat) and c2 = mean(dp pv), dp = k (dh + rh (a - hhat c1))
        // with k = scale act: one round of sums, c2 = s[1] - c1 s[2].
        float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hh = x.h[j].get(i) * x.rh;
                const float a = x.dy[j].get(i) * (p.w_pre ? w_pre[j].get(i) : 1.0f);
                s[0] = fmaf(a, hh, s[0]);
                if (p.post) {
                    float k = p.scale * x.u[j].get(i) * x.ru * (p.w_post ? w_post[j].get(i) : 1.0f);
                    if (p.gate) k *= act(x.gate[j].get(i), p.gate_act);
                    s[1] = fmaf(k, fmaf(x.rh, a, x.dh[j].get(i)), s[1]);
                    s[2] = fmaf(k, x.rh * hh, s[2]);
                }
            }
        team.sum(s);
        const float c1 = s[0] * inv_d, c2 = (s[1] - c1 * s[2]) * inv_d;
        const bool last = p.gate_rows && ((uint32_t)(t + 1) % p.gate_rows == 0 || t + 1 == p.T);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float dh[V], du[V], dg[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hh = x.h[j].get(i) * x.rh;
                const float dy = x.dy[j].get(i), a = dy * (p.w_pre ? w_pre[j].get(i) : 1.0f);
                dh[i] = fmaf(x.rh, a - hh * c1, x.dh[j].get(i));
                dw_pre[j][i] = fmaf(dy, hh, dw_pre[j][i]);
                const float uh = x.u[j].get(i) * x.ru, wp = p.w_post ? w_post[j].get(i) : 1.0f;
                const float dz = p.scale * dh[i];
                float dp = dz, der = 1.0f;
                if (p.gate) {
                    const float g = act(x.gate[j].get(i), p.gate_act);
                    dp *= g;
                    if (p.gate_act) der = g * (1.0f - g);
                }
                dw_post[j][i] = fmaf(dp, uh, dw_post[j][i]);
                du[i] = p.post ? x.ru * (dp * wp - uh * c2) : dp;
                dgate[j][i] = fmaf(dz * der, uh * wp, dgate[j][i]);
                dg[i] = dgate[j][i];
            }
            const uint32_t i = (j * team.size + team.rank) * V;
            if (i < p.D) {
                if (p.dresid) put<V>(static_cast<R*>(p.dresid) + t * p.ld_dresid + i, dh);
                if (p.du) put<V>(p.du + t * p.ld_du + i, du);
                if (p.dgate && last && !c.per_gate)
                    put<V>(p.dgate + (uint32_t)t / p.gate_rows * p.ld_dgate + i, dg);
            }
            if (last && !c.per_gate)
#pragma unroll
                for (int e = 0; e < V; ++e) dgate[j][e] = 0.0f;
        }
    }
    const uint64_t plane = (uint64_t)c.count * p.D;
    float* ws = p.ws + (uint64_t)team.index * p.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t i = (j * team.size + team.rank) * V;
        if (i >= p.D) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {  // the workspace's rows are not aligned for vectors
            if (p.dw_pre) ws[i + e] = dw_pre[j][e];
            if (p.dw_post) ws[plane + i + e] = dw_post[j][e];
            if (p.dgate && c.per_gate) ws[2 * plane + i + e] = dgate[j][e];
        }
    }
}

// Adds the chunks' sums: blockIdx.y 0 and 1 dw_pre and dw_post, 2 + g gate row
// g.  32 columns a CTA, 8 warps that take every eighth chunk; the warps' sums
// are added in order.
__global__ void __launch_bounds__(256) sum_chunks(const Backward p, const Chunks c) {
    __shared__ float part[8][32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, i = blockIdx.x * 32u + lane;
    for (uint32_t what = blockIdx.y; what < 2u + c.gates; what += gridDim.y) {
        if ((what == 0 && !p.dw_pre) || (what == 1 && !p.dw_post)) continue;
        const uint32_t first = what < 2u ? 0u : (what - 2u) * c.per_gate, n = what < 2u ? c.count : c.per_gate;
        const float* ws = p.ws + ((uint64_t)min(what, 2u) * c.count + first) * p.D + i;
        float s = 0.0f;
        if (i < p.D)
#pragma unroll 4
            for (uint32_t k = warp; k < n; k += 8) s += ws[(uint64_t)k * p.D];
        __syncthreads();
        part[warp][lane] = s;
        __syncthreads();
        if (warp != 0 || i >= p.D) continue;
        for (int k = 1; k < 8; ++k) s += part[k][lane];
        if (what == 0)
            p.dw_pre[i] = s;
        else if (what == 1)
            p.dw_post[i] = s;
        else
            p.dgate[(uint64_t)(what - 2u) * p.ld_dgate + i] = (uint16_t)(cvt_bf16x2(s, 0.0f) & 0xffffu);
    }
}

// Widest vector (8, 2 or 1 channels) that every tensor in use allows.
struct Width {
    int v = 8;
    void use(const void* p, uint64_t ld, uint64_t elem) {
        if (!p) return;
        while (v > 1 && ((uintptr_t)p % (v * elem < 16 ? v * elem : 16) || ld % v)) v = v == 8 ? 2 : 1;
    }
    explicit Width(uint32_t D) {
        // Few channels: narrower vectors keep a warp's lanes busy.
        while (v > 1 && (D % v || D < 32u * v)) v = v == 8 ? 2 : 1;
    }
};

template <class K, class... Args>
cudaError_t launch(K kernel, dim3 grid, uint32_t threads, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid, cfg.blockDim = dim3(threads, 1, 1), cfg.stream = s;
    cudaLaunchAttribute la[1];
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = la, cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) foil_count_launch();
    return e;
}

// Threads of a row's team for E channels each, and CTAs' threads: warps that
// are teams of their own share a CTA of 4.
uint32_t team_threads(uint32_t D, uint32_t E) { return (D + 32 * E - 1) / (32 * E) * 32; }

template <class R, int V>
cudaError_t forward_typed(const Forward& p, cudaStream_t s) {
    const uint32_t sms = (uint32_t)foil_sm_count();
    const bool wide = p.D > 2048;  // 16 channels a thread
    const uint32_t team = team_threads(p.D, wide ? 16 : 8), threads = team == 32 ? 128 : team;
    const uint64_t ctas = team == 32 ? (p.T + 3) / 4 : p.T, most = (uint64_t)sms * (2048 / threads);
    const dim3 grid((unsigned)(ctas < most ? ctas : most));
    if (!wide) return launch(forward_kernel<R, V, 8 / V, 256>, grid, threads, s, p, team);
    return threads <= 512 ? launch(forward_kernel<R, V, 16 / V, 512>, grid, threads, s, p, team)
                          : launch(forward_kernel<R, V, 16 / V, 1024>, grid, threads, s, p, team);
}

template <class R, int V>
cudaError_t backward_typed(const Backward& p, const Chunks& c, cudaStream_t s) {
    const bool wide = p.D > 4096;
    const uint32_t team = team_threads(p.D, wide ? 16 : 8), threads = team == 32 ? 128 : team;
    const dim3 grid(team == 32 ? (c.count + 3) / 4 : c.count);
    if (!wide) return launch(backward_kernel<R, V, 8 / V, 512>, grid, threads, s, p, c, team);
    return threads <= 512 ? launch(backward_kernel<R, V, 16 / V, 512>, grid, threads, s, p, c, team)
                          : launch(backward_kernel<R, V, 16 / V, 1024>, grid, threads, s, p, c, team);
}

}  // namespace

uint64_t backward_ws_bytes(uint32_t T, uint32_t D, uint32_t gate_rows) {
    if (T == 0 || D == 0) return 0;
    const Chunks c = plan_chunks(T, D, gate_rows, (uint32_t)foil_sm_count());
    return (uint64_t)c.count * D * 4 * (c.per_gate ? 3 : 2);
}

cudaError_t forward(const Forward& p, bool fp32, cudaStream_t s) {
    Width w(p.D);
    w.use(p.resid, p.ld_resid, fp32 ? 4 : 2), w.use(p.h, p.ld_h, fp32 ? 4 : 2);
    w.use(p.u, p.ld_u, 2), w.use(p.gate, p.ld_gate, 2), w.use(p.y, p.ld_y, 2);
    w.use(p.w_post, 0, 2), w.use(p.w_pre, 0, 2);
    if (fp32)
        return w.v == 8 ? forward_typed<float, 8>(p, s)
                        : w.v == 2 ? forward_typed<float, 2>(p, s) : forward_typed<float, 1>(p, s);
    return w.v == 8 ? forward_typed<uint16_t, 8>(p, s)
                    : w.v == 2 ? forward_typed<uint16_t, 2>(p, s) : forward_typed<uint16_t, 1>(p, s);
}

cudaError_t backward(const Backward& p, bool fp32, cudaStream_t s) {
    if (p.T == 0) {
        for (float* d : {p.dw_pre, p.dw_post})
            if (d) {
                const cudaError_t e = cudaMemsetAsync(d, 0, 4ull * p.D, s);
                if (e != cudaSuccess) return e;
            }
        return cudaSuccess;
    }
    const Chunks c = plan_chunks(p.T, p.D, p.gate_rows, (uint32_t)foil_sm_count());
    Width w(p.D);
    w.use(p.dh, p.ld_dh, fp32 ? 4 : 2), w.use(p.h, p.ld_h, fp32 ? 4 : 2), w.use(p.dresid, p.ld_dresid, fp32 ? 4 : 2);
    w.use(p.dy, p.ld_dy, 2), w.use(p.u, p.ld_u, 2), w.use(p.gate, p.ld_gate, 2), w.use(p.du, p.ld_du, 2);
    w.use(p.dgate, p.ld_dgate, 2), w.use(p.w_post, 0, 2), w.use(p.w_pre, 0, 2);
    cudaError_t e;
    if (fp32)
        e = w.v == 8 ? backward_typed<float, 8>(p, c, s)
                     : w.v == 2 ? backward_typed<float, 2>(p, c, s) : backward_typed<float, 1>(p, c, s);
    else
        e = w.v == 8 ? backward_typed<uint16_t, 8>(p, c, s)
                     : w.v == 2 ? backward_typed<uint16_t, 2>(p, c, s) : backward_typed<uint16_t, 1>(p, c, s);
    const bool shared_gate = p.dgate && c.per_gate;
    if (e != cudaSuccess || !(p.dw_pre || p.dw_post || shared_gate)) return e;
    Chunks sums = c;
    if (!shared_gate) sums.gates = 0;
    const uint32_t rows = 2 + sums.gates;
    return launch(sum_chunks, dim3((p.D + 31) / 32, rows < 32768 ? rows : 32768), 256, s, p, sums);
}

}  // namespace norm
}  // namespace foil
