// The norms after a residual block and before the next one, fused with the
// block's gate, its scale and the residual addition; and their gradients.
// The formulas stand at foil_block_norm_dev in include/foil_c.h.
//
// Bound by HBM, closely followed by instruction issue: every tensor is read
// and written once, with 10 (forward) to 30 instructions a channel.  A row lives
// in the registers of one warp, one CTA or a cluster of CTAs (its team), 8 or 16
// channels a thread; a team goes over many rows, the next ones on their way to L2
// or to registers while the present one is worked on.  (A ring of three rows in
// shared memory, tried: 10 to 50 % slower, for the instructions it takes.)
// Channels are moved in vectors of 16 bytes where D, the strides and
// the pointers allow, else of 4 bytes (even D), else one by one.
#include "block_norm.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "gemm_ptx.cuh"

namespace foil {
namespace norm {
namespace {

using gemm::cluster_sync;
using gemm::map_to_rank;

// V values of type T (uint16_t: bf16 bits) as loaded.
template <class T, int V>
struct Raw {
    static constexpr int kWords = (sizeof(T) * V + 3) / 4;
    uint32_t w[kWords];
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

__device__ __forceinline__ float sum2(float2 v) { return v.x + v.y; }

// Channels 2 i and 2 i + 1 of a thread's.
template <class T, int V, int NV>
__device__ __forceinline__ float2 get2(const Raw<T, V> (&r)[NV], int i) {
    if constexpr (V == 1) return make_float2(r[2 * i].get(0), r[2 * i + 1].get(0));
    const Raw<T, V>& v = r[2 * i / V];
    return make_float2(v.get(2 * i % V), v.get(2 * i % V + 1));
}

// Channels of vector j, from pairs.
template <int V>
__device__ __forceinline__ void put(uint16_t* p, const float2* v, int j) {
    if constexpr (V == 8) {
        v += 4 * j;
        *reinterpret_cast<uint4*>(p) = make_uint4(cvt_bf16x2(v[0].x, v[0].y), cvt_bf16x2(v[1].x, v[1].y),
                                                  cvt_bf16x2(v[2].x, v[2].y), cvt_bf16x2(v[3].x, v[3].y));
    } else if constexpr (V == 2) {
        *reinterpret_cast<uint32_t*>(p) = cvt_bf16x2(v[j].x, v[j].y);
    } else {
        *p = (uint16_t)(cvt_bf16x2(j % 2 ? v[j / 2].y : v[j / 2].x, 0.0f) & 0xffffu);
    }
}
template <int V>
__device__ __forceinline__ void put(float* p, const float2* v, int j) {
    if constexpr (V == 8) {
        v += 4 * j;
        if (((uintptr_t)p & 31u) == 0) {  // one store of whole sectors
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(i % 2 ? v[i / 2].y : v[i / 2].x);
            gemm::st_global_v8(p, w);
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
        }
    } else if constexpr (V == 2) {
        *reinterpret_cast<float2*>(p) = v[j];
    } else {
        *p = j % 2 ? v[j / 2].y : v[j / 2].x;
    }
}
// A row's share of this thread to memory (nowhere if p is null).
template <int V, int NV, class T, class Team>
__device__ __forceinline__ void store_row(T* p, const float2 (&v)[V * NV / 2], const Team& t, uint32_t D) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t i = (j * t.size + t.rank) * V;
        if (p && i < D) put<V>(p + i, v, j);
    }
}

// The same without vectors: the workspace's rows are not aligned for them.
template <int V, int NV, class Team>
__device__ __forceinline__ void store_plain(float* p, const float2 (&v)[V * NV / 2], const Team& t, uint32_t D) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t i = (j * t.size + t.rank) * V;
        if (i >= D) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) p[i + e] = (j * V + e) % 2 ? v[(j * V + e) / 2].y : v[(j * V + e) / 2].x;
    }
}

// The logistic function of gates: act(g) = 1 / (1 + e) with e = exp(-g), and for its
// derivative act(g) act(-g) the other factor is e act(g), without the cancellation
// of 1 - act(g).  Gates are bf16, so e = 2^t (1 + c) with t = -g H exact (8 bits
// times the 16 upper bits H of log2 e) and c = -g ln 2 (log2 e - H), below 2^-11, so
// that what follows c does not count.  ex2.approx is within 2^-22, rcp.approx within
// 2^-23; with the operations' roundings act and the derivative are within 2^-20
// relative, to 0 below 2^-126.  (By expf and a division: 8192 x 5120 118 us, with
// this 104.)
constexpr float kLog2e = 47274.0f / 32768.0f;
constexpr float kRest = (float)((1.4426950408889634 - 47274.0 / 32768.0) * 0.6931471805599453);
__device__ __forceinline__ float2 exp2(float2 x) {
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x.y));
    return x;
}
__device__ __forceinline__ float2 reciprocal2(float2 x) {
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x.y));
    return x;
}
// g, at least -88 and at most 128; NaN stays.
__device__ __forceinline__ float between(float g) {
    asm("min.NaN.f32 %0, %0, 0f43000000;\n\tmax.NaN.f32 %0, %0, 0fc2b00000;" : "+f"(g));
    return g;
}
// exp(-g) of gates 2 i and 2 i + 1, between exp(-128) = 0 and exp(88), a number
// whose reciprocal is 0; NaN stays.
template <int V, int NV>
__device__ __forceinline__ float2 exp_minus2(const Raw<uint16_t, V> (&r)[NV], int i) {
    float2 g = get2(r, i);
    if constexpr (V == 1) {
        g = make_float2(between(g.x), between(g.y));
    } else {
        uint32_t w = r[2 * i / V].w[i % (V / 2)];
        asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0x43004300u));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0xc2b0c2b0u));
        g = make_float2(bf16_bits_to_f32(w & 0xffffu), __uint_as_float(w & 0xffff0000u));
    }
    return mul2(exp2(mul2(g, both(-kLog2e))), fma2(g, both(-kRest), both(1.0f)));
}
__device__ __forceinline__ float2 act2(float2 e) { return reciprocal2(add2(e, both(1.0f))); }
template <int V, int NV>
__device__ __forceinline__ float2 sigmoid2(const Raw<uint16_t, V> (&r)[NV], int i) {
    return act2(exp_minus2(r, i));
}

// The threads that hold one row: 4 to 32 lanes of a warp, a CTA, or the CTAs of
// a cluster.
struct Team {
    uint32_t size, rank;    // threads, this thread
    uint32_t lane;
    uint32_t ctas;          // CTAs of a team (0: the team is in a warp)
    uint32_t index, count;  // this team, teams of the grid
    float* shared;          // two sets of kSumFloats floats
    uint32_t flip;

    // Sums of N (1 to 4) values over the team, the same bits in every thread.
    // A warp's lanes first halve the values they hold (lanes with bit 16 clear
    // go on with values 0 and 1, and so on), so four sums take 6 shuffles
    // instead of 20; then 8 lanes add the warps' sums of one value.
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N]) {
        constexpr uint32_t kAll = 0xffffffffu;
        float s;
        if (size < 32u) {  // the warp's other teams may be elsewhere
            const uint32_t mask = ((1u << size) - 1u) << (lane & ~(size - 1u));
            for (uint32_t o = size / 2u; o; o >>= 1)
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(mask, v[n], o);
            return;
        }
        if constexpr (N == 1) {
            s = v[0];
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
            if (ctas == 0) {
                v[0] = s;
                return;
            }
        } else {
            const float v3 = N > 3 ? v[N - 1] : 0.0f, v2 = N > 2 ? v[2] : 0.0f;
            const bool up = lane & 16u, odd = lane & 8u;
            const float a = (up ? v2 : v[0]) + __shfl_xor_sync(kAll, up ? v[0] : v2, 16);
            const float b = (up ? v3 : v[1]) + __shfl_xor_sync(kAll, up ? v[1] : v3, 16);
            s = (odd ? b : a) + __shfl_xor_sync(kAll, odd ? a : b, 8);
#pragma unroll
            for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        }
        // s: the warp's sum of value lane / 8 (N > 1).
        if (ctas) {
            const uint32_t warps = blockDim.x / 32u, all = warps * ctas;
            float* part = shared + flip * kSumFloats;  // [value][warp], two sets in turn: one barrier a sum
            flip ^= 1u;
            const uint32_t value = N == 1 ? 0u : lane / 8u;
            if (N == 1 ? lane == 0 : lane % 8u == 0 && value < (uint32_t)N) {
                float* at = part + value * kMaxTeamWarps + rank / 32u;
                if (ctas == 1u)
                    *at = s;
                else
                    for (uint32_t c = 0; c < ctas; ++c)
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_rank(at, c)), "f"(s) : "memory");
            }
            if (ctas == 1u)
                __syncthreads();
            else
                cluster_sync();
            s = 0.0f;
            if (value < (uint32_t)N)
                for (uint32_t w = lane % 8u; w < all; w += 8u) s += part[value * kMaxTeamWarps + w];
#pragma unroll
            for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = __shfl_sync(kAll, s, 8 * n);
    }
    static constexpr uint32_t kMaxTeamWarps = 64, kSumFloats = 4 * kMaxTeamWarps;
};

// A team as the host planned it: `ctas` CTAs, or (0) `lanes` lanes of a warp.
struct TeamPlan {
    uint32_t ctas, lanes;
};
__device__ __forceinline__ Team team_of(const TeamPlan& t, float* shared) {
    const uint32_t lane = threadIdx.x % 32u;
    if (t.ctas == 0) {
        const uint32_t per = blockDim.x / t.lanes;
        return Team{t.lanes, lane & (t.lanes - 1u), lane, 0u, blockIdx.x * per + threadIdx.x / t.lanes,
                    gridDim.x * per, shared, 0u};
    }
    return Team{t.ctas * blockDim.x, blockIdx.x % t.ctas * blockDim.x + threadIdx.x, lane, t.ctas,
                blockIdx.x / t.ctas, gridDim.x / t.ctas, shared, 0u};
}

// Element of vector j of this thread.  Threads past D read the last vector
// again, so that loads need no branch; what they hold must not enter a sum.
template <int V>
__device__ __forceinline__ uint32_t column(int j, const Team& t, uint32_t D) {
    return min((j * t.size + t.rank) * V, D - V);
}
template <int V>
__device__ __forceinline__ bool inside(int j, const Team& t, uint32_t D) {
    return (j * t.size + t.rank) * V < D;
}

template <class T, int V>
__device__ __forceinline__ void clear(Raw<T, V>& r) {
#pragma unroll
    for (int k = 0; k < Raw<T, V>::kWords; ++k) r.w[k] = 0u;
}

// bf16 weights of the thread's channels: ones where there are none, zeros past D.
template <int V, int NV>
__device__ __forceinline__ void load_weights(Raw<uint16_t, V> (&r)[NV], const uint16_t* p, const Team& t, uint32_t D) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t none = inside<V>(j, t, D) ? 0x3f803f80u : 0u;
        if (p && none)
            r[j].load(p + column<V>(j, t, D));
        else
#pragma unroll
            for (int k = 0; k < Raw<uint16_t, V>::kWords; ++k) r[j].w[k] = none;
    }
}

// A row of zeros, read where a tensor is not given; a factor of one.
__device__ uint4 g_zeros[kMaxD * 4 / 16];
__device__ float g_one = 1.0f;

// A tensor as a team reads it.  Row strides are below 2^32, so a row's offset
// is one multiplication.
template <class T, int V, int NV>
struct Input {
    const T* p;
    uint32_t ld;
    __device__ __forceinline__ Input(const void* base, uint64_t stride)
        : p(static_cast<const T*>(base ? base : g_zeros)), ld(base ? (uint32_t)stride : 0u) {}
    __device__ __forceinline__ void load(Raw<T, V> (&r)[NV], uint32_t row, const Team& team, uint32_t D) const {
        const T* q = p + (uint64_t)row * ld;
#pragma unroll
        for (int j = 0; j < NV; ++j) r[j].load(q + column<V>(j, team, D));
    }
};

// A row of a tensor towards L2: each of a team's first threads asks for one
// tensor's, the whole 16-byte pieces of it.  Forward, 8192 x 5120: 121 us
// without, 104 with.
struct Ahead {
    uint64_t at;            // row 0
    uint32_t pitch, bytes;  // bytes 0: nothing to ask for
    template <class T, int V, int NV>
    __device__ __forceinline__ void use(const Input<T, V, NV>& in, uint32_t D) {
        if (in.ld >= 1u << 30) return;
        at = reinterpret_cast<uint64_t>(in.p), pitch = in.ld * (uint32_t)sizeof(T);
        bytes = D * (uint32_t)sizeof(T) - (V == 8 ? 0u : 16u) & ~15u;
    }
    __device__ __forceinline__ void operator()(uint32_t row) const {
        const uint64_t from = at + (uint64_t)row * pitch + 15u & ~15ull;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(bytes) : "memory");
    }
};
// This thread's part of a row's sum of squares.
template <int V, int NV>
__device__ __forceinline__ float sum_squares(const float2 (&v)[V * NV / 2], const Team& t, uint32_t D) {
    float s = 0.0f;
    if constexpr (V == 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const float x = j % 2 ? v[j / 2].y : v[j / 2].x;
            s += inside<V>(j, t, D) ? x * x : 0.0f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float2 q = mul2(v[j * (V / 2)], v[j * (V / 2)]);
#pragma unroll
            for (int i = 1; i < V / 2; ++i) q = fma2(v[j * (V / 2) + i], v[j * (V / 2) + i], q);
            s += inside<V>(j, t, D) ? sum2(q) : 0.0f;
        }
    }
    return s;
}

// Gates: none, as they are, through the logistic function.
enum { kNoGate = 0, kPlainGate = 1, kSigmoidGate = 2 };
template <int GATE, int V, int NV>
__device__ __forceinline__ float2 gate2(const Raw<uint16_t, V> (&r)[NV], int i) {
    return GATE == kSigmoidGate ? sigmoid2(r, i) : get2(r, i);
}

template <class R, int V, int NV, int THREADS, int CTAS, int GATE>
__global__ void __launch_bounds__(THREADS, CTAS) forward_kernel(const Forward p, const TeamPlan plan) {
    __shared__ float shared[2 * Team::kSumFloats];
    Team team = team_of(plan, shared);
    if (plan.ctas > 1) cluster_sync();  // every CTA of the team runs before its memory is written
    griddep_wait();                     // launched with programmatic stream serialization
    griddep_launch_dependents();
    const float inv_d = 1.0f / (float)p.D;
    const Input<R, V, NV> resid_in(p.resid, p.ld_resid);
    const Input<uint16_t, V, NV> u_in(p.u, p.ld_u), gate_in(p.gate, p.ld_gate);
    Ahead ahead{};
    if (p.D >= 2048u) {
        if (team.rank == 0 && p.resid) ahead.use(resid_in, p.D);
        if (team.rank == 1 && p.u) ahead.use(u_in, p.D);
        if (GATE && team.rank == 2 && p.gate_rows == 1) ahead.use(gate_in, p.D);
    }
    for (uint64_t row = team.index; row < p.T; row += team.count) {
        const uint32_t t = (uint32_t)row;
        Raw<R, V> resid[NV];
        Raw<uint16_t, V> u[NV], gate[NV];
        u_in.load(u, t, team, p.D);
        resid_in.load(resid, t, team, p.D);
        if constexpr (GATE) gate_in.load(gate, p.gate_rows == 1 ? t : t / p.gate_rows, team, p.D);
        if (ahead.bytes && row + team.count < p.T) ahead((uint32_t)(row + team.count));
        constexpr int kPairs = V * NV / 2;
        float k = p.scale;
        if (p.post) {
            float2 v[kPairs];
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = get2(u, i);
            float s[1] = {sum_squares<V, NV>(v, team, p.D)};
            team.sum(s);
            const float rp = 1.0f / sqrtf(s[0] * inv_d + p.eps);
            if (p.rstd_post && team.rank == 0) p.rstd_post[t] = rp;
            k *= rp;
        }
        // The weights come from the first-level cache for every row: registers
        // for them would cost a resident CTA.
        Raw<uint16_t, V> w[NV];
        load_weights(w, p.w_post, team, p.D);
        float2 h[kPairs];
        // Without a branch u is zeros (and k a number), so h = resid.
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            float2 b = mul2(get2(u, i), get2(w, i));
            if constexpr (GATE) b = mul2(b, gate2<GATE>(gate, i));
            h[i] = fma2(b, both(k), get2(resid, i));
        }
        if (p.h) store_row<V, NV>(static_cast<R*>(p.h) + (uint64_t)t * (uint32_t)p.ld_h, h, team, p.D);
        if (!p.y) continue;
        load_weights(w, p.w_pre, team, p.D);
        float s[1] = {sum_squares<V, NV>(h, team, p.D)};
        team.sum(s);
        const float r = 1.0f / sqrtf(s[0] * inv_d + p.eps);
        if (p.rstd_pre && team.rank == 0) p.rstd_pre[t] = r;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) h[i] = mul2(mul2(h[i], both(r)), get2(w, i));
        store_row<V, NV>(p.y + (uint64_t)t * (uint32_t)p.ld_y, h, team, p.D);
    }
}

// A row's team of E channels a thread in CTAs of at most `most` threads: lanes
// of a warp (a CTA has 128), a CTA, or a cluster of CTAs.
constexpr uint32_t kBackwardThreads = 512;  // of an SM, by registers
struct Shape {
    uint32_t threads, teams;  // threads and teams of a CTA
    TeamPlan plan;
    Shape(uint32_t D, uint32_t E, uint32_t most) {
        const uint32_t team = (D + 32 * E - 1) / (32 * E) * 32;
        plan.ctas = team == 32 ? 0 : (team + most - 1) / most;
        plan.lanes = 32;
        while (team == 32 && plan.lanes > 4 && plan.lanes / 2 * E >= D) plan.lanes /= 2;
        threads = plan.ctas ? ((team + plan.ctas - 1) / plan.ctas + 31) / 32 * 32 : 128;
        teams = plan.ctas ? 1 : 128 / plan.lanes;
    }
    // CTAs (or clusters) that run at once with `per_sm` threads on an SM.
    uint32_t resident(uint32_t per_sm) const {
        const uint32_t sms = (uint32_t)foil_sm_count(), n = per_sm / threads ? per_sm / threads : 1;
        return plan.ctas > 1 ? foil_resident_clusters(plan.ctas) * n : sms * n;
    }
};

// Backward.  A team takes a chunk of consecutive tokens and sums dw_pre,
// dw_post and, for a gate row that several tokens share, dgate in its
// registers.  Chunks do not cross the tokens of a gate row unless they hold
// all of them, so a gate row's gradient is either complete in a chunk or a
// run of chunks.  The chunks' sums go to the workspace and sum_chunks adds
// them in order.
struct Chunks {
    uint32_t rows, count;     // tokens of a chunk, chunks
    uint32_t parts;           // sums of dw_pre and dw_post: of a chunk, or of a CTA of several
    uint32_t per_gate;        // chunks of a gate row, 0: a chunk holds whole gate rows
    uint32_t gates;           // gate rows
};
Chunks plan_chunks(uint32_t T, uint32_t D, uint32_t gate_rows) {
    // As many teams as run at once: a chunk writes and reads 3 x 4 bytes a
    // channel beside the 12 and more of each token.
    const Shape sh(D, 8, 512);
    const uint32_t teams = sh.resident(kBackwardThreads) * sh.teams;
    uint32_t rows = (T + teams - 1) / teams;
    Chunks c{};
    if (gate_rows > T) gate_rows = T;
    c.gates = gate_rows ? (T + gate_rows - 1) / gate_rows : 0;
    if (gate_rows > rows) {
        // Not more chunks than teams, if there are fewer gate rows.
        c.per_gate = c.gates < teams ? teams / c.gates : 1;
        c.rows = (gate_rows + c.per_gate - 1) / c.per_gate;
        c.per_gate = (gate_rows + c.rows - 1) / c.rows;
        c.count = c.per_gate * c.gates;
    } else {
        c.rows = gate_rows ? rows / gate_rows * gate_rows : rows;
        c.count = (T + c.rows - 1) / c.rows;
    }
    c.parts = sh.plan.ctas ? c.count : (c.count + sh.teams - 1) / sh.teams;
    return c;
}

// GATE: kNoGate where a gate row serves several tokens or there is none (then
// the gate's part is taken out of the sums over its tokens: with A = sum dz
// uhat, dw_post gains act A and dgate is act' w_post A), else a gate row for
// each token.
// AHEAD: the next row arrives in registers while the present one is worked on.
template <class R, int V, int NV, int THREADS, int GATE, bool AHEAD>
__global__ void __launch_bounds__(THREADS) backward_kernel(const Backward p, const Chunks c, const TeamPlan plan) {
    constexpr int kPairs = V * NV / 2;
    // Rows asked for from L2.  Beside the row in registers it pays where a row
    // takes a cluster (2000 x 8192: 78 us, 85 without), elsewhere it costs registers
    // (16384 x 4096 without gates: 182 us, 167 without).
    constexpr bool kAhead = !AHEAD || GATE;
    constexpr uint32_t kAheadBy = AHEAD ? 3u : 2u, kAheadMin = AHEAD ? 4097u : 256u;
    __shared__ float shared[2 * Team::kSumFloats];
    __shared__ float2 post_sum[GATE ? 1 : kPairs * THREADS];  // dw_post of the gate rows done, a slot for each thread
    Team team = team_of(plan, shared);
    if (plan.ctas > 1) cluster_sync();  // every CTA of the team runs before its memory is written
    griddep_wait();                     // launched with programmatic stream serialization
    griddep_launch_dependents();
    // Tokens [t0, t1); none past the last chunk.
    uint32_t t0, t1;
    if (team.index >= c.count) {
        t0 = t1 = 0;
    } else if (c.per_gate) {
        const uint64_t gate0 = (uint64_t)(team.index / c.per_gate) * p.gate_rows;
        const uint64_t end = min((uint64_t)p.T, gate0 + p.gate_rows);
        const uint64_t first = min(end, gate0 + (uint64_t)(team.index % c.per_gate) * c.rows);
        t0 = (uint32_t)first, t1 = (uint32_t)min(end, first + c.rows);
    } else {
        const uint64_t first = (uint64_t)team.index * c.rows;
        t0 = (uint32_t)first, t1 = (uint32_t)min((uint64_t)p.T, first + c.rows);
    }
    Raw<uint16_t, V> w_pre[NV], w_post[GATE ? NV : 1];
    load_weights(w_pre, p.w_pre, team, p.D);
    if constexpr (GATE) load_weights(w_post, p.w_post, team, p.D);
    float2 dw_pre[kPairs], dw_post[kPairs], gw[GATE ? 1 : kPairs];  // dw_post: A; gw: act(gate) w_post
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        dw_post[i] = dw_pre[i] = both(0.0f);
        if constexpr (!GATE) post_sum[i * blockDim.x + threadIdx.x] = both(0.0f);
    }
    const float inv_d = 1.0f / (float)p.D;
    struct Row {
        Raw<R, V> dh[NV], h[NV];
        Raw<uint16_t, V> dy[NV], u[NV], gate[GATE ? NV : 1];
        float rh, ru;
    };
    const Input<R, V, NV> dh_in(p.dh, p.ld_dh), h_in(p.dy ? p.h : nullptr, p.ld_h);
    const Input<uint16_t, V, NV> dy_in(p.dy, p.ld_dy), u_in(p.u, p.ld_u), gate_in(p.gate, p.ld_gate);
    const bool post = p.post && p.u;
    const float* const rstd_pre = p.dy ? p.rstd_pre : reinterpret_cast<const float*>(g_zeros);
    const float* const rstd_post = post ? p.rstd_post : &g_one;
    const uint32_t pre_step = p.dy ? 1u : 0u, post_step = post ? 1u : 0u;
    // In shared memory: registers for it would spill others.
    __shared__ Ahead ahead[5];
    if (kAhead && threadIdx.x < 5u) {
        Ahead a{};
        if (p.D >= kAheadMin && team.rank < 5u) {
            if (threadIdx.x == 0 && p.dy) a.use(dy_in, p.D);
            if (threadIdx.x == 1 && p.dy) a.use(h_in, p.D);
            if (threadIdx.x == 2 && p.u) a.use(u_in, p.D);
            if (threadIdx.x == 3 && p.dh) a.use(dh_in, p.D);
            if (GATE && threadIdx.x == 4) a.use(gate_in, p.D);
        }
        ahead[threadIdx.x] = a;
    }
    auto fetch = [&](Row& x, uint32_t t) {
        dy_in.load(x.dy, t, team, p.D);
        h_in.load(x.h, t, team, p.D);
        u_in.load(x.u, t, team, p.D);
        dh_in.load(x.dh, t, team, p.D);
        if constexpr (GATE) gate_in.load(x.gate, t, team, p.D);
        x.rh = rstd_pre[(uint64_t)t * pre_step];
        x.ru = rstd_post[(uint64_t)t * post_step];
    };
    // A gate row that several tokens share: before and after its tokens here.
    uint32_t gate_row = 0, gate_left = 0xffffffffu;  // of token t, and its tokens from t on
    auto start_gate = [&] {
        Raw<uint16_t, V> g[NV], wp[NV];
        load_weights(wp, p.w_post, team, p.D);
        if (p.gate) gate_in.load(g, gate_row, team, p.D);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            gw[i] = get2(wp, i);
            if (p.gate) gw[i] = mul2(gw[i], p.gate_act ? sigmoid2(g, i) : get2(g, i));
        }
    };
    auto end_gate = [&] {
        Raw<uint16_t, V> g[NV], wp[NV];
        load_weights(wp, p.w_post, team, p.D);
        if (p.gate) gate_in.load(g, gate_row, team, p.D);
        float2 dgate[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            float2 a = dw_post[i];
            dgate[i] = mul2(get2(wp, i), a);
            if (p.gate) {
                float2 ga = get2(g, i);
                if (p.gate_act) {
                    const float2 e = exp_minus2(g, i);
                    ga = act2(e);
                    dgate[i] = mul2(dgate[i], mul2(ga, mul2(ga, e)));
                }
                a = mul2(a, ga);
            }
            float2& sum = post_sum[i * blockDim.x + threadIdx.x];
            sum = fma2(a, both(1.0f), sum);
            dw_post[i] = both(0.0f);
        }
        if (!p.gate || !p.dgate) return;
        if (c.per_gate)
            store_plain<V, NV>(p.ws + (2ull * c.parts + team.index) * p.D, dgate, team, p.D);
        else
            store_row<V, NV>(p.dgate + (uint64_t)gate_row * (uint32_t)p.ld_dgate, dgate, team, p.D);
    };
    // Threads past D read the last vector again, and if it is infinite or NaN no
    // weight of zero keeps it out of the sums.  Cleared before it is used where the row
    // has just been asked for; with the next row on its way that would wait for both
    // (16384 x 4096: 214 us, this 171), so the sums go on without the last vector,
    // the only one that can be outside there (see backward_launch).
    const bool edge = !inside<V>(NV - 1, team, p.D);
    // One token: x is its row, which arrived while the one before was worked
    // on; the one after it goes to `next`.
    auto step = [&](Row& x, Row& next, uint32_t t) {
        if (AHEAD && t + 1u < t1) fetch(next, t + 1u);
        if (!AHEAD && edge)
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (!inside<V>(j, team, p.D)) clear(x.dy[j]), clear(x.h[j]), clear(x.u[j]), clear(x.dh[j]);
        // c1 = mean(a hhat) and c2 = mean(dp pv), dp = k (dh + rh (a - hhat c1))
        // with k = scale act: one round of sums, c2 = ru (S1 - c1 rh S2).
        const float ks = p.scale * x.ru;
        const float2 rh = both(x.rh);
        float2 e[kPairs], hh[kPairs], ga[GATE ? kPairs : 1];  // ga: the gate, or exp(-gate)
        float2 s0 = both(0.0f), s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            hh[i] = mul2(get2(x.h, i), rh);
            const float2 dy = get2(x.dy, i), a = mul2(dy, get2(w_pre, i));
            dw_pre[i] = fma2(dy, hh[i], dw_pre[i]);
            const float2 s0_before = s0, s1_before = s1, s2_before = s2;
            s0 = fma2(a, hh[i], s0);
            e[i] = fma2(rh, a, get2(x.dh, i));
            float2 k;
            if constexpr (GATE) {
                ga[i] = GATE == kSigmoidGate ? exp_minus2(x.gate, i) : get2(x.gate, i);
                k = mul2(mul2(get2(x.u, i), get2(w_post, i)), GATE == kSigmoidGate ? act2(ga[i]) : ga[i]);
            } else {
                k = mul2(get2(x.u, i), gw[i]);
            }
            s1 = fma2(k, e[i], s1);
            s2 = fma2(k, hh[i], s2);
            if (AHEAD && V == 2 && i == kPairs - 1 && edge) s0 = s0_before, s1 = s1_before, s2 = s2_before;
        }
        float s[3] = {sum2(s0), sum2(s1), sum2(s2)};
        if (AHEAD && NV == 1 && edge) s[0] = s[1] = s[2] = 0.0f;
        team.sum(s);
        const float c1 = x.rh * s[0] * inv_d;
        const float c2 = post ? x.ru * x.ru * ks * (s[1] - c1 * s[2]) * inv_d : 0.0f;
        const float2 m1 = both(-c1), m2 = both(-c2), k2 = both(ks);
        // e becomes dh, hh becomes du.
        float2 dgate[GATE ? kPairs : 1];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            e[i] = fma2(m1, hh[i], e[i]);
            const float2 u = get2(x.u, i), dz = mul2(e[i], k2);
            if constexpr (GATE) {
                const float2 act = GATE == kSigmoidGate ? act2(ga[i]) : ga[i];
                const float2 wp = get2(w_post, i), dp = mul2(dz, act);
                dgate[i] = mul2(GATE == kSigmoidGate ? mul2(dp, mul2(ga[i], act)) : dz, mul2(u, wp));
                dw_post[i] = fma2(dp, u, dw_post[i]);
                hh[i] = fma2(m2, u, mul2(dp, wp));
            } else {
                dw_post[i] = fma2(dz, u, dw_post[i]);
                hh[i] = fma2(m2, u, mul2(dz, gw[i]));
            }
        }
        // Without the post norm u has no part in du, but 0 times an infinity has: made
        // anew in a row whose u is not finite (its sums are not, either).
        if (!post && !(fabsf(s[1]) + fabsf(s[2]) < INFINITY))
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                const float2 dz = mul2(e[i], k2);
                if constexpr (GATE)
                    hh[i] = mul2(mul2(dz, GATE == kSigmoidGate ? act2(ga[i]) : ga[i]), get2(w_post, i));
                else
                    hh[i] = mul2(dz, gw[i]);
            }
        store_row<V, NV>(p.dresid ? static_cast<R*>(p.dresid) + (uint64_t)t * (uint32_t)p.ld_dresid : nullptr, e, team,
                         p.D);
        store_row<V, NV>(p.du ? p.du + (uint64_t)t * (uint32_t)p.ld_du : nullptr, hh, team, p.D);
        if (kAhead && threadIdx.x < 5u && t + kAheadBy < t1) {
            const Ahead a = ahead[threadIdx.x];
            if (a.bytes) a(t + kAheadBy);
        }
        if constexpr (GATE) {
            if (p.dgate) store_row<V, NV>(p.dgate + (uint64_t)t * (uint32_t)p.ld_dgate, dgate, team, p.D);
        } else if (--gate_left == 0u) {
            end_gate();
            ++gate_row;
            gate_left = p.gate_rows;
            if (t + 1u < t1) start_gate();
        }
    };
    if (t0 < t1) {
        Row a, b;
        if (AHEAD) fetch(a, t0);
        if constexpr (!GATE) {
            if (p.gate) gate_row = t0 / p.gate_rows, gate_left = p.gate_rows - t0 % p.gate_rows;
            start_gate();
        }
        for (uint32_t t = t0; t < t1; t += 2u) {
            if (!AHEAD) fetch(a, t);
            step(a, b, t);
            if (!AHEAD && t + 1u < t1) fetch(b, t + 1u);
            if (t + 1u < t1) step(b, a, t + 1u);
        }
        if constexpr (!GATE)
            if (!p.gate || gate_left != p.gate_rows) end_gate();  // the last row's tokens go on in another chunk, or end
    } else if (!GATE && c.per_gate && p.dgate && team.index < c.count) {
        store_plain<V, NV>(p.ws + (2ull * c.parts + team.index) * p.D, dw_post, team, p.D);  // no tokens: zeros
    }
    if constexpr (!GATE)
#pragma unroll
        for (int i = 0; i < kPairs; ++i) dw_post[i] = post_sum[i * blockDim.x + threadIdx.x];
    if (plan.ctas) {
        if (p.dw_pre) store_plain<V, NV>(p.ws + (uint64_t)team.index * p.D, dw_pre, team, p.D);
        if (p.dw_post) store_plain<V, NV>(p.ws + ((uint64_t)c.parts + team.index) * p.D, dw_post, team, p.D);
        return;
    }
    // The sums of the CTA's teams, in order.
    __shared__ float2 all[kPairs][128];
    const uint32_t per = 128u / team.size;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (w ? !p.dw_post : !p.dw_pre) continue;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPairs; ++i) all[i][threadIdx.x] = w ? dw_post[i] : dw_pre[i];
        __syncthreads();
        if (threadIdx.x < team.size) {  // the first team adds
            float2 sum[kPairs];
#pragma unroll
            for (int i = 0; i < kPairs; ++i) sum[i] = all[i][threadIdx.x];
            for (uint32_t k = 1; k < per; ++k)
#pragma unroll
                for (int i = 0; i < kPairs; ++i) sum[i] = add2(sum[i], all[i][k * team.size + threadIdx.x]);
            store_plain<V, NV>(p.ws + ((uint64_t)w * c.parts + blockIdx.x) * p.D, sum, team, p.D);
        }
    }
}

// Adds the chunks' sums: blockIdx.y 0 and 1 dw_pre and dw_post, 2 + g gate row
// g.  32 columns a CTA, 32 warps that take every 32nd chunk; the warps' sums
// are added in order.
constexpr uint32_t kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps) sum_chunks(const Backward p, const Chunks c) {
    __shared__ float part[kSumWarps][32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, i = blockIdx.x * 32u + lane;
    for (uint32_t what = blockIdx.y; what < 2u + c.gates; what += gridDim.y) {
        if ((what == 0 && !p.dw_pre) || (what == 1 && !p.dw_post)) continue;
        const uint32_t first = what < 2u ? 0u : (what - 2u) * c.per_gate, n = what < 2u ? c.parts : c.per_gate;
        const float* ws = p.ws + ((uint64_t)min(what, 2u) * c.parts + first) * p.D + i;
        float s = 0.0f;
        if (i < p.D)
#pragma unroll 8
            for (uint32_t k = warp; k < n; k += kSumWarps) s += ws[(uint64_t)k * p.D];
        __syncthreads();
        part[warp][lane] = s;
        __syncthreads();
        if (warp != 0 || i >= p.D) continue;
#pragma unroll
        for (uint32_t k = 1; k < kSumWarps; ++k) s += part[k][lane];
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
        while (v > 1 && D % v) v = v == 8 ? 2 : 1;
    }
};

template <class K, class... Args>
cudaError_t launch(K kernel, dim3 grid, uint32_t threads, uint32_t cluster, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid, cfg.blockDim = dim3(threads, 1, 1), cfg.stream = s;
    cudaLaunchAttribute la[2];
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = cluster, la[1].val.clusterDim.y = 1, la[1].val.clusterDim.z = 1;
    cfg.attrs = la, cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) foil_count_launch();
    return e;
}

template <class R, int V, int E, int THREADS, int CTAS, int GATE>
cudaError_t forward_launch(const Forward& p, const Shape& sh, cudaStream_t s) {
    const uint32_t resident = sh.resident(THREADS * CTAS);
    const uint32_t teams = (p.T + sh.teams - 1) / sh.teams < resident ? (p.T + sh.teams - 1) / sh.teams : resident;
    const dim3 grid(teams * (sh.plan.ctas ? sh.plan.ctas : 1));
    return launch(forward_kernel<R, V, E / V, THREADS, CTAS, GATE>, grid, sh.threads, sh.plan.ctas, s, p, sh.plan);
}

// 8 channels a thread up to 2048 channels, then 16: one CTA up to 6144, above
// that two to four of up to 256 threads (one of 512 leaves an SM a single row at
// a time: 2000 x 8192 53 us).  As many CTAs on an SM as about 85 registers a thread
// allow (with 64 they spill, with more too few rows are on their way).
template <class R, int V, int GATE>
cudaError_t forward_gated(const Forward& p, cudaStream_t s) {
    if (p.D <= 2048) return forward_launch<R, V, 8, 256, 4, GATE>(p, Shape(p.D, 8, 512), s);
    if (p.D <= 4096) return forward_launch<R, V, 16, 256, 3, GATE>(p, Shape(p.D, 16, 512), s);
    if (p.D <= 6144) return forward_launch<R, V, 16, 384, 2, GATE>(p, Shape(p.D, 16, 512), s);
    return forward_launch<R, V, 16, 256, 3, GATE>(p, Shape(p.D, 16, 256), s);
}

template <class R, int V>
cudaError_t forward_typed(const Forward& p, cudaStream_t s) {
    if (!p.gate) return forward_gated<R, V, kNoGate>(p, s);
    return p.gate_act ? forward_gated<R, V, kSigmoidGate>(p, s) : forward_gated<R, V, kPlainGate>(p, s);
}

// The next row in registers where those suffice (4096 x 4096, bf16 in vectors of 8:
// 59 us with, 70 without; 4099 x 2050 in vectors of 2: 57 and 66), else towards L2 only
// (fp32: 98 us with, 80 without; 4000 x 4095 one by one: 160 and 101; bf16 with logistic
// gates: 90 and 72).
template <class R, int V, int GATE>
constexpr bool next_row_ahead() {
    return sizeof(R) == 2 && ((V == 8 && GATE != kSigmoidGate) || (V == 2 && GATE == kNoGate));
}

template <class R, int V, int GATE>
cudaError_t backward_launch(const Backward& p, const Chunks& c, cudaStream_t s) {
    const Shape sh(p.D, 8, 512);
    const uint32_t ctas = sh.plan.ctas ? sh.plan.ctas : 1;
    const dim3 grid((c.count + sh.teams - 1) / sh.teams * ctas);
    auto go = [&](auto ahead) {
        return launch(backward_kernel<R, V, 8 / V, 512, GATE, decltype(ahead)::value>, grid, sh.threads, sh.plan.ctas,
                      s, p, c, sh.plan);
    };
    if constexpr (!next_row_ahead<R, V, GATE>()) {
        return go(std::false_type());
    } else if constexpr (V == 8) {
        return go(std::true_type());
    } else {
        // Every vector but a thread's last has to be inside: not so for some rows of
        // fewer than 768 channels.
        const uint32_t team = sh.plan.ctas ? ctas * sh.threads : sh.plan.lanes;
        return (8 / V - 1) * V * team <= p.D ? go(std::true_type()) : go(std::false_type());
    }
}

template <class R, int V>
cudaError_t backward_typed(const Backward& p, const Chunks& c, cudaStream_t s) {
    if (!p.gate || p.gate_rows > 1) return backward_launch<R, V, kNoGate>(p, c, s);
    return p.gate_act ? backward_launch<R, V, kSigmoidGate>(p, c, s) : backward_launch<R, V, kPlainGate>(p, c, s);
}

}  // namespace

uint64_t backward_ws_bytes(uint32_t T, uint32_t D, uint32_t gate_rows) {
    if (T == 0 || D == 0) return 0;
    // Bounds of plan_chunks for T tokens or fewer.  There are at most `teams` chunks
    // of T tokens, one token or more each; where gate rows are shared, at most `teams`
    // of parts of them (the last gate row may have fewer tokens than chunks: 2 T), or
    // less than twice `teams` of whole ones (a chunk is more than half of T / teams).
    const Shape sh(D, 8, 512);
    const uint64_t teams = (uint64_t)sh.resident(kBackwardThreads) * sh.teams, shared = gate_rows > 1;
    const uint64_t count = std::min((1 + shared) * T, (1 + shared) * teams);
    const uint64_t parts = sh.plan.ctas ? count : (count + sh.teams - 1) / sh.teams;
    return (2 * parts + (shared ? std::min<uint64_t>(2ull * T, teams) : 0)) * D * 4;
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
    const Chunks c = plan_chunks(p.T, p.D, p.gate_rows);
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
    return launch(sum_chunks, dim3((p.D + 31) / 32, rows < 32768 ? rows : 32768), 32 * kSumWarps, 1, s, p, sums);
}

}  // namespace norm
}  // namespace foil
