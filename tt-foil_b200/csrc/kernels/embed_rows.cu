// Embedding rows: scaled lookup, and the table's gradient by sorted tokens.
//
// Lookup: bound by HBM, a gather of whole rows: a few threads of one CTA a row,
// four vectors of 8 channels each on their way.
//
// Gradient, three launches:
//  1. sort_tokens: a stable radix sort of (id, token) in one cluster (one CTA
//     for few tokens), the digits' counts exchanged through distributed shared
//     memory.  Meanwhile the other SMs write the zeros of the table's rows that
//     no token names (each CTA looks through the ids for its rows), so the
//     table is written once.
//  2. sum_runs: CTAs take a run of 8 to 32 consecutive sorted tokens, add the rows of one
//     id in registers in that order and write an id's sum to the table where
//     all of its tokens are in the run; the sums of the first and the last id,
//     where they go on beyond it, go to the workspace.
//  3. join_runs: adds the parts of the ids that several runs share, in order.
// Bound by HBM (the table's rows written, the tokens' rows read).  The order of
// every sum is fixed by the ids alone; there are no floating-point atomics.
#include "embed_rows.cuh"

#include <algorithm>
#include <cstring>

#include "gemm_ptx.cuh"

namespace foil {
namespace embed {
namespace {

using gemm::cluster_sync;
using gemm::map_to_rank;

__device__ __forceinline__ int64_t load_id(const void* ids, int32_t id_bytes, uint64_t t) {
    return id_bytes == 8 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
}

// V values of type T (uint16_t: bf16 bits) to fp32 and back.
template <int V>
__device__ __forceinline__ void load(const uint16_t* p, float (&v)[V]) {
    if constexpr (V == 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = bf16_bits_to_f32(a[i] & 0xffffu);
            v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    } else if constexpr (V == 2) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        v[0] = bf16_bits_to_f32(w & 0xffffu), v[1] = __uint_as_float(w & 0xffff0000u);
    } else {
        v[0] = bf16_bits_to_f32(*p);
    }
}
template <int V>
__device__ __forceinline__ void load(const float* p, float (&v)[V]) {
    if constexpr (V == 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else if constexpr (V == 2) {
        const float2 a = *reinterpret_cast<const float2*>(p);
        v[0] = a.x, v[1] = a.y;
    } else {
        v[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void store(uint16_t* p, const float (&v)[V]) {
    if constexpr (V == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3]),
                                                  cvt_bf16x2(v[4], v[5]), cvt_bf16x2(v[6], v[7]));
    else if constexpr (V == 2)
        *reinterpret_cast<uint32_t*>(p) = cvt_bf16x2(v[0], v[1]);
    else
        *p = (uint16_t)(cvt_bf16x2(v[0], 0.0f) & 0xffffu);
}
template <int V>
__device__ __forceinline__ void store(float* p, const float (&v)[V]) {
    if constexpr (V == 8) {
        // One store of whole sectors where the address allows (two of half
        // sectors each reached two thirds of the bandwidth).
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
        if (((uintptr_t)p & 31u) == 0) {
            gemm::st_global_v8(p, w);
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else if constexpr (V == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
        *p = v[0];
    }
}

// Widest vector (8, 2 or 1 channels) for rows of D that every tensor allows.
struct Width {
    int v = 8;
    explicit Width(uint32_t D) {
        while (v > 1 && D % v) v = v == 8 ? 2 : 1;
    }
    void use(const void* p, uint64_t ld, uint64_t elem) {
        while (v > 1 && ((uintptr_t)p % (v * elem < 16 ? v * elem : 16) || ld % v)) v = v == 8 ? 2 : 1;
    }
};

template <class K, class... Args>
cudaError_t launch(K kernel, dim3 grid, uint32_t threads, uint32_t smem, uint32_t cluster, cudaStream_t s,
                   Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid, cfg.blockDim = dim3(threads, 1, 1), cfg.dynamicSmemBytes = smem, cfg.stream = s;
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

// ------------------------------------------------------------------ lookup ---
constexpr uint32_t kThreads = 256;

// A CTA holds kThreads / team rows at a time, `team` threads each.
template <class O, int V>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const Lookup p, uint32_t team) {
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x % team, per = kThreads / team;
    for (uint64_t t = (uint64_t)blockIdx.x * per + threadIdx.x / team; t < p.T; t += (uint64_t)gridDim.x * per) {
        const int64_t id = load_id(p.ids, p.id_bytes, t);
        const bool ok = id != p.pad_id && id >= 0 && id < (int64_t)p.V;
        if (!ok && id != p.pad_id && lane == 0) atomicOr(p.err, kErrBadIndex);
        const uint16_t* row = p.table + (ok ? (uint64_t)id * p.ld_table : 0u);
        O* out = static_cast<O*>(p.out) + t * p.ld_out;
        for (uint32_t i0 = lane * V; i0 < p.D; i0 += 4u * team * V) {
            float v[4][V];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t i = i0 + j * team * V;
#pragma unroll
                for (int e = 0; e < V; ++e) v[j][e] = 0.0f;
                if (ok && i < p.D) load<V>(row + i, v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t i = i0 + j * team * V;
                if (i >= p.D) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) v[j][e] *= p.scale;
                store<V>(out + i, v[j]);
            }
        }
    }
}

template <class O, int V>
cudaError_t lookup_launch(const Lookup& p, cudaStream_t s) {
    uint32_t team = 1;
    while (team < kThreads && (uint64_t)team * 4 * V < p.D) team *= 2;
    const uint64_t ctas = ((uint64_t)p.T + kThreads / team - 1) / (kThreads / team);
    const uint64_t most = (uint64_t)foil_sm_count() * 8;
    return launch(lookup_kernel<O, V>, dim3((unsigned)(ctas < most ? ctas : most)), kThreads, 0, 1, s, p, team);
}

// -------------------------------------------------------------------- sort ---
constexpr uint32_t kMaxRun = 32;      // sorted tokens of a run, at most
constexpr uint32_t kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCtas = 8;
constexpr uint32_t kSortAhead = 8;  // rounds of 32 tokens of a warp whose keys are on their way
constexpr uint32_t kMaxBits = 9, kMaxRadix = 1u << kMaxBits;
// A warp's counts of each digit, every CTA's, and the scan's; or the marks of
// a clearing CTA's rows.
constexpr uint32_t kSortSmem = (kSortWarps * kMaxRadix + kSortCtas * kMaxRadix + 32) * 4;
constexpr uint32_t kMarkRows = kSortSmem * 8 / 32 * 32;  // rows that one CTA can clear

struct Plan {
    uint32_t run, runs, slabs, joined;  // tokens of a run, runs, column slabs of a run, runs a CTA joins
    uint32_t ctas, clear;              // CTAs of the sort, CTAs that clear rows
    uint32_t passes, bits;             // passes of `bits` bits
    uint32_t *key0, *token0, *key1, *token1;  // buffers of the sort, in turn
    uint32_t *key, *token;             // those that hold the result
    float *head, *tail;                // [run][D]: sums that begin before, or end after, the run
};
uint64_t align16(uint64_t b) { return (b + 15u) / 16u * 16u; }

// Tokens of a run: short runs where there are few tokens, so that they fill the
// SMs; one run where one can hold them, which needs no join.
uint32_t run_length(uint32_t T, uint32_t D) {
    uint32_t run = kMaxRun;
    while (run > 8 && T > kMaxRun && (uint64_t)T * ((D + 2047) / 2048) < 512ull * run) run /= 2;
    return run;
}
// The most runs of T tokens or fewer: of T, or of as many as have shorter runs.
uint32_t most_runs(uint32_t T, uint32_t D) {
    uint32_t most = 0;
    for (uint32_t run = 8; run <= kMaxRun; run *= 2) {
        const uint32_t t = std::min(T, (512u * 2 * run - 1) / ((D + 2047) / 2048));
        for (uint32_t n : {t, T}) most = std::max(most, (n + run_length(n, D) - 1) / run_length(n, D));
    }
    return most;
}

Plan make_plan(const Gradient& p) {
    Plan q{};
    q.run = run_length(p.T, p.D);
    q.runs = (p.T + q.run - 1) / q.run;
    // One CTA sorts few tokens as fast (2048 of them).  Clusters of 4 leave 128 SMs
    // to the zeros, of 8 only 112 (a cluster stays inside a GPC) but sort in half the
    // time: taken where the table has less than 16 KB a token (4 and 8 CTAs: 32768
    // tokens, 32000 x 1024: 77 and 60 us; 8192 tokens, 32000 x 4096: 115 and 122).
    q.ctas = p.T <= 2048 ? 1 : p.accumulate || (uint64_t)p.V * p.D <= 4096ull * p.T ? kSortCtas : kSortCtas / 2;
    uint32_t bits = 1;
    while (bits < 32 && (p.V >> bits)) ++bits;  // ids 0 .. V - 1, and V for the rows that do not count
    q.passes = (bits + kMaxBits - 1) / kMaxBits;
    q.bits = (bits + q.passes - 1) / q.passes;
    char* at = static_cast<char*>(p.ws);
    uint64_t off = 0;
    auto take = [&](uint64_t n) {
        char* r = at + off;
        off += align16(n);
        return r;
    };
    q.key0 = (uint32_t*)take(4ull * p.T), q.token0 = (uint32_t*)take(4ull * p.T);
    q.key1 = (uint32_t*)take(4ull * p.T), q.token1 = (uint32_t*)take(4ull * p.T);
    q.key = q.passes % 2 ? q.key1 : q.key0, q.token = q.passes % 2 ? q.token1 : q.token0;
    if (q.runs > 1) q.head = (float*)take(4ull * q.runs * p.D), q.tail = (float*)take(4ull * q.runs * p.D);
    return q;
}

// Zeros to the rows [v0, v1) that no token names.
template <int V>
__device__ __forceinline__ void clear_rows(const Gradient& p, uint32_t* marks, uint32_t v0, uint32_t v1) {
    const uint32_t tid = threadIdx.x, warp = tid / 32u, lane = tid % 32u;
    for (uint32_t i = tid; i < (v1 - v0 + 31u) / 32u; i += kSortThreads) marks[i] = 0u;
    __syncthreads();
#pragma unroll 4
    for (uint32_t t = tid; t < p.T; t += kSortThreads) {
        const int64_t id = load_id(p.ids, p.id_bytes, t);
        if (id >= (int64_t)v0 && id < (int64_t)v1 && id != p.pad_id)
            atomicOr(&marks[((uint32_t)id - v0) / 32u], 1u << ((uint32_t)id - v0) % 32u);
    }
    __syncthreads();
    const float zero[V] = {};
    for (uint32_t r = warp; r < v1 - v0; r += kSortWarps) {
        if (marks[r / 32u] >> r % 32u & 1u) continue;
        float* row = p.dtable + (uint64_t)(v0 + r) * p.ld_dtable;
        for (uint32_t i = lane * V; i < p.D; i += 32u * V) store<V>(row + i, zero);
    }
}

template <int V>
__global__ void __launch_bounds__(kSortThreads, 1) sort_tokens(const Gradient p, const Plan q) {
    extern __shared__ __align__(16) uint32_t smem[];
    __shared__ uint32_t warp_sum[kMaxRadix / 32];
    uint32_t* const count = smem;                                // [warp][digit]: counts, then next places
    uint32_t* const total = smem + kSortWarps * kMaxRadix;       // [CTA][digit]
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, rank = blockIdx.x, ctas = q.ctas;
    const uint32_t radix = 1u << q.bits, tid = threadIdx.x;
    auto sync_all = [&] {
        if (ctas > 1)
            cluster_sync();
        else
            __syncthreads();
    };
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    if (rank >= ctas) {
        const uint64_t c = rank - ctas;
        clear_rows<V>(p, smem, (uint32_t)(p.V * c / q.clear), (uint32_t)(p.V * (c + 1) / q.clear));
        return;
    }
    // This warp's tokens, in order.
    const uint32_t part = rank * kSortWarps + warp, parts = ctas * kSortWarps;
    const uint32_t first = (uint32_t)((uint64_t)p.T * part / parts), last = (uint32_t)((uint64_t)p.T * (part + 1) / parts);
    uint32_t* const mine = count + warp * kMaxRadix;
    if (ctas > 1) cluster_sync();  // every CTA runs before its memory is written
    for (uint32_t pass = 0; pass < q.passes; ++pass) {
        const uint32_t *key_in = pass % 2 ? q.key1 : q.key0, *token_in = pass % 2 ? q.token1 : q.token0;
        uint32_t *key_out = pass % 2 ? q.key0 : q.key1, *token_out = pass % 2 ? q.token0 : q.token1;
        const uint32_t shift = pass * q.bits;
        auto key_of = [&](uint32_t i) {
            if (pass) return __ldcg(key_in + i);
            const int64_t id = load_id(p.ids, p.id_bytes, i);
            if (id == p.pad_id) return p.V;
            if (id >= 0 && id < (int64_t)p.V) return (uint32_t)id;
            atomicOr(p.err, kErrBadIndex);
            return p.V;
        };
        for (uint32_t d = lane; d < radix; d += 32u) mine[d] = 0u;
        __syncwarp();
        for (uint32_t i0 = first; i0 < last; i0 += 32u * kSortAhead) {
            uint32_t key[kSortAhead];
#pragma unroll
            for (uint32_t b = 0; b < kSortAhead; ++b)
                key[b] = i0 + 32u * b + lane < last ? key_of(i0 + 32u * b + lane) : ~0u;
#pragma unroll
            for (uint32_t b = 0; b < kSortAhead; ++b) {
                if (i0 + 32u * b >= last) break;  // the whole warp
                const bool in = i0 + 32u * b + lane < last;
                const uint32_t d = in ? key[b] >> shift & (radix - 1u) : ~0u;
                const uint32_t peers = __match_any_sync(0xffffffffu, d);
                if (in && (peers & ((1u << lane) - 1u)) == 0u) mine[d] += __popc(peers);
                __syncwarp();
            }
        }
        __syncthreads();
        // Digit tid: the tokens of the warps before each warp, and of the CTA.
        uint32_t n[kSortWarps];
        if (tid < radix) {
            uint32_t sum = 0;
#pragma unroll
            for (uint32_t w = 0; w < kSortWarps; ++w) n[w] = count[w * kMaxRadix + tid];
#pragma unroll
            for (uint32_t w = 0; w < kSortWarps; ++w) {
                const uint32_t k = n[w];
                n[w] = sum;
                sum += k;
            }
            if (ctas == 1)
                total[tid] = sum;
            else
                for (uint32_t c = 0; c < ctas; ++c)
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank(total + rank * kMaxRadix + tid, c)),
                                 "r"(sum)
                                 : "memory");
        }
        sync_all();
        // The places of digit tid: after all smaller digits, after the CTAs before.
        uint32_t all = 0, before = 0, incl = 0;
        if (tid < kMaxRadix) {
            if (tid < radix)
                for (uint32_t c = 0; c < ctas; ++c) {
                    const uint32_t k = total[c * kMaxRadix + tid];
                    all += k;
                    before += c < rank ? k : 0u;
                }
            incl = all;
            for (uint32_t o = 1; o < 32u; o <<= 1) {
                const uint32_t k = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += k;
            }
            if (lane == 31u) warp_sum[warp] = incl;
        }
        __syncthreads();
        if (tid < radix) {
            uint32_t base = incl - all + before;
            for (uint32_t w = 0; w < warp; ++w) base += warp_sum[w];
#pragma unroll
            for (uint32_t w = 0; w < kSortWarps; ++w) count[w * kMaxRadix + tid] = n[w] + base;
        }
        __syncthreads();
        for (uint32_t i0 = first; i0 < last; i0 += 32u * kSortAhead) {
            uint32_t key[kSortAhead], token[kSortAhead];
#pragma unroll
            for (uint32_t b = 0; b < kSortAhead; ++b) {
                const uint32_t i = i0 + 32u * b + lane;
                key[b] = i < last ? key_of(i) : ~0u;
                token[b] = i >= last ? 0u : pass ? __ldcg(token_in + i) : i;
            }
#pragma unroll
            for (uint32_t b = 0; b < kSortAhead; ++b) {
                if (i0 + 32u * b >= last) break;  // the whole warp
                const bool in = i0 + 32u * b + lane < last;
                const uint32_t d = in ? key[b] >> shift & (radix - 1u) : ~0u;
                const uint32_t peers = __match_any_sync(0xffffffffu, d), lower = peers & ((1u << lane) - 1u);
                uint32_t at = 0;
                if (in) at = mine[d] + __popc(lower);
                __syncwarp();
                if (in) {
                    if (lower == 0u) mine[d] += __popc(peers);
                    key_out[at] = key[b];
                    token_out[at] = token[b];
                }
                __syncwarp();
            }
        }
        sync_all();
    }
}

// -------------------------------------------------------------------- sums ---
constexpr uint32_t kAhead = 8;  // rows of tokens on their way

template <class I, int V>
__global__ void __launch_bounds__(kThreads) sum_runs(const Gradient p, const Plan q) {
    __shared__ uint32_t key[kMaxRun + 2], token[kMaxRun];
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    const uint32_t run = (uint32_t)(blockIdx.x / q.slabs), first = run * q.run, n = min(q.run, p.T - first);
    const uint32_t *keys = q.key, *tokens = q.token;
    if (threadIdx.x < q.run + 2u) {  // the keys before and after the run too
        const uint32_t i = first + threadIdx.x - 1u;
        key[threadIdx.x] = first + threadIdx.x >= 1u && i < p.T ? __ldcg(keys + i) : ~0u;
        if (threadIdx.x >= 1u && threadIdx.x <= q.run && i < p.T) token[threadIdx.x - 1u] = __ldcg(tokens + i);
    }
    __syncthreads();
    const uint32_t col = (blockIdx.x % q.slabs * kThreads + threadIdx.x) * V;
    if (col >= p.D) return;
    const I* dout = static_cast<const I*>(p.dout) + col;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    bool before = key[0] == key[1];  // the id began before the run
    for (uint32_t r0 = 0; r0 < n; r0 += kAhead) {
        float x[kAhead][V];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t r = min(r0 + j, n - 1u);  // past the end: read again, not used
            load<V>(dout + (uint64_t)token[r] * p.ld_dout, x[j]);
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t r = r0 + j;
            if (r >= n || key[r + 1] >= p.V) return;  // padding and bad ids come last
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += x[j][e];
            const bool ends = key[r + 2] != key[r + 1];
            if (!ends && r + 1u < n) continue;
            if (ends && !before) {
                float* row = p.dtable + (uint64_t)key[r + 1] * p.ld_dtable + col;
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = 0.0f;
                if (p.accumulate) load<V>(row, v);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = fmaf(p.scale, acc[e], v[e]);
                store<V>(row, v);
            } else {
                float* part = (before ? q.head : q.tail) + (uint64_t)run * p.D + col;
#pragma unroll
                for (int e = 0; e < V; ++e) part[e] = acc[e];
            }
            before = false;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = 0.0f;
        }
    }
}

// blockIdx.x: one or eight runs, of which those count whose last id begins there
// and goes on; blockIdx.y: 256 columns.  8 warps take every eighth part, their sums
// are added in order.
constexpr uint32_t kJoinColumns = 256, kJoinRuns = 8;
constexpr uint32_t kJoinAhead = 4;  // parts of a warp on their way

__global__ void __launch_bounds__(kThreads) join_runs(const Gradient p, const Plan q) {
    __shared__ float part[kThreads / 32][kJoinColumns];
    __shared__ uint32_t ids[kJoinRuns], ends[kJoinRuns];  // the id (~0: nothing to do), the run after its last part
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    const uint32_t *keys = q.key, warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    // Warp w looks at run w.
    {
        const uint64_t run = (uint64_t)blockIdx.x * q.joined + warp, first = run * q.run, end = first + q.run;
        uint32_t found = ~0u, lo = (uint32_t)run + 1u, hi = q.runs;
        if (warp < q.joined && end < p.T) {
            const uint32_t id = __ldcg(keys + end - 1u), next = __ldcg(keys + end), begin = __ldcg(keys + first);
            const uint32_t previous = first ? __ldcg(keys + first - 1u) : ~0u;
            if (id < p.V && next == id && !(begin == id && previous == id)) found = id;
        }
        // Runs after this one that begin with the id: lo begins with it, hi does
        // not; 32 places between them at a time.
        while (found != ~0u && hi - lo > 1u) {
            const uint32_t step = (hi - lo + 32u) / 33u, at = lo + (lane + 1u) * step;
            const uint32_t in =
                __popc(__ballot_sync(0xffffffffu, at < hi && __ldcg(keys + (uint64_t)at * q.run) == found));
            hi = min(hi, lo + (in + 1u) * step);
            lo += in * step;
        }
        if (lane == 0) ids[warp] = found, ends[warp] = hi;
    }
    __syncthreads();
    const uint32_t col = blockIdx.y * kJoinColumns + lane;
    constexpr int kEach = kJoinColumns / 32;
    for (uint32_t w = 0; w < q.joined; ++w) {
        const uint32_t id = ids[w], run = blockIdx.x * q.joined + w, hi = ends[w];
        if (id == ~0u) continue;
        float s[kEach] = {};
        for (uint32_t r0 = run + warp; r0 < hi; r0 += kJoinAhead * (kThreads / 32u)) {
            float v[kJoinAhead][kEach];
#pragma unroll
            for (uint32_t k = 0; k < kJoinAhead; ++k) {
                const uint32_t r = r0 + k * (kThreads / 32u);
                const float* row = (r == run ? q.tail : q.head) + (uint64_t)r * p.D + col;
#pragma unroll
                for (int j = 0; j < kEach; ++j) v[k][j] = r < hi && col + 32u * j < p.D ? row[32 * j] : 0.0f;
            }
#pragma unroll
            for (uint32_t k = 0; k < kJoinAhead; ++k)
#pragma unroll
                for (int j = 0; j < kEach; ++j) s[j] += v[k][j];
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) part[warp][lane + 32 * j] = s[j];
        __syncthreads();
        const uint32_t i = blockIdx.y * kJoinColumns + threadIdx.x;
        if (i < p.D) {
            float sum = 0.0f;
            for (uint32_t k = 0; k < kThreads / 32u; ++k) sum += part[k][threadIdx.x];
            float* at = p.dtable + (uint64_t)id * p.ld_dtable + i;
            *at = fmaf(p.scale, sum, p.accumulate ? *at : 0.0f);
        }
        __syncthreads();
    }
}
static_assert(kJoinColumns == kThreads && kJoinRuns == kThreads / 32, "a thread a column, a warp a run");

template <int V>
cudaError_t sort_launch(const Gradient& p, Plan& q, cudaStream_t s) {
    // The other SMs clear rows, as many CTAs as run beside the sort.
    const uint32_t sms = (uint32_t)foil_sm_count(), fit = q.ctas > 1 ? foil_resident_clusters(q.ctas) * q.ctas : sms;
    q.clear = 0;
    if (!p.accumulate) {
        q.clear = fit > q.ctas ? fit - q.ctas : q.ctas;
        while ((uint64_t)q.clear * kMarkRows < p.V + q.clear) q.clear += q.ctas;
    }
    const cudaError_t e = foil_smem_optin(reinterpret_cast<const void*>(sort_tokens<V>), (int)kSortSmem);
    if (e != cudaSuccess) return e;
    return launch(sort_tokens<V>, dim3(q.ctas + q.clear), kSortThreads, kSortSmem, q.ctas, s, p, q);
}

template <class I>
cudaError_t sum_launch(const Gradient& p, Plan q, int v, cudaStream_t s) {
    q.slabs = (p.D + kThreads * v - 1) / (kThreads * v);
    const uint64_t grid = (uint64_t)q.runs * q.slabs;
    if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    const dim3 g((unsigned)grid);
    if (v == 8) return launch(sum_runs<I, 8>, g, kThreads, 0, 1, s, p, q);
    return v == 2 ? launch(sum_runs<I, 2>, g, kThreads, 0, 1, s, p, q)
                  : launch(sum_runs<I, 1>, g, kThreads, 0, 1, s, p, q);
}

}  // namespace

uint64_t gradient_ws_bytes(uint32_t T, uint32_t V, uint32_t D) {
    if (T == 0 || V == 0 || D == 0) return 0;
    // Enough for fewer tokens too, whose runs may be shorter.
    const uint64_t runs = most_runs(T, D);
    return 4 * align16(4ull * T) + (runs > 1 ? 2 * align16(4 * runs * D) : 0);
}

cudaError_t lookup(const Lookup& p, bool fp32, cudaStream_t s) {
    Width w(p.D);
    w.use(p.table, p.ld_table, 2), w.use(p.out, p.ld_out, fp32 ? 4 : 2);
    if (fp32)
        return w.v == 8 ? lookup_launch<float, 8>(p, s)
                        : w.v == 2 ? lookup_launch<float, 2>(p, s) : lookup_launch<float, 1>(p, s);
    return w.v == 8 ? lookup_launch<uint16_t, 8>(p, s)
                    : w.v == 2 ? lookup_launch<uint16_t, 2>(p, s) : lookup_launch<uint16_t, 1>(p, s);
}

cudaError_t gradient(const Gradient& p, bool fp32, cudaStream_t s) {
    if (p.T == 0)
        return p.accumulate ? cudaSuccess
                            : cudaMemset2DAsync(p.dtable, p.ld_dtable * 4, 0, (size_t)p.D * 4, p.V, s);
    Plan q = make_plan(p);
    Width w(p.D);
    w.use(p.dtable, p.ld_dtable, 4);
    cudaError_t e = w.v == 8 ? sort_launch<8>(p, q, s) : w.v == 2 ? sort_launch<2>(p, q, s) : sort_launch<1>(p, q, s);
    if (e != cudaSuccess) return e;
    w.use(p.dout, p.ld_dout, fp32 ? 4 : 2);
    e = fp32 ? sum_launch<float>(p, q, w.v, s) : sum_launch<uint16_t>(p, q, w.v, s);
    if (e != cudaSuccess || q.runs < 2) return e;
    const uint32_t columns = (p.D + kJoinColumns - 1) / kJoinColumns;
    // A run a CTA where those are few: an id's parts are found and added in a chain
    // (3592 tokens of 439 channels 29 and 21 us), else eight, for the launch of so many
    // CTAs (65536 of 1024 channels 104 and 96 us).
    q.joined = (uint64_t)q.runs * columns <= 2048 ? 1 : kJoinRuns;
    const dim3 grid((q.runs + q.joined - 1) / q.joined, columns);
    return launch(join_runs, grid, kThreads, 0, 1, s, p, q);
}

}  // namespace embed
}  // namespace foil
