// 4-bit weights with group scales: storage, conversion from and to tile
// streams, and products with a few rows.  The storage format is described at
// foil_w4_pack_dev in include/foil_c.h.
#include "w4.cuh"

#include "gemm_ptx.cuh"

namespace foil {
namespace w4 {
namespace {

using gemm::cluster_sync;
using gemm::cp_async16;
using gemm::map_to_rank;
using gemm::smem_u32;

// Element index of (row r, column c) in a tile stream of ct tile columns.
__device__ __forceinline__ uint64_t tile_index(uint32_t r, uint32_t c, uint32_t ct) {
    return ((uint64_t)(r / 32u) * ct + c / 32u) * 1024u + ((r % 32u / 16u) * 2u + c % 32u / 16u) * 256u +
           (r % 16u) * 16u + c % 16u;
}

// Byte offset of the 32-bit word of codes that holds (n, k..k+7), k % 8 == 0.
__device__ __forceinline__ uint64_t word_offset(uint32_t n, uint32_t k, uint32_t kb, uint32_t bytes) {
    return ((uint64_t)(n / kBlockN) * kb + k / kBlockK) * bytes +
           4u * ((n % 16u) * 16u + (k % 32u / 8u) * 4u + k % 128u / 32u);
}
__device__ __forceinline__ uint64_t scale_offset(uint32_t n, uint32_t k, uint32_t kb, uint32_t bytes, uint32_t group) {
    return ((uint64_t)(n / kBlockN) * kb + k / kBlockK) * bytes + kCodeBytes +
           2u * ((k % 128u / group) * 16u + n % 16u);
}
__device__ __forceinline__ uint64_t zero_offset(uint32_t n, uint32_t k, uint32_t kb, uint32_t bytes, uint32_t group) {
    return ((uint64_t)(n / kBlockN) * kb + k / kBlockK) * bytes + kCodeBytes + 32u * (128u / group) +
           (k % 128u / group) * 16u + n % 16u;
}
// Bit position in its word of the code of k % 8 = i: order 0 2 4 6 1 3 5 7.
__device__ __forceinline__ uint32_t nibble_shift(uint32_t i) { return 4u * (i / 2u + 4u * (i % 2u)); }

// One thread for each word of codes.
__global__ void pack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                            const uint8_t* __restrict__ zero_points, uint8_t* __restrict__ packed, Weights w,
                            uint32_t kb, uint64_t words) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= words) return;
    const uint32_t per_n = kb * 16u;  // words of a column
    const uint32_t n = (uint32_t)(i / per_n), k = (uint32_t)(i % per_n) * 8u;
    const uint32_t bytes = block_bytes(w.group, w.zeros);
    uint32_t v = 0;
    for (uint32_t j = 0; j < 8; ++j)
        if (n < w.N && k + j < w.K) v |= (codes[(uint64_t)n * w.K + k + j] & 15u) << nibble_shift(j);
    *reinterpret_cast<uint32_t*>(packed + word_offset(n, k, kb, bytes)) = v;
    if (k % w.group == 0) {
        const uint32_t groups = (w.K + w.group - 1) / w.group;
        const bool in = n < w.N && k < w.K;
        const uint64_t g = (uint64_t)n * groups + k / w.group;
        *reinterpret_cast<uint16_t*>(packed + scale_offset(n, k, kb, bytes, w.group)) = in ? scales[g] : 0;
        if (w.zeros) packed[zero_offset(n, k, kb, bytes, w.group)] = in ? zero_points[g] & 15u : 0;
    }
}

// One thread for each (column, group).
__global__ void quantize_kernel(const uint16_t* __restrict__ tiles, uint8_t* __restrict__ packed, Weights w,
                                uint32_t kb, uint64_t groups) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= groups) return;
    const uint32_t np = (w.N + 15u) / 16u * 16u;
    const uint32_t n = (uint32_t)(i % np), k0 = (uint32_t)(i / np) * w.group;
    const uint32_t bytes = block_bytes(w.group, w.zeros), ct = w.N / 32u;
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
    for (uint32_t k = k0; k < k0 + w.group && k < w.K && n < w.N; ++k) {
        const float v = bf16_bits_to_f32(tiles[tile_index(k, n, ct)]);
        bad |= !isfinite(v);
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    float s = w.zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f;
    const uint32_t s_bits = bad ? 0x7fc0u : f32_to_bf16_bits(s);
    s = bf16_bits_to_f32(s_bits);
    const bool ok = s > 0.0f && isfinite(s);
    const float z = !w.zeros || !ok ? 8.0f : fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f);
    for (uint32_t k = k0; k < k0 + w.group; k += 8) {
        uint32_t word = 0;
        for (uint32_t j = 0; j < 8; ++j) {
            float q = z;
            if (ok && k + j < w.K && n < w.N) {
                q = rintf(bf16_bits_to_f32(tiles[tile_index(k + j, n, ct)]) / s) + z;
                q = fminf(fmaxf(q, 0.0f), 15.0f);
            }
            word |= (uint32_t)q << nibble_shift(j);
        }
        *reinterpret_cast<uint32_t*>(packed + word_offset(n, k, kb, bytes)) = word;
    }
    *reinterpret_cast<uint16_t*>(packed + scale_offset(n, k0, kb, bytes, w.group)) = (uint16_t)s_bits;
    if (w.zeros) packed[zero_offset(n, k0, kb, bytes, w.group)] = (uint8_t)z;
}

__device__ __forceinline__ float weight(const uint8_t* packed, uint32_t n, uint32_t k, const Weights& w, uint32_t kb,
                                        uint32_t bytes) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(packed + word_offset(n, k / 8u * 8u, kb, bytes));
    const int q = (int)((word >> nibble_shift(k % 8u)) & 15u);
    const int z = w.zeros ? packed[zero_offset(n, k, kb, bytes, w.group)] : 8;
    return bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(packed + scale_offset(n, k, kb, bytes, w.group))) *
           (float)(q - z);
}

// One thread for each element of the tile stream.
__global__ void dequantize_kernel(const uint8_t* __restrict__ packed, uint16_t* __restrict__ tiles, Weights w,
                                  uint32_t kb, uint32_t transpose, uint64_t total) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const uint32_t ct = ((transpose ? w.K : w.N) + 31u) / 32u;
    const uint64_t tile = i / 1024u;
    const uint32_t e = (uint32_t)(i % 1024u), face = e / 256u;
    const uint32_t r = (uint32_t)(tile / ct) * 32u + face / 2u * 16u + e % 256u / 16u;
    const uint32_t c = (uint32_t)(tile % ct) * 32u + face % 2u * 16u + e % 16u;
    const uint32_t k = transpose ? c : r, n = transpose ? r : c;
    uint32_t bits = 0;
    if (k < w.K && n < w.N)
        bits = cvt_bf16x2(weight(packed, n, k, w, kb, block_bytes(w.group, w.zeros)), 0.0f) & 0xffffu;
    tiles[i] = (uint16_t)bits;
}

// ------------------------------------------------------------------ matvec ---
// y = x W for up to 16 rows of x at a time.  HBM-bound: 4-bit weights are read
// once, so everything else is laid around that stream.
//
//  * A warp takes one or two tiles of 16 columns n (what it reads of x serves
//    both) and a run of their storage blocks along k, one contiguous piece of
//    memory each, through a ring of its own: 16-byte asynchronous copies, 4 to
//    6 blocks (1056 to 1216 bytes each: codes, scales, zero points) ahead, no
//    other warp involved.  (Bulk copies of one block each, measured: 80 to 140 ns of an SM's copy
//    engine apiece, 1.2 to 2 TB/s in all.)
//  * mma.m16n8k16 with the weights as the 16-row operand: 16 + q is made in
//    bf16 by one shift and one logical operation for two codes (0x4180 is 16,
//    a code at bits 3..6 of its mantissa adds q, exact), laid out in storage
//    so that a lane's 16-byte words are its operand registers.  x is the other
//    operand, one 16-byte shared-memory read for two MMAs.
//  * The group's scale and zero point come after the MMAs in fp32:
//    s * (sum (16 + q) x - (16 + z) sum x), sum x of each group made once when
//    x is staged.  Nothing is rounded to fewer than 32 bits before the output.
//  * K is split over the CTAs of a cluster (S) where x would not fit one SM's
//    shared memory, and over the warps of a CTA (WK) where there are few
//    columns; the parts are added in a fixed order through (distributed)
//    shared memory.  Clusters take contiguous, near-equal runs of tiles: the
//    grid is one CTA per SM, whatever N is.
constexpr int kMvWarps = 16;
constexpr int kMvThreads = 32 * kMvWarps;
// Tiles of a warp at a time: two for up to 8 rows of x, one for up to 16 (the
// accumulators of two would not fit the registers); and the slots in flight.
__host__ __device__ constexpr int mv_tiles(int nt) { return nt == 1 ? 2 : 1; }
__host__ __device__ constexpr int mv_ahead(int rt) { return rt == 2 ? 3 : 4; }
constexpr uint32_t kMaxSmem = 232448;

struct Matvec {
    const uint16_t* x;
    const uint8_t* packed;
    const uint16_t* bias;
    uint16_t* y;
    uint64_t ld_x, ld_y;
    uint32_t M, K, N, kb, tiles;
    uint32_t S, WK, clusters, pass_runs;           // split (host)
    uint32_t x_pitch, off_sum, off_red, off_ring;  // shared-memory plan (host)
    uint32_t relu, x_vec;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes number I and I + 4 of a word as 16 + q in bf16.
template <int I>
__device__ __forceinline__ uint32_t codes16(uint32_t w) {
    const uint32_t v = I == 0 ? w << 3 : w >> (4 * I - 3);
    uint32_t r;  // (v & mask) | magic in one instruction
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "r"(0x00780078u), "r"(0x41804180u));
    return r;
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
__device__ __forceinline__ void st_cluster_f4(uint32_t addr, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
                 : "memory");
}

// The x rows of this CTA's blocks into shared memory (zeros past M and K) and
// the sum of each group of each row, times -24 (codes stand as 16 + q, and q - 8 is
// wanted) where there are no zero points.
template <int NT, int GROUP, bool ZEROS>
__device__ __forceinline__ void stage_x(const Matvec& p, uint8_t* smem, uint32_t m0, uint32_t kb0, uint32_t nkb) {
    float* sums = reinterpret_cast<float*>(smem + p.off_sum);
    const uint32_t rows = min(p.M - m0, 8u * NT);
    const uint32_t per_row = nkb * 16u, total = rows * per_row;  // 16-byte pieces
    for (uint32_t i = rows * p.x_pitch + threadIdx.x * 16u; i < 8u * NT * p.x_pitch; i += kMvThreads * 16u)
        *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
    for (uint32_t i0 = 0; i0 < total; i0 += kMvThreads) {
        const uint32_t i = i0 + threadIdx.x, row = i / per_row, c = i - row * per_row;
        uint4 v = make_uint4(0, 0, 0, 0);
        const uint32_t k = kb0 * kBlockK + c * 8u;
        if (i < total && k < p.K) {
            const uint16_t* src = p.x + (m0 + row) * p.ld_x + k;
            if (p.x_vec && k + 8u <= p.K) {
                v = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t e[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) e[j] = k + j < p.K ? src[j] : 0u;
                v = make_uint4(pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]),
                               pack_bf16x2(e[6], e[7]));
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = word_of(v, j);
            s += bf16_bits_to_f32(w & 0xffffu) + bf16_bits_to_f32(w >> 16);
        }
#pragma unroll
        for (int o = 1; o < GROUP / 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (i < total) {
            *reinterpret_cast<uint4*>(smem + row * p.x_pitch + c * 16u) = v;
            if (c % (GROUP / 8) == 0) sums[c / (GROUP / 8) * (8u * NT) + row] = ZEROS ? s : -24.0f * s;
        }
    }
}

template <int NT>
__device__ __forceinline__ void put(const Matvec& p, uint32_t m0, uint32_t tile, uint32_t nt, uint32_t lane,
                                    const float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t n = tile * 16u + lane / 4u + (j / 2) * 8u, m = m0 + nt * 8u + lane % 4u * 2u + j % 2;
        if (n >= p.N || m >= p.M) continue;
        float o = v[j];
        if (p.bias) o += bf16_bits_to_f32(p.bias[n]);
        if (p.relu && o < 0.0f) o = 0.0f;
        p.y[m * p.ld_y + n] = (uint16_t)(cvt_bf16x2(o, 0.0f) & 0xffffu);
    }
}

// -(16 + z) for a zero point z, in the bits of a float: 16 + z is 16 with z at
// bits 19..22 of the mantissa.
__device__ __forceinline__ float minus16(uint32_t z) { return __uint_as_float(0xc1800000u | (z & 15u) << 19); }

template <int NT, int RT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kMvThreads, 1) matvec_kernel(const __grid_constant__ Matvec p) {
    constexpr uint32_t kBytes = block_bytes(GROUP, ZEROS);
    constexpr int kGroups = 128 / GROUP;  // groups of a block
    constexpr int kAhead = mv_ahead(RT);
    constexpr uint32_t kSlot = RT * kBytes, kPlace = 512 * RT * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, g = lane / 4u, t = lane % 4u;
    const uint32_t rank = blockIdx.x % p.S, cluster = blockIdx.x / p.S, clusters = p.clusters;
    const uint32_t m0 = blockIdx.y * 8u * NT;
    // This CTA's blocks of k and its cluster's tiles, in runs of RT.
    const uint32_t kb0 = (uint32_t)((uint64_t)p.kb * rank / p.S);
    const uint32_t nkb = (uint32_t)((uint64_t)p.kb * (rank + 1) / p.S) - kb0;
    const uint32_t t0 = (uint32_t)((uint64_t)p.tiles * cluster / clusters);
    const uint32_t t1 = (uint32_t)((uint64_t)p.tiles * (cluster + 1) / clusters);
    const uint32_t runs = (t1 - t0 + RT - 1) / RT;
    // This warp's share: runs wn, wn + WN, ... and blocks [b0, b0 + nb) of kb0 ...
    const uint32_t WN = kMvWarps / p.WK, wn = warp / p.WK, wk = warp % p.WK;
    const uint32_t b0 = nkb * wk / p.WK, nb = nkb * (wk + 1) / p.WK - b0;
    const bool joined = p.S * p.WK > 1;
    const uint64_t tile_bytes = (uint64_t)p.kb * kBytes;

    uint8_t* const ring = smem + p.off_ring + warp * (kAhead * kSlot);
    uint8_t* const ring_end = ring + kAhead * kSlot;
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();

    // The warp's blocks in order, one commit group for a block of each tile of
    // the run (empty past the end).
    uint32_t is_run = wn, is_block = 0;
    const uint8_t* src = p.packed + (uint64_t)(t0 + RT * wn) * tile_bytes + (uint64_t)(kb0 + b0) * kBytes + lane * 16u;
    auto issue = [&](uint8_t* slot) {
        if (is_run < runs && nb) {
            const uint32_t dst = smem_u32(slot) + lane * 16u;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if (r && t0 + RT * is_run + r >= t1) break;
                const uint8_t* s = src + r * tile_bytes;
                cp_async16(dst + r * kBytes, s, 16);
                cp_async16(dst + r * kBytes + 512u, s + 512, 16);
                if (lane < (kBytes - kCodeBytes) / 16u)
                    cp_async16(dst + r * kBytes + kCodeBytes, s + kCodeBytes, 16);
            }
            src += kBytes;
            if (++is_block == nb) is_block = 0, is_run += WN, src += RT * WN * tile_bytes - (uint64_t)nb * kBytes;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) issue(ring + i * kSlot);

    stage_x<NT, GROUP, ZEROS>(p, smem, m0, kb0, nkb);
    if (p.S > 1)
        cluster_sync();  // also: every CTA of the cluster runs before its memory is written
    else
        __syncthreads();

    const uint8_t* const xrow = smem + g * p.x_pitch + t * 16u + b0 * 256u;
    const float* const sums =
        reinterpret_cast<const float*>(smem + p.off_sum) + b0 * kGroups * (8u * NT) + 2u * t;
    uint8_t* slot = ring;
    for (uint32_t pass = 0; pass < runs; pass += p.pass_runs) {
        const uint32_t pass_end = min(runs, pass + p.pass_runs);
        // pass_runs is a multiple of WN, so a warp's runs keep their stride.
        for (uint32_t run = pass + wn; run < pass_end; run += WN) {
            const uint32_t tile = t0 + RT * run, n_tiles = min((uint32_t)RT, t1 - tile);
            float acc[RT][NT][4];
#pragma unroll
            for (int i = 0; i < 4 * RT * NT; ++i) acc[i / (4 * NT)][i / 4 % NT][i % 4] = 0.0f;
            const uint8_t* xb = xrow;
            const float* xs = sums;
#pragma unroll 1
            for (uint32_t b = 0; b < nb; ++b, xb += 256, xs += kGroups * 8 * NT) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
                __syncwarp();  // every lane's copies have landed
                uint4 wa[RT], wb[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    wa[r] = *reinterpret_cast<const uint4*>(slot + r * kBytes + lane * 16u);
                    wb[r] = *reinterpret_cast<const uint4*>(slot + r * kBytes + 512u + lane * 16u);
                }
#pragma unroll
                for (int gi = 0; gi < kGroups; ++gi) {
                    float part[RT][NT][4];
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        // Start from minus (16 + z) times the group's sum of x.
                        float z0 = 1.0f, z1 = 1.0f;
                        if constexpr (ZEROS) {
                            const uint8_t* zp = slot + r * kBytes + kCodeBytes + 32 * kGroups + gi * 16;
                            z0 = minus16(zp[g]), z1 = minus16(zp[g + 8]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const float2 x2 = *reinterpret_cast<const float2*>(xs + (gi * NT + n) * 8);
                            part[r][n][0] = z0 * x2.x, part[r][n][1] = z0 * x2.y;
                            part[r][n][2] = z1 * x2.x, part[r][n][3] = z1 * x2.y;
                        }
                    }
#pragma unroll
                    for (int q = gi * (GROUP / 32); q < (gi + 1) * (GROUP / 32); ++q) {
                        uint4 xv[NT];
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            xv[n] = *reinterpret_cast<const uint4*>(xb + n * 8u * p.x_pitch + q * 64u);
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            if (r && r >= (int)n_tiles) break;
                            const uint32_t a = word_of(wa[r], q), c = word_of(wb[r], q);
                            const uint32_t a0 = codes16<0>(a), a1 = codes16<1>(a), a2 = codes16<2>(a),
                                           a3 = codes16<3>(a);
                            const uint32_t c0 = codes16<0>(c), c1 = codes16<1>(c), c2 = codes16<2>(c),
                                           c3 = codes16<3>(c);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma_bf16(part[r][n], a0, c0, a1, c1, xv[n].x, xv[n].y);
                                mma_bf16(part[r][n], a2, c2, a3, c3, xv[n].z, xv[n].w);
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint16_t* sc = reinterpret_cast<const uint16_t*>(slot + r * kBytes + kCodeBytes) + gi * 16;
                        const float s0 = bf16_bits_to_f32(sc[g]), s1 = bf16_bits_to_f32(sc[g + 8]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            acc[r][n][0] = fmaf(s0, part[r][n][0], acc[r][n][0]);
                            acc[r][n][1] = fmaf(s0, part[r][n][1], acc[r][n][1]);
                            acc[r][n][2] = fmaf(s1, part[r][n][2], acc[r][n][2]);
                            acc[r][n][3] = fmaf(s1, part[r][n][3], acc[r][n][3]);
                        }
                    }
                }
                __syncwarp();  // every lane has read the slot
                issue(slot);
                slot += kSlot;
                if (slot == ring_end) slot = ring;
            }
            if (!joined) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    if (r < (int)n_tiles)
#pragma unroll
                        for (int n = 0; n < NT; ++n) put<NT>(p, m0, tile + r, n, lane, acc[r][n]);
                continue;
            }
            // Run i of the pass belongs to CTA i % S, place i / S, part rank * WK + wk.
            const uint32_t i = run - pass;
            uint8_t* place = smem + p.off_red + (((i / p.S) * p.S + rank) * p.WK + wk) * kPlace + lane * 16u;
            const uint32_t dst = p.S > 1 ? map_to_rank(place, i % p.S) : smem_u32(place);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    st_cluster_f4(dst + 512u * (r * NT + n), acc[r][n][0], acc[r][n][1], acc[r][n][2], acc[r][n][3]);
        }
        if (!joined) continue;
        if (p.S > 1)
            cluster_sync();
        else
            __syncthreads();
        // Add the parts of this CTA's runs in order and finish them.
        const uint32_t n_pass = pass_end - pass;
        const uint32_t mine = n_pass > rank ? (n_pass - rank + p.S - 1) / p.S : 0u, parts = p.S * p.WK;
        for (uint32_t i = warp; i < mine * RT * NT; i += kMvWarps) {
            const uint32_t place = i / (RT * NT), tile = t0 + RT * (pass + place * p.S + rank) + i / NT % RT;
            const uint8_t* part = smem + p.off_red + place * parts * kPlace + i % (RT * NT) * 512u + lane * 16u;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t k = 0; k < parts; ++k) {
                const float4 f = *reinterpret_cast<const float4*>(part + k * kPlace);
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            }
            if (tile < t1) put<NT>(p, m0, tile, i % NT, lane, v);
        }
        if (pass_end < runs) {  // the places are free again
            if (p.S > 1)
                cluster_sync();
            else
                __syncthreads();
        }
    }
}

using MatvecKernel = void (*)(const Matvec);
template <int NT>
MatvecKernel pick_matvec(const Weights& w) {
    constexpr int RT = mv_tiles(NT);
    if (w.group == 32) return w.zeros ? matvec_kernel<NT, RT, 32, true> : matvec_kernel<NT, RT, 32, false>;
    if (w.group == 64) return w.zeros ? matvec_kernel<NT, RT, 64, true> : matvec_kernel<NT, RT, 64, false>;
    return w.zeros ? matvec_kernel<NT, RT, 128, true> : matvec_kernel<NT, RT, 128, false>;
}

uint32_t blocks_k(const Weights& w) { return (w.K + kBlockK - 1) / kBlockK; }
uint32_t padded_n(const Weights& w) { return (w.N + kBlockN - 1) / kBlockN * kBlockN; }
unsigned ctas(uint64_t threads) { return (unsigned)((threads + 255u) / 256u); }

cudaError_t count(cudaError_t e) {
    if (e == cudaSuccess) foil_count_launch();
    return e;
}

}  // namespace

cudaError_t pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zero_points, uint8_t* packed,
                 const Weights& w, cudaStream_t s) {
    const uint64_t words = (uint64_t)padded_n(w) * blocks_k(w) * 16u;
    pack_kernel<<<ctas(words), 256, 0, s>>>(codes, scales, zero_points, packed, w, blocks_k(w), words);
    return count(cudaGetLastError());
}

cudaError_t quantize_tiles(const uint16_t* tiles, uint8_t* packed, const Weights& w, cudaStream_t s) {
    const uint64_t groups = (uint64_t)padded_n(w) * blocks_k(w) * (128u / w.group);
    quantize_kernel<<<ctas(groups), 256, 0, s>>>(tiles, packed, w, blocks_k(w), groups);
    return count(cudaGetLastError());
}

cudaError_t dequantize_tiles(const uint8_t* packed, uint16_t* tiles, const Weights& w, bool transpose,
                             cudaStream_t s) {
    const uint64_t total = (uint64_t)((w.K + 31) / 32) * ((w.N + 31) / 32) * 1024u;
    dequantize_kernel<<<ctas(total), 256, 0, s>>>(packed, tiles, w, blocks_k(w), transpose ? 1u : 0u, total);
    return count(cudaGetLastError());
}

// The split of K over the CTAs of a cluster (S) and the warps of a CTA (WK):
// the one whose busiest warp reads the fewest storage blocks, among those
// whose slice of x fits.  A cluster barrier costs about as much as two blocks
// a warp, the join of a CTA's warps about half a block.
static bool plan_matvec(Matvec& p, uint32_t nt, uint32_t bytes, uint32_t group, uint32_t sms) {
    const uint32_t width = 8 * nt, rt = mv_tiles((int)nt), ring = kMvWarps * mv_ahead((int)rt) * rt * bytes;
    float best = 0.0f;
    for (uint32_t S = 1; S <= 8; S *= 2) {
        const uint32_t ks = (p.kb + S - 1) / S;
        if (S > 1 && S > p.kb) break;
        const uint32_t pitch = ks * 256 + 64;  // 64 bytes more: rows of an 8-lane read phase on distinct banks
        const uint32_t off_sum = width * pitch, sums = ks * (128 / group) * width * 4;
        const uint32_t off_red = (off_sum + sums + 127) / 128 * 128;
        const uint32_t fit = (S == 1 ? sms : foil_resident_clusters(S)), clusters = fit < p.tiles ? fit : p.tiles;
        const uint32_t tc = ((p.tiles + clusters - 1) / clusters + rt - 1) / rt;  // runs of rt tiles
        for (uint32_t wk = 1; wk <= kMvWarps && wk <= ks; wk *= 2) {
            // A run's set-up and join cost about as much as one of its steps.
            const uint32_t wn = kMvWarps / wk, units = (tc + wn - 1) / wn * ((ks + wk - 1) / wk + 1);
            const uint32_t place = S * wk * 512 * rt * nt;  // one run's parts
            const uint32_t min_red = S * wk > 1 ? (wn + S - 1) / S * place : 0;
            if (off_red + min_red + ring > kMaxSmem - 1024) continue;
            // What the ring leaves joins tiles.
            uint32_t red = kMaxSmem - 1024 - off_red - ring, pass = tc;
            if (S * wk > 1) {
                const uint32_t cap = red / place * S;
                if (cap < tc) pass = cap / wn * wn;
                red = (pass + S - 1) / S * place;
            } else {
                red = 0;
            }
            const uint32_t passes = (tc + pass - 1) / pass;
            const float cost = units + passes * (S > 1 ? 2.0f : wk > 1 ? 0.5f : 0.0f);
            if (best > 0.0f && cost >= best) continue;
            best = cost;
            p.S = S, p.WK = wk, p.clusters = clusters, p.x_pitch = pitch, p.off_sum = off_sum, p.off_red = off_red;
            p.off_ring = (off_red + red + 127) / 128 * 128;
            p.pass_runs = pass < tc ? pass : (tc + wn - 1) / wn * wn;
        }
    }
    return best > 0.0f;
}

cudaError_t matvec(const uint16_t* x, uint64_t ld_x, const uint8_t* packed, const uint16_t* bias, uint16_t* y,
                   uint64_t ld_y, uint32_t M, const Weights& w, bool relu, cudaStream_t s) {
    Matvec p{};
    p.x = x, p.packed = packed, p.bias = bias, p.y = y, p.ld_x = ld_x, p.ld_y = ld_y, p.M = M, p.K = w.K, p.N = w.N;
    p.kb = blocks_k(w), p.tiles = (w.N + 15) / 16, p.relu = relu ? 1 : 0;
    p.x_vec = (uintptr_t)x % 16 == 0 && ld_x % 8 == 0;
    const uint32_t bytes = block_bytes(w.group, w.zeros), sms = (uint32_t)foil_sm_count();
    // 16 rows at a time where there are more than 8 and their x fits, else 8.
    const uint32_t nt = M > 8 && plan_matvec(p, 2, bytes, w.group, sms) ? 2 : 1;
    if (nt == 1 && !plan_matvec(p, 1, bytes, w.group, sms)) return cudaErrorInvalidConfiguration;
    const uint32_t rt = mv_tiles((int)nt), smem = p.off_ring + kMvWarps * mv_ahead((int)rt) * rt * bytes;
    const MatvecKernel kernel = nt == 2 ? pick_matvec<2>(w) : pick_matvec<1>(w);
    const cudaError_t e = foil_smem_optin(reinterpret_cast<const void*>(kernel), (int)kMaxSmem - 512);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.clusters * p.S, (M + 8 * nt - 1) / (8 * nt), 1);
    cfg.blockDim = dim3(kMvThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute la[2]{};
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = p.S, la[1].val.clusterDim.y = 1, la[1].val.clusterDim.z = 1;
    cfg.attrs = la;
    cfg.numAttrs = p.S > 1 ? 2 : 1;
    return count(cudaLaunchKernelEx(&cfg, kernel, p));
}

}  // namespace w4
}  // namespace foil
