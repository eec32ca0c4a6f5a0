// 4-bit weights with group scales: storage, conversion from and to tile
// streams, and products with a few rows.  The storage format is described at
// foil_w4_pack_dev in include/foil_c.h.
#include "w4.cuh"

#include <cstring>
#include <type_traits>

#include "gemm_ptx.cuh"

namespace foil {
namespace w4 {
namespace {

using gemm::cluster_sync;
using gemm::cp_async16;
using gemm::map_to_rank;
using gemm::smem_u32;

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

// ---------------------------------------------------- tile stream <-> codes ---
// One warp a storage block: 16 columns n by 128 k are the same face column of
// four tiles, eight faces of 512 contiguous bytes.  Lane l of a face holds its
// row k = l / 2, columns 8 (l % 2) + 0..7; in the storage a lane holds words
// of one column and 8 k.  Between the two lies an 8 x 8 transpose of codes
// over the 8 lanes of equal l % 2 and l / 16, three exchanges of half a word.
// Bound by HBM; no shared memory, 16-byte accesses in whole sectors.

// Codes in word position i + 4 j stand for element 2 i + j (column or k), so
// that bits i and i + 16 are a bf16 pair's.  With e the element's bits: position
// bit 2 is e0, bit 1 is e2, bit 0 is e1; the lane's bits 1, 2, 3 are e0, e1, e2.
__device__ __forceinline__ uint32_t swap_codes(uint32_t w, uint32_t lane, uint32_t lane_bit, uint32_t shift,
                                               uint32_t low) {
    const uint32_t o = __shfl_xor_sync(0xffffffffu, w, lane_bit);
    return lane & lane_bit ? (w & ~low) | (o >> shift & low) : (w & low) | (o & low) << shift;
}
__device__ __forceinline__ uint32_t transpose_codes(uint32_t w, uint32_t lane) {
    w = swap_codes(w, lane, 2, 16, 0x0000ffffu);
    w = swap_codes(w, lane, 8, 8, 0x00ff00ffu);
    return swap_codes(w, lane, 4, 4, 0x0f0f0f0fu);
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
__device__ __forceinline__ void word_set(uint4& v, int i, uint32_t w) {
    if (i == 0) v.x = w;
    if (i == 1) v.y = w;
    if (i == 2) v.z = w;
    if (i == 3) v.w = w;
}

// Face (k face f of block kb, column tile n16) in a stream of ct tile columns.
__device__ __forceinline__ uint64_t face_offset(uint32_t kb, uint32_t f, uint32_t n16, uint32_t ct) {
    const uint32_t kt = kb * 4u + f / 2u;
    return ((uint64_t)kt * ct + n16 / 2u) * 1024u + ((f % 2u) * 2u + n16 % 2u) * 256u;
}

// w / s: the product with the reciprocal, corrected once by its residual
// (Newton's iteration for a quotient).  Where the quotient is k + 1/2, which
// decides the rounding, it is representable and comes out exact; anywhere else
// two bf16 values' quotient is at least 2^-12 away from k + 1/2.
__device__ __forceinline__ float2 quotient(float2 w, float2 s, float2 inv) {
    const float2 t = mul2(w, inv);
    return fma2(fma2(make_float2(-t.x, -t.y), s, w), inv, t);
}

// A column's scale (its bits), the scale's reciprocal and the zero point from
// the largest value and the largest magnitude below zero (bf16 bits).
struct Column {
    uint32_t s_bits, zero;
    float s, inv;
};
template <bool ZEROS>
__device__ __forceinline__ Column column_of(uint32_t hi, uint32_t lo) {
    Column c;
    const float fh = bf16_bits_to_f32(hi), fl = bf16_bits_to_f32(lo);
    c.s_bits = f32_to_bf16_bits(ZEROS ? (fh + fl) / 15.0f : fmaxf(fh, fl) / 7.0f);
    // An infinity or NaN among them, or a range that overflows: NaN, not an infinity,
    // which times a sum that is not exactly zero would be one.
    if (max(hi, lo) >= 0x7f80u || c.s_bits >= 0x7f80u) c.s_bits = 0x7fc0u;
    c.s = bf16_bits_to_f32(c.s_bits);
    c.zero = 8;
    if (!(c.s > 0.0f)) {
        c.s = 0.0f, c.inv = 0.0f;  // every code is the zero point
        return c;
    }
    c.inv = 1.0f / c.s;
    if (ZEROS) c.zero = (uint32_t)fminf(fmaxf(rintf(fl / c.s), 0.0f), 15.0f);
    return c;
}

template <int GROUP, bool ZEROS>
__global__ void __launch_bounds__(256) quantize_kernel(const uint16_t* __restrict__ tiles, uint8_t* __restrict__ packed,
                                                       Weights w, uint32_t kb_count, uint64_t blocks) {
    constexpr int kGroups = 128 / GROUP, kFaces = GROUP / 16;  // of a block, of a group
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x % 32u, nt = (w.N + 15u) / 16u, ct = w.N / 32u;
    const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 32u);
    for (uint64_t b = (uint64_t)blockIdx.x * (blockDim.x / 32u) + threadIdx.x / 32u; b < blocks; b += step) {
        const uint32_t kb = (uint32_t)(b / nt), n16 = (uint32_t)(b % nt);
        uint4 x[8];
#pragma unroll
        for (int f = 0; f < 8; ++f) {
            x[f] = make_uint4(0, 0, 0, 0);
            if (kb * 128u + f * 16u < w.K)
                x[f] = __ldcs(reinterpret_cast<const uint4*>(tiles + face_offset(kb, f, n16, ct)) + lane);
        }
        uint8_t* const block = packed + ((uint64_t)n16 * kb_count + kb) * block_bytes(GROUP, ZEROS);
        uint4 out[2];  // words of k = 32 i + 8 (lane / 16), and 16 more
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
            // Largest value (or magnitude) of each column, two columns a word:
            // magnitudes' bits order like integers.
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hi[i] = lo[i] = 0;
#pragma unroll
                for (int f = gi * kFaces; f < (gi + 1) * kFaces; ++f) {
                    const uint32_t v = word_of(x[f], i), mag = v & 0x7fff7fffu;
                    if constexpr (ZEROS) {
                        const uint32_t neg = (v >> 15 & 0x00010001u) * 0xffffu;  // halves that are negative
                        hi[i] = __vmaxu2(hi[i], mag & ~neg);
                        lo[i] = __vmaxu2(lo[i], mag & neg);
                    } else {
                        hi[i] = __vmaxu2(hi[i], mag);
                    }
                }
#pragma unroll
                for (int o = 2; o < 32; o <<= 1) {
                    hi[i] = __vmaxu2(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
                    if constexpr (ZEROS) lo[i] = __vmaxu2(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
                }
            }
            // Lane l makes column 8 (l % 2) + l / 2 % 8, then all lanes ask for theirs.
            const uint32_t e = lane / 2u % 8u;
            const uint32_t eh = e < 4u ? (e < 2u ? hi[0] : hi[1]) : (e < 6u ? hi[2] : hi[3]);
            const uint32_t el = e < 4u ? (e < 2u ? lo[0] : lo[1]) : (e < 6u ? lo[2] : lo[3]);
            const Column c = column_of<ZEROS>(e % 2u ? eh >> 16 : eh & 0xffffu, e % 2u ? el >> 16 : el & 0xffffu);
            if (lane < 16u) {
                const uint32_t n = lane % 2u * 8u + e;
                reinterpret_cast<uint16_t*>(block + kCodeBytes)[gi * 16 + n] = (uint16_t)c.s_bits;
                if constexpr (ZEROS) block[kCodeBytes + 32 * kGroups + gi * 16 + n] = (uint8_t)c.zero;
            }
            float2 s[4], inv[4], zero[ZEROS ? 4 : 1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int from = (int)(lane % 2u) + 4 * j;
                s[j] = make_float2(__shfl_sync(0xffffffffu, c.s, from), __shfl_sync(0xffffffffu, c.s, from + 2));
                inv[j] = make_float2(__shfl_sync(0xffffffffu, c.inv, from), __shfl_sync(0xffffffffu, c.inv, from + 2));
                if constexpr (ZEROS)
                    zero[j] = make_float2((float)__shfl_sync(0xffffffffu, c.zero, from),
                                          (float)__shfl_sync(0xffffffffu, c.zero, from + 2));
            }
            // Without zero points |w / s| is below 7.2 where the reciprocal is a number (a
            // scale above 2^-128 is within 2^-6 of max / 7).  Smaller scales, which divide,
            // have few bits: w / s reaches 10 and is clamped.
            auto face_codes = [&](int f, auto divide) {
                uint32_t word = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t v = word_of(x[f], j);
                    const float2 wf = make_float2(bf16_bits_to_f32(v & 0xffffu), __uint_as_float(v & 0xffff0000u));
                    float2 t = quotient(wf, s[j], inv[j]);
                    if constexpr (decltype(divide)::value) {
                        t = make_float2(s[j].x > 0.0f ? wf.x / s[j].x : 0.0f, s[j].y > 0.0f ? wf.y / s[j].y : 0.0f);
                        if constexpr (!ZEROS)
                            t = make_float2(fminf(fmaxf(t.x, -8.0f), 7.0f), fminf(fmaxf(t.y, -8.0f), 7.0f));
                    }
                    // To integers, ties to even: 1.5 * 2^23 leaves no fraction bits.
                    const float2 kRound = both(12582912.0f);
                    if constexpr (ZEROS) {
                        t = add2(add2(add2(t, kRound), both(-12582912.0f)), zero[j]);
                        t = make_float2(fminf(fmaxf(t.x, 0.0f), 15.0f), fminf(fmaxf(t.y, 0.0f), 15.0f));
                        t = add2(t, kRound);
                    } else {
                        t = add2(t, both(12582920.0f));  // + 8
                    }
                    const uint32_t codes = __byte_perm(__float_as_uint(t.x), __float_as_uint(t.y), 0x5410);
                    word |= (codes & 0x000f000fu) << (4 * j);
                }
                word_set(out[f % 2], f / 2, transpose_codes(word, lane));
            };
            if (__any_sync(0xffffffffu, !isfinite(c.inv))) {  // a reciprocal overflows: divide
#pragma unroll
                for (int f = gi * kFaces; f < (gi + 1) * kFaces; ++f) face_codes(f, std::true_type());
            } else {
#pragma unroll
                for (int f = gi * kFaces; f < (gi + 1) * kFaces; ++f) face_codes(f, std::false_type());
            }
        }
        // Lane l holds column 8 (l % 2) + l / 2 % 8.
        uint4* const dst = reinterpret_cast<uint4*>(block) + (lane % 2u * 8u + lane / 2u % 8u) * 4u + lane / 16u;
        dst[0] = out[0];
        dst[2] = out[1];
    }
}

// Two weights of a word of codes: (q - z) s in bf16, (16 + q) - (16 + z) exact
// and the product rounded once.
template <int I>
__device__ __forceinline__ uint32_t weights2(uint32_t w, uint32_t z16, uint32_t s) {
    const uint32_t v = I == 0 ? w << 3 : w >> (4 * I - 3);
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\t"
        "lop3.b32 t, %1, 0x00780078, %2, 0xea;\n\t"
        "sub.rn.bf16x2 t, t, %3;\n\t"
        "mul.rn.bf16x2 %0, t, %4;\n\t}"
        : "=r"(r)
        : "r"(v), "r"(0x41804180u), "r"(z16), "r"(s));
    return r;
}
// 16 + z in bf16 for both halves' zero points.
__device__ __forceinline__ uint32_t sixteen(uint32_t z0, uint32_t z1) {
    return 0x41804180u | (z0 & 15u) << 3 | (z1 & 15u) << 19;
}

template <int GROUP, bool ZEROS, bool TRANSPOSE>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ packed, uint16_t* __restrict__ tiles,
                                                         Weights w, uint32_t kb_count, uint64_t blocks) {
    constexpr int kGroups = 128 / GROUP, kFaces = GROUP / 16;
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();
    const uint32_t lane = threadIdx.x % 32u;
    // Tile columns of the output; 16-column blocks up to whole tiles (the one
    // past N, if any, is zeros).
    const uint32_t nt = (w.N + 31u) / 32u * 2u, stored = (w.N + 15u) / 16u;
    const uint32_t kt = (w.K + 31u) / 32u, ct = TRANSPOSE ? kt : nt / 2u;
    const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 32u);
    for (uint64_t b = (uint64_t)blockIdx.x * (blockDim.x / 32u) + threadIdx.x / 32u; b < blocks; b += step) {
        const uint32_t kb = (uint32_t)(TRANSPOSE ? b % kb_count : b / nt), n16 = (uint32_t)(TRANSPOSE ? b / kb_count : b % nt);
        const uint8_t* const block = packed + ((uint64_t)n16 * kb_count + kb) * block_bytes(GROUP, ZEROS);
        // The column whose words this lane reads, and those it writes.
        const uint32_t row = TRANSPOSE ? lane / 2u : lane % 2u * 8u + lane / 2u % 8u;
        const uint32_t half = TRANSPOSE ? lane % 2u : lane / 16u;
        uint4 in[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        const bool there = n16 < stored;
        if (there) {
            const uint4* src = reinterpret_cast<const uint4*>(block) + row * 4u + half;
            in[0] = __ldcs(src), in[1] = __ldcs(src + 2);
        }
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
            uint32_t s[4] = {0, 0, 0, 0}, z[4] = {0x41c041c0u, 0x41c041c0u, 0x41c041c0u, 0x41c041c0u};
            if (there) {
                const uint8_t* scales = block + kCodeBytes + gi * 32;
                const uint8_t* zeros = block + kCodeBytes + 32 * kGroups + gi * 16;
                if constexpr (TRANSPOSE) {
                    const uint32_t one = reinterpret_cast<const uint16_t*>(scales)[row];
                    s[0] = s[1] = s[2] = s[3] = one * 0x00010001u;
                    if constexpr (ZEROS) z[0] = z[1] = z[2] = z[3] = sixteen(zeros[row], zeros[row]);
                } else {
                    const uint4 v = reinterpret_cast<const uint4*>(scales)[lane % 2u];
                    s[0] = v.x, s[1] = v.y, s[2] = v.z, s[3] = v.w;
                    if constexpr (ZEROS) {
                        const uint2 q = reinterpret_cast<const uint2*>(zeros)[lane % 2u];
                        z[0] = sixteen(q.x, q.x >> 8), z[1] = sixteen(q.x >> 16, q.x >> 24);
                        z[2] = sixteen(q.y, q.y >> 8), z[3] = sixteen(q.y >> 16, q.y >> 24);
                    }
                }
            }
#pragma unroll
            for (int f = gi * kFaces; f < (gi + 1) * kFaces; ++f) {
                uint32_t word = word_of(in[f % 2], f / 2);
                if constexpr (!TRANSPOSE) word = transpose_codes(word, lane);
                uint4 v = make_uint4(weights2<0>(word, z[0], s[0]), weights2<1>(word, z[1], s[1]),
                                     weights2<2>(word, z[2], s[2]), weights2<3>(word, z[3], s[3]));
                const uint32_t k0 = kb * 128u + f * 16u;
                if (k0 / 32u >= kt) continue;
                // Zeros past K and N.
                const uint32_t r = TRANSPOSE ? n16 * 16u + lane / 2u : k0 + lane / 2u;
                const uint32_t c = (TRANSPOSE ? k0 : n16 * 16u) + lane % 2u * 8u;
                const uint32_t rows = TRANSPOSE ? w.N : w.K, cols = TRANSPOSE ? w.K : w.N;
                if (r >= rows || c >= cols) {
                    v = make_uint4(0, 0, 0, 0);
                } else if (c + 8u > cols) {
                    const uint32_t n = cols - c;  // values of this lane that count, 1 to 7
                    v.x = n > 1u ? v.x : v.x & 0xffffu;
                    v.y = n > 3u ? v.y : n > 2u ? v.y & 0xffffu : 0u;
                    v.z = n > 5u ? v.z : n > 4u ? v.z & 0xffffu : 0u;
                    v.w = n > 6u ? v.w & 0xffffu : 0u;
                }
                const uint64_t face = TRANSPOSE ? ((uint64_t)(n16 / 2u) * ct + k0 / 32u) * 1024u +
                                                      ((n16 % 2u) * 2u + k0 / 16u % 2u) * 256u
                                                : face_offset(kb, f, n16, ct);
                __stcs(reinterpret_cast<uint4*>(tiles + face) + lane, v);
            }
        }
    }
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
//  * mma.m16n8k16 with the weights as the 16-row operand.  bf16 bits 0 to 255
//    (subnormal numbers and the first binade) stand for 0 to 255 times 2^-133,
//    so a code needs no conversion: five integer operations make the operands
//    of a word's eight codes, four masks and one shift, every second pair 16
//    times too large.  x is the other operand, one 16-byte shared-memory read
//    for two MMAs, in bf16 times 2^100, and 2^96 against the pairs that are too
//    large: exact, and the products, q x 2^-33, are ordinary fp32 numbers.
//    Rows of x whose largest value is not between 2^-69 and 2^21 get a power of
//    two of their own.  (With 16 + q made in bf16 by a shift and a logical
//    operation for two codes, eight operations a word, the integer pipe was the
//    limit: 11.5 us for 16384 x 4096, one row.)
//  * The accumulators start from minus z sum(x), made once for each group when
//    x is staged, and end as sum((q - z) x); the group's scale follows in fp32.
//    Nothing is rounded to fewer than 32 bits before the output.
//  * K is split over the CTAs of a cluster (S) where x would not fit one SM's
//    shared memory, and over the warps of a CTA (WK) where there are few
//    columns; the parts are added in a fixed order through (distributed)
//    shared memory.  Clusters take contiguous, near-equal runs of tiles: the
//    grid is one CTA per SM, whatever N is.
constexpr int kMvWarps = 16, kMvLog = 4;
constexpr int kMvThreads = 32 * kMvWarps;
// Blocks of each of a warp's tiles that are on their way.
__host__ __device__ constexpr int mv_ahead(int rt) { return rt == 2 ? 3 : 4; }
constexpr uint32_t kMaxSmem = 232448;

struct Matvec {
    const uint16_t* x;
    const uint8_t* packed;
    const uint16_t* bias;
    uint16_t* y;
    uint64_t ld_x, ld_y;
    uint32_t M, K, N, kb, tiles;
    uint32_t nt, rt;                               // rows of x / 8 and tiles that a warp takes at a time
    uint32_t S, WK, clusters, pass_runs;           // split (host)
    uint32_t S_log, WK_log;                        // both are powers of two
    uint32_t kb_each, kb_more, tiles_each, tiles_more;  // shares of a CTA / cluster, and how many have one more
    uint32_t x_pitch, off_sum, off_red, off_ring;  // shared-memory plan (host)
    uint32_t relu, x_vec, x_log;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes number I and I + 4 of a word in place: q (even I) or 16 q (odd I).
template <int I>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
    return (I < 2 ? w : w >> 8) & (I % 2 ? 0x00f000f0u : 0x000f000fu);
}
__device__ __forceinline__ void st_cluster_f4(uint32_t addr, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
                 : "memory");
}

// 16 bytes at an address that is a multiple of 2, out of the two aligned vectors
// that hold them.  Up to 14 bytes before and after them are read too.
__device__ __forceinline__ uint4 load_any(const uint16_t* p) {
    const uint32_t off = (uint32_t)((uintptr_t)p & 15u);
    const uint4* at = reinterpret_cast<const uint4*>((uintptr_t)p - off);
    const uint4 a = at[0], b = off ? at[1] : make_uint4(0, 0, 0, 0);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = off & 8u ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = off & 4u ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], off & 2u ? 16u : 0u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row's powers of two: x is multiplied by up1 up2, its sums by down1 down2
// (2^133 over the former); two factors each, as their product may not be a
// number.
struct RowScale {
    float up1, up2, down1, down2;
};
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// For a row whose largest exponent field is `field`: the largest value to 2^120.
__device__ __forceinline__ RowScale row_scale(uint32_t field) {
    const int up = 120 - max((int)field - 127, -126), down = 133 - up;  // -8 .. 246, -113 .. 141
    const int u = min(up, 120), d = min(down, 120);
    return RowScale{power(u), power(up - u), power(d), power(down - d)};
}
constexpr int kScale = 100;                                          // of ordinary rows
constexpr uint32_t kTopLow = 127 - 69, kTopHigh = 127 + 20;          // exponent fields of their largest values

// The x rows of this CTA's blocks into shared memory (zeros past M and K) and
// the sum of each group of each row, times -8 where there are no zero points,
// in the units of the products (2^100 x 2^-133 = 2^-33).  OWN: scaled by each row's own powers, else by
// 2^kScale, and the largest exponent field of each row is noted in `top`.
template <int NT, int GROUP, bool ZEROS, bool OWN>
__device__ __forceinline__ void stage_x(const Matvec& p, uint8_t* smem, uint32_t m0, uint32_t kb0, uint32_t nkb,
                                        uint32_t* top, const RowScale* own) {
    float* sums = reinterpret_cast<float*>(smem + p.off_sum);
    const uint32_t rows = min(p.M - m0, 8u * NT), per_row = nkb * 16u;  // 16-byte pieces
    for (uint32_t i = rows * p.x_pitch + threadIdx.x * 16u; i < 8u * NT * p.x_pitch; i += kMvThreads * 16u)
        *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
    // 2^x_log threads (16 and more) side by side on a row, kMvThreads / 2^x_log
    // rows at a time; eight pieces of a thread on their way.
    const uint32_t side = 1u << p.x_log, c0 = threadIdx.x & (side - 1u), r0 = threadIdx.x >> p.x_log;
    const uint32_t row_step = kMvThreads >> p.x_log, along = (per_row + side - 1u) >> p.x_log;
    const uint32_t steps = (rows + row_step - 1u) / row_step * along;
    constexpr uint32_t kBatch = 8;
    uint32_t row = r0, c = c0;
    for (uint32_t i0 = 0; i0 < steps; i0 += kBatch) {
        uint4 v[kBatch];
        uint32_t rows_of[kBatch], cs[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            v[b] = make_uint4(0, 0, 0, 0);
            const bool in = i0 + b < steps && row < rows && c < per_row;
            rows_of[b] = in ? row : ~0u, cs[b] = c;
            const uint32_t k = kb0 * kBlockK + c * 8u;
            if (in && k < p.K) {
                const uint16_t* src = p.x + (m0 + row) * p.ld_x + k;
                if (p.x_vec && k + 8u <= p.K) {
                    v[b] = *reinterpret_cast<const uint4*>(src);
                } else if (!p.x_vec && k >= 8u && k + 16u <= p.K) {
                    v[b] = load_any(src);
                } else {
                    uint32_t e[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) e[j] = k + j < p.K ? src[j] : 0u;
                    v[b] = make_uint4(pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]),
                                      pack_bf16x2(e[6], e[7]));
                }
            }
            c += side;
            if (c >= along << p.x_log) c = c0, row += row_step;
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            if (i0 + b >= steps) break;  // every thread
            const bool in = rows_of[b] != ~0u;
            float s = 0.0f;
            uint32_t h[4];
            if constexpr (OWN) {
                const float up1 = in ? own[rows_of[b]].up1 : 1.0f, up2 = in ? own[rows_of[b]].up2 : 1.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = word_of(v[b], j);
                    float lo = bf16_bits_to_f32(w & 0xffffu) * up1 * up2;
                    float hi = __uint_as_float(w & 0xffff0000u) * up1 * up2;
                    s += lo + hi;
                    if (j % 2) lo *= 0.0625f, hi *= 0.0625f;
                    h[j] = cvt_bf16x2(lo, hi);
                }
                s *= power(-100);  // 2^-133 in two steps, with what follows
            } else {
                uint32_t most = 0;
                float2 sum = both(0.0f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = word_of(v[b], j);
                    // 2^100 or 2^96 times the pair, exact.
                    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(h[j]) : "r"(w), "r"(j % 2 ? 0x6f806f80u : 0x71807180u));
                    sum = add2(sum, make_float2(bf16_bits_to_f32(w & 0xffffu), __uint_as_float(w & 0xffff0000u)));
                    most = __vmaxu2(most, w & 0x7f807f80u);
                }
                s = sum.x + sum.y;
                most = max(most & 0xffffu, most >> 16);
                if (p.x_log >= 5u) {  // a warp on one row
                    most = __reduce_max_sync(0xffffffffu, most);
                    if ((threadIdx.x & 31u) == 0u && in) atomicMax(&top[rows_of[b]], most >> 7);
                } else {
                    if (in) atomicMax(&top[rows_of[b]], most >> 7);
                }
            }
#pragma unroll
            for (int o = 1; o < GROUP / 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (in) {
                *reinterpret_cast<uint4*>(smem + rows_of[b] * p.x_pitch + cs[b] * 16u) =
                    make_uint4(h[0], h[1], h[2], h[3]);
                if (cs[b] % (GROUP / 8) == 0)
                    sums[cs[b] / (GROUP / 8) * (8u * NT) + rows_of[b]] = (ZEROS ? power(-33) : -8.0f * power(-33)) * s;
            }
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

// -z for a zero point z.
__device__ __forceinline__ float minus(uint32_t z) { return 8388608.0f - __uint_as_float(0x4b000000u | (z & 15u)); }

template <int NT, int RT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kMvThreads, 1) matvec_kernel(const __grid_constant__ Matvec p) {
    constexpr uint32_t kBytes = block_bytes(GROUP, ZEROS);
    constexpr int kGroups = 128 / GROUP;  // groups of a block
    constexpr int kAhead = mv_ahead(RT);
    constexpr uint32_t kSlot = RT * kBytes, kPlace = 512 * RT * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t top[8 * NT];
    __shared__ RowScale own[8 * NT];
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u, g = lane / 4u, t = lane % 4u;
    const uint32_t rank = blockIdx.x & (p.S - 1u), cluster = blockIdx.x >> p.S_log;
    const uint32_t m0 = blockIdx.y * 8u * NT;
    // This CTA's blocks of k and its cluster's tiles, in runs of RT.
    const uint32_t kb0 = rank * p.kb_each + min(rank, p.kb_more), nkb = p.kb_each + (rank < p.kb_more ? 1u : 0u);
    const uint32_t t0 = cluster * p.tiles_each + min(cluster, p.tiles_more);
    const uint32_t t1 = t0 + p.tiles_each + (cluster < p.tiles_more ? 1u : 0u);
    const uint32_t runs = (t1 - t0 + RT - 1) / RT;
    // This warp's share: runs wn, wn + WN, ... and blocks [b0, b0 + nb) of kb0 ...
    const uint32_t WN = kMvWarps >> p.WK_log, wn = warp >> p.WK_log, wk = warp & (p.WK - 1u);
    const uint32_t b0 = nkb * wk >> p.WK_log, nb = (nkb * (wk + 1) >> p.WK_log) - b0;
    const bool joined = p.S * p.WK > 1;
    const uint64_t tile_bytes = (uint64_t)p.kb * kBytes;

    uint8_t* const ring = smem + p.off_ring + warp * (kAhead * kSlot);
    uint8_t* const ring_end = ring + kAhead * kSlot;
    if (threadIdx.x < 8u * NT) top[threadIdx.x] = 0u;
    __syncthreads();
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();

    // The warp's blocks in order, one commit group for a block of each tile of
    // the run (empty past the end).
    const uint32_t my_runs = nb && wn < runs ? (runs - wn + WN - 1) >> (kMvLog - p.WK_log) : 0u;
    uint32_t left = my_runs * nb, in_run = nb, is_tile = t0 + RT * wn;
    const uint8_t* src = p.packed + (uint64_t)is_tile * tile_bytes + (uint64_t)(kb0 + b0) * kBytes + lane * 16u;
    auto issue = [&](uint8_t* slot) {
        if (left) {
            const uint32_t dst = smem_u32(slot) + lane * 16u;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                // Past the cluster's last tile: the one before once more, not used.
                const uint8_t* s = r && is_tile + r < t1 ? src + r * tile_bytes : src;
                cp_async16(dst + r * kBytes, s, 16);
                cp_async16(dst + r * kBytes + 512u, s + 512, 16);
                if (lane < (kBytes - kCodeBytes) / 16u)
                    cp_async16(dst + r * kBytes + kCodeBytes, s + kCodeBytes, 16);
            }
            src += kBytes;
            --left;
            if (--in_run == 0) in_run = nb, is_tile += RT * WN, src += RT * WN * tile_bytes - (uint64_t)nb * kBytes;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) issue(ring + i * kSlot);

    stage_x<NT, GROUP, ZEROS, false>(p, smem, m0, kb0, nkb, top, own);
    __syncthreads();
    const uint32_t most = lane < 8u * NT ? top[lane] : 0u;
    const bool unusual = __any_sync(0xffffffffu, most > kTopHigh || (most != 0u && most < kTopLow));
    if (unusual) {
        if (threadIdx.x < 8u * NT) own[threadIdx.x] = row_scale(top[threadIdx.x]);
        __syncthreads();
        stage_x<NT, GROUP, ZEROS, true>(p, smem, m0, kb0, nkb, top, own);
        __syncthreads();
    }
    if (p.S > 1) cluster_sync();  // every CTA of the cluster runs before its memory is written

    const uint32_t x_rows = 8u * p.x_pitch;
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
                        // Start from minus z times the group's sum of x.
                        float z0 = 1.0f, z1 = 1.0f;
                        if constexpr (ZEROS) {
                            const uint8_t* zp = slot + r * kBytes + kCodeBytes + 32 * kGroups + gi * 16;
                            z0 = minus(zp[g]), z1 = minus(zp[g + 8]);
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
                            xv[n] = *reinterpret_cast<const uint4*>(xb + n * x_rows + q * 64u);
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            const uint32_t a = word_of(wa[r], q), c = word_of(wb[r], q);
                            const uint32_t a0 = codes<0>(a), a1 = codes<1>(a), a2 = codes<2>(a), a3 = codes<3>(a);
                            const uint32_t c0 = codes<0>(c), c1 = codes<1>(c), c2 = codes<2>(c), c3 = codes<3>(c);
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
            // Out of the products' units.
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                RowScale d0{0.0f, 0.0f, power(133 - kScale), 1.0f}, d1 = d0;
                if (unusual) d0 = own[8 * n + 2 * t], d1 = own[8 * n + 2 * t + 1];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    acc[r][n][0] *= d0.down1, acc[r][n][2] *= d0.down1;
                    acc[r][n][1] *= d1.down1, acc[r][n][3] *= d1.down1;
                    if (unusual) {
                        acc[r][n][0] *= d0.down2, acc[r][n][2] *= d0.down2;
                        acc[r][n][1] *= d1.down2, acc[r][n][3] *= d1.down2;
                    }
                }
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
template <int NT, int RT>
MatvecKernel pick_matvec(const Weights& w) {
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

// One warp a block, 8 a CTA, at most `most` CTAs an SM.
template <class K, class... Args>
static cudaError_t launch_blocks(K kernel, uint64_t blocks, cudaStream_t s, Args... args) {
    const uint64_t ctas = (blocks + 7) / 8, most = (uint64_t)foil_sm_count() * 8;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(ctas < most ? ctas : most), 1, 1), cfg.blockDim = dim3(256, 1, 1), cfg.stream = s;
    cudaLaunchAttribute la[1]{};
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = la, cfg.numAttrs = 1;
    return count(cudaLaunchKernelEx(&cfg, kernel, args..., blocks));
}

template <int GROUP, bool ZEROS>
static cudaError_t quantize_typed(const uint16_t* tiles, uint8_t* packed, const Weights& w, cudaStream_t s) {
    const uint64_t blocks = (uint64_t)padded_n(w) / 16 * blocks_k(w);
    return launch_blocks(quantize_kernel<GROUP, ZEROS>, blocks, s, tiles, packed, w, blocks_k(w));
}

cudaError_t quantize_tiles(const uint16_t* tiles, uint8_t* packed, const Weights& w, cudaStream_t s) {
    if (w.group == 32)
        return w.zeros ? quantize_typed<32, true>(tiles, packed, w, s) : quantize_typed<32, false>(tiles, packed, w, s);
    if (w.group == 64)
        return w.zeros ? quantize_typed<64, true>(tiles, packed, w, s) : quantize_typed<64, false>(tiles, packed, w, s);
    return w.zeros ? quantize_typed<128, true>(tiles, packed, w, s) : quantize_typed<128, false>(tiles, packed, w, s);
}

template <int GROUP, bool ZEROS>
static cudaError_t dequantize_typed(const uint8_t* packed, uint16_t* tiles, const Weights& w, bool transpose,
                                    cudaStream_t s) {
    const uint64_t blocks = (uint64_t)((w.N + 31) / 32) * 2 * blocks_k(w);
    return transpose
               ? launch_blocks(dequantize_kernel<GROUP, ZEROS, true>, blocks, s, packed, tiles, w, blocks_k(w))
               : launch_blocks(dequantize_kernel<GROUP, ZEROS, false>, blocks, s, packed, tiles, w, blocks_k(w));
}

cudaError_t dequantize_tiles(const uint8_t* packed, uint16_t* tiles, const Weights& w, bool transpose, cudaStream_t s) {
    if (w.group == 32)
        return w.zeros ? dequantize_typed<32, true>(packed, tiles, w, transpose, s)
                       : dequantize_typed<32, false>(packed, tiles, w, transpose, s);
    if (w.group == 64)
        return w.zeros ? dequantize_typed<64, true>(packed, tiles, w, transpose, s)
                       : dequantize_typed<64, false>(packed, tiles, w, transpose, s);
    return w.zeros ? dequantize_typed<128, true>(packed, tiles, w, transpose, s)
                   : dequantize_typed<128, false>(packed, tiles, w, transpose, s);
}

// The rows of x (8 nt) and the tiles (rt) that a warp takes at a time, the
// split of K over the CTAs of a cluster (S) and the warps of a CTA (WK): the
// plan of least estimated time, where the slice of x fits.  The terms, in ns,
// are fitted to what 1 to 16 rows measured over all plans at 2048 x 2048 to
// 65536 x 4096 (the plan taken is within 5 % of the best there):
//  staging: 10 a row and block of k (30 if rows are not aligned), so that more
//  rows want a larger S;
//  the warps' steps: 25 to 37 a block for each warp at work, 160 at least;
//  250 for each run of tiles of a warp, 400 for a join in a CTA, 1000 in a
//  cluster and 6 for each part;
//  HBM: 43 bytes an SM, with fewer SMs at work for larger clusters, and less
//  with fewer than 48,000 bytes on their way to an SM.
static bool plan_matvec(Matvec& p, uint32_t bytes, uint32_t group, uint32_t sms) {
    float best = 0.0f;
    for (uint32_t kind = 0; kind < 4; ++kind) {
        const uint32_t nt = 1 + kind / 2, rt = 1 + kind % 2, width = 8 * nt;
        if ((nt == 2) != (p.M > 8) && best > 0.0f) continue;  // 8 rows at a time only where 16 do not fit
        const uint32_t rows = p.M < width ? p.M : width, groups_of_rows = (p.M + width - 1) / width;
        const float block = (nt == 2 ? (rt == 2 ? 33.0f : 37.0f) : (rt == 2 ? 25.0f : 26.0f)) * (group == 32 ? 1.3f : 1.0f);
        const uint32_t ring = kMvWarps * mv_ahead((int)rt) * rt * bytes;
        for (uint32_t S = 1; S <= 8 && S <= p.kb; S *= 2) {
            const uint32_t ks = (p.kb + S - 1) / S;
            const uint32_t pitch = ks * 256 + 64;  // 64 bytes more: rows of an 8-lane read phase on distinct banks
            const uint32_t off_sum = width * pitch, sums = ks * (128 / group) * width * 4;
            const uint32_t off_red = (off_sum + sums + 127) / 128 * 128;
            const uint32_t fit = S == 1 ? sms : foil_resident_clusters(S), clusters = fit < p.tiles ? fit : p.tiles;
            const uint32_t tc = ((p.tiles + clusters - 1) / clusters + rt - 1) / rt;  // runs of rt tiles
            const float staging = 300.0f + (float)(rows * ks) * (p.x_vec ? 10.0f : 30.0f);
            const float hbm = (float)p.tiles * p.kb * bytes / (43.0f * clusters * S);
            for (uint32_t wk = 1; wk <= kMvWarps && wk <= ks; wk *= 2) {
                const uint32_t wn = kMvWarps / wk, rounds = (tc + wn - 1) / wn, rest = tc % wn * wk;
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
                const float last = rest == 0 ? 0.0f : block * rest > 160.0f ? block * rest : 160.0f;
                const float steps = (float)((ks + wk - 1) / wk * rt) * (tc / wn * block * kMvWarps + last);
                const float join = (float)passes * (S > 1 ? 1000.0f : wk > 1 ? 400.0f : 0.0f) + 6.0f * tc * wk * rt * nt;
                const uint32_t busy = tc < wn ? tc * wk : kMvWarps;
                const float ahead = (float)busy * mv_ahead((int)rt) * rt * bytes;
                const float read = ahead < 48000.0f ? hbm * (48000.0f / ahead) : hbm;
                const float cost = (staging + (steps > read ? steps : read) + 250.0f * rounds + join) * groups_of_rows;
                if (best > 0.0f && cost >= best && p.nt == nt) continue;
                best = cost;
                p.nt = nt, p.rt = rt, p.S = S, p.WK = wk, p.clusters = clusters;
                p.x_pitch = pitch, p.off_sum = off_sum, p.off_red = off_red;
                p.off_ring = (off_red + red + 127) / 128 * 128;
                p.pass_runs = pass < tc ? pass : (tc + wn - 1) / wn * wn;
            }
        }
    }
    return best > 0.0f;
}

cudaError_t matvec(const uint16_t* x, uint64_t ld_x, const uint8_t* packed, const uint16_t* bias, uint16_t* y,
                   uint64_t ld_y, uint32_t M, const Weights& w, bool relu, uint32_t* err, cudaStream_t s) {
    // More rows than two of the warps' MMAs take: on tcgen05, which reads x in
    // 16-byte pieces (32 rows of 4096 x 4096: 15 us in two passes here, 9 there).
    if (M > kWarpRows && (uintptr_t)x % 16 == 0 && ld_x % 8 == 0)
        return matvec_batch(x, ld_x, packed, bias, y, ld_y, M, w, relu, err, s);
    Matvec p{};
    p.x = x, p.packed = packed, p.bias = bias, p.y = y, p.ld_x = ld_x, p.ld_y = ld_y, p.M = M, p.K = w.K, p.N = w.N;
    p.kb = blocks_k(w), p.tiles = (w.N + 15) / 16, p.relu = relu ? 1 : 0;
    p.x_vec = (uintptr_t)x % 16 == 0 && ld_x % 8 == 0;
    const uint32_t bytes = block_bytes(w.group, w.zeros), sms = (uint32_t)foil_sm_count();
    // The plan depends on the sizes alone; each thread keeps its latest ones
    // (making one takes as long as a launch).
    struct Known {
        uint32_t key[7];
        Matvec plan;
    };
    static thread_local Known known[16];
    const uint32_t key[7] = {M, w.K, w.N, w.group, w.zeros + 2 * p.x_vec, sms, 1};
    Known& k = known[(M + w.K / 32 + w.N / 16 * 5 + w.group / 32) % 16];
    if (memcmp(k.key, key, sizeof key) != 0) {
        k.key[6] = 0;
        k.plan = p;
        if (!plan_matvec(k.plan, bytes, w.group, sms)) return cudaErrorInvalidConfiguration;
        memcpy(k.key, key, sizeof key);
    }
    p = k.plan;
    p.x = x, p.packed = packed, p.bias = bias, p.y = y, p.ld_x = ld_x, p.ld_y = ld_y, p.relu = relu ? 1 : 0;
    while (1u << p.S_log < p.S) ++p.S_log;
    while (1u << p.WK_log < p.WK) ++p.WK_log;
    p.kb_each = p.kb / p.S, p.kb_more = p.kb % p.S;
    p.tiles_each = p.tiles / p.clusters, p.tiles_more = p.tiles % p.clusters;
    for (p.x_log = 4; p.x_log < 9 && (1u << p.x_log) < (p.kb + p.S - 1) / p.S * 16; ++p.x_log) {
    }
    const uint32_t smem = p.off_ring + kMvWarps * mv_ahead((int)p.rt) * p.rt * bytes;
    const MatvecKernel kernel = p.nt == 2 ? (p.rt == 2 ? pick_matvec<2, 2>(w) : pick_matvec<2, 1>(w))
                                          : (p.rt == 2 ? pick_matvec<1, 2>(w) : pick_matvec<1, 1>(w));
    const cudaError_t e = foil_smem_optin(reinterpret_cast<const void*>(kernel), (int)kMaxSmem - 512);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.clusters * p.S, (M + 8 * p.nt - 1) / (8 * p.nt), 1);
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
