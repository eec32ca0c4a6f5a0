// 4-bit weights with group scales: storage, conversion from and to tile
// streams, and products with a few rows.  The storage format is described at
// foil_w4_pack_dev in include/foil_c.h.
#include "w4.cuh"

#include "common.cuh"

namespace foil {
namespace w4 {
namespace {

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

// One warp for each column n and row m.
__global__ void matvec_kernel(const uint16_t* __restrict__ x, uint64_t ld_x, const uint8_t* __restrict__ packed,
                              const uint16_t* __restrict__ bias, uint16_t* __restrict__ y, uint64_t ld_y, uint32_t M,
                              Weights w, uint32_t kb, uint32_t relu) {
    const uint32_t n = blockIdx.x * (blockDim.x / 32u) + threadIdx.x / 32u, m = blockIdx.y, lane = threadIdx.x % 32u;
    if (n >= w.N) return;
    float acc = 0.0f;
    const uint32_t bytes = block_bytes(w.group, w.zeros);
    for (uint32_t k = lane; k < w.K; k += 32)
        acc += bf16_bits_to_f32(x[m * ld_x + k]) * weight(packed, n, k, w, kb, bytes);
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) {
        if (bias) acc += bf16_bits_to_f32(bias[n]);
        if (relu && acc < 0.0f) acc = 0.0f;
        y[m * ld_y + n] = (uint16_t)(cvt_bf16x2(acc, 0.0f) & 0xffffu);
    }
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

cudaError_t matvec(const uint16_t* x, uint64_t ld_x, const uint8_t* packed, const uint16_t* bias, uint16_t* y,
                   uint64_t ld_y, uint32_t M, const Weights& w, bool relu, uint32_t* err, cudaStream_t s) {
    (void)err;
    matvec_kernel<<<dim3((w.N + 7) / 8, M), 256, 0, s>>>(x, ld_x, packed, bias, y, ld_y, M, w, blocks_k(w),
                                                         relu ? 1u : 0u);
    return count(cudaGetLastError());
}

}  // namespace w4
}  // namespace foil
