// Launchers of the 4-bit weight kernels (w4.cu).  Arguments are checked by
// the caller; each returns a cudaError_t.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace foil {
namespace w4 {

constexpr uint32_t kBlockN = 16;         // columns of a storage block
constexpr uint32_t kBlockK = 128;        // k of a storage block
constexpr uint32_t kCodeBytes = 1024;    // codes of a block
constexpr uint32_t kMaxRows = 64;        // rows of one matvec call
constexpr uint32_t kWarpRows = 16;       // rows the warps' MMAs take in one pass
constexpr uint32_t kMaxK = 32768;        // K of one matvec call

struct Weights {
    uint32_t K, N, group;
    uint32_t zeros;  // 1: the storage has zero points
};

__host__ __device__ constexpr uint32_t block_bytes(uint32_t group, uint32_t zeros) {
    return kCodeBytes + kBlockK / group * kBlockN * (zeros ? 3u : 2u);
}
inline uint64_t packed_bytes(const Weights& w) {
    return (uint64_t)((w.N + kBlockN - 1) / kBlockN) * ((w.K + kBlockK - 1) / kBlockK) *
           block_bytes(w.group, w.zeros);
}

cudaError_t pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zero_points, uint8_t* packed,
                 const Weights& w, cudaStream_t s);
cudaError_t quantize_tiles(const uint16_t* tiles, uint8_t* packed, const Weights& w, cudaStream_t s);
cudaError_t dequantize_tiles(const uint8_t* packed, uint16_t* tiles, const Weights& w, bool transpose,
                             cudaStream_t s);
cudaError_t matvec(const uint16_t* x, uint64_t ld_x, const uint8_t* packed, const uint16_t* bias, uint16_t* y,
                   uint64_t ld_y, uint32_t M, const Weights& w, bool relu, uint32_t* err, cudaStream_t s);
// The same on tcgen05 (w4_batch.cu): x 16-byte aligned, ld_x a multiple of 8.
cudaError_t matvec_batch(const uint16_t* x, uint64_t ld_x, const uint8_t* packed, const uint16_t* bias, uint16_t* y,
                         uint64_t ld_y, uint32_t M, const Weights& w, bool relu, uint32_t* err, cudaStream_t s);

}  // namespace w4
}  // namespace foil
