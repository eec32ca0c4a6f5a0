// Launchers of the embedding row kernels (embed_rows.cu).  Arguments are
// checked by the caller; each returns a cudaError_t.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace foil {
namespace embed {

constexpr uint32_t kMaxRows = 1u << 24;  // T and V
constexpr uint32_t kMaxD = 1u << 20;     // columns are counted in 32 bits, 16 Ki at a time

struct Lookup {
    const void* ids;
    const uint16_t* table;
    void* out;
    uint64_t ld_table, ld_out;
    uint32_t T, V, D;
    int32_t id_bytes;
    float scale;
    int64_t pad_id;
    uint32_t* err;
};

struct Gradient {
    const void* ids;
    const void* dout;
    float* dtable;
    void* ws;
    uint64_t ld_dout, ld_dtable;
    uint32_t T, V, D;
    int32_t id_bytes;
    float scale;
    int64_t pad_id;
    uint32_t accumulate;
    uint32_t* err;
};

uint64_t gradient_ws_bytes(uint32_t T, uint32_t V, uint32_t D);
cudaError_t lookup(const Lookup& p, bool fp32, cudaStream_t s);
cudaError_t gradient(const Gradient& p, bool fp32, cudaStream_t s);

}  // namespace embed
}  // namespace foil
