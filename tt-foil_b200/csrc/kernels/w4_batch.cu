// y = x W of 4-bit weights for batches of rows: the product that w4.cu makes on
// the warps' MMA pipe, on tcgen05.
//
// That pipe does an m16n8k16 in about 4 cycles of an SM, so from 16 rows on it
// bounds the kernel of w4.cu (64 rows of 8192 x 24576: 118 us; reading the
// weights takes 16).  Here a CTA takes 128 columns and a share of K:
//
//  * Eight warps read the storage blocks of 16 columns each through rings of
//    their own (16-byte asynchronous copies) and write (q - z) 2^-11, exact in
//    bf16, to shared memory as the MMA's operand of 128 rows: K-major in the
//    128-byte swizzle, 128 k a stage, or 64 where 64 rows leave no room for more
//    (32 rows of 8192 x 24576: 61 us with 64, 56 with 128).  A word of a storage
//    block is 8 consecutive k of a column, one 16-byte piece of that layout.  12
//    operations a word: shift, mask and 16 + q, minus 16 + z.
//  * x comes by tensor copies, zeros past M and K, as the operand of 32, 48 or
//    64 columns.
//  * One thread issues tcgen05.mma 128 x MT x 16.  Each group of k has an
//    accumulator of its own in TMEM (four in turn), which the eight warps read
//    back, multiply by the group's scales in fp32 and add to their registers: a
//    thread holds a column n and half of the rows.  No rounding but the last.
//  * K is split over a cluster's CTAs; each adds the parts of its columns in
//    order.  Two CTAs share an SM, so one's start and join overlap the other's
//    products.
//
// 64 rows, us (the warps' MMAs): 4096 x 4096 11 (29), 16384 x 4096 26 (67),
// 8192 x 24576 68 (117), 8192 x 65536 143 (280); 48 rows: 9.5 (22), 22 (51), 59 (88); 32
// rows: 9 (15), 19 (34), 56 (60).
// Bound by the instructions of the conversion (some 350 a storage block, of which
// 130 make the operand and 40 add its products) and by shared memory, where a
// block's 1 KB of codes is written and read as 4 KB.  Tried, for 64 rows of 8192 x
// 24576 at a time when this took 85: the weights' operand in TMEM instead, x by
// 4-byte copies in the order of the weights' fragments: 87 to 99; one CTA of 16
// warps and 256 columns: 84, but 17 against 14 for 4096 x 4096.
#include "w4.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "gemm_ptx.cuh"

namespace foil {
namespace w4 {
namespace {

using namespace gemm;

constexpr uint32_t kColumns = 128;   // of W a CTA takes: the MMA's rows
constexpr uint32_t kWorkers = 8, kMmaWarp = 8, kCopyWarp = 9, kThreads = 320;
// Halves of 64 k in a stage, stages, storage blocks of a warp on their way: what
// two CTAs of an SM have room for.
__host__ __device__ constexpr uint32_t halves(uint32_t mt) { return mt == 64 ? 1 : 2; }
__host__ __device__ constexpr uint32_t stages(uint32_t mt) { return mt == 64 ? 3 : 2; }
__host__ __device__ constexpr uint32_t ring(uint32_t mt) { return mt == 64 ? 3 : 2; }
constexpr uint32_t kUnits = 4;       // accumulators
constexpr uint32_t kScaleSlots = 4;  // blocks whose scales are kept: warps are at most three blocks apart
constexpr uint32_t kWHalf = kColumns * 128;

struct Batch {
    const uint8_t* packed;
    const uint16_t* bias;
    uint16_t* y;
    uint32_t* err;
    uint64_t ld_y, wait_ns;
    uint32_t M, N, kb, tiles, relu;   // blocks of k, tiles of 16 columns
    uint32_t S, kb_each, kb_more;     // CTAs of a cluster, blocks of each, how many have one more
};

__host__ __device__ constexpr uint32_t stage_bytes(uint32_t mt) { return halves(mt) * (kWHalf + mt * 128u); }
constexpr uint32_t smem_bytes(uint32_t mt, uint32_t group, uint32_t zeros) {
    return 1024u + stages(mt) * stage_bytes(mt) + kWorkers * ring(mt) * block_bytes(group, zeros) +
           kScaleSlots * (128u / group) * kColumns * 2u;
}

// Instruction descriptor: fp32 accumulators, bf16 operands, both K-major.
__host__ __device__ constexpr uint32_t instruction(uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// N (8 or 16) consecutive values of this thread's row.
template <int N>
__device__ __forceinline__ void tmem_values(uint32_t at, float* v) {
    uint32_t r[16];
    if constexpr (N == 16)
        tmem_ld16(at, r);
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(at));
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared memory by its own addresses (from generic ones: more instructions).
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t ld_shared_u8(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

// True in one lane of a converged warp, always the same.
__device__ __forceinline__ bool elect() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ uint32_t word(const uint4& v, uint32_t i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Codes number I and I + 4 of a word minus the zero point, times 2^-11, as bf16:
// (16 + q) 2^-11 by a mask, minus (16 + z) 2^-11, both exact.  Sums of a group stay
// below 128 x 15 x 2^-11 < 1 times its largest x, so no finite x overflows them;
// the 2^11 is put back at the end.
constexpr uint32_t kSixteen = 0x3c003c00u;  // twice 16 x 2^-11, whose steps of one are bits 3 to 6
constexpr float kUnit = 2048.0f;
template <int I>
__device__ __forceinline__ uint32_t difference(uint32_t w, uint32_t z16) {
    const uint32_t v = I == 0 ? w << 3 : w >> (4 * I - 3);
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\t"
        "lop3.b32 t, %1, 0x00780078, %2, 0xea;\n\t"
        "sub.rn.bf16x2 %0, t, %3;\n\t}"
        : "=r"(r)
        : "r"(v), "r"(kSixteen), "r"(z16));
    return r;
}

template <int MT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kThreads, 2)
    batch_kernel(const Batch p, const __grid_constant__ CUtensorMap map_x) {
    constexpr uint32_t kBytes = block_bytes(GROUP, ZEROS), kGroups = 128 / GROUP;
    constexpr uint32_t kStages = stages(MT), kRing = ring(MT), kHalves = halves(MT);
    constexpr uint32_t kStageBytes = stage_bytes(MT), kWBytes = kHalves * kWHalf;
    constexpr uint32_t kTmem = MT == 32 ? 128 : 256;  // columns, a power of two
    constexpr int kAcc = MT / 2;  // rows of x a thread holds
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kStages], x_full[kStages], empty[kStages], d_full[kUnits], d_empty[kUnits], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;
    uint8_t* const smem =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem), rings = base + kStages * kStageBytes;
    const uint32_t scales = rings + kWorkers * kRing * kBytes;
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
    const uint32_t rank = blockIdx.x % p.S, n0 = blockIdx.x / p.S * kColumns, m0 = blockIdx.y * MT;
    const uint32_t kb0 = rank * p.kb_each + min(rank, p.kb_more), nkb = p.kb_each + (rank < p.kb_more ? 1u : 0u);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], kWorkers);
            mbar_init(&x_full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t u = 0; u < kUnits; ++u) {
            mbar_init(&d_full[u], 1);
            mbar_init(&d_empty[u], kWorkers);
        }
        mbar_init(&drain, 1);
        abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    griddep_wait();  // launched with programmatic stream serialization
    griddep_launch_dependents();

    float acc[kAcc];
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i] = 0.0f;
    // Workers: the thread's column of the CTA's, its first row of x.
    const uint32_t column = warp % 4u * 32u + lane, row0 = warp / 4u * kAcc;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        // Most waits are short: without the clock and its instructions at first.
        if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
            if (mbar_try_wait_sleep(bar, parity)) return true;
        return mbar_wait(bar, parity, &abort_flag, p.err, p.wait_ns);
    };

    if (warp < kWorkers) {
        const uint32_t g = lane / 4u, t = lane % 4u;
        const uint32_t slots = rings + warp * kRing * kBytes;
        // Past the last tile: that one once more, not stored.
        const uint32_t tile = min(n0 / kBlockN + warp, p.tiles - 1u);
        const uint8_t* src = p.packed + ((uint64_t)tile * p.kb + kb0) * kBytes + lane * 16u;
        uint32_t left = nkb;
        auto issue = [&](uint32_t slot) {
            if (left) {
                const uint32_t dst = slot + lane * 16u;
                cp_async16(dst, src, 16);
                cp_async16(dst + 512u, src + 512, 16);
                if (lane < (kBytes - kCodeBytes) / 16u) cp_async16(dst + kCodeBytes, src + kCodeBytes, 16);
                src += kBytes, --left;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (uint32_t i = 0; i < kRing; ++i) issue(slots + i * kBytes);

        // After a wait that ran out the workers go on, with whatever there is, to
        // the end.
        // Accumulator u (of the group gi of block b), times its scales, to registers.
        auto take = [&](uint32_t u, uint32_t b, uint32_t gi) {
            wait(&d_full[u % kUnits], u / kUnits & 1u);
            __syncwarp();
            tc_fence_after();
            const float s = bf16_bits_to_f32(
                ld_shared_u16(scales + ((b % kScaleSlots * kGroups + gi) * kColumns + column) * 2u));
            const uint32_t at = tmem + (warp % 4u * 32u << 16) + u % kUnits * MT + row0;
#pragma unroll
            for (int c = 0; c < kAcc; c += 16) {
                float v[16];
                if (c + 16 <= kAcc)
                    tmem_values<16>(at + c, v);
                else
                    tmem_values<8>(at + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (c + i < kAcc) acc[c + i] = fmaf(s, v[i], acc[c + i]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&d_empty[u % kUnits]);
        };
        // The accumulators that are complete with half h of block b.
        auto take_half = [&](uint32_t b, uint32_t h) {
            if constexpr (GROUP == 128) {
                if (h == 1u) take(b, b, 0u);
            } else if constexpr (GROUP == 64) {
                take(2u * b + h, b, h);
            } else {
                take(4u * b + 2u * h, b, 2u * h);
                take(4u * b + 2u * h + 1u, b, 2u * h + 1u);
            }
        };

        // Odd columns take each two words in the other order, so that eight
        // lanes' 16-byte stores fall on distinct banks.
        const uint32_t odd = g & 1u;
        uint32_t eight;  // (16 + 8) 2^-11 twice, in one register for good
        asm volatile("mov.b32 %0, 0x3c403c40;" : "=r"(eight));
        uint32_t slot = slots;
        uint32_t stage = 0, phase = 1;  // phase of the stage's previous round
        for (uint32_t b = 0; b < nkb; ++b) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            __syncwarp();  // every lane's copies have landed
            const uint4 a4 = ld_shared_v4(slot + lane * 16u), c4 = ld_shared_v4(slot + 512u + lane * 16u);
            uint32_t za[ZEROS ? kGroups : 1], zb[ZEROS ? kGroups : 1];
            if constexpr (ZEROS) {
                const uint32_t z = slot + kCodeBytes + 32u * kGroups;
#pragma unroll
                for (uint32_t i = 0; i < kGroups; ++i) {
                    const uint32_t at = (GROUP == 32 ? i ^ odd : i) * 16u + g;
                    za[i] = kSixteen | (ld_shared_u8(z + at) & 15u) * 0x00080008u;
                    zb[i] = kSixteen | (ld_shared_u8(z + at + 8u) & 15u) * 0x00080008u;
                }
            }
            if (lane < 2u * kGroups)  // 8 scales a lane
                st_shared_v4(scales + (b % kScaleSlots * kGroups + lane / 2u) * (kColumns * 2u) + warp * 32u +
                                 lane % 2u * 16u,
                             ld_shared_v4(slot + kCodeBytes + lane * 16u));
            __syncwarp();  // every lane has read the slot
            issue(slot);
            slot = slot + kBytes == slots + kRing * kBytes ? slots : slot + kBytes;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                if (h % kHalves == 0) {
                    if (2u * b + h >= kStages * kHalves) wait(&empty[stage], phase);
                    __syncwarp();
                }
                // 64 k of 128 rows in the 128-byte swizzle.
                const uint32_t rows = base + stage * kStageBytes + h % kHalves * kWHalf + warp * 2048u + g * 128u;
                const uint32_t at0 = ((odd * 4u + t) ^ g) * 16u;  // of the first word written; the other: 64 bytes off
#pragma unroll
                for (uint32_t s = 2 * h; s < 2 * h + 2; ++s) {
                    // Word s, or s ^ 1 in odd columns.
                    const uint32_t a = odd ? word(a4, s ^ 1u) : word(a4, s), c = odd ? word(c4, s ^ 1u) : word(c4, s);
                    const uint32_t gi = s * 32 / GROUP;
                    const uint32_t z0 = ZEROS ? za[ZEROS ? gi : 0] : eight, z1 = ZEROS ? zb[ZEROS ? gi : 0] : eight;
                    const uint32_t to = rows + (at0 ^ s % 2u * 64u);
                    st_shared_v4(to, make_uint4(difference<0>(a, z0), difference<1>(a, z0), difference<2>(a, z0),
                                                difference<3>(a, z0)));
                    st_shared_v4(to + 1024u, make_uint4(difference<0>(c, z1), difference<1>(c, z1),
                                                        difference<2>(c, z1), difference<3>(c, z1)));
                }
                if (h % kHalves == kHalves - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[stage]);
                    if (++stage == kStages) stage = 0, phase ^= 1u;
                }
                if (b) take_half(b - 1u, h);
            }
        }
        take_half(nkb - 1u, 0u);
        take_half(nkb - 1u, 1u);
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kMmaWarp) {
        // One lane of the warp issues; all wait, so that the others' way is the same.
        const bool one = elect();
        constexpr uint64_t kmaj = smem_desc_sw128_kmajor();
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (uint32_t b = 0; b < nkb && ok; ++b) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                if (h % kHalves == 0) ok = ok && wait(&full[stage], phase) && wait(&x_full[stage], phase);
                // W was written by the generic proxy, the MMA reads through the async
                // one.  (A fence by every writer: 75 us instead of 68, 64 rows of 8192 x 24576.)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                const uint32_t w_at = base + stage * kStageBytes + h % kHalves * kWHalf >> 4;
                const uint32_t x_at = base + stage * kStageBytes + kWBytes + h % kHalves * (MT * 128u) >> 4;
                const uint64_t w_desc = kmaj | (uint64_t)(w_at & 0x3fffu), x_desc = kmaj | (uint64_t)(x_at & 0x3fffu);
#pragma unroll
                for (uint32_t k0 = 0; k0 < 4; k0 += GROUP == 32 ? 2 : 4) {  // 16 k each
                    const uint32_t in = (4 * h + k0) % (GROUP / 16);  // the group
                    const uint32_t u = b * kGroups + (4 * h + k0) / (GROUP / 16);
                    if (in == 0 && u >= kUnits) ok = ok && wait(&d_empty[u % kUnits], (u / kUnits - 1u) & 1u);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                    if (one && ok) {
#pragma unroll
                        for (uint32_t k = k0; k < k0 + (GROUP == 32 ? 2 : 4); ++k)
                            tc_mma(tmem + u % kUnits * MT, w_desc + k * 2u, x_desc + k * 2u, instruction(MT),
                                   in == 0 && k == k0 ? 0u : 1u);
                        if (GROUP < 128 || h == 1) tc_commit(&d_full[u % kUnits]);
                        if (k0 + (GROUP == 32 ? 2 : 4) == 4 && h % kHalves == kHalves - 1) tc_commit(&empty[stage]);
                    }
                }
                if (h % kHalves == kHalves - 1 && ++stage == kStages) stage = 0, phase ^= 1u;
            }
        }
        // Every MMA ends before TMEM is released.
        if (one) {
            tc_commit(&drain);
            mbar_drain(&drain, 0, 100000000ull);
        }
    } else if (warp == kCopyWarp && lane == 0) {
        uint32_t stage = 0, phase = 1, i = 0;
        for (; i < 2u / kHalves * nkb; ++i) {
            if (i >= kStages && !wait(&empty[stage], phase)) break;
            mbar_expect_tx(&x_full[stage], kHalves * MT * 128u);
#pragma unroll
            for (uint32_t h = 0; h < kHalves; ++h)
                tma_load_2d(base + stage * kStageBytes + kWBytes + h * (MT * 128u), &map_x,
                            (int32_t)(kb0 * kBlockK + (i * kHalves + h) * 64u), (int32_t)m0, &x_full[stage]);
            if (++stage == kStages) stage = 0, phase ^= 1u;
        }
        // Every copy ends before the block does.
        for (uint32_t k = i > kStages ? i - kStages : 0u; k < i; ++k)
            mbar_drain(&x_full[k % kStages], k / kStages & 1u, 100000000ull);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
    }
    auto put = [&](uint32_t n, uint32_t m, float v) {
        if (n >= p.N || m >= p.M) return;
        v *= kUnit;
        if (p.bias) v += bf16_bits_to_f32(p.bias[n]);
        if (p.relu && v < 0.0f) v = 0.0f;
        p.y[m * p.ld_y + n] = (uint16_t)(cvt_bf16x2(v, 0.0f) & 0xffffu);
    };
    if (p.S == 1) {
        if (warp < kWorkers)
#pragma unroll
            for (int i = 0; i < kAcc; ++i) put(n0 + column, m0 + row0 + i, acc[i]);
        return;
    }
    // CTA c of the cluster adds the parts of columns [c own, (c + 1) own) in
    // order: [CTA][rows / 4][column][4 rows] where the stages were.
    const uint32_t own = kColumns / p.S;
    cluster_sync();  // every CTA's products are done
    if (warp < kWorkers) {
        const uint32_t to = map_to_rank(smem, column / own) +
                          ((rank * (MT / 4u) + row0 / 4u) * own + column % own) * 16u;
#pragma unroll
        for (int i = 0; i < kAcc; i += 4)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(to + i / 4 * own * 16u), "f"(acc[i]),
                         "f"(acc[i + 1]), "f"(acc[i + 2]), "f"(acc[i + 3])
                         : "memory");
    }
    cluster_sync();
    for (uint32_t i = threadIdx.x; i < own * (MT / 4u); i += kThreads) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t c = 0; c < p.S; ++c) {
            const float4 f = reinterpret_cast<const float4*>(smem)[c * (MT / 4u) * own + i];
            v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) put(n0 + rank * own + i % own, m0 + i / own * 4u + j, v[j]);
    }
}

using BatchKernel = void (*)(const Batch, const CUtensorMap);
template <int MT>
BatchKernel pick(const Weights& w) {
    if (w.group == 32) return w.zeros ? batch_kernel<MT, 32, true> : batch_kernel<MT, 32, false>;
    if (w.group == 64) return w.zeros ? batch_kernel<MT, 64, true> : batch_kernel<MT, 64, false>;
    return w.zeros ? batch_kernel<MT, 128, true> : batch_kernel<MT, 128, false>;
}

PFN_cuTensorMapEncodeTiled encoder() {
    static PFN_cuTensorMapEncodeTiled encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", (void**)&encode, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            encode = nullptr;
    });
    return encode;
}

// CTAs that share K: the least estimated time, in us, two CTAs on an SM.  A CTA
// takes 0.8 a block of k alone and 1.15 beside another, 2 to begin and end, and
// 0.3 for each part to join (64 rows).  (64 rows of 4096 x 4096: 28, 17, 11 and 11
// us with 1, 2, 4 and 8; of 8192 x 24576: 76, 67, 68, 84; estimates within a
// fifth.)
uint32_t split(uint32_t tiles, uint32_t kb, uint32_t mt) {
    const uint32_t sms = (uint32_t)foil_sm_count();
    uint32_t best = 1;
    float least = 0.0f;
    for (uint32_t S = 1; S <= 8 && S <= kb; S *= 2) {
        const uint32_t blocks = (kb + S - 1) / S, ctas = tiles * S, last = ctas % (2 * sms);
        const float join = 2.0f + (S > 1 ? 0.3f * S * mt / 64 : 0.0f);
        float t = (float)(ctas / (2 * sms)) * (join + 1.15f * blocks);
        if (last) t += join + (last > sms ? 1.15f : 0.8f) * blocks;
        if (S == 1 || t < least) best = S, least = t;
    }
    return best;
}

}  // namespace

cudaError_t matvec_batch(const uint16_t* x, uint64_t ld_x, const uint8_t* packed, const uint16_t* bias, uint16_t* y,
                         uint64_t ld_y, uint32_t M, const Weights& w, bool relu, uint32_t* err, cudaStream_t s) {
    const PFN_cuTensorMapEncodeTiled encode = encoder();
    if (!encode) return cudaErrorNotSupported;
    const uint32_t mt = M <= 32 ? 32 : M <= 48 ? 48 : 64;
    Batch p{};
    p.packed = packed, p.bias = bias, p.y = y, p.err = err, p.ld_y = ld_y, p.wait_ns = foil_wait_limit_ns();
    p.M = M, p.N = w.N, p.kb = (w.K + kBlockK - 1) / kBlockK, p.tiles = (w.N + kBlockN - 1) / kBlockN, p.relu = relu;
    const uint32_t columns = (w.N + kColumns - 1) / kColumns;
    p.S = split(columns * ((M + mt - 1) / mt), p.kb, mt);
    p.kb_each = p.kb / p.S, p.kb_more = p.kb % p.S;
    CUtensorMap map;
    const cuuint64_t dims[2] = {w.K, M}, strides[1] = {ld_x * 2};
    const cuuint32_t box[2] = {64, mt}, steps[2] = {1, 1};
    if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t*>(x), dims, strides, box, steps,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    const BatchKernel kernel = mt == 32 ? pick<32>(w) : mt == 48 ? pick<48>(w) : pick<64>(w);
    const uint32_t smem = smem_bytes(mt, w.group, w.zeros);
    const cudaError_t e = foil_smem_optin(reinterpret_cast<const void*>(kernel), (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(columns * p.S, (M + mt - 1) / mt, 1), cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute la[2]{};
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = p.S, la[1].val.clusterDim.y = 1, la[1].val.clusterDim.z = 1;
    cfg.attrs = la, cfg.numAttrs = p.S > 1 ? 2 : 1;
    const cudaError_t launched = cudaLaunchKernelEx(&cfg, kernel, p, map);
    if (launched == cudaSuccess) foil_count_launch();
    return launched;
}

}  // namespace w4
}  // namespace foil
