// q4_gemm.cu -- products of many activation rows with 4-bit weights on tcgen05 tensor cores.
//
//   c[r, o] = (accumulate ? c[r, o] : 0) + scale * act(s_r sum_g d[o, g] S[r, o, g] + bias[o]),
//   S[r, o, g] = sum over the inputs i of group g of a[r, i] (code[o, i] - zero[o, g]).
//
// Weights are never rounded: the matrix instructions multiply the integers code - zero, which bf16
// and fp16 hold exactly, group by group, and each group's f32 sum is multiplied by its f32 scale
// and added up in f32 registers. (Operands code * scale would round each weight to 8 or 11 bits,
// as large an error as the output's own rounding.) bf16 and fp16 activations are operands as they
// are. f32 activations are first written as two fp16 planes hi + lo of 22 significant bits, scaled
// by a power of two per row (s_r) so that the row's largest value lies in [2^14, 2^15); both planes
// are multiplied into the same accumulators.
//
// The instruction computes the transposed tile: A is 128 weight rows (outputs), B is BN
// activation rows; TMEM lane i holds output n0 + i, column j row m0 + j. CG = 2 runs CTA pairs: M =
// 256, each CTA holding its own 128 outputs and half of the activation rows, so the activations'
// share of the L2 reads is halved.
//
// One CTA per SM, persistent, 16 warps:
//   warp 0        TMA: 128 inputs of BN / CG activation rows (per plane) a stage
//   warp 1        issues the products: eight K = 16 instructions per stage and plane
//   warp 2        bulk copies of the codes (and zero points): 8 KB per 128 outputs and 128 inputs
//   warps 4-7     take the codes apart and store them into the stage's swizzled A tile
//   warps 8-15    add up: a group's sums from TMEM times its scale into registers (each thread one
//                 output and BN / 2 rows), and after the last group the epilogue
// TMEM holds several groups' accumulators, so the additions run behind the products. Registers are
// dealt out by role (setmaxnreg; 56 + 88 + 2 * 184 a thread and warpgroup = 4 * 128 at launch). Few
// tiles are split along the inputs: the CTAs of a cluster take a share of the chunks each, exchange
// their sums through distributed shared memory and finish a slice of the rows each, adding in rank
// order. Every wait is bounded; on timeout the kernel records kErrWaitTimeout and returns.
//
// Measured: 4096 rows of bf16, 4096 -> 8192 in groups of 128: 214 us in a short run, 1285 TFLOP/s (77% of the
// library's dense bf16 product), about 200 cycles an instruction of 256 x 256 x 16; 251 us after seconds under the
// power cap (1627 MHz), 1095 TFLOP/s (79% of the library's rate so). 1500 rows of f32, 1024 -> 4096: 36.9 us in a
// stream of calls, 34.3 captured, with their split, where eight chunks a tile leave its beginning and end uncovered
// (tensor pipe 34%).
#include "ptx.cuh"
#include "q4_device.cuh"
#include "tma.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace telmo {

namespace {

constexpr int kThreads = 512;
constexpr int kHalfK = 64;                    // inputs of one 128-byte swizzled row of 16-bit values
constexpr int kAHalf = 128 * kHalfK * 2;      // one CTA's A tile of 64 inputs
constexpr int kCodeBytes = 128 * 64;          // the codes of 128 outputs and one 128-input chunk
constexpr int kCodeStage = kCodeBytes + 512;  // and their zero points
constexpr int kCodeStages = 4;
constexpr int kDrainWarps = 8;
constexpr int kDequantWarps = 4;
constexpr int kStageBudget = 192 << 10;

template <int P, int BN, int CG>
struct Shape {
    static constexpr int kBRows = BN / CG;  // activation rows a CTA stages, per plane
    static constexpr int kBHalf = kBRows * kHalfK * 2;  // of one plane and 64 inputs
    static constexpr int kStageBytes = 2 * kAHalf + 2 * P * kBHalf;
    static constexpr int kStages = std::min(4, kStageBudget / kStageBytes);
    static constexpr int kBufs = std::min(4, 512 / BN);  // accumulators in TMEM
    static constexpr int kTmemCols = BN == 192 ? 512 : kBufs * BN;  // a power of two
    static constexpr int kSmemBytes = kStages * kStageBytes + kCodeStages * kCodeStage + 512;
};

struct GemmParams {
    const uint4* codes;
    const __half* scales;
    const uint8_t* zeros;
    int n, k, chunks;
    int per_chunk;  // groups per 128 inputs
    int m;
    const float* row_scale;  // [m] with two planes
    const float* bias;
    int act;
    float scale;
    int accumulate;
    void* c;
    int c_type;
    int64_t ldc;
    int tiles, num_n;
    int splits;        // CTAs of one cluster that share a tile's inputs
    int split_chunks;  // chunks of each
    bool planes;       // a was made by the kernel before
    uint32_t* error;
};

__device__ __forceinline__ void gave_up(const GemmParams& p, volatile int* abort_flag) {
    if (p.error) atomicCAS(p.error, 0u, static_cast<uint32_t>(kErrWaitTimeout));
    *abort_flag = 1;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// (x, y) = (x, y) + d (a, b), each rounded once.
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t d2, uint32_t a, uint32_t b) {
    const uint64_t ab = (static_cast<uint64_t>(b) << 32) | a;
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(d2), "l"(ab));
}

template <bool BF16>
__device__ __forceinline__ uint4 dequant_word(uint32_t word, uint32_t base) {
    return make_uint4(code_pair<BF16>(word, 0, base), code_pair<BF16>(word, 1, base), code_pair<BF16>(word, 2, base),
                      code_pair<BF16>(word, 3, base));
}

// Every thread of the cluster, at its own time (cluster_sync wants whole warps).
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Arrives on a barrier of either CTA of the pair. With DATA it announces what the arriving CTA's threads wrote to
// their shared memory (each lane's fence.proxy.async comes first) to an instruction that the other CTA issues, so
// the release is at cluster scope. It is restricted to this CTA's shared memory (4096 rows, 4096 -> 8192: 217 us; a
// full one, which covers the epilogue's stores to global memory too, 320). Without
// DATA it says that TMEM has been read, which the tcgen05 fences around an arrival and a wait order.
template <bool DATA>
__device__ __forceinline__ void arrive_pair(uint32_t cluster_bar) {
    if (DATA) asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// mbar_wait with a longer run of polls before it sleeps: these waits are short and follow one another.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kWaitPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (i > 4096) __nanosleep(256);
    }
    return false;
}

// The same for a barrier on which the other CTA of a pair arrives, or its products; with DATA what arrive_pair
// releases is acquired.
template <int CG, bool DATA>
__device__ __forceinline__ bool wait_for_pair(uint64_t* bar, uint32_t parity) {
    if constexpr (CG == 1) {
        return wait_for(bar, parity);
    } else {
        for (uint32_t i = 0; i < kWaitPolls; ++i) {
            uint32_t ok;
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.b32 %0, 1, 0, p;\n\t}"
                : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
            if (ok) {
                if (DATA) asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
                return true;
            }
            if (i > 4096) __nanosleep(256);
        }
        return false;
    }
}

// Arrives on the same barrier of both CTAs of the pair once this thread's products are complete.
__device__ __forceinline__ void commit_both(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
}

// A ring position and its phase.
template <int N>
struct Ring {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) {
            at = 0;
            phase ^= 1;
        }
    }
};

// Stores one output of N rows (those below m).
template <typename T, int N>
__device__ __forceinline__ void store_rows(const GemmParams& p, float (&v)[N], int row, int n) {
    T* out = static_cast<T*>(p.c) + static_cast<int64_t>(row) * p.ldc + n;
    const int rows = min(N, p.m - row);
    if (p.accumulate) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < rows) v[j] += static_cast<float>(out[j * p.ldc]);
    }
    if (rows == N) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            *out = static_cast<T>(v[j]);
            out += p.ldc;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < rows) out[j * p.ldc] = static_cast<T>(v[j]);
    }
}

// The epilogue of one output's sums over N rows, a multiple of four (those below m).
template <int P, int N>
__device__ __forceinline__ void finish_rows(const GemmParams& p, float (&v)[N], int row, int n, float bias) {
    if (P == 2) {
        const float4* rs = reinterpret_cast<const float4*>(p.row_scale + row);  // padded to whole tiles
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
            const float4 s = rs[j];
            v[4 * j] *= s.x;
            v[4 * j + 1] *= s.y;
            v[4 * j + 2] *= s.z;
            v[4 * j + 3] *= s.w;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += bias;
    if (p.act == kActRelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];
    } else if (p.act == kActSilu) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = mul_sigmoid(v[j], v[j]);
    }
    if (p.scale != 1.0f) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] *= p.scale;
    }
    if (p.c_type == kQ4F32) store_rows<float, N>(p, v, row, n);
    else if (p.c_type == kQ4BF16) store_rows<__nv_bfloat16, N>(p, v, row, n);
    else store_rows<__half, N>(p, v, row, n);
}

// One dequantizing warp's whole work: 32 of the CTA's 128 outputs.
template <bool BF16, int STAGES, int STAGE_BYTES, int CG, bool ZEROS>
__device__ __forceinline__ bool dequant_role(const GemmParams& p, uint8_t* smem, const uint8_t* code_ring, uint64_t* full,
                                             uint64_t* empty, uint64_t* code_full, uint64_t* code_empty, int first,
                                             int stride, int c0, int c1) {
    const int dw = (threadIdx.x / 32) & 3, lane = threadIdx.x % 32;
    const int g = lane >> 2, t4 = lane & 3, odd = g & 1;
    // Row r's 16-byte segment s lies at s ^ (r % 8) of its 128 bytes. Rows of odd g store their
    // second word first, so the two rows that share a store's phase use different banks.
    const uint32_t row = static_cast<uint32_t>((dw * 32 + g) * 128);
    const uint32_t at_a = row + static_cast<uint32_t>((4 * odd + t4) ^ g) * 16;
    const uint32_t at_b = row + static_cast<uint32_t>((4 * (odd ^ 1) + t4) ^ g) * 16;
    const uint32_t full0 = CG == 2 ? cluster_addr(full, 0) : smem_u32(full);
    const uint32_t stage0 = smem_u32(smem);
    Ring<STAGES> st;
    Ring<kCodeStages> cs;
    for (int t = first; t < p.tiles; t += stride) {
        for (int c = c0; c < c1; ++c) {
            if (!wait_for(&code_full[cs.at], cs.phase)) return false;
            const uint8_t* src = code_ring + cs.at * kCodeStage;
            uint4 v[4];
            uint32_t z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = reinterpret_cast<const uint4*>(src)[(dw * 4 + i) * 32 + lane];
                if (ZEROS) {
                    // One byte per word: a group spans 4 / per_chunk of a lane's four words.
                    const uint8_t* zs = src + kCodeBytes + ((dw * 4 + i) * 8 + g) * p.per_chunk;
                    z[i] = p.per_chunk == 4   ? *reinterpret_cast<const uint32_t*>(zs)
                           : p.per_chunk == 2 ? __byte_perm(*reinterpret_cast<const uint16_t*>(zs), 0, 0x1100)
                                              : *zs * 0x01010101u;
                }
            }
            if (!wait_for_pair<CG, true>(&empty[st.at], st.phase ^ 1)) return false;
            const uint32_t a = stage0 + st.at * STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t w0 = h ? v[i].z : v[i].x, w1 = h ? v[i].w : v[i].y;
                    uint32_t b0 = code_base<BF16>(8), b1 = b0;
                    if (ZEROS) {
                        b0 = code_base<BF16>((z[i] >> (16 * h)) & 0xffu);
                        b1 = code_base<BF16>((z[i] >> (16 * h + 8)) & 0xffu);
                    }
                    const uint32_t at = a + h * kAHalf + i * 1024;
                    st_shared_v4(at + at_a, dequant_word<BF16>(odd ? w1 : w0, ZEROS && odd ? b1 : b0));
                    st_shared_v4(at + at_b, dequant_word<BF16>(odd ? w0 : w1, ZEROS && odd ? b0 : b1));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (CG == 1) mbar_arrive(&full[st.at]);
                else arrive_pair<true>(full0 + static_cast<uint32_t>(st.at * sizeof(uint64_t)));
                // Only now: the codes have reached registers, since their operands are stored.
                mbar_arrive(&code_empty[cs.at]);
            }
            st.next();
            cs.next();
        }
    }
    return true;
}

// The issuing warp's whole work. All lanes walk the loops, so that addresses and descriptors stay in
// uniform registers; the elected one issues. PER_CHUNK groups of 128 / PER_CHUNK inputs to a stage.
template <bool BF16, int P, int BN, int CG, int PER_CHUNK>
__device__ __forceinline__ bool issue_role(const GemmParams& p, uint8_t* smem, uint64_t* full, uint64_t* empty,
                                           uint64_t* acc_full, uint64_t* acc_empty, uint32_t tmem_base, int first,
                                           int stride, int c0, int c1) {
    using S = Shape<P, BN, CG>;
    constexpr uint32_t idesc = idesc_f16(CG * 128, BN, false) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
    constexpr int kSteps = 8 / PER_CHUNK;  // K = 16 instructions to a group
    const bool issuer = elect_one();
    Ring<S::kStages> st;
    Ring<S::kBufs> acc;
    const uint64_t a0 = sw128_desc(smem_u32(smem)), b0 = sw128_desc(smem_u32(smem) + 2 * kAHalf);
    for (int t = first; t < p.tiles; t += stride) {
        for (int c = c0; c < c1; ++c) {
            if (!wait_for_pair<CG, true>(&full[st.at], st.phase)) return false;
            tc_fence_after();
            const uint64_t off = static_cast<uint64_t>(st.at * S::kStageBytes) >> 4;
#pragma unroll
            for (int q = 0; q < PER_CHUNK; ++q) {
                if (q > 0 && c * 128 + q * (128 / PER_CHUNK) >= p.k) break;
                if (!wait_for_pair<CG, false>(&acc_empty[acc.at], acc.phase ^ 1)) return false;
                tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc.at * BN);
                if (issuer) {
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        const int kk = q * kSteps + i;  // of the stage's eight
#pragma unroll
                        for (int pl = 0; pl < P; ++pl) {
                            const uint64_t da = a0 + off + static_cast<uint64_t>(((kk / 4) * kAHalf + (kk % 4) * 32) >> 4);
                            const uint64_t db = b0 + off + static_cast<uint64_t>(((pl * 2 + kk / 4) * S::kBHalf + (kk % 4) * 32) >> 4);
                            if (CG == 1) mma_f16(d, da, db, idesc, i + pl > 0);
                            else mma_f16_pair(d, da, db, idesc, i + pl > 0);
                        }
                    }
                    if (CG == 1) mma_commit(&acc_full[acc.at]);
                    else commit_both(&acc_full[acc.at]);
                }
                acc.next();
            }
            if (issuer) {
                if (CG == 1) mma_commit(&empty[st.at]);
                else commit_both(&empty[st.at]);
            }
            st.next();
        }
    }
    return true;
}

// SPLIT: the CTAs of a cluster share a tile's inputs (a kernel of its own, since the exchange's code costs the
// adding warps registers: prompt of 4096 rows, groups of 32, 588 us with it, 470 without).
template <bool BF16, int P, int BN, int CG, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
q4_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const GemmParams p) {
    using S = Shape<P, BN, CG>;
    constexpr int kCols = BN / 2;  // activation rows per adding thread
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw;
    if (smem_u32(smem) % 1024 != 0) {  // the declaration's alignment, which the swizzled tiles rely on
        if (threadIdx.x == 0 && p.error) atomicCAS(p.error, 0u, static_cast<uint32_t>(kErrWaitTimeout));
        return;
    }
    uint8_t* code_ring = smem + S::kStages * S::kStageBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(code_ring + kCodeStages * kCodeStage);
    uint64_t* empty = full + S::kStages;
    uint64_t* code_full = empty + S::kStages;
    uint64_t* code_empty = code_full + kCodeStages;
    uint64_t* acc_full = code_empty + kCodeStages;
    uint64_t* acc_empty = acc_full + S::kBufs;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kBufs);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // A cluster is a pair (CG = 2) or the CTAs that share a tile's inputs (SPLIT).
    static_assert(CG == 1 || !SPLIT, "pairs do not share inputs");
    const int splits = SPLIT ? p.splits : 1;
    const uint32_t rank = CG == 2 || SPLIT ? cluster_rank() : 0;
    const int pair = CG == 2 ? static_cast<int>(rank) : 0;  // this CTA's 128 of the tile's outputs
    const bool leader = pair == 0;
    const int split = SPLIT ? static_cast<int>(rank) : 0;
    const int first = blockIdx.x / (CG * splits), stride = gridDim.x / (CG * splits);
    const int c0 = split * p.split_chunks, c1 = min(p.chunks, c0 + p.split_chunks);
    const int per_chunk = p.per_chunk;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&full[s], 1 + CG * kDequantWarps);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kCodeStages; ++s) {
            mbar_init(&code_full[s], 1);
            mbar_init(&code_empty[s], kDequantWarps);
        }
        for (int b = 0; b < S::kBufs; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], CG * kDrainWarps);
        }
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tensormap(&map_a);
    }
    if (warp == 1) {
        if (CG == 1) {
            tmem_alloc(tmem_slot, S::kTmemCols);
            tmem_relinquish();
        } else {
            tmem_alloc_pair(tmem_slot, S::kTmemCols);
            tmem_relinquish_pair();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();  // both CTAs' barriers exist before either signals the other's
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp < 4) {
        regs_dec<56>();
        if (warp == 0 && lane == 0) {
            // ---- activations by TMA ----------------------------------------------------------
            Ring<S::kStages> st;
            bool ok = true;
            wait_for_previous();
            for (int t = first; t < p.tiles && ok; t += stride) {
                const int m0 = t / p.num_n * BN + pair * S::kBRows;
                for (int c = c0; c < c1; ++c) {
                    if (!(ok = wait_for_pair<CG, true>(&empty[st.at], st.phase ^ 1))) break;
                    uint8_t* b = smem + st.at * S::kStageBytes + 2 * kAHalf;
                    // Both CTAs' loads of a pair count on the first CTA's barrier, which expects them all.
                    const uint32_t bar = CG == 2 ? cluster_addr(&full[st.at], 0) : 0;
                    if (leader) mbar_arrive_expect_tx(&full[st.at], CG * P * 2 * S::kBHalf);
#pragma unroll
                    for (int i = 0; i < 2 * P; ++i) {  // plane i / 2, inputs 64 (i % 2) ..
                        const int x = c * 128 + (i % 2) * kHalfK, y = m0 + (i / 2) * p.m;
                        if (CG == 1) tma_load_2d(&map_a, &full[st.at], b + i * S::kBHalf, x, y);
                        else tma_load_2d_pair(&map_a, bar, b + i * S::kBHalf, x, y);
                    }
                    st.next();
                }
            }
            if (!ok) gave_up(p, abort_flag);
        } else if (warp == 1 && leader) {
            // ---- products (the pair's first CTA issues for both) -----------------------------
            const auto role = [&](auto per) {
                return issue_role<BF16, P, BN, CG, decltype(per)::value>(p, smem, full, empty, acc_full, acc_empty, tmem_base,
                                                                         first, stride, c0, c1);
            };
            const bool ok = per_chunk == 4   ? role(std::integral_constant<int, 4>())
                            : per_chunk == 2 ? role(std::integral_constant<int, 2>())
                                             : role(std::integral_constant<int, 1>());
            if (!ok) gave_up(p, abort_flag);
        } else if (warp == 2 && lane == 0) {
            // ---- codes and zero points: contiguous per 128 outputs and chunk ------------------
            Ring<kCodeStages> cs;
            bool ok = true;
            const uint32_t zero_bytes = p.zeros ? 128u * static_cast<uint32_t>(per_chunk) : 0u;
            for (int t = first; t < p.tiles && ok; t += stride) {
                // A pair's second CTA may have no outputs of its own: it repeats the last ones.
                const int block = min(t % p.num_n * CG + pair, (p.n + 127) / 128 - 1);
                for (int c = c0; c < c1; ++c) {
                    if (!(ok = wait_for(&code_empty[cs.at], cs.phase ^ 1))) break;
                    uint8_t* dst = code_ring + cs.at * kCodeStage;
                    const int64_t at = static_cast<int64_t>(block) * p.chunks + c;
                    mbar_arrive_expect_tx(&code_full[cs.at], kCodeBytes + zero_bytes);
                    bulk_load(dst, reinterpret_cast<const uint8_t*>(p.codes) + at * kCodeBytes, kCodeBytes, &code_full[cs.at]);
                    if (zero_bytes) bulk_load(dst + kCodeBytes, p.zeros + at * zero_bytes, zero_bytes, &code_full[cs.at]);
                    cs.next();
                }
            }
            if (!ok) gave_up(p, abort_flag);
        }
    } else if (warp < 8) {
        regs_dec<88>();
        const bool ok =
            p.zeros ? dequant_role<BF16, S::kStages, S::kStageBytes, CG, true>(p, smem, code_ring, full, empty, code_full,
                                                                               code_empty, first, stride, c0, c1)
                    : dequant_role<BF16, S::kStages, S::kStageBytes, CG, false>(p, smem, code_ring, full, empty, code_full,
                                                                                code_empty, first, stride, c0, c1);
        if (!ok) gave_up(p, abort_flag);
    } else {
        regs_inc<184>();
        // ---- sums and epilogue: thread = one output, kCols activation rows --------------------
        const int quad = warp & 3, half = (warp - 8) / 4;
        const int lane_row = quad * 32 + lane;
        Ring<S::kBufs> ab;
        wait_for_previous();
        const uint32_t acc_empty0 = CG == 2 ? cluster_addr(&acc_empty[0], 0) : 0;
        for (int t = first; t < p.tiles; t += stride) {
            const int m0 = t / p.num_n * BN + half * kCols;
            const int n = (t % p.num_n * CG + pair) * 128 + lane_row;
            const bool n_ok = n < p.n;
            // This output's scales, 2 per_chunk bytes a chunk, loaded a chunk ahead.
            const uint8_t* sc = reinterpret_cast<const uint8_t*>(p.scales) +
                                ((static_cast<int64_t>(n / 128) * p.chunks + c0) * 128 + lane_row) * per_chunk * 2;
            const auto load_scales = [&]() -> uint64_t {
                uint64_t v = 0;
                if (n_ok)
                    v = per_chunk == 4   ? __ldg(reinterpret_cast<const unsigned long long*>(sc))
                        : per_chunk == 2 ? __ldg(reinterpret_cast<const uint32_t*>(sc))
                                         : __ldg(reinterpret_cast<const uint16_t*>(sc));
                sc += 256 * per_chunk;
                return v;
            };
            uint64_t next = c0 < c1 ? load_scales() : 0;
            uint64_t acc[kCols / 2];
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) acc[j] = 0;
            bool ok = true;
            const auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) mbar_arrive(&acc_empty[ab.at]);
                    else arrive_pair<false>(acc_empty0 + static_cast<uint32_t>(ab.at * sizeof(uint64_t)));
                }
                ab.next();
            };
#pragma unroll 1
            for (int c = c0; c < c1 && ok; ++c) {
                uint64_t now = next;
                if (c + 1 < c1) next = load_scales();
                const int left = p.k - c * 128, size = 128 / per_chunk;
#pragma unroll 1
                for (int i = 0; i < left && i < 128; i += size, now >>= 16) {
                    const float d = __half2float(__ushort_as_half(static_cast<unsigned short>(now & 0xffff)));
                    ok = wait_for_pair<CG, false>(&acc_full[ab.at], ab.phase);
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                                           static_cast<uint32_t>(ab.at * BN + half * kCols);
                    const uint64_t d2 = pack_f2(make_float2(d, d));
                    // Two warps of a scheduler take turns: one's loads are under way while the other adds. The
                    // accumulator is released with its last columns' additions still to come (prompt of
                    // 4096 rows, 4096 -> 8192: 257 us with the release after them, 230 before).
                    const bool last = c == c1 - 1 && i + size >= left;  // the tile's last accumulator is kept
#pragma unroll
                    for (int q = 0; q < kCols / 32; ++q) {
                        uint32_t r[32];
                        tmem_ld32(taddr + q * 32, r);
                        tmem_ld_wait();
                        if (q == kCols / 32 - 1 && !last) release();
#pragma unroll
                        for (int j = 0; j < 16; ++j) fma2(acc[q * 16 + j], d2, r[2 * j], r[2 * j + 1]);
                    }
                }
            }
            if (!ok) {
                gave_up(p, abort_flag);
                if (SPLIT) {
                    cluster_meet();
                    cluster_meet();
                }
                break;
            }
            const float bias = p.bias && n_ok ? __ldg(p.bias + n) : 0.0f;
            // The sums go back to the last accumulator's columns, from where rolled loops can take them
            // (registers cannot be indexed): code that runs once a tile stays small. Its fetching is what
            // short products wait for (unrolled over the columns: 1500 rows, 1024 -> 4096: 89 us; 256 rows on pairs
            // split in four: 41 us).
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                                   static_cast<uint32_t>(ab.at * BN + half * kCols);
#pragma unroll
            for (int q = 0; q < kCols / 32; ++q) {
                uint32_t r[32];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    r[2 * j] = static_cast<uint32_t>(acc[q * 16 + j]);
                    r[2 * j + 1] = static_cast<uint32_t>(acc[q * 16 + j] >> 32);
                }
                tmem_st32(taddr + q * 32, r);
            }
            tmem_st_wait();
            // The CTAs that share a tile each finish a slice of its rows: every one sends its sums of a slice to
            // the slice's CTA, which adds them in rank order. The stages are free: all of a CTA's products
            // have been added up, here and, after the meeting, in the others.
            const int slice = kCols / splits, log = __ffs(slice) - 1;
            if (SPLIT) cluster_meet();
#pragma unroll 1
            for (int q = 0; q < kCols / 16; ++q) {
                const int row = m0 + q * 16;
                if (row >= p.m) break;
                uint32_t r[16];
                tmem_ld16(taddr + q * 16, r);
                tmem_ld_wait();
                if (!SPLIT) {
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                    if (n_ok) finish_rows<P, 16>(p, v, row, n, bias);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int col = q * 16 + j;
                        const uint32_t to = cluster_addr(smem, static_cast<uint32_t>(col >> log));
                        const int at = ((split * 2 + half) * slice + (col & (slice - 1))) * 128 + lane_row;
                        st_cluster_f32(to + static_cast<uint32_t>(at * 4), __uint_as_float(r[j]));
                    }
                }
                __syncwarp();
            }
            if (!SPLIT) {
                release();
                continue;
            }
            cluster_meet();
            const float* parts = reinterpret_cast<const float*>(smem);
#pragma unroll 1
            for (int j = 0; j < slice; j += 4) {  // a slice is four rows or more
                const int row = m0 + split * slice + j;
                if (row >= p.m || !n_ok) break;
                float v[4] = {};
                for (int q = 0; q < splits; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += parts[((q * 2 + half) * slice + j + i) * 128 + lane_row];
                finish_rows<P, 4>(p, v, row, n, bias);
            }
        }
    }

    if (SPLIT && warp < 8) {
        // The two meetings of the adding warps' exchange, which count every thread of the cluster.
        cluster_meet();
        cluster_meet();
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag)  // copies that were under way land before the shared memory is given back
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    // A pair's CTAs leave together: the first CTA's products read the second's shared memory and
    // write its TMEM, and the second's loads signal the first's barriers.
    if (CG == 2) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if (CG == 1) tmem_dealloc(tmem_base, S::kTmemCols);
        else tmem_dealloc_pair(tmem_base, S::kTmemCols);
    }
}

// The rows of a as the products read them. f32: two fp16 planes and the row's power of two, one block per
// row, which keeps the row's first values in registers between looking for the largest and splitting.
// 16-bit types: a copy with rows that start on 16-byte boundaries, 2048 values a block. (With few rows
// these wait for loads alone: 24 rows of 11009 took 14 us in one block of 256 threads a row, a value at a time.)
constexpr int kKeep = 4;  // fours of values a thread keeps

__device__ __forceinline__ float4 load_four(const float* row, int i, int k, bool vec) {
    if (vec && i + 4 <= k) return __ldg(reinterpret_cast<const float4*>(row + i));
    float4 v;
    v.x = i < k ? __ldg(row + i) : 0.0f;
    v.y = i + 1 < k ? __ldg(row + i + 1) : 0.0f;
    v.z = i + 2 < k ? __ldg(row + i + 2) : 0.0f;
    v.w = i + 3 < k ? __ldg(row + i + 3) : 0.0f;
    return v;
}

__global__ void __launch_bounds__(1024) q4_split_kernel(const float* a, int64_t lda, int m, int k, bool vec, __half* planes,
                                                        int64_t ld, float* row_scale) {
    let_next_start();
    const int64_t row = blockIdx.x;
    const float* src = a + row * lda;
    const int step = static_cast<int>(blockDim.x) * 4, i0 = static_cast<int>(threadIdx.x) * 4;
    __shared__ float tops[32];
    float4 kept[kKeep];
    float top = 0.0f;  // fmaxf passes NaNs over
    const auto look = [&](const float4& v) {
        top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
    };
#pragma unroll
    for (int q = 0; q < kKeep; ++q) kept[q] = load_four(src, i0 + q * step, k, vec);
#pragma unroll
    for (int q = 0; q < kKeep; ++q) look(kept[q]);
    for (int i = i0 + kKeep * step; i < k; i += step) look(load_four(src, i, k, vec));
#pragma unroll
    for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) top = fmaxf(top, tops[w]);
    // 2^e with the largest value 2^e times a number in [2^14, 2^15). e stops at -126, so that 2^-e
    // stays a normal f32: a row below 2^-112 keeps its values to 2^-150. An infinity's exponent makes e
    // 114, which holds every finite value below 2^14 and leaves the infinity one.
    const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -126);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    if (threadIdx.x == 0) row_scale[row] = up;
    __half* hi = planes + row * ld;
    __half* lo = hi + static_cast<int64_t>(m) * ld;
    const auto write = [&](const float4& v, int i) {  // ld is a multiple of 8: whole fours
        if (i >= ld) return;
        const float x[4] = {v.x * down, v.y * down, v.z * down, v.w * down};
        __half h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = __float2half_rn(x[j]);
            l[j] = __float2half_rn(x[j] - __half2float(h[j]));
        }
        *reinterpret_cast<uint2*>(hi + i) = *reinterpret_cast<const uint2*>(h);
        *reinterpret_cast<uint2*>(lo + i) = *reinterpret_cast<const uint2*>(l);
    };
#pragma unroll
    for (int q = 0; q < kKeep; ++q) write(kept[q], i0 + q * step);
    for (int i = i0 + kKeep * step; i < ld; i += step) write(load_four(src, i, k, vec), i);
}

constexpr int kAlignThreads = 256, kAlignValues = 2048;

__global__ void __launch_bounds__(kAlignThreads) q4_align_kernel(const uint16_t* a, int64_t lda, int k, uint16_t* out,
                                                                 int64_t ld) {
    const int64_t row = blockIdx.x;
    // One turn, but for rows of more pieces than a grid has blocks along y.
    for (int64_t begin = static_cast<int64_t>(blockIdx.y) * kAlignValues; begin < ld;
         begin += static_cast<int64_t>(gridDim.y) * kAlignValues) {
        const int base = static_cast<int>(begin) + threadIdx.x;
        uint16_t v[kAlignValues / kAlignThreads];
#pragma unroll
        for (int j = 0; j < kAlignValues / kAlignThreads; ++j) {
            const int i = base + j * kAlignThreads;
            v[j] = i < k ? __ldg(a + row * lda + i) : uint16_t(0);
        }
#pragma unroll
        for (int j = 0; j < kAlignValues / kAlignThreads; ++j) {
            const int i = base + j * kAlignThreads;
            if (i < ld) out[row * ld + i] = v[j];
        }
    }
    // At the end: blocks of the product that come while these still hold SMs lie unevenly (24 rows, 11009 ->
    // 4096: 27.6 us with this at the beginning, 24.6 without it, 22.6 here).
    let_next_start();
}

// A launch of the kernel with clusters of `cluster` CTAs.
struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    Launch(int cluster, unsigned grid, size_t smem, cudaStream_t stream, bool early = false) {
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        add_attributes(cfg, attr, cluster, early);
    }
};

// How many clusters of 1, 2, 4 or 8 CTAs the device runs at once (fewer than its SMs would hold: a cluster
// stays within a GPC; 15 of eight CTAs on 148 SMs). Asked once per device, with the kernel's attributes set.
template <bool BF16, int P, int BN, int CG, bool SPLIT>
cudaError_t clusters_at_once(int cluster, int sms, int* count) {
    using S = Shape<P, BN, CG>;
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices][4];
    static DeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const auto kernel = q4_gemm_kernel<BF16, P, BN, CG, SPLIT>;
    if (!once.done(dev)) {
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes)) != cudaSuccess)
            return e;
        once.mark(dev);
    }
    const int at = cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3;
    int n = dev < kDevices ? known[dev][at].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        if (cluster == 1) {
            n = sms;
        } else {
            const Launch l(cluster, static_cast<unsigned>(cluster), S::kSmemBytes, nullptr);
            if ((e = cudaOccupancyMaxActiveClusters(&n, kernel, &l.cfg)) != cudaSuccess) return e;
            n = std::max(n, 1);
        }
        if (dev < kDevices) known[dev][at].store(n, std::memory_order_relaxed);
    }
    *count = n;
    return cudaSuccess;
}

template <bool BF16, int P, int BN, int CG, bool SPLIT>
cudaError_t launch_gemm(const void* a, int64_t lda, GemmParams p, int splits, int at_once, cudaStream_t stream) {
    using S = Shape<P, BN, CG>;
    CUtensorMap map;
    if (!encode_map_2d(&map, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a,
                       static_cast<uint64_t>(p.k), static_cast<uint64_t>(p.m) * P, static_cast<uint64_t>(lda) * 2, kHalfK,
                       S::kBRows, CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    p.num_n = (p.n + CG * 128 - 1) / (CG * 128);
    const int64_t tiles = static_cast<int64_t>((p.m + BN - 1) / BN) * p.num_n;
    if (tiles > (1 << 28)) return cudaErrorInvalidValue;
    p.tiles = static_cast<int>(tiles);
    p.splits = splits;
    p.split_chunks = (p.chunks + splits - 1) / splits;
    const int cluster = CG * splits;
    const Launch l(cluster, static_cast<unsigned>(cluster * (splits > 1 ? p.tiles : std::min(p.tiles, at_once))), S::kSmemBytes,
                   stream, p.planes);
    return cudaLaunchKernelEx(&l.cfg, q4_gemm_kernel<BF16, P, BN, CG, SPLIT>, map, p);
}

template <int BN, bool SPLIT>
struct Kernel {
    static constexpr int kBN = BN, kCG = BN >= 192 ? 2 : 1;
    static constexpr bool kSplit = SPLIT;
};

// Calls f with the kernel's constants.
template <bool BF16, int P, typename F>
cudaError_t with_shape(int bn, int splits, F f) {
    if (splits > 1) return bn == 128 ? f(Kernel<128, true>()) : f(Kernel<64, true>());
    return bn == 256   ? f(Kernel<256, false>())
           : bn == 192 ? f(Kernel<192, false>())
           : bn == 128 ? f(Kernel<128, false>())
                       : f(Kernel<64, false>());
}

// The tile and the number of CTAs that share its inputs. Up to 192 rows a chunk's time is that of
// taking 128 outputs' codes apart, about 1450 cycles whatever the rows (so larger tiles win even where they are
// not filled, and tiles split among CTAs that exchange their sums, before the codes are taken apart again);
// then it is the products', and with two planes from 128 rows on the activations' way from L2. Pairs do not
// share inputs: their exchange of 128 KB a CTA cost more than it saved (200 rows, 4096 -> 8192: 40 us split in two,
// 33 whole). The rounds of
// tiles over the GPU count too: 1500 rows of f32, 1024 -> 4096, are 96 tiles of 256 rows on 74 pairs (42 us) or 128
// of 192 (35 us). Against each of the ten choices forced, for 40 to 4096 rows and six shapes (640 -> 1000 to 4096 ->
// 8192 and 8192 -> 2048, both types): the best one or within 5%, but for 100 and 128 rows of 1024 -> 4096 (10.3 us for
// 9.4, f32 12.5 for 11.8); the worst choice takes 1.5 to 7 times as long.
template <bool BF16, int P>
cudaError_t launch_shape(const void* a, int64_t lda, const GemmParams& p, int sms, cudaStream_t stream) {
    int best_bn = 0, best_splits = 1, best_at_once = 1;
    double best = 0.0;
    for (const int bn : {64, 128, 192, 256}) {
        const int cg = bn >= 192 ? 2 : 1;
        const double tiles = static_cast<double>((p.m + bn - 1) / bn) * ((p.n + cg * 128 - 1) / (cg * 128));
        const int most_splits = cg == 2 ? 1 : 8;
        for (int splits = 1; splits <= most_splits && (splits == 1 || p.chunks >= 2 * splits); splits *= 2) {
            int at_once = 0;
            const cudaError_t e = with_shape<BF16, P>(bn, splits, [&](auto shape) {
                using K = decltype(shape);
                return clusters_at_once<BF16, P, K::kBN, K::kCG, K::kSplit>(cg * splits, sms, &at_once);
            });
            if (e != cudaSuccess) return e;
            const double chunk = P == 2 ? (bn == 64 ? 1700.0 : bn < 256 ? 2400.0 : 3200.0) : (bn < 256 ? 1450.0 : 1700.0);
            // A first chunk's way through the roles, the epilogue, and the exchange of sums.
            const double tile = 4000.0 + ((p.chunks + splits - 1) / splits) * chunk + bn * 10.0 / splits +
                                (splits > 1 ? 4500.0 + bn * 25.0 : 0.0);
            const double time = std::ceil(tiles / at_once) * tile;
            if (best_bn == 0 || time < best) {
                best = time;
                best_bn = bn;
                best_splits = splits;
                best_at_once = at_once;
            }
        }
    }
    return with_shape<BF16, P>(best_bn, best_splits, [&](auto shape) {
        using K = decltype(shape);
        return launch_gemm<BF16, P, K::kBN, K::kCG, K::kSplit>(a, lda, p, best_splits, best_at_once, stream);
    });
}

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace

size_t q4_planes_bytes(const Q4Args& g) {
    const size_t m = static_cast<size_t>(g.m), ld = round_up(static_cast<size_t>(g.w->k), 8);
    if (g.a_type != kQ4F32) return m * ld * 2;
    return round_up(2 * m * ld * sizeof(__half), 256) + round_up(m, 256) * sizeof(float);
}

cudaError_t q4_make_planes(const Q4Args& g, void* workspace, Q4Planes* planes, cudaStream_t stream) {
    const int64_t ld = static_cast<int64_t>(round_up(static_cast<size_t>(g.w->k), 8));
    planes->a = workspace;
    planes->ld = ld;
    if (g.a_type == kQ4F32) {
        float* rs = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                             round_up(2 * static_cast<size_t>(g.m) * ld * sizeof(__half), 256));
        planes->row_scale = rs;
        const int threads = std::min<int>(1024, static_cast<int>(round_up((static_cast<size_t>(g.w->k) + 7) / 8, 32)));
        q4_split_kernel<<<g.m, threads, 0, stream>>>(static_cast<const float*>(g.a), g.lda, g.m, g.w->k, q4_rows_aligned(g),
                                                     static_cast<__half*>(workspace), ld, rs);
    } else {
        const dim3 grid(g.m, static_cast<unsigned>(std::min<int64_t>(65535, (ld + kAlignValues - 1) / kAlignValues)));
        q4_align_kernel<<<grid, kAlignThreads, 0, stream>>>(static_cast<const uint16_t*>(g.a), g.lda, g.w->k,
                                                            static_cast<uint16_t*>(workspace), ld);
    }
    return cudaGetLastError();
}

cudaError_t q4_linear_gemm(const Q4Args& g, const Q4Planes* planes, cudaStream_t stream) {
    GemmParams p = {};
    p.codes = g.w->codes;
    p.scales = g.w->scales;
    p.zeros = g.w->zeros;
    p.n = g.w->n;
    p.k = g.w->k;
    p.chunks = g.w->chunks;
    p.per_chunk = 128 / g.w->group;
    p.m = g.m;
    p.row_scale = planes ? planes->row_scale : nullptr;
    p.planes = planes != nullptr;
    p.bias = g.bias;
    p.act = g.act;
    p.scale = g.scale;
    p.accumulate = g.accumulate;
    p.c = g.c;
    p.c_type = g.c_type;
    p.ldc = g.ldc;
    p.error = g.error;
    const void* a = planes ? planes->a : g.a;
    const int64_t lda = planes ? planes->ld : g.lda;
    if (g.a_type == kQ4F32) return launch_shape<false, 2>(a, lda, p, g.sms, stream);
    return g.a_type == kQ4BF16 ? launch_shape<true, 1>(a, lda, p, g.sms, stream)
                               : launch_shape<false, 1>(a, lda, p, g.sms, stream);
}

}  // namespace telmo
