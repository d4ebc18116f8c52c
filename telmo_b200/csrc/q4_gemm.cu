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
//   warp 0        TMA producer: 64 inputs of BN / CG activation rows (per plane) a stage
//   warp 1        MMA issuer: four K = 16 instructions per stage and plane
//   warps 4-7     take the codes of 128 outputs apart: 16-byte loads of the tiled layout, one
//                 chunk ahead in registers, and 16-byte stores into the stage's swizzled A tile
//   warps 8-15    add up: a group's sums from TMEM times its scale into registers (each thread one
//                 output and BN / 2 rows), and after the last group the epilogue
// TMEM holds several groups' accumulators, so the additions run behind the products. Registers are
// dealt out by role (setmaxnreg; 40 + 104 + 2 * 184 a thread and warpgroup = 4 * 128 at launch). Every
// wait is bounded; on timeout the kernel records kErrWaitTimeout and returns.
#include "ptx.cuh"
#include "q4_device.cuh"
#include "tma.h"

#include <algorithm>
#include <cstring>

namespace telmo {

namespace {

constexpr int kThreads = 512;
constexpr int kStepK = 64;                    // inputs per stage: one 128-byte swizzled row of 16-bit values
constexpr int kABytes = 128 * kStepK * 2;     // one CTA's A tile
constexpr int kDrainWarps = 8;
constexpr int kDequantWarps = 4;
constexpr int kSmemBudget = 224 << 10;

template <int P, int BN, int CG>
struct Shape {
    static constexpr int kBRows = BN / CG;                     // activation rows a CTA stages, per plane
    static constexpr int kBPlane = kBRows * kStepK * 2;
    static constexpr int kStageBytes = kABytes + P * kBPlane;
    static constexpr int kStages = std::min(8, (kSmemBudget - 2048) / kStageBytes);
    static constexpr int kBufs = std::min(4, 512 / BN);        // accumulators in TMEM
    static constexpr int kTmemCols = kBufs * BN;
    static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 512;
};

struct GemmParams {
    const uint4* codes;
    const __half* scales;
    const uint8_t* zeros;
    int n, k, chunks, tiles8;  // tiles8: 8-output tile rows of the layout
    int m;
    const float* row_scale;  // [m] with two planes
    const float* bias;
    int act;
    float scale;
    int accumulate;
    void* c;
    int c_type;
    int64_t ldc;
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

// (x, y) = (x, y) + d (a, b), each rounded once.
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t d2, uint32_t a, uint32_t b) {
    const uint64_t ab = (static_cast<uint64_t>(b) << 32) | a;
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(d2), "l"(ab));
}

// Zero points of one output row in one chunk, a byte per group.
template <int GROUPS>
__device__ __forceinline__ uint32_t load_zeros(const uint8_t* zeros, int64_t tile, int g) {
    const uint8_t* z = zeros + (tile * 8 + g) * GROUPS;
    if (GROUPS == 4) return __ldg(reinterpret_cast<const uint32_t*>(z));
    if (GROUPS == 2) return __ldg(reinterpret_cast<const uint16_t*>(z));
    return __ldg(z);
}

// One warp's codes of a chunk: four 8-output tiles.
struct Codes {
    uint4 v[4];
    uint32_t z[4];
};

template <int GROUPS>
__device__ __forceinline__ void load_codes(const GemmParams& p, int tile8, int c, int lane, Codes& w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t8 = tile8 + i;
        w.v[i] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        w.z[i] = 0x08080808u;
        if (t8 < p.tiles8) {
            const int64_t tile = static_cast<int64_t>(t8) * p.chunks + c;
            w.v[i] = __ldg(p.codes + tile * 32 + lane);
            if (p.zeros) w.z[i] = load_zeros<GROUPS>(p.zeros, tile, lane >> 2);
        }
    }
}

template <bool BF16>
__device__ __forceinline__ uint4 dequant_word(uint32_t word, uint32_t zero) {
    const uint32_t base = code_base<BF16>(zero);
    return make_uint4(code_pair<BF16>(word, 0, base), code_pair<BF16>(word, 1, base), code_pair<BF16>(word, 2, base),
                      code_pair<BF16>(word, 3, base));
}

template <bool BF16, int P, int BN, int CG, int GROUPS>
__global__ void __launch_bounds__(kThreads, 1)
q4_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const GemmParams p) {
    using S = Shape<P, BN, CG>;
    constexpr int kCols = BN / 2;  // activation rows per adding thread
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStageBytes);
    uint64_t* empty = full + S::kStages;
    uint64_t* acc_full = empty + S::kStages;
    uint64_t* acc_empty = acc_full + S::kBufs;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kBufs);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const bool leader = rank == 0;
    const int unit = blockIdx.x / CG, units = gridDim.x / CG;
    const int num_n = (p.n + CG * 128 - 1) / (CG * 128);
    const int64_t tiles = static_cast<int64_t>((p.m + BN - 1) / BN) * num_n;
    const int steps = (p.k + kStepK - 1) / kStepK;
    const int groups = (p.k + 128 / GROUPS - 1) / (128 / GROUPS);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&full[s], 1 + CG * kDequantWarps);
            mbar_init(&empty[s], 1);
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
        regs_dec<40>();
        if (warp == 0 && lane == 0) {
            // ---- activations by TMA ----------------------------------------------------------
            int stage = 0;
            uint32_t phase = 0;
            for (int64_t t = unit; t < tiles && !*abort_flag; t += units) {
                const int m0 = static_cast<int>(t / num_n) * BN + static_cast<int>(rank) * S::kBRows;
                for (int s = 0; s < steps; ++s) {
                    if (!mbar_wait(&empty[stage], phase ^ 1)) {
                        gave_up(p, abort_flag);
                        break;
                    }
                    uint8_t* b = smem + stage * S::kStageBytes + kABytes;
                    if (CG == 1) {
                        mbar_arrive_expect_tx(&full[stage], P * S::kBPlane);
                        for (int pl = 0; pl < P; ++pl)
                            tma_load_2d(&map_a, &full[stage], b + pl * S::kBPlane, s * kStepK, m0 + pl * p.m);
                    } else {
                        // Both CTAs' loads count on the first CTA's barrier, which expects them all.
                        const uint32_t bar = cluster_addr(&full[stage], 0);
                        if (leader) mbar_arrive_expect_tx(&full[stage], 2 * P * S::kBPlane);
                        for (int pl = 0; pl < P; ++pl)
                            tma_load_2d_pair(&map_a, bar, b + pl * S::kBPlane, s * kStepK, m0 + pl * p.m);
                    }
                    if (++stage == S::kStages) { stage = 0; phase ^= 1; }
                }
            }
        } else if (warp == 1 && leader) {
            // ---- products (the pair's first CTA issues for both) -----------------------------
            constexpr uint32_t idesc = idesc_f16(CG * 128, BN, false) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
            constexpr int kHalves = GROUPS == 4 ? 2 : 1;      // groups that start within a step
            constexpr int kPerHalf = kStepK / 16 / kHalves;   // K = 16 instructions of each
            int stage = 0, buf = 0;
            uint32_t phase = 0, acc_phase = 0;
            const uint32_t peer_empty = CG == 2 ? cluster_addr(&empty[0], 1) : 0;
            const uint32_t peer_acc_full = CG == 2 ? cluster_addr(&acc_full[0], 1) : 0;
            for (int64_t t = unit; t < tiles && !*abort_flag; t += units) {
                bool ok = true;
                for (int s = 0; s < steps && ok; ++s) {
                    if (!(ok = mbar_wait(&full[stage], phase))) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + stage * S::kStageBytes), b = a + kABytes;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) {
                        if (GROUPS == 4 && h == 1 && s * kStepK + 32 >= p.k) break;
                        const bool first = GROUPS != 1 || s % 2 == 0;
                        const bool last = GROUPS != 1 || s % 2 == 1 || s == steps - 1;
                        if (first) {
                            if (!(ok = mbar_wait(&acc_empty[buf], acc_phase ^ 1))) break;
                            tc_fence_after();
                        }
                        if (lane == 0) {
                            const uint32_t d = tmem_base + static_cast<uint32_t>(buf * BN);
#pragma unroll
                            for (int i = 0; i < kPerHalf; ++i) {
                                const int kk = h * kPerHalf + i;
#pragma unroll
                                for (int pl = 0; pl < P; ++pl) {
                                    const uint64_t da = sw128_desc(a + kk * 32);
                                    const uint64_t db = sw128_desc(b + pl * S::kBPlane + kk * 32);
                                    const uint32_t add = first && i == 0 && pl == 0 ? 0u : 1u;
                                    if (CG == 1) mma_f16(d, da, db, idesc, add);
                                    else mma_f16_pair(d, da, db, idesc, add);
                                }
                            }
                            if (last) {
                                if (CG == 1) {
                                    mma_commit(&acc_full[buf]);
                                } else {
                                    mma_commit_pair(smem_u32(&acc_full[buf]));
                                    mma_commit_pair(peer_acc_full + static_cast<uint32_t>(buf * sizeof(uint64_t)));
                                }
                            }
                        }
                        __syncwarp();
                        if (last && ++buf == S::kBufs) { buf = 0; acc_phase ^= 1; }
                    }
                    if (!ok) break;
                    if (lane == 0) {
                        if (CG == 1) {
                            mma_commit(&empty[stage]);
                        } else {
                            mma_commit_pair(smem_u32(&empty[stage]));
                            mma_commit_pair(peer_empty + static_cast<uint32_t>(stage * sizeof(uint64_t)));
                        }
                    }
                    __syncwarp();
                    if (++stage == S::kStages) { stage = 0; phase ^= 1; }
                }
                if (!ok) {
                    gave_up(p, abort_flag);
                    break;
                }
            }
        }
    } else if (warp < 8) {
        regs_dec<104>();
        // ---- weights: codes to operands ------------------------------------------------------
        const int dw = warp - 4;
        const int g = lane >> 2, t4 = lane & 3, odd = g & 1;
        int stage = 0;
        uint32_t phase = 0;
        const uint32_t full0 = CG == 2 ? cluster_addr(&full[0], 0) : 0;
        const auto first_tile = [&](int64_t t) {
            return (static_cast<int>(t % num_n) * CG + static_cast<int>(rank)) * 16 + dw * 4;
        };
        Codes now, next;
        int64_t t = unit;
        int c = 0;
        if (t < tiles) load_codes<GROUPS>(p, first_tile(t), 0, lane, now);
        while (t < tiles && !*abort_flag) {
            int64_t tn = t;
            int cn = c + 1;
            if (cn == p.chunks) {
                cn = 0;
                tn = t + units;
            }
            if (tn < tiles) load_codes<GROUPS>(p, first_tile(tn), cn, lane, next);
            bool ok = true;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && c * 128 + kStepK >= p.k) break;
                if (!(ok = mbar_wait(&empty[stage], phase ^ 1))) break;
                const uint32_t a = smem_u32(smem + stage * S::kStageBytes);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w0 = h ? now.v[i].z : now.v[i].x, w1 = h ? now.v[i].w : now.v[i].y;
                    // Groups of the two words' inputs within the chunk.
                    const int q0 = GROUPS == 4 ? 2 * h : GROUPS == 2 ? h : 0, q1 = GROUPS == 4 ? 2 * h + 1 : q0;
                    const uint32_t z0 = (now.z[i] >> (8 * q0)) & 0xffu, z1 = (now.z[i] >> (8 * q1)) & 0xffu;
                    // Row r's 16-byte segment s lies at s ^ (r % 8). Rows of odd g store their second
                    // word first, so the two rows that share a store's phase use different banks.
                    const uint32_t row = a + static_cast<uint32_t>(((dw * 4 + i) * 8 + g) * 128);
                    const uint32_t sa = static_cast<uint32_t>((4 * odd + t4) ^ g), sb = static_cast<uint32_t>((4 * (odd ^ 1) + t4) ^ g);
                    st_shared_v4(row + sa * 16, dequant_word<BF16>(odd ? w1 : w0, odd ? z1 : z0));
                    st_shared_v4(row + sb * 16, dequant_word<BF16>(odd ? w0 : w1, odd ? z0 : z1));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) mbar_arrive(&full[stage]);
                    else mbar_arrive_cluster(full0 + static_cast<uint32_t>(stage * sizeof(uint64_t)));
                }
                if (++stage == S::kStages) { stage = 0; phase ^= 1; }
            }
            if (!ok) {
                gave_up(p, abort_flag);
                break;
            }
            now = next;
            t = tn;
            c = cn;
        }
    } else {
        regs_inc<184>();
        // ---- sums and epilogue: thread = one output, kCols activation rows --------------------
        const int quad = warp & 3, half = (warp - 8) / 4;
        int buf = 0;
        uint32_t acc_phase = 0;
        const uint32_t acc_empty0 = CG == 2 ? cluster_addr(&acc_empty[0], 0) : 0;
        for (int64_t t = unit; t < tiles && !*abort_flag; t += units) {
            const int m0 = static_cast<int>(t / num_n) * BN + half * kCols;
            const int n = (static_cast<int>(t % num_n) * CG + static_cast<int>(rank)) * 128 + quad * 32 + lane;
            const bool n_ok = n < p.n;
            // This output's scales: GROUPS per chunk, the next group's loaded a group ahead.
            const __half* sc = p.scales + (static_cast<int64_t>(n / 8) * p.chunks * 8 + n % 8) * GROUPS;
            float d = n_ok ? __half2float(__ldg(sc)) : 0.0f;
            uint64_t acc[kCols / 2];
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) acc[j] = 0;
            bool ok = true;
#pragma unroll 1
            for (int gi = 0; gi < groups; ++gi) {
                const float d_now = d;
                if (gi + 1 < groups && n_ok)
                    d = __half2float(__ldg(sc + static_cast<int64_t>((gi + 1) / GROUPS) * 8 * GROUPS + (gi + 1) % GROUPS));
                ok = mbar_wait(&acc_full[buf], acc_phase);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                                       static_cast<uint32_t>(buf * BN + half * kCols);
                const uint64_t d2 = pack_f2(make_float2(d_now, d_now));
#pragma unroll
                for (int q = 0; q < kCols / 32; ++q) {
                    uint32_t r[32];
                    tmem_ld32(taddr + q * 32, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) fma2(acc[q * 16 + j], d2, r[2 * j], r[2 * j + 1]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) mbar_arrive(&acc_empty[buf]);
                    else mbar_arrive_cluster(acc_empty0 + static_cast<uint32_t>(buf * sizeof(uint64_t)));
                }
                if (++buf == S::kBufs) { buf = 0; acc_phase ^= 1; }
            }
            if (!ok) {
                gave_up(p, abort_flag);
                break;
            }
            const float bias = p.bias && n_ok ? __ldg(p.bias + n) : 0.0f;
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                const int row = m0 + j;
                if (row >= p.m || !n_ok) continue;
                const float2 pair = unpack_f2(acc[j / 2]);
                float v = j % 2 ? pair.y : pair.x;
                if (P == 2) v *= __ldg(p.row_scale + row);
                v = q4_act(v + bias, p.act) * p.scale;
                const int64_t at = static_cast<int64_t>(row) * p.ldc + n;
                if (p.accumulate) v += q4_load(p.c, p.c_type, at);
                q4_store(p.c, p.c_type, at, v);
            }
            __syncwarp();
        }
    }

    tc_fence_before();
    __syncthreads();
    // A pair's CTAs leave together: the first CTA's products read the second's shared memory and
    // write its TMEM, and the second's loads signal the first's barriers.
    if (CG == 2) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if (CG == 1) tmem_dealloc(tmem_base, S::kTmemCols);
        else tmem_dealloc_pair(tmem_base, S::kTmemCols);
    }
}

// The rows of a as the products read them: one block per row. f32: two fp16 planes and the row's
// power of two. 16-bit types: a copy with rows that start on 16-byte boundaries.
constexpr int kPrepThreads = 256;

__global__ void __launch_bounds__(kPrepThreads) q4_split_kernel(const float* a, int64_t lda, int m, int k, __half* planes,
                                                                int64_t ld, float* row_scale) {
    const int64_t row = blockIdx.x;
    const float* src = a + row * lda;
    __shared__ float tops[kPrepThreads / 32];
    float top = 0.0f;  // fmaxf passes NaNs over
    for (int i = threadIdx.x; i < k; i += kPrepThreads) top = fmaxf(top, fabsf(__ldg(src + i)));
#pragma unroll
    for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    for (int w = 0; w < kPrepThreads / 32; ++w) top = fmaxf(top, tops[w]);
    // 2^e with the largest value 2^e times a number in [2^14, 2^15). e stops at -126, so that 2^-e
    // stays a normal f32: a row below 2^-112 keeps its values to 2^-150. An infinity's exponent makes e
    // 114, which holds every finite value below 2^14 and leaves the infinity one.
    const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -126);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    if (threadIdx.x == 0) row_scale[row] = up;
    __half* hi = planes + row * ld;
    __half* lo = hi + static_cast<int64_t>(m) * ld;
    for (int i = threadIdx.x; i < ld; i += kPrepThreads) {
        const float x = i < k ? __ldg(src + i) * down : 0.0f;
        const __half h = __float2half_rn(x);
        hi[i] = h;
        lo[i] = __float2half_rn(x - __half2float(h));
    }
}

__global__ void __launch_bounds__(kPrepThreads) q4_align_kernel(const uint16_t* a, int64_t lda, int k, uint16_t* out,
                                                                int64_t ld) {
    const int64_t row = blockIdx.x;
    for (int i = threadIdx.x; i < ld; i += kPrepThreads) out[row * ld + i] = i < k ? __ldg(a + row * lda + i) : uint16_t(0);
}

template <bool BF16, int P, int BN, int CG, int GROUPS>
cudaError_t launch_gemm(const void* a, int64_t lda, const GemmParams& p, int sms, cudaStream_t stream) {
    using S = Shape<P, BN, CG>;
    static DeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!once.done(dev)) {
        if ((e = cudaFuncSetAttribute(q4_gemm_kernel<BF16, P, BN, CG, GROUPS>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes)) != cudaSuccess)
            return e;
        once.mark(dev);
    }
    CUtensorMap map;
    if (!encode_map_2d(&map, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a,
                       static_cast<uint64_t>(p.k), static_cast<uint64_t>(p.m) * P, static_cast<uint64_t>(lda) * 2, kStepK,
                       S::kBRows, CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    const int64_t tiles = static_cast<int64_t>((p.m + BN - 1) / BN) * ((p.n + CG * 128 - 1) / (CG * 128));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CG * static_cast<unsigned>(std::min<int64_t>(tiles, sms / CG)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CG == 2 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, q4_gemm_kernel<BF16, P, BN, CG, GROUPS>, map, p);
}

template <bool BF16, int P, int BN, int CG>
cudaError_t launch_group(const void* a, int64_t lda, const GemmParams& p, int group, int sms, cudaStream_t stream) {
    if (group == 32) return launch_gemm<BF16, P, BN, CG, 4>(a, lda, p, sms, stream);
    if (group == 64) return launch_gemm<BF16, P, BN, CG, 2>(a, lda, p, sms, stream);
    return launch_gemm<BF16, P, BN, CG, 1>(a, lda, p, sms, stream);
}

template <bool BF16, int P>
cudaError_t launch_shape(const void* a, int64_t lda, const GemmParams& p, int group, int sms, cudaStream_t stream) {
    // Pairs on 256 x 256 tiles where they fill the GPU, else smaller tiles on single CTAs.
    const auto tiles = [&](int bn, int features) {
        return static_cast<int64_t>((p.m + bn - 1) / bn) * ((p.n + features - 1) / features);
    };
    if (tiles(256, 256) * 2 >= sms) return launch_group<BF16, P, 256, 2>(a, lda, p, group, sms, stream);
    if (tiles(128, 128) >= sms) return launch_group<BF16, P, 128, 1>(a, lda, p, group, sms, stream);
    return launch_group<BF16, P, 64, 1>(a, lda, p, group, sms, stream);
}

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace

size_t q4_gemm_workspace(const Q4Args& g) {
    const size_t m = static_cast<size_t>(g.m), ld = round_up(static_cast<size_t>(g.w->k), 8);
    if (g.a_type == kQ4F32) return round_up(2 * m * ld * sizeof(__half), 256) + m * sizeof(float);
    const bool aligned = reinterpret_cast<uintptr_t>(g.a) % 16 == 0 && g.lda % 8 == 0;
    return aligned ? 0 : m * ld * 2;
}

cudaError_t q4_linear_gemm(const Q4Args& g, void* workspace, cudaStream_t stream) {
    GemmParams p;
    p.codes = g.w->codes;
    p.scales = g.w->scales;
    p.zeros = g.w->zeros;
    p.n = g.w->n;
    p.k = g.w->k;
    p.chunks = g.w->chunks;
    p.tiles8 = (g.w->n + 15) / 16 * 2;
    p.m = g.m;
    p.row_scale = nullptr;
    p.bias = g.bias;
    p.act = g.act;
    p.scale = g.scale;
    p.accumulate = g.accumulate;
    p.c = g.c;
    p.c_type = g.c_type;
    p.ldc = g.ldc;
    p.error = g.error;
    const int64_t ld = static_cast<int64_t>(round_up(static_cast<size_t>(p.k), 8));
    if (g.a_type == kQ4F32) {
        __half* planes = static_cast<__half*>(workspace);
        float* rs = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                             round_up(2 * static_cast<size_t>(p.m) * ld * sizeof(__half), 256));
        q4_split_kernel<<<p.m, kPrepThreads, 0, stream>>>(static_cast<const float*>(g.a), g.lda, p.m, p.k, planes, ld, rs);
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
        p.row_scale = rs;
        return launch_shape<false, 2>(planes, ld, p, g.w->group, g.sms, stream);
    }
    const void* a = g.a;
    int64_t lda = g.lda;
    if (workspace) {
        q4_align_kernel<<<p.m, kPrepThreads, 0, stream>>>(static_cast<const uint16_t*>(g.a), g.lda, p.k,
                                                          static_cast<uint16_t*>(workspace), ld);
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
        a = workspace;
        lda = ld;
    }
    return g.a_type == kQ4BF16 ? launch_shape<true, 1>(a, lda, p, g.w->group, g.sms, stream)
                               : launch_shape<false, 1>(a, lda, p, g.w->group, g.sms, stream);
}

}  // namespace telmo
