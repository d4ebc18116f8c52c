// q4_rows.cuh -- products of few activation rows with 4-bit weights.
//
//   c[r, o] = (accumulate ? c[r, o] : 0) + scale * act(s_r sum_g d[o, g] S[r, o, g] + bias[o]),
//   S[r, o, g] = sum over the inputs i of group g of a[r, i] (code[o, i] - zero[o, g]).
//
// A product of a few rows reads each weight once and is bound by those bytes: n k / 2 of codes
// and 2 n k / group of scales. What stands against the memory's rate is the work of taking the
// codes apart, so they go to the matrix pipe (mma.sync m16n8k16, f32 accumulators) as the
// integers code - zero, which bf16 and fp16 hold exactly: one logic operation makes the pair
// 0x4300 | code (bf16 128 + code; fp16: 0x6400, 1024 + code) and one subtraction of 128 + zero
// leaves two exact operands. tcgen05 would need the operands in shared memory first and a tile of
// 128 outputs by 8 rows leaves its accumulators almost empty; here they go from the load to the
// instruction in registers. The scale multiplies the group's f32 sum, so weights are never
// rounded.
//
// Activations: bf16 and fp16 are operands as they are. An f32 activation becomes three bf16
// parts of 8 significant bits by truncation, x = hi + mid + lo, which is exact (24 bits; parts
// below 2^-126 vanish), and three products are summed. More than eight f32 rows come as two fp16 planes
// (q4_split) and a power of two per row s_r, two instructions.
//
// A warp takes 16 or 32 outputs and a share of the 128-input chunks, with its next chunks under way
// while it works on one: in registers (q4_rows_kernel, rows of any alignment and f32), or in a ring
// in shared memory together with the activations (q4_rows_staged_kernel). Warps that share outputs
// add up in shared memory, in order. Where n gives too few blocks, the blocks of a cluster take a
// share of the chunks each and add up through distributed shared memory, in rank order (24 rows,
// 4096 -> 4096 in groups of 64: 10.7 us, 22.2 without).
//
// Measured (captured, weights from memory): 8 rows of bf16, 4096 -> 4096: 8.3 us (1.1 TB/s of codes and
// scales); 24 rows of f16, 11009 -> 4096 with zero points: 21.2 us with the copy of its rows, 1.1 TB/s; 8 rows of
// f32, 4096 -> 8192: 17.5 us, 1.0 TB/s (every block reads and splits the activations for itself, and three
// products take a step). A launch, the first loads' way and the sums are 3 us of it; then the chunks'
// latencies: up to 24 rows an SM holds two blocks, 16 warps at up to 128 registers, beyond that one, and about
// 35% of its issue slots are used.
#pragma once

#include "ptx.cuh"
#include "q4_async.cuh"
#include "q4_device.cuh"

#include <algorithm>
#include <type_traits>

namespace telmo {

namespace q4rows {

enum RowsMode : int {
    kModeF16 = 0,     // fp16 activations
    kModeBF16 = 1,    // bf16 activations
    kModeF32 = 2,     // f32 activations, three instructions
    kModePlanes = 3,  // two fp16 planes, two instructions
};

constexpr int kWarps = 8;

struct RowsParams {
    const uint4* codes;
    const __half* scales;
    const uint8_t* zeros;
    int n, k, chunks;
    const void* a;
    int64_t lda;
    int m;
    bool vec;                // rows of a start on 16-byte boundaries
    const float* row_scale;  // [m] with planes
    bool planes;             // a was made by the kernel before
    const float* bias;
    int act;
    float scale;
    int accumulate;
    void* c;
    int c_type;
    int64_t ldc;
    int splits;     // blocks of a cluster that share the chunks
    int split_chunks;
};

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight activations of one row from `src` on, `left` of which (may be negative) lie in the matrix; 0 for
// the others. `vec`: src is 16-byte aligned.
__device__ __forceinline__ uint4 load_a16(const uint16_t* src, bool row_ok, bool vec, int left) {
    if (!row_ok) return make_uint4(0, 0, 0, 0);
    if (vec && left >= 8) return __ldg(reinterpret_cast<const uint4*>(src));
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? __ldg(src + j) : 0u;
    return make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16), v[6] | (v[7] << 16));
}

template <int N>
__device__ __forceinline__ void load_a32(const float* src, bool row_ok, bool vec, int left, float (&x)[N]) {
    if (row_ok && vec && left >= N) {
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
            const float4 u = __ldg(reinterpret_cast<const float4*>(src) + j);
            x[4 * j] = u.x;
            x[4 * j + 1] = u.y;
            x[4 * j + 2] = u.z;
            x[4 * j + 3] = u.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = row_ok && j < left ? __ldg(src + j) : 0.0f;
}

// f32 values as pairs of bf16 parts. Truncation leaves 8 of the 24 significant bits to each part
// and every difference is exact. An infinity or a NaN makes its other parts NaN, so the row's outputs
// are not finite.
__device__ __forceinline__ float bf16_rest(float x) {
    return __fsub_rn(x, __uint_as_float(__float_as_uint(x) & 0xffff0000u));
}
__device__ __forceinline__ uint32_t bf16_tops(float x0, float x1) {
    return __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
}
template <int N>
__device__ __forceinline__ void split_parts(const float (&x)[N], uint32_t (&hi)[N / 2], uint32_t (&mid)[N / 2],
                                            uint32_t (&lo)[N / 2]) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        const float r0 = bf16_rest(x[2 * j]), r1 = bf16_rest(x[2 * j + 1]);
        hi[j] = bf16_tops(x[2 * j], x[2 * j + 1]);
        mid[j] = bf16_tops(r0, r1);
        lo[j] = bf16_tops(bf16_rest(r0), bf16_rest(r1));
    }
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr)
                 : "memory");
    return v;
}

// A chunk's codes, scales and zero points of this lane's two rows, as loaded.
template <int GROUPS, bool ZEROS>
struct Chunk {
    uint4 words[2];
    uint32_t d[2][GROUPS == 4 ? 2 : 1];  // f16 pairs
    uint32_t z[2];                       // bytes
};

template <int GROUPS, bool ZEROS>
__device__ __forceinline__ void load_chunk(Chunk<GROUPS, ZEROS>& x, const uint4* codes, const uint8_t* scales,
                                           const uint8_t* zeros) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        // Tiles of the same 128 outputs follow one another: 512 bytes of codes, 16 GROUPS of scales.
        x.words[r] = __ldg(codes + r * 32);
        const uint8_t* s = scales + r * (8 * GROUPS * 2);
        if (GROUPS == 4) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(s));
            x.d[r][0] = v.x;
            x.d[r][GROUPS == 4 ? 1 : 0] = v.y;
        } else if (GROUPS == 2) {
            x.d[r][0] = __ldg(reinterpret_cast<const uint32_t*>(s));
        } else {
            x.d[r][0] = __ldg(reinterpret_cast<const uint16_t*>(s));
        }
        if (ZEROS) {
            const uint8_t* z = zeros + r * (8 * GROUPS);
            if (GROUPS == 4) x.z[r] = __ldg(reinterpret_cast<const uint32_t*>(z));
            else if (GROUPS == 2) x.z[r] = __ldg(reinterpret_cast<const uint16_t*>(z));
            else x.z[r] = __ldg(z);
        }
    }
}

// The loops over a chunk's four words stay rolled: unrolled, a warp runs through several KB of code a
// few times only, and fetching it took longer than running it (32 rows, 4096 -> 8192: 36 us unrolled).
// So scales and zero points are taken from the low end of their registers and shifted down.
template <int GROUPS>
__device__ __forceinline__ float next_scale(uint32_t (&d)[GROUPS == 4 ? 2 : 1]) {
    const float v = __half2float(__ushort_as_half(static_cast<unsigned short>(d[0] & 0xffffu)));
    if (GROUPS == 4) {
        d[0] = __funnelshift_r(d[0], d[GROUPS == 4 ? 1 : 0], 16);
        d[GROUPS == 4 ? 1 : 0] >>= 16;
    } else if (GROUPS == 2) {
        d[0] >>= 16;
    }
    return v;
}

// part times the group's scales onto acc, and part to zero.
template <int GROUPS, int R, int CB>
__device__ __forceinline__ void add_group(float (&acc)[R][CB][4], float (&part)[R][CB][4],
                                          uint32_t (&d)[2 * R][GROUPS == 4 ? 2 : 1]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float d0 = next_scale<GROUPS>(d[2 * r]), d1 = next_scale<GROUPS>(d[2 * r + 1]);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            acc[r][cb][0] = fmaf(d0, part[r][cb][0], acc[r][cb][0]);
            acc[r][cb][1] = fmaf(d0, part[r][cb][1], acc[r][cb][1]);
            acc[r][cb][2] = fmaf(d1, part[r][cb][2], acc[r][cb][2]);
            acc[r][cb][3] = fmaf(d1, part[r][cb][3], acc[r][cb][3]);
            part[r][cb][0] = part[r][cb][1] = part[r][cb][2] = part[r][cb][3] = 0.0f;
        }
    }
}

// Two output rows' words as the A operands of two instructions.
template <bool BF16>
__device__ __forceinline__ void operands(uint32_t x0, uint32_t x1, uint32_t z0, uint32_t z1, uint32_t (&a)[2][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        a[h][0] = code_pair<BF16>(x0, 2 * h, z0);
        a[h][1] = code_pair<BF16>(x1, 2 * h, z1);
        a[h][2] = code_pair<BF16>(x0, 2 * h + 1, z0);
        a[h][3] = code_pair<BF16>(x1, 2 * h + 1, z1);
    }
}

// The sums of a block's shares, and of a cluster's blocks, and the epilogue, four outputs a thread at a
// time. `sums`: [share][column][output of the block] in shared memory, written and synchronised.
template <bool SCALED, int SHARES, int OUTS, int COLS>
__device__ __forceinline__ void finish_block(const RowsParams& p, float* sums, int64_t out0, int split) {
    constexpr int kAll = OUTS * COLS / 4;
    float4* s4 = reinterpret_cast<float4*>(sums);
    const auto add = [](float4& a, const float4& b) {
        a.x += b.x;
        a.y += b.y;
        a.z += b.z;
        a.w += b.w;
    };
    const auto finish = [&](int e, const float4& s) {
        const int row = e / (OUTS / 4);
        if (row >= p.m) return;
        const float rs = SCALED ? p.row_scale[row] : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t out = out0 + e % (OUTS / 4) * 4 + j;
            if (out >= p.n) return;
            float v = (j == 0 ? s.x : j == 1 ? s.y : j == 2 ? s.z : s.w) * rs;
            if (p.bias) v += __ldg(p.bias + out);
            v = q4_act(v, p.act) * p.scale;
            const int64_t at = static_cast<int64_t>(row) * p.ldc + out;
            if (p.accumulate) v += q4_load(p.c, p.c_type, at);
            q4_store(p.c, p.c_type, at, v);
        }
    };
    for (int e = threadIdx.x; e < kAll; e += 32 * kWarps) {
        float4 v = s4[e];
#pragma unroll
        for (int s = 1; s < SHARES; ++s) add(v, s4[s * kAll + e]);
        if (p.splits == 1) finish(e, v);
        else s4[e] = v;  // into the first share's place
    }
    if (p.splits == 1) return;
    __syncwarp();
    cluster_sync();
    // Each block of the cluster finishes a part of the outputs. All blocks' sums are asked for at once.
    for (int e = split * 32 * kWarps + threadIdx.x; e < kAll; e += p.splits * 32 * kWarps) {
        float4 v[8];
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s < p.splits) v[s] = ld_cluster_v4(cluster_addr(s4 + e, static_cast<uint32_t>(s)));
#pragma unroll
        for (int s = 1; s < 8; ++s)
            if (s < p.splits) add(v[0], v[s]);
        finish(e, v[0]);
    }
    __syncwarp();
    cluster_sync();  // the other blocks have read this one's sums
}

// Up to eight rows: a block's warps share the chunks of 16 outputs.
template <int MODE, int GROUPS, bool ZEROS>
__global__ void __launch_bounds__(32 * kWarps) q4_rows_kernel(const RowsParams p) {
    constexpr bool BF16 = MODE != kModeF16;
    constexpr int kParts = MODE == kModeF32 ? 3 : 1;
    constexpr int kWordsPerGroup = 4 / GROUPS;
    constexpr int kOuts = 16, kCols = 8;  // outputs and activation rows of the block
    __shared__ __align__(16) float sums[kWarps * kOuts * kCols];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int g = lane >> 2, t = lane & 3;
    const int64_t out0 = static_cast<int64_t>(blockIdx.x) * kOuts;
    int c = warp;
    // The compiler is not to know that rows are 0..7: with that it orders the loads of rows off 16-byte boundaries
    // worse (3 rows of bf16, 4096 -> 8192: 15.4 us, 13.8 so).
    int row = g;
    asm("" : "+r"(row));

    float acc[1][1][4] = {}, part[1][1][4] = {};
    if (c < p.chunks) {
        const int64_t first = q4_tile(out0 / 8, p.chunks, c);
        const uint4* codes = p.codes + first * 32 + lane;
        const uint8_t* scales = reinterpret_cast<const uint8_t*>(p.scales) + (first * 8 + g) * GROUPS * 2;
        const uint8_t* zeros = ZEROS ? p.zeros + (first * 8 + g) * GROUPS : nullptr;
        Chunk<GROUPS, ZEROS> now, next;
        load_chunk(now, codes, scales, zeros);
        next = now;
        for (; c < p.chunks; c += kWarps) {
            codes += kWarps * (16 * 32);
            scales += kWarps * (16 * 8 * GROUPS * 2);
            if (ZEROS) zeros += kWarps * (16 * 8 * GROUPS);
            if (c + kWarps < p.chunks) load_chunk(next, codes, scales, zeros);

#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
                const int i = c * 128 + 32 * w + 8 * t;
                uint32_t b[kParts][4];
                if (MODE == kModeF32) {
                    float x[8];
                    load_a32<8>(static_cast<const float*>(p.a) + row * p.lda + i, row < p.m, p.vec, p.k - i, x);
                    split_parts<8>(x, b[0], b[kParts > 1 ? 1 : 0], b[kParts > 2 ? 2 : 0]);
                } else {
                    const uint4 v = load_a16(static_cast<const uint16_t*>(p.a) + row * p.lda + i, row < p.m, p.vec, p.k - i);
                    b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w;
                }
                uint32_t a[2][4];
                operands<BF16>(now.words[0].x, now.words[1].x, code_base<BF16>(ZEROS ? now.z[0] & 0xffu : 8u),
                               code_base<BF16>(ZEROS ? now.z[1] & 0xffu : 8u), a);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int pl = 0; pl < kParts; ++pl)
                        mma_16816<BF16>(part[0][0], a[h], b[pl][2 * h], b[pl][2 * h + 1]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    now.words[r].x = now.words[r].y;
                    now.words[r].y = now.words[r].z;
                    now.words[r].z = now.words[r].w;
                }
                if ((w + 1) % kWordsPerGroup == 0) {
                    add_group<GROUPS, 1, 1>(acc, part, now.d);
                    if (ZEROS) {
                        now.z[0] >>= 8;
                        now.z[1] >>= 8;
                    }
                }
            }
            now = next;
        }
    }

    // sums[warp][column][output of the block]
#pragma unroll
    for (int j = 0; j < 4; ++j)
        sums[(warp * kCols + 2 * t + (j & 1)) * kOuts + g + 8 * (j >> 1)] = acc[0][0][j];
    __syncthreads();
    finish_block<false, kWarps, kOuts, kCols>(p, sums, out0, 0);
}

// Rows that start on 16-byte boundaries (16-bit activations, or planes): activations and codes come
// through a ring of chunks in shared memory (cp.async), filled by the warps of a share together.
// The rows' pitch of 320 bytes puts the two rows of an 8-lane phase on different banks.
constexpr int kRing = 3;
constexpr int kPitch = 320;

template <int MODE, int R, int CB>
struct Staged {
    static constexpr int kParts = MODE == kModePlanes ? 2 : 1;
    static constexpr int kActBytes = kParts * 8 * CB * kPitch;
    static constexpr int kCodeBytes = 2 * R * 512;  // of one warp
    // Warps side by side on outputs: they share the activations; the others share the chunks.
    static constexpr int kRowWarps = CB == 1 ? 2 : 4;
    static constexpr int kShares = kWarps / kRowWarps;
    static constexpr int kStageBytes = kActBytes + kRowWarps * kCodeBytes;
    static constexpr int kSmem = std::max(kShares * kRing * kStageBytes, kWarps * 16 * R * 8 * CB * 4);
    // Blocks per SM, which bounds the registers (24 rows, 4096 -> 8192: 13.9 us with two, 15.0 with one; two of
    // 32 rows spill).
    static constexpr int kBlocks = CB * kParts <= 3 ? 2 : 1;
};

template <int MODE, int GROUPS, bool ZEROS, int R, int CB>
__global__ void __launch_bounds__(32 * kWarps, Staged<MODE, R, CB>::kBlocks) q4_rows_staged_kernel(const RowsParams p) {
    using S = Staged<MODE, R, CB>;
    constexpr bool BF16 = MODE == kModeBF16;
    constexpr int kParts = S::kParts, kWordsPerGroup = 4 / GROUPS, kCols = 8 * CB;
    extern __shared__ __align__(128) uint8_t ring[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int g = lane >> 2, t = lane & 3;
    constexpr int row_warps = S::kRowWarps, shares = S::kShares;
    const int rw = warp % row_warps, share = warp / row_warps;
    const int split = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int block = p.splits > 1 ? blockIdx.x / p.splits : blockIdx.x;
    const int64_t out0 = static_cast<int64_t>(block) * (16 * R * row_warps);
    const int64_t tile0 = out0 / 8 + rw * 2 * R;
    const bool live = tile0 * 8 < p.n;  // tiles past the last 128 outputs do not exist
    const int c_end = min(p.chunks, (split + 1) * p.split_chunks);
    const int c0 = split * p.split_chunks + share;

    constexpr int stage_bytes = S::kStageBytes;
    const uint32_t mine = smem_u32(ring) + static_cast<uint32_t>(share * kRing * stage_bytes);
    const int64_t first = q4_tile(live ? tile0 : 0, p.chunks, 0);
    const uint4* codes = p.codes + first * 32 + lane;
    const uint8_t* scales = reinterpret_cast<const uint8_t*>(p.scales) + (first * 8 + g) * GROUPS * 2;
    const uint8_t* zeros = ZEROS ? p.zeros + (first * 8 + g) * GROUPS : nullptr;

    // Start the copies of chunk c into a ring place: the codes, and 16 pieces of 16 bytes to each row of
    // activations.
    const auto fetch_codes = [&](int c, int place) {
        if (c < c_end && live) {
            const uint32_t to = mine + static_cast<uint32_t>(place * stage_bytes + S::kActBytes + rw * S::kCodeBytes + lane * 16);
#pragma unroll
            for (int r = 0; r < 2 * R; ++r)
                cp_async16(to + r * 512, codes + static_cast<int64_t>(c) * 512 + r * 32, 16);
        }
    };
    const auto fetch_rows = [&](int c, int place) {
        if (c < c_end) {
            const uint32_t at = mine + static_cast<uint32_t>(place * stage_bytes);
            for (int e = rw * 32 + lane; e < kParts * kCols * 16; e += row_warps * 32) {
                const int row = e / 16, piece = e % 16, m = row % kCols;
                const int left = m < p.m ? max(0, min(8, p.k - c * 128 - piece * 8)) : 0;
                const uint16_t* src = static_cast<const uint16_t*>(p.a);
                if (left) src += (static_cast<int64_t>(row / kCols) * p.m + m) * p.lda + c * 128 + piece * 8;
                cp_async16(at + row * kPitch + piece * 16, src, left * 2);
            }
        }
        cp_commit();  // of both; an empty group where there is no such chunk, so that the counts stay even
    };
    const auto load_scales = [&](int c, uint32_t (&d)[2 * R][GROUPS == 4 ? 2 : 1], uint32_t (&z)[2 * R]) {
#pragma unroll
        for (int r = 0; r < 2 * R; ++r) {
            const uint8_t* s = scales + static_cast<int64_t>(c) * (16 * 8 * GROUPS * 2) + r * (8 * GROUPS * 2);
            if (GROUPS == 4) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(s));
                d[r][0] = v.x;
                d[r][GROUPS == 4 ? 1 : 0] = v.y;
            } else if (GROUPS == 2) {
                d[r][0] = __ldg(reinterpret_cast<const uint32_t*>(s));
            } else {
                d[r][0] = __ldg(reinterpret_cast<const uint16_t*>(s));
            }
            if (ZEROS) {
                const uint8_t* y = zeros + static_cast<int64_t>(c) * (16 * 8 * GROUPS) + r * (8 * GROUPS);
                z[r] = GROUPS == 4   ? __ldg(reinterpret_cast<const uint32_t*>(y))
                       : GROUPS == 2 ? __ldg(reinterpret_cast<const uint16_t*>(y))
                                     : __ldg(y);
            }
        }
    };

    float acc[R][CB][4] = {}, part[R][CB][4] = {};
    uint32_t d_next[2 * R][GROUPS == 4 ? 2 : 1], z_next[2 * R] = {};
    for (int i = 0; i < kRing - 1; ++i) fetch_codes(c0 + i * shares, i);
    if (c0 < c_end) load_scales(c0, d_next, z_next);
    wait_for_previous();
    for (int i = 0; i < kRing - 1; ++i) fetch_rows(c0 + i * shares, i);
    int place = 0;
    for (int c = c0; c < c_end; c += shares) {
        uint32_t d[2 * R][GROUPS == 4 ? 2 : 1], z[2 * R];
#pragma unroll
        for (int r = 0; r < 2 * R; ++r) {
            d[r][0] = d_next[r][0];
            if (GROUPS == 4) d[r][GROUPS == 4 ? 1 : 0] = d_next[r][GROUPS == 4 ? 1 : 0];
            z[r] = z_next[r];
        }
        cp_wait<kRing - 2>();
        // The share's copies are complete, and its warps are done with the place that is filled next.
        asm volatile("bar.sync %0, %1;" ::"r"(1 + share), "r"(32 * row_warps) : "memory");
        const int ahead = place == 0 ? kRing - 1 : place - 1;
        fetch_codes(c + (kRing - 1) * shares, ahead);
        fetch_rows(c + (kRing - 1) * shares, ahead);
        if (c + shares < c_end) load_scales(c + shares, d_next, z_next);
        const uint32_t at = mine + static_cast<uint32_t>(place * stage_bytes);
        const uint32_t acts = at + static_cast<uint32_t>(g * kPitch + t * 16);
        const uint32_t mine_codes = at + S::kActBytes + rw * S::kCodeBytes + lane * 16;
        if (++place == kRing) place = 0;
        if (!live) continue;
#pragma unroll 1
        for (int w = 0; w < 4; ++w) {
            uint32_t a[R][2][4];
#pragma unroll
            for (int r = 0; r < R; ++r)
                operands<BF16>(ld_shared_u32(mine_codes + (2 * r) * 512 + w * 4), ld_shared_u32(mine_codes + (2 * r + 1) * 512 + w * 4),
                               code_base<BF16>(ZEROS ? z[2 * r] & 0xffu : 8u), code_base<BF16>(ZEROS ? z[2 * r + 1] & 0xffu : 8u), a[r]);
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int pl = 0; pl < kParts; ++pl) {
                    const uint4 b = ld_shared_v4(acts + (pl * kCols + cb * 8) * kPitch + w * 64);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        mma_16816<BF16>(part[r][cb], a[r][0], b.x, b.y);
                        mma_16816<BF16>(part[r][cb], a[r][1], b.z, b.w);
                    }
                }
            if ((w + 1) % kWordsPerGroup == 0) {
                add_group<GROUPS, R, CB>(acc, part, d);
                if (ZEROS)
#pragma unroll
                    for (int r = 0; r < 2 * R; ++r) z[r] >>= 8;
            }
        }
    }
    cp_wait<0>();
    __syncthreads();  // the ring's bytes now hold the sums
    float* sums = reinterpret_cast<float*>(ring);
    const int outs = 16 * R * row_warps;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sums[(share * kCols + 8 * cb + 2 * t + (j & 1)) * outs + rw * 16 * R + 16 * r + g + 8 * (j >> 1)] = acc[r][cb][j];
    __syncthreads();
    finish_block<MODE == kModePlanes, S::kShares, 16 * R * S::kRowWarps, kCols>(p, sums, out0, split);
}

// `outs`: outputs of a block, or of a cluster of p.splits blocks.
inline cudaError_t rows_launch(void (*kernel)(RowsParams), const RowsParams& p, int outs, size_t smem, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((p.n + outs - 1) / outs) * p.splits);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    add_attributes(cfg, attr, p.splits, p.planes);
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int MODE, int GROUPS, bool ZEROS, int R, int CB>
cudaError_t launch_staged(const RowsParams& p, cudaStream_t stream) {
    using S = Staged<MODE, R, CB>;
    static DeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!once.done(dev)) {
        e = cudaFuncSetAttribute(q4_rows_staged_kernel<MODE, GROUPS, ZEROS, R, CB>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e != cudaSuccess) return e;
        once.mark(dev);
    }
    return rows_launch(q4_rows_staged_kernel<MODE, GROUPS, ZEROS, R, CB>, p, 16 * R * S::kRowWarps, S::kSmem, stream);
}

template <int MODE, int GROUPS, bool ZEROS>
cudaError_t launch_direct(const RowsParams& p, cudaStream_t stream) {
    return rows_launch(q4_rows_kernel<MODE, GROUPS, ZEROS>, p, 16, 0, stream);
}

// Calls f with the group's and the zero points' constants.
template <typename F>
cudaError_t by_group(const RowsParams& p, int group, F f) {
    using std::integral_constant;
    if (p.zeros) {
        if (group == 32) return f(integral_constant<int, 4>(), std::true_type());
        if (group == 64) return f(integral_constant<int, 2>(), std::true_type());
        return f(integral_constant<int, 1>(), std::true_type());
    }
    if (group == 32) return f(integral_constant<int, 4>(), std::false_type());
    if (group == 64) return f(integral_constant<int, 2>(), std::false_type());
    return f(integral_constant<int, 1>(), std::false_type());
}

// Up to 8 rows as they are (q4_rows.cu); up to 32 aligned rows (q4_rows_staged.cu).
cudaError_t launch_small(const RowsParams& p, int mode, int group, cudaStream_t stream);
cudaError_t launch_aligned(const RowsParams& p, int mode, int group, cudaStream_t stream);

}  // namespace q4rows

}  // namespace telmo
