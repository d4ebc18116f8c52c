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
// below 2^-126 vanish), and three products are summed: in three instructions, or for one and two
// rows in one, the parts in columns of their own. More than eight f32 rows come as two fp16 planes
// (q4_split) and a power of two per row s_r, two instructions.
//
// A warp takes 16 R outputs and a share of the 128-input chunks, with the codes of its next chunk
// under way while it works on one. Warps that share outputs add up in shared memory, in order.
// Where n gives too few blocks, the blocks of a cluster take a share of the chunks each and add up
// through distributed shared memory, in rank order.
#pragma once

#include "ptx.cuh"
#include "q4_device.cuh"

#include <algorithm>

namespace telmo {

namespace q4rows {

enum RowsMode : int {
    kModeF16 = 0,        // fp16 activations
    kModeBF16 = 1,       // bf16 activations
    kModeF32 = 2,        // f32 activations, three instructions
    kModeF32Packed = 3,  // f32 activations of one or two rows: part p of row r in column 2 p + r
    kModePlanes = 4,     // two fp16 planes, two instructions
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
    const float* bias;
    int act;
    float scale;
    int accumulate;
    void* c;
    int c_type;
    int64_t ldc;
    int row_warps;  // warps side by side on outputs; kWarps / row_warps share the chunks
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

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// A chunk's codes, scales and zero points of this lane's 2 R rows, as loaded.
template <int GROUPS, bool ZEROS, int R>
struct Chunk {
    uint4 words[2 * R];
    uint32_t d[2 * R][GROUPS == 4 ? 2 : 1];  // f16 pairs
    uint32_t z[2 * R];                       // bytes
};

template <int GROUPS, bool ZEROS, int R>
__device__ __forceinline__ void load_chunk(Chunk<GROUPS, ZEROS, R>& x, const uint4* codes, const uint8_t* scales,
                                           const uint8_t* zeros) {
#pragma unroll
    for (int r = 0; r < 2 * R; ++r) {
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

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) {
    return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w;
}

template <int MODE, int GROUPS, bool ZEROS, int R, int CB>
__global__ void __launch_bounds__(32 * kWarps) q4_rows_kernel(const RowsParams p) {
    constexpr bool BF16 = MODE != kModeF16 && MODE != kModePlanes;
    constexpr bool kPacked = MODE == kModeF32Packed;
    constexpr int kParts = MODE == kModeF32 ? 3 : MODE == kModePlanes ? 2 : 1;
    constexpr int kWordsPerGroup = 4 / GROUPS;
    constexpr int kCols = kPacked ? 2 : 8 * CB;  // activation rows of the block
    constexpr int kPackedRow = 128 + 32;         // a part's 128 values, and what keeps rows off each other's banks
    __shared__ float sums[kWarps * 16 * R * kCols];
    __shared__ __align__(16) uint16_t packed[kPacked ? kWarps * 6 * kPackedRow : 8];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int g = lane >> 2, t = lane & 3;
    const int row_warps = p.row_warps, shares = kWarps / row_warps;
    const int rw = warp % row_warps, share = warp / row_warps;
    const int split = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int block = p.splits > 1 ? blockIdx.x / p.splits : blockIdx.x;
    const int m0 = blockIdx.y * kCols;
    const int64_t out0 = static_cast<int64_t>(block) * (16 * R * row_warps);  // the block's first output
    const int64_t tile0 = out0 / 8 + rw * 2 * R;                              // the warp's first 8-output tile
    const int c_end = min(p.chunks, (split + 1) * p.split_chunks);
    int c = split * p.split_chunks + share;

    float acc[R][CB][4] = {};
    // Tiles past the last 128 outputs do not exist: such a warp has nothing to do.
    if (tile0 * 8 < p.n && c < c_end) {
        const int64_t first = q4_tile(tile0, p.chunks, c);
        const uint4* codes = p.codes + first * 32 + lane;
        const uint8_t* scales = reinterpret_cast<const uint8_t*>(p.scales) + (first * 8 + g) * GROUPS * 2;
        const uint8_t* zeros = ZEROS ? p.zeros + (first * 8 + g) * GROUPS : nullptr;
        Chunk<GROUPS, ZEROS, R> now, next;
        load_chunk(now, codes, scales, zeros);
        next = now;
        for (; c < c_end; c += shares) {
            codes += shares * (16 * 32);
            scales += shares * (16 * 8 * GROUPS * 2);
            if (ZEROS) zeros += shares * (16 * 8 * GROUPS);
            if (c + shares < c_end) load_chunk(next, codes, scales, zeros);

            if (kPacked) {
                // Each lane splits four inputs of each row; lane (g, t) then reads row g % 2 of part g / 2.
                uint16_t* mine = packed + warp * 6 * kPackedRow;
                __syncwarp();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x[4];
                    const int i = c * 128 + lane * 4;
                    load_a32<4>(static_cast<const float*>(p.a) + (m0 + r) * p.lda + i, m0 + r < p.m, p.vec, p.k - i, x);
                    uint32_t parts[3][2];
                    split_parts<4>(x, parts[0], parts[1], parts[2]);
#pragma unroll
                    for (int pl = 0; pl < 3; ++pl)
                        *reinterpret_cast<uint2*>(mine + (pl * 2 + r) * kPackedRow + lane * 4) =
                            make_uint2(parts[pl][0], parts[pl][1]);
                }
                __syncwarp();
            }
#pragma unroll
            for (int q = 0; q < GROUPS; ++q) {
                float part[R][CB][4] = {};
#pragma unroll
                for (int ww = 0; ww < kWordsPerGroup; ++ww) {
                    const int w = q * kWordsPerGroup + ww;
                    const int i = c * 128 + 32 * w + 8 * t;
                    uint32_t b[kParts][CB][4];
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        const int row = m0 + 8 * cb + g;
                        if (MODE == kModeF32) {
                            float x[8];
                            load_a32<8>(static_cast<const float*>(p.a) + row * p.lda + i, row < p.m, p.vec, p.k - i, x);
                            split_parts<8>(x, b[0][cb], b[kParts > 1 ? 1 : 0][cb], b[kParts > 2 ? 2 : 0][cb]);
                        } else if (kPacked) {
                            uint4 v = make_uint4(0, 0, 0, 0);
                            if (g < 6)
                                v = *reinterpret_cast<const uint4*>(packed + (warp * 6 + g) * kPackedRow + 32 * w + 8 * t);
                            b[0][cb][0] = v.x; b[0][cb][1] = v.y; b[0][cb][2] = v.z; b[0][cb][3] = v.w;
                        } else {
#pragma unroll
                            for (int pl = 0; pl < kParts; ++pl) {
                                const uint4 v = load_a16(static_cast<const uint16_t*>(p.a) +
                                                             (row + static_cast<int64_t>(pl) * p.m) * p.lda + i,
                                                         row < p.m, p.vec, p.k - i);
                                b[pl][cb][0] = v.x; b[pl][cb][1] = v.y; b[pl][cb][2] = v.z; b[pl][cb][3] = v.w;
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const uint32_t x0 = word_of(now.words[2 * r], w), x1 = word_of(now.words[2 * r + 1], w);
                        const uint32_t z0 = code_base<BF16>(ZEROS ? (now.z[2 * r] >> (8 * q)) & 0xffu : 8u);
                        const uint32_t z1 = code_base<BF16>(ZEROS ? (now.z[2 * r + 1] >> (8 * q)) & 0xffu : 8u);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t a[4] = {code_pair<BF16>(x0, 2 * h, z0), code_pair<BF16>(x1, 2 * h, z1),
                                                   code_pair<BF16>(x0, 2 * h + 1, z0), code_pair<BF16>(x1, 2 * h + 1, z1)};
#pragma unroll
                            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                                for (int pl = 0; pl < kParts; ++pl)
                                    mma_16816<BF16>(part[r][cb], a, b[pl][cb][2 * h], b[pl][cb][2 * h + 1]);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const auto scale_of = [&](int row) {
                        const uint32_t pair = now.d[row][GROUPS == 4 ? q / 2 : 0];
                        return __half2float(__ushort_as_half(static_cast<unsigned short>(q % 2 ? pair >> 16 : pair & 0xffff)));
                    };
                    const float d0 = scale_of(2 * r), d1 = scale_of(2 * r + 1);
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        acc[r][cb][0] = fmaf(d0, part[r][cb][0], acc[r][cb][0]);
                        acc[r][cb][1] = fmaf(d0, part[r][cb][1], acc[r][cb][1]);
                        acc[r][cb][2] = fmaf(d1, part[r][cb][2], acc[r][cb][2]);
                        acc[r][cb][3] = fmaf(d1, part[r][cb][3], acc[r][cb][3]);
                    }
                }
            }
            now = next;
        }
    }

    if (kPacked) {
        // Columns 2 p and 2 p + 1 hold part p of the two rows; 6 and 7 hold zeros.
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = acc[r][0][j];
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                acc[r][0][j] = v;
            }
    }
    // sums[share][column][output of the block]
    const int outs = 16 * R * row_warps;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = 8 * cb + 2 * t + (j & 1);
                if (!kPacked || t == 0)
                    sums[(share * kCols + col) * outs + rw * 16 * R + 16 * r + g + 8 * (j >> 1)] = acc[r][cb][j];
            }
    __syncthreads();
    const int all = outs * kCols;
    const auto finish = [&](int e, float v) {
        const int64_t out = out0 + e % outs;
        const int row = m0 + e / outs;
        if (out >= p.n || row >= p.m) return;
        if (MODE == kModePlanes) v *= __ldg(p.row_scale + row);
        if (p.bias) v += __ldg(p.bias + out);
        v = q4_act(v, p.act) * p.scale;
        const int64_t at = static_cast<int64_t>(row) * p.ldc + out;
        if (p.accumulate) v += q4_load(p.c, p.c_type, at);
        q4_store(p.c, p.c_type, at, v);
    };
    if (p.splits == 1) {
        for (int e = threadIdx.x; e < all; e += 32 * kWarps) {
            float v = 0.0f;
            for (int s = 0; s < shares; ++s) v += sums[s * all + e];
            finish(e, v);
        }
        return;
    }
    // The block's own sums into its first share's place, then each block finishes a part of the outputs.
    for (int e = threadIdx.x; e < all; e += 32 * kWarps) {
        float v = 0.0f;
        for (int s = 0; s < shares; ++s) v += sums[s * all + e];
        sums[e] = v;
    }
    __syncwarp();
    cluster_sync();
    for (int e = split * 32 * kWarps + threadIdx.x; e < all; e += p.splits * 32 * kWarps) {
        float v = 0.0f;
        for (int s = 0; s < p.splits; ++s) v += ld_cluster_f32(cluster_addr(sums + e, static_cast<uint32_t>(s)));
        finish(e, v);
    }
    __syncwarp();
    cluster_sync();  // the other blocks have read this one's sums
}

template <int MODE, int GROUPS, bool ZEROS, int R, int CB>
cudaError_t launch(const RowsParams& p, cudaStream_t stream) {
    constexpr int kCols = MODE == kModeF32Packed ? 2 : 8 * CB;
    const int outs = 16 * R * p.row_warps;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((p.n + outs - 1) / outs) * p.splits, (p.m + kCols - 1) / kCols);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, q4_rows_kernel<MODE, GROUPS, ZEROS, R, CB>, p);
}

template <int MODE, int R, int CB>
cudaError_t launch_group(const RowsParams& p, int group, cudaStream_t stream) {
    if (p.zeros) {
        if (group == 32) return launch<MODE, 4, true, R, CB>(p, stream);
        if (group == 64) return launch<MODE, 2, true, R, CB>(p, stream);
        return launch<MODE, 1, true, R, CB>(p, stream);
    }
    if (group == 32) return launch<MODE, 4, false, R, CB>(p, stream);
    if (group == 64) return launch<MODE, 2, false, R, CB>(p, stream);
    return launch<MODE, 1, false, R, CB>(p, stream);
}

// Up to 8 rows (q4_rows.cu), 9 to 32 rows (q4_rows_mid.cu).
cudaError_t launch_small(const RowsParams& p, int mode, int group, int r, cudaStream_t stream);
cudaError_t launch_mid(const RowsParams& p, int mode, int group, cudaStream_t stream);

}  // namespace q4rows

}  // namespace telmo
