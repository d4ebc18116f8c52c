// q4_rows.cu -- products of few activation rows with 4-bit weights, and the weights' layout.
//
//   c[r, o] = (accumulate ? c[r, o] : 0) + scale * act(sum_g d[o, g] S[r, o, g] + bias[o]),
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
// rows in one, the parts in columns of their own.
#include "q4_device.cuh"

#include <algorithm>

namespace telmo {

namespace {

enum RowsMode : int {
    kModeF16 = 0,        // fp16 activations
    kModeBF16 = 1,       // bf16 activations
    kModeF32 = 2,        // f32 activations, three instructions
    kModeF32Packed = 3,  // f32 activations of one or two rows: part p of row r in column 2 p + r
};

constexpr int kMaxWarps = 8;

struct RowsParams {
    const uint4* codes;
    const __half* scales;
    const uint8_t* zeros;
    int n, k, chunks;
    const void* a;
    int64_t lda;
    int m;
    bool vec;  // rows of a start on 16-byte boundaries
    const float* bias;
    int act;
    float scale;
    int accumulate;
    void* c;
    int c_type;
    int64_t ldc;
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

// Eight 16-bit activations of one row from input i on; 0 outside the row and the matrix.
__device__ __forceinline__ uint4 load_a16(const RowsParams& p, int row, int i) {
    if (row >= p.m) return make_uint4(0, 0, 0, 0);
    const uint16_t* src = static_cast<const uint16_t*>(p.a) + static_cast<int64_t>(row) * p.lda + i;
    if (p.vec && i + 8 <= p.k) return __ldg(reinterpret_cast<const uint4*>(src));
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < p.k ? __ldg(src + j) : 0u;
    return make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16), v[6] | (v[7] << 16));
}

__device__ __forceinline__ void load_a32(const RowsParams& p, int row, int i, float (&x)[8]) {
    if (row >= p.m) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.0f;
        return;
    }
    const float* src = static_cast<const float*>(p.a) + static_cast<int64_t>(row) * p.lda + i;
    if (p.vec && i + 8 <= p.k) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(src));
        const float4 v = __ldg(reinterpret_cast<const float4*>(src) + 1);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < p.k ? __ldg(src + j) : 0.0f;
}

// Part `part` (0 hi, 1 mid, 2 lo) of eight f32 values as four bf16 pairs. Truncation leaves 8 of the 24
// significant bits to each part and every difference is exact. An infinity or a NaN makes its
// other parts NaN, so the row's outputs are not finite.
__device__ __forceinline__ float bf16_rest(float x) {
    return __fsub_rn(x, __uint_as_float(__float_as_uint(x) & 0xffff0000u));
}
__device__ __forceinline__ uint32_t bf16_tops(float x0, float x1) {
    return __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
}
__device__ __forceinline__ void split_parts(const float (&x)[8], uint32_t (&hi)[4], uint32_t (&mid)[4],
                                            uint32_t (&lo)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float r0 = bf16_rest(x[2 * j]), r1 = bf16_rest(x[2 * j + 1]);
        hi[j] = bf16_tops(x[2 * j], x[2 * j + 1]);
        mid[j] = bf16_tops(r0, r1);
        lo[j] = bf16_tops(bf16_rest(r0), bf16_rest(r1));
    }
}

// One tile's scales and zero points of this lane's row: GROUPS of each.
template <int GROUPS>
struct RowScales {
    float d[GROUPS];
    uint32_t z[GROUPS];
};

template <int GROUPS, bool ZEROS>
__device__ __forceinline__ RowScales<GROUPS> load_scales(const RowsParams& p, int64_t tile, int g) {
    RowScales<GROUPS> s;
    const int64_t at = (tile * 8 + g) * GROUPS;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        s.d[i] = __half2float(__ldg(p.scales + at + i));
        s.z[i] = ZEROS ? __ldg(p.zeros + at + i) : 8u;
    }
    return s;
}

// A block of up to 8 warps takes 16 R outputs and 8 CB rows; its warps take the 128-input chunks
// in turn and their sums meet in shared memory.
template <int MODE, int GROUPS, bool ZEROS, int R, int CB>
__global__ void __launch_bounds__(32 * kMaxWarps) q4_rows_kernel(const RowsParams p) {
    constexpr bool BF16 = MODE != kModeF16;
    constexpr int kWordsPerGroup = 4 / GROUPS;
    constexpr int kCols = 8 * CB;
    __shared__ float sums[kMaxWarps][16 * R][kCols + 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    const int g = lane >> 2, t = lane & 3;
    const int64_t tile0 = static_cast<int64_t>(blockIdx.x) * 2 * R;  // first 8-output tile row
    const int m0 = blockIdx.y * kCols;

    float acc[R][CB][4] = {};
    for (int c = warp; c < p.chunks; c += warps) {
        uint4 words[2 * R];
        RowScales<GROUPS> sc[2 * R];
#pragma unroll
        for (int r = 0; r < 2 * R; ++r) {
            const int64_t tile = q4_tile(tile0 + r, p.chunks, c);
            words[r] = __ldg(p.codes + tile * 32 + lane);
            sc[r] = load_scales<GROUPS, ZEROS>(p, tile, g);
        }
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            float part[R][CB][4] = {};
#pragma unroll
            for (int ww = 0; ww < kWordsPerGroup; ++ww) {
                const int w = q * kWordsPerGroup + ww;
                const int i = c * 128 + 32 * w + 8 * t;
                uint32_t b[MODE == kModeF32 ? 3 : 1][CB][4];
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    const int row = m0 + 8 * cb + g;
                    if (MODE == kModeF16 || MODE == kModeBF16) {
                        const uint4 v = load_a16(p, row, i);
                        b[0][cb][0] = v.x; b[0][cb][1] = v.y; b[0][cb][2] = v.z; b[0][cb][3] = v.w;
                    } else if (MODE == kModeF32) {
                        float x[8];
                        load_a32(p, row, i, x);
                        split_parts(x, b[0][cb], b[MODE == kModeF32 ? 1 : 0][cb], b[MODE == kModeF32 ? 2 : 0][cb]);
                    } else {
                        float x[8];
                        load_a32(p, g < 6 ? m0 + (g & 1) : p.m, i, x);
                        uint32_t hi[4], mid[4], lo[4];
                        split_parts(x, hi, mid, lo);
#pragma unroll
                        for (int j = 0; j < 4; ++j) b[0][cb][j] = g < 2 ? hi[j] : g < 4 ? mid[j] : lo[j];
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t x0 = w == 0 ? words[2 * r].x : w == 1 ? words[2 * r].y : w == 2 ? words[2 * r].z
                                                                                              : words[2 * r].w;
                    const uint32_t x1 = w == 0 ? words[2 * r + 1].x : w == 1 ? words[2 * r + 1].y
                                                : w == 2 ? words[2 * r + 1].z : words[2 * r + 1].w;
                    const uint32_t z0 = code_base<BF16>(sc[2 * r].z[q]), z1 = code_base<BF16>(sc[2 * r + 1].z[q]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t a[4] = {code_pair<BF16>(x0, 2 * h, z0), code_pair<BF16>(x1, 2 * h, z1),
                                               code_pair<BF16>(x0, 2 * h + 1, z0), code_pair<BF16>(x1, 2 * h + 1, z1)};
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                            for (int pl = 0; pl < (MODE == kModeF32 ? 3 : 1); ++pl)
                                mma_16816<BF16>(part[r][cb], a, b[pl][cb][2 * h], b[pl][cb][2 * h + 1]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    acc[r][cb][0] = fmaf(sc[2 * r].d[q], part[r][cb][0], acc[r][cb][0]);
                    acc[r][cb][1] = fmaf(sc[2 * r].d[q], part[r][cb][1], acc[r][cb][1]);
                    acc[r][cb][2] = fmaf(sc[2 * r + 1].d[q], part[r][cb][2], acc[r][cb][2]);
                    acc[r][cb][3] = fmaf(sc[2 * r + 1].d[q], part[r][cb][3], acc[r][cb][3]);
                }
        }
    }

    if (MODE == kModeF32Packed) {
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
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sums[warp][16 * r + g + 8 * (j >> 1)][8 * cb + 2 * t + (j & 1)] = acc[r][cb][j];
    __syncthreads();
    const int cols = MODE == kModeF32Packed ? 2 : kCols;
    for (int e = threadIdx.x; e < 16 * R * cols; e += blockDim.x) {
        const int o = e % (16 * R), col = e / (16 * R);
        const int64_t out = tile0 * 8 + o;
        const int row = m0 + col;
        if (out >= p.n || row >= p.m) continue;
        float v = 0.0f;
        for (int w = 0; w < warps; ++w) v += sums[w][o][col];
        if (p.bias) v += __ldg(p.bias + out);
        v = q4_act(v, p.act) * p.scale;
        const int64_t at = static_cast<int64_t>(row) * p.ldc + out;
        if (p.accumulate) v += q4_load(p.c, p.c_type, at);
        q4_store(p.c, p.c_type, at, v);
    }
}

template <int MODE, int GROUPS, bool ZEROS, int R, int CB>
cudaError_t launch_rows(const RowsParams& p, cudaStream_t stream) {
    constexpr int kRowsPerBlock = MODE == kModeF32Packed ? 2 : 8 * CB;
    const dim3 grid((p.n + 16 * R - 1) / (16 * R), (p.m + kRowsPerBlock - 1) / kRowsPerBlock);
    q4_rows_kernel<MODE, GROUPS, ZEROS, R, CB><<<grid, 32 * std::min(kMaxWarps, p.chunks), 0, stream>>>(p);
    return cudaGetLastError();
}

template <int MODE, int R, int CB>
cudaError_t launch_rows_group(const RowsParams& p, int group, cudaStream_t stream) {
    if (p.zeros) {
        if (group == 32) return launch_rows<MODE, 4, true, R, CB>(p, stream);
        if (group == 64) return launch_rows<MODE, 2, true, R, CB>(p, stream);
        return launch_rows<MODE, 1, true, R, CB>(p, stream);
    }
    if (group == 32) return launch_rows<MODE, 4, false, R, CB>(p, stream);
    if (group == 64) return launch_rows<MODE, 2, false, R, CB>(p, stream);
    return launch_rows<MODE, 1, false, R, CB>(p, stream);
}

// One thread per 32-bit word of the layout (four words to a lane).
__global__ void q4_repack_kernel(const uint8_t* codes, const float* scales, const uint8_t* zeros, Q4Weights w,
                                 int64_t tiles) {
    const int64_t word = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (word >= tiles * 128) return;
    const int64_t tile = word / 128;
    const int in = static_cast<int>(word % 128);
    const int lane = in / 4, wi = in % 4;
    const int64_t o0 = (tile / 16 / w.chunks * 16 + tile % 16) * 8;
    const int64_t o = o0 + lane / 4;
    const int c = static_cast<int>(tile / 16 % w.chunks);
    const int i0 = c * 128 + 32 * wi + 8 * (lane % 4);
    const int64_t row_bytes = (static_cast<int64_t>(w.k) + 1) / 2;
    uint32_t v = 0;
    for (int j = 0; j < 8; ++j) {
        uint32_t q = 8;
        if (o < w.n && i0 + j < w.k) {
            const uint8_t b = codes[o * row_bytes + (i0 + j) / 2];
            q = ((i0 + j) & 1) ? b >> 4 : b & 15;
        }
        v |= q << (4 * (j / 2 + 4 * (j & 1)));
    }
    reinterpret_cast<uint32_t*>(w.codes)[word] = v;
    // The first of a tile's threads write its scales and zero points.
    const int per = 128 / w.group;
    if (in < 8 * per) {
        const int64_t so = o0 + in / per;
        const int64_t groups = (static_cast<int64_t>(w.k) + w.group - 1) / w.group;
        const int64_t q = static_cast<int64_t>(c) * per + in % per;
        const bool ok = so < w.n && q < groups;
        w.scales[tile * 8 * per + in] = __float2half_rn(ok ? scales[so * groups + q] : 0.0f);
        if (w.zeros) w.zeros[tile * 8 * per + in] = ok ? zeros[so * groups + q] : 8;
    }
}

}  // namespace

cudaError_t q4_repack(const uint8_t* codes, const float* scales, const uint8_t* zeros, const Q4Weights& w,
                      cudaStream_t stream) {
    const int64_t tiles = (static_cast<int64_t>(w.n) + 127) / 128 * 16 * w.chunks;
    const int64_t blocks = (tiles * 128 + 255) / 256;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    q4_repack_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(codes, scales, zeros, w, tiles);
    return cudaGetLastError();
}

cudaError_t q4_linear_rows(const Q4Args& g, cudaStream_t stream) {
    RowsParams p;
    p.codes = g.w->codes;
    p.scales = g.w->scales;
    p.zeros = g.w->zeros;
    p.n = g.w->n;
    p.k = g.w->k;
    p.chunks = g.w->chunks;
    p.a = g.a;
    p.lda = g.lda;
    p.m = g.m;
    const int size = g.a_type == kQ4F32 ? 4 : 2;
    p.vec = reinterpret_cast<uintptr_t>(g.a) % 16 == 0 && g.lda * size % 16 == 0;
    p.bias = g.bias;
    p.act = g.act;
    p.scale = g.scale;
    p.accumulate = g.accumulate;
    p.c = g.c;
    p.c_type = g.c_type;
    p.ldc = g.ldc;
    if (g.a_type == kQ4F32) {
        if (g.m <= 2) return launch_rows_group<kModeF32Packed, 1, 1>(p, g.w->group, stream);
        return launch_rows_group<kModeF32, 1, 1>(p, g.w->group, stream);
    }
    if (g.a_type == kQ4BF16) return launch_rows_group<kModeBF16, 1, 1>(p, g.w->group, stream);
    return launch_rows_group<kModeF16, 1, 1>(p, g.w->group, stream);
}

}  // namespace telmo
