// q4_vec.cu -- products of one or two activation rows with 4-bit weights, in integers.
//
//   c[r, o] = (accumulate ? c[r, o] : 0) + scale * act(s_r sum_g d[o, g] S[r, o, g] + bias[o])
//
// A single row's product is bound by the weights' bytes (n k / 2), if taking the codes apart keeps
// up with them: at 6.5 TB/s an SM gets about 50 codes per clock, and the integer pipe's half rate
// leaves it two operations for each eight. Making 16-bit operands of codes (q4_rows.cuh) takes
// seven integer and four half-precision operations per eight codes. Here they become 8-bit
// operands in three: a byte with a code in its upper half is 16 code - 256 [code > 7], so storing
// codes with their top bit flipped (two's complement of code - 8) makes (word << 4) & 0xf0f0f0f0 and
// word & 0xf0f0f0f0 the bytes 16 (code - 8), exactly.
//
// The activations are integers too: a row is scaled by a power of two so that its largest value
// lies in [2^26, 2^27), and integer and fraction (the latter times 2^28) are rounded and written as
// four digits of base 128 each, -64..63: every value to 2^-55 of the row's largest, so an f32 value
// within 2^-31 of it is exact. The eight digits are the eight columns of the B operand, which a single
// row would leave empty otherwise: mma.sync m16n8k32 (s8 x s8 -> s32) gives all digits' exact sums of 16
// outputs and 32 inputs in one instruction. The accumulators start at 0x4b400000, the f32 bits of
// 1.5 2^23, where an integer added is the same integer added to the float (|sum| <= 16 * 8 * 64 * 128 =
// 2^20): a subtraction and a fused multiply-add bring a group's sum, times its scale, to f32. Zero
// points subtract 16 (zero - 8) times the group's sum of digits, in integers that f32 holds exactly.
//
// Each block writes the digits of the whole rows into shared memory once and walks over blocks of
// 32 outputs; its eight warps share the chunks, each with a ring of chunks of codes, scales and
// zero points in shared memory (cp.async), and add up in order.
//
// Measured: one bf16 row, 4096 -> 32768, 69 MB of codes and scales from memory, 15.9 us captured: 4.3 TB/s
// (67% of a copy's rate); the digits of the first block and the rings' first chunks take 3 us before the
// stream runs. An SM holds two blocks, 16 warps: their digits and rings take 102,400 bytes each (75 registers
// would let three in).
#include "q4_device.cuh"
#include "ptx.cuh"
#include "q4_async.cuh"

#include <algorithm>
#include <type_traits>

namespace telmo {

namespace {

constexpr int kWarps = 8;
constexpr int kRing = 4;
constexpr int kTiles = 4;    // 8-output tiles of a block: 32 outputs
constexpr int kDigits = 8;

struct VecParams {
    const uint4* codes;
    const uint8_t* scales;
    const uint8_t* zeros;
    int n, k, chunks;
    const void* a;
    int a_type;
    int64_t lda;
    bool vec;  // rows of a start on 16-byte boundaries
    const float* bias;
    int act;
    float scale;
    int accumulate;
    void* c;
    int c_type;
    int64_t ldc;
    int blocks;
};

template <int M, int GROUPS, bool ZEROS>
struct Layout {
    static constexpr int kScaleBytes = kTiles * 8 * GROUPS * 2;
    static constexpr int kZeroBytes = ZEROS ? kTiles * 8 * GROUPS : 0;
    static constexpr int kStage = kTiles * 512 + kScaleBytes + kZeroBytes;
    static constexpr int kSums = 2 * kWarps * M * 32 * 4;  // two blocks' [warp][row][output]
    static size_t smem(int chunks) {
        return static_cast<size_t>(kWarps) * kRing * kStage + kSums +
               static_cast<size_t>(chunks) * M * (1024 + (ZEROS ? GROUPS * 32 : 0));
    }
};

// Eight inputs of a row from i on (a multiple of 8), zeros behind the row's end.
__device__ __forceinline__ void load_eight(const VecParams& p, int row, int i, float (&x)[8]) {
    const int64_t at = static_cast<int64_t>(row) * p.lda + i;
    if (p.a_type == kQ4F32) {
        const float* src = static_cast<const float*>(p.a) + at;
        if (p.vec && i + 8 <= p.k) {
            const float4 u = __ldg(reinterpret_cast<const float4*>(src)), v = __ldg(reinterpret_cast<const float4*>(src) + 1);
            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
            x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = i + j < p.k ? __ldg(src + j) : 0.0f;
        }
        return;
    }
    const uint16_t* src = static_cast<const uint16_t*>(p.a) + at;
    uint16_t h[8];
    if (p.vec && i + 8 <= p.k) {
        *reinterpret_cast<uint4*>(h) = __ldg(reinterpret_cast<const uint4*>(src));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = i + j < p.k ? __ldg(src + j) : uint16_t(0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        x[j] = p.a_type == kQ4BF16 ? __uint_as_float(static_cast<uint32_t>(h[j]) << 16) : __half2float(__ushort_as_half(h[j]));
}

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

template <int M, int GROUPS, bool ZEROS>
__global__ void __launch_bounds__(32 * kWarps, 2) q4_vec_kernel(const VecParams p) {
    using L = Layout<M, GROUPS, ZEROS>;
    constexpr int kWordsPerGroup = 4 / GROUPS;
    constexpr int kBase = 0x4b400000;  // 12582912.0f
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t tops[kWarps][M];
    float* sums = reinterpret_cast<float*>(smem + kWarps * kRing * L::kStage);
    uint2* digits = reinterpret_cast<uint2*>(smem + kWarps * kRing * L::kStage + L::kSums);  // [row][chunk][word][lane]
    float* digit_sums = reinterpret_cast<float*>(digits + static_cast<size_t>(M * p.chunks) * 128);  // [row][group][digit]
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int g = lane >> 2, t = lane & 3;

    // ---- the warp's ring: chunk `warp`, `warp` + 8 .. of each of the block's outputs in turn -------
    const uint32_t ring = smem_u32(smem) + static_cast<uint32_t>(warp * kRing * L::kStage);
    int fetch_block = blockIdx.x, fetch_chunk = warp, fetch_place = 0;
    const auto fetch = [&] {
        if (warp < p.chunks && fetch_block < p.blocks) {
            const int64_t tile = q4_tile(static_cast<int64_t>(fetch_block) * kTiles, p.chunks, fetch_chunk);
            const uint32_t to = ring + static_cast<uint32_t>(fetch_place * L::kStage);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) cp_async16(to + i * 512 + lane * 16, p.codes + (tile + i) * 32 + lane, 16);
            if (lane < L::kScaleBytes / 16)
                cp_async16(to + kTiles * 512 + lane * 16, p.scales + tile * (8 * GROUPS * 2) + lane * 16, 16);
            if (ZEROS && lane < L::kZeroBytes / 16)
                cp_async16(to + kTiles * 512 + L::kScaleBytes + lane * 16, p.zeros + tile * (8 * GROUPS) + lane * 16, 16);
            if ((fetch_chunk += kWarps) >= p.chunks) {
                fetch_chunk = warp;
                fetch_block += gridDim.x;
            }
            if (++fetch_place == kRing) fetch_place = 0;
        }
        cp_commit();  // an empty group where nothing is left, so that the counts stay even
    };
    for (int i = 0; i < kRing - 1; ++i) fetch();

    // ---- the rows' digits --------------------------------------------------------------------------
    // A thread has every 256th unit of eight inputs (of row 0, then of row 1) and keeps the first
    // kKeep in registers between looking for the rows' largest values and writing digits.
    constexpr int kKeep = 4;
    const int units = p.chunks * 16, all_units = units * M;
    float kept[kKeep][8];
    uint32_t top[M] = {};  // |x| as bits: infinities and NaNs are the largest
    const auto look = [&](const float (&x)[8], int u) {
        uint32_t v = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) v = max(v, __float_as_uint(x[j]) & 0x7fffffffu);
        if (M == 2 && u >= units) top[M - 1] = max(top[M - 1], v);
        else top[0] = max(top[0], v);
    };
    const auto load_unit = [&](int u, float (&x)[8]) {
        const int r = M == 2 && u >= units, v = r ? u - units : u;
        load_eight(p, r, v * 8, x);
    };
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int u = threadIdx.x + i * 32 * kWarps;
        if (u < all_units) load_unit(u, kept[i]);
    }
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int u = threadIdx.x + i * 32 * kWarps;
        if (u < all_units) look(kept[i], u);
    }
    for (int u = threadIdx.x + kKeep * 32 * kWarps; u < all_units; u += 32 * kWarps) {
        float x[8];
        load_unit(u, x);
        look(x, u);
    }
#pragma unroll
    for (int r = 0; r < M; ++r) {
        top[r] = __reduce_max_sync(0xffffffffu, top[r]);
        if (lane == 0) tops[warp][r] = top[r];
    }
    __syncthreads();
    float up[M], unit[M];  // what brings a row's largest value to [2^26, 2^27), and s_r / 16
#pragma unroll
    for (int r = 0; r < M; ++r) {
        uint32_t v = 0;
        for (int w = 0; w < kWarps; ++w) v = max(v, tops[w][r]);
        // v = 2^e times 1..2, e held to -96 so that every factor is a normal f32 (a row below that keeps
        // its values to 2^-150).
        const int e = max(static_cast<int>(v >> 23) - 127, -96);
        up[r] = e > 127 ? 0.0f : pow2(26 - e);
        // A row with an infinity or a NaN has outputs that are all NaN.
        unit[r] = e > 127 ? __uint_as_float(0x7fc00000u) : pow2(e - 30);
    }
    const auto write_digits = [&](int u, const float (&in)[8]) {
        // Unit v of row r is word v / 4 % 4 of chunk v / 16, lane place t = v % 4.
        const int r = M == 2 && u >= units, v = r ? u - units : u;
        const float f = r ? up[M - 1] : up[0];
        constexpr int kHalfUnit = 64 + (64 << 7) + (64 << 14);  // makes the digits' remainders -64..63
        int x[2][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = f != 0.0f ? in[j] * f : 0.0f;
            const float whole = rintf(a);
            x[0][j] = static_cast<int>(whole) + kHalfUnit;
            x[1][j] = __float2int_rn((a - whole) * 268435456.0f) + kHalfUnit;
        }
#pragma unroll
        for (int l = 0; l < kDigits; ++l) {
            const auto digit = [&](int j) {
                const int y = x[l / 4][j] >> (7 * (3 - l % 4));
                return l % 4 == 0 ? y : (y & 127) - 64;
            };
            // The bytes in the order in which the codes come: inputs 0 4 1 5 of (word << 4), 2 6 3 7 of word.
            const auto pack = [&](int a, int b, int c, int d) {
                return __byte_perm(__byte_perm(digit(a), digit(b), 0x0040), __byte_perm(digit(c), digit(d), 0x0040), 0x5410);
            };
            const uint2 w = make_uint2(pack(0, 4, 1, 5), pack(2, 6, 3, 7));
            digits[(r * p.chunks * 4 + v / 4) * 32 + l * 4 + v % 4] = w;
            if (ZEROS) {
                // A group's places are neighbouring lanes; half warps (16 places to a chunk) take part whole.
                int sum = __dp4a(static_cast<int>(w.x), 0x01010101, __dp4a(static_cast<int>(w.y), 0x01010101, 0));
                const unsigned half = 0xffffu << (lane & 16);
#pragma unroll
                for (int d = 1; d < 4 * kWordsPerGroup; d *= 2) sum += __shfl_xor_sync(half, sum, d);
                if (v % (4 * kWordsPerGroup) == 0)
                    digit_sums[(r * p.chunks * GROUPS + v / (4 * kWordsPerGroup)) * 8 + l] = static_cast<float>(sum);
            }
        }
    };
#pragma unroll 1
    for (int i = 0; i < kKeep; ++i) {
        const int u = threadIdx.x + i * 32 * kWarps;
        if (u < all_units) write_digits(u, kept[0]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int o = 0; o + 1 < kKeep; ++o) kept[o][j] = kept[o + 1][j];
    }
    for (int u = threadIdx.x + kKeep * 32 * kWarps; u < all_units; u += 32 * kWarps) {
        float x[8];
        load_unit(u, x);
        write_digits(u, x);
    }
    __syncthreads();

    // ---- the outputs, 32 at a time -------------------------------------------------------------------
    const float weight[2] = {pow2(7 * (3 - 2 * t)), pow2(7 * (2 - 2 * t))};  // of this lane's two digits
    int place = 0, parity = 0;
    for (int block = blockIdx.x; block < p.blocks; block += gridDim.x, parity ^= 1) {
        float acc[M][2][4] = {};
        for (int c = warp; c < p.chunks; c += kWarps) {
            cp_wait<kRing - 2>();
            __syncwarp();  // every lane's copies are complete, and every lane is done with the place filled next
            fetch();
            const uint32_t at = ring + static_cast<uint32_t>(place * L::kStage);
            if (++place == kRing) place = 0;
            uint4 words[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) words[i] = ld_shared_v4(at + i * 512 + lane * 16);
            const uint32_t sc = at + kTiles * 512 + g * GROUPS * 2, zp = at + kTiles * 512 + L::kScaleBytes + g * GROUPS;
            int part[M][2][4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int q = w / kWordsPerGroup;
                if (w % kWordsPerGroup == 0)
#pragma unroll
                    for (int e = 0; e < M * 8; ++e) part[e / 8][e / 4 % 2][e % 4] = kBase;
                uint2 b[M];
#pragma unroll
                for (int m = 0; m < M; ++m) b[m] = digits[((m * p.chunks + c) * 4 + w) * 32 + lane];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint4 &x = words[2 * r], &y = words[2 * r + 1];
                    const uint32_t x0 = w == 0 ? x.x : w == 1 ? x.y : w == 2 ? x.z : x.w;
                    const uint32_t y0 = w == 0 ? y.x : w == 1 ? y.y : w == 2 ? y.z : y.w;
                    const uint32_t a[4] = {(x0 << 4) & 0xf0f0f0f0u, (y0 << 4) & 0xf0f0f0f0u, x0 & 0xf0f0f0f0u, y0 & 0xf0f0f0f0u};
#pragma unroll
                    for (int m = 0; m < M; ++m) mma_s8(part[m][r], a, b[m].x, b[m].y);
                }
                if ((w + 1) % kWordsPerGroup == 0) {
                    float2 ds[M];
                    if (ZEROS)
#pragma unroll
                        for (int m = 0; m < M; ++m)
                            ds[m] = *reinterpret_cast<const float2*>(digit_sums + ((m * p.chunks + c) * GROUPS + q) * 8 + 2 * t);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {  // output rows g + 8 e of the block
                        const float d = __half2float(__ushort_as_half(ld_shared_u16(sc + e * (8 * GROUPS * 2) + q * 2)));
                        float z = 0.0f;
                        if (ZEROS) z = static_cast<float>(128 - 16 * static_cast<int>(ld_shared_u8(zp + e * (8 * GROUPS) + q)));
#pragma unroll
                        for (int m = 0; m < M; ++m)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                float f = __int_as_float(part[m][e / 2][e % 2 * 2 + j]) - 12582912.0f;
                                if (ZEROS) f = fmaf(z, j ? ds[m].y : ds[m].x, f);
                                acc[m][e / 2][e % 2 * 2 + j] = fmaf(d, f, acc[m][e / 2][e % 2 * 2 + j]);
                            }
                    }
                }
            }
        }
        // Digits onto one another, then the warps.
        float* mine = sums + (parity * kWarps + warp) * (M * 32);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = fmaf(acc[m][e / 2][e % 2 * 2], weight[0], acc[m][e / 2][e % 2 * 2 + 1] * weight[1]);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                if (t == 0) mine[m * 32 + e * 8 + g] = v;
            }
        // One meeting a block of outputs: the sums alternate between two places.
        __syncthreads();
        if (threadIdx.x < 32 * M) {
            const int row = threadIdx.x / 32, out = block * 32 + threadIdx.x % 32;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += sums[(parity * kWarps + w) * (M * 32) + threadIdx.x];
            if (out < p.n) {
                v *= M == 2 && row ? unit[M - 1] : unit[0];
                if (p.bias) v += __ldg(p.bias + out);
                v = q4_act(v, p.act) * p.scale;
                const int64_t at = static_cast<int64_t>(row) * p.ldc + out;
                if (p.accumulate) v += q4_load(p.c, p.c_type, at);
                q4_store(p.c, p.c_type, at, v);
            }
        }
    }
    cp_wait<0>();
}

template <int M, int GROUPS, bool ZEROS>
cudaError_t launch(const VecParams& p, int sms, cudaStream_t stream) {
    using L = Layout<M, GROUPS, ZEROS>;
    static DeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!once.done(dev)) {
        e = cudaFuncSetAttribute(q4_vec_kernel<M, GROUPS, ZEROS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kQ4VecSmem);
        if (e != cudaSuccess) return e;
        once.mark(dev);
    }
    const size_t smem = L::smem(p.chunks);
    const int resident = (smem <= kQ4VecSmem / 2 ? 2 : 1) * sms;
    q4_vec_kernel<M, GROUPS, ZEROS><<<std::min(p.blocks, resident), 32 * kWarps, smem, stream>>>(p);
    return cudaGetLastError();
}

// Calls f with the constants of the product's rows, groups and zero points.
template <typename F>
auto by_shape(int m, int group, bool zeros, F f) {
    using std::integral_constant;
    const auto by_group = [&](auto rows, auto z) {
        if (group == 32) return f(rows, integral_constant<int, 4>(), z);
        if (group == 64) return f(rows, integral_constant<int, 2>(), z);
        return f(rows, integral_constant<int, 1>(), z);
    };
    const auto by_zeros = [&](auto rows) {
        return zeros ? by_group(rows, std::true_type()) : by_group(rows, std::false_type());
    };
    return m == 1 ? by_zeros(integral_constant<int, 1>()) : by_zeros(integral_constant<int, 2>());
}

}  // namespace

// One or two rows whose digits and rings fit into shared memory. 4096 -> 8192, bf16: one row 8.5 us, 10.7 on the
// row kernels; two rows 10.4 against 11.1. 1024 -> 4096, f32: 3.0 against 4.1, two rows 3.5 against 4.2.
bool q4_vec_fits(const Q4Args& g) {
    if (g.m > 2) return false;
    return by_shape(g.m, g.w->group, g.w->zeros != nullptr, [&](auto m, auto groups, auto zeros) {
        return Layout<decltype(m)::value, decltype(groups)::value, decltype(zeros)::value>::smem(g.w->chunks) <= kQ4VecSmem;
    });
}

cudaError_t q4_linear_vec(const Q4Args& g, cudaStream_t stream) {
    VecParams p;
    p.codes = g.w->codes;
    p.scales = reinterpret_cast<const uint8_t*>(g.w->scales);
    p.zeros = g.w->zeros;
    p.n = g.w->n;
    p.k = g.w->k;
    p.chunks = g.w->chunks;
    p.a = g.a;
    p.a_type = g.a_type;
    p.lda = g.lda;
    p.vec = q4_rows_aligned(g);
    p.bias = g.bias;
    p.act = g.act;
    p.scale = g.scale;
    p.accumulate = g.accumulate;
    p.c = g.c;
    p.c_type = g.c_type;
    p.ldc = g.ldc;
    p.blocks = (p.n + 31) / 32;
    return by_shape(g.m, g.w->group, p.zeros != nullptr, [&](auto m, auto groups, auto zeros) {
        return launch<decltype(m)::value, decltype(groups)::value, decltype(zeros)::value>(p, g.sms, stream);
    });
}

}  // namespace telmo
