// q4.h -- 4-bit weights with a scale (and, where given, a zero point) per group of inputs:
// their device layout and the products that read it (internal to libtelmo_b200).
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace telmo {

// w[o, i] = (code[o, i] - zero[o, i / group]) * scale[o, i / group], codes and zero points 0..15.
//
// Codes are stored in tiles of 8 outputs by 128 inputs (a chunk), 512 bytes each; the 16 tiles of
// 128 outputs and one chunk lie together (8 KB, one bulk copy), chunk after chunk. Lane l = 4 g + t
// of a warp owns bytes 16 l .. 16 l + 15 of a tile: four 32-bit words of output row g, word w holding
// inputs 32 w + 8 t + 0..7 of the chunk (input 2 p in nibble p, input 2 p + 1 in nibble p + 4), each code with
// its top bit flipped (code - 8 in two's complement). So a
// tile is one coalesced 16-byte load per lane; (word >> 4 p) & 0x000f000f leaves two neighbouring
// inputs in the two halves of a register; and one word of the four lanes of a row spans 32 inputs, the
// smallest group, so a 16-input matrix instruction never mixes two groups. Scales and zero points lie
// in the tiles' order, [8 outputs][128 / group] a tile. Outputs and inputs are padded to multiples of
// 128 with code 8, zero point 8 and scale 0.
struct Q4Weights {
    int n = 0, k = 0, group = 0;
    int chunks = 0;             // 128-input chunks per output
    uint4* codes = nullptr;     // [ceil(n / 128)][chunks][16 tiles][32 lanes]
    __half* scales = nullptr;   // [ceil(n / 128)][chunks][16 tiles][8][128 / group]
    uint8_t* zeros = nullptr;   // the same shape, or null: 8 everywhere
};

// The tile of outputs 8 t8 .. 8 t8 + 7 and chunk c.
__host__ __device__ inline int64_t q4_tile(int64_t t8, int chunks, int c) {
    return (t8 / 16 * chunks + c) * 16 + t8 % 16;
}

enum Q4Type : int { kQ4F32 = 0, kQ4BF16 = 1, kQ4F16 = 2 };

struct Q4Args {
    const Q4Weights* w = nullptr;
    const void* a = nullptr;  // [m, lda] of a_type
    int a_type = kQ4F32;
    int64_t lda = 0;
    int m = 0;
    const float* bias = nullptr;  // [n] or null
    int act = 0;                  // Act
    float scale = 1.0f;
    int accumulate = 0;
    void* c = nullptr;  // [m, ldc] of c_type
    int c_type = kQ4F32;
    int64_t ldc = 0;
    int sms = 148;
    uint32_t* error = nullptr;  // device error word
};

// Codes as the host gives them ([n, ceil(k / 2)] bytes, the even input in the low half), scales
// and zero points [n, groups], all in device memory, into the layout above.
cudaError_t q4_repack(const uint8_t* codes, const float* scales, const uint8_t* zeros, const Q4Weights& w,
                      cudaStream_t stream);

// The activations as the kernels for more rows read them where they cannot read the caller's: f32 as
// two fp16 planes (rows 0..m-1 hi, m..2m-1 lo, both times row_scale[r], a power of two), 16-bit
// values copied to rows that start on 16-byte boundaries (row_scale null).
struct Q4Planes {
    const void* a = nullptr;
    int64_t ld = 0;
    const float* row_scale = nullptr;
};

inline bool q4_rows_aligned(const Q4Args& g) {
    return reinterpret_cast<uintptr_t>(g.a) % 16 == 0 && g.lda * (g.a_type == kQ4F32 ? 4 : 2) % 16 == 0;
}

// Whether the product wants Q4Planes, their bytes, and their making.
bool q4_rows_planes(const Q4Args& g);  // up to 32 rows, f32 up to 16
inline bool q4_gemm_planes(const Q4Args& g) { return g.a_type == kQ4F32 || !q4_rows_aligned(g); }
size_t q4_planes_bytes(const Q4Args& g);
cudaError_t q4_make_planes(const Q4Args& g, void* workspace, Q4Planes* planes, cudaStream_t stream);

// The product for one or two rows whose digits fit shared memory (kQ4VecSmem bytes at most).
constexpr size_t kQ4VecSmem = 222 << 10;
bool q4_vec_fits(const Q4Args& g);
cudaError_t q4_linear_vec(const Q4Args& g, cudaStream_t stream);

// The product for up to 32 rows (f32: 16), and for any number of rows on tcgen05 tiles. `planes`: null where not wanted.
cudaError_t q4_linear_rows(const Q4Args& g, const Q4Planes* planes, cudaStream_t stream);
cudaError_t q4_linear_gemm(const Q4Args& g, const Q4Planes* planes, cudaStream_t stream);

}  // namespace telmo
