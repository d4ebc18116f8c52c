// q4_rows.cu -- the layout of 4-bit weights, and products of up to 32 activation rows with them: the
// choice of a kernel's shape, and its instances for up to 8 rows (q4_rows.cuh).
#include "q4_rows.cuh"

namespace telmo {

namespace {

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
        v |= (q ^ 8) << (4 * (j / 2 + 4 * (j & 1)));
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

namespace q4rows {

namespace {

template <int MODE>
cudaError_t by_shape(const RowsParams& p, int group, cudaStream_t stream) {
    return by_group(p, group, [&](auto groups, auto zeros) {
        return launch_direct<MODE, decltype(groups)::value, decltype(zeros)::value>(p, stream);
    });
}

}  // namespace

cudaError_t launch_small(const RowsParams& p, int mode, int group, cudaStream_t stream) {
    if (mode == kModeF32) return by_shape<kModeF32>(p, group, stream);
    if (mode == kModeBF16) return by_shape<kModeBF16>(p, group, stream);
    return by_shape<kModeF16>(p, group, stream);
}

}  // namespace q4rows

bool q4_rows_planes(const Q4Args& g) { return g.m > 8 && (g.a_type == kQ4F32 || !q4_rows_aligned(g)); }

cudaError_t q4_linear_rows(const Q4Args& g, const Q4Planes* planes, cudaStream_t stream) {
    using namespace q4rows;
    RowsParams p;
    p.codes = g.w->codes;
    p.scales = g.w->scales;
    p.zeros = g.w->zeros;
    p.n = g.w->n;
    p.k = g.w->k;
    p.chunks = g.w->chunks;
    p.a = planes ? planes->a : g.a;
    p.lda = planes ? planes->ld : g.lda;
    p.m = g.m;
    p.vec = planes || q4_rows_aligned(g);
    p.planes = planes != nullptr;
    p.row_scale = planes ? planes->row_scale : nullptr;
    p.bias = g.bias;
    p.act = g.act;
    p.scale = g.scale;
    p.accumulate = g.accumulate;
    p.c = g.c;
    p.c_type = g.c_type;
    p.ldc = g.ldc;
    p.splits = 1;
    const int mode = g.a_type == kQ4BF16 ? kModeBF16 : g.a_type == kQ4F16 ? kModeF16 : kModeF32;
    // Up to 8 rows of f32 or of any alignment are read as they are (f32, 1024 -> 4096: 3.9 us, as two planes 7.8;
    // 4096 -> 8192: 17.5 and 17.7. 16-bit rows off 16-byte boundaries, copied first: 5.4 us against 4.1, and 12.2
    // against 13.6), and aligned ones where a warp has one chunk at most, so that a ring has nothing to run ahead
    // to (1024 -> 4096: 3.3 us, staged 4.2; 4096 -> 4096: 8.7 us, staged 8.3).
    if (!p.vec || mode == kModeF32 ? g.m <= 8 : g.m <= 8 && p.chunks <= kWarps)
        return launch_small(p, mode, g.w->group, stream);
    // Warps side by side read the same activations; the chunks are split over clusters as long as the SMs have
    // places for all blocks (fewer clusters may fit) and a share keeps two chunks (4096 -> 4096: 24 rows 10.7 us,
    // 22.2 without; 8 rows 8.3, 10.6 without; 4096 -> 8192, 32 rows: 17.1, 26.4 without).
    const int row_warps = g.m <= 8 ? 2 : 4, shares = kWarps / row_warps;
    const int blocks = (p.n + 32 * row_warps - 1) / (32 * row_warps);
    const int resident = (mode != kModeF32 && g.m <= 24 ? 2 : 1) * g.sms;
    while (p.splits < 8 && blocks * p.splits * 2 <= resident && p.chunks >= 4 * shares * p.splits) p.splits *= 2;
    p.split_chunks = (p.chunks + p.splits - 1) / p.splits;
    return launch_aligned(p, mode == kModeF32 ? kModePlanes : mode, g.w->group, stream);
}

}  // namespace telmo
