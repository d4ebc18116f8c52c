// q4_api.cu -- the C ABI of 4-bit weights: encoding, upload and the product.
#include "../../include/telmo_b200.h"
#include "api_internal.h"
#include "q4.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

using namespace telmo;

namespace {

bool group_ok(size_t group) { return group == 32 || group == 64 || group == 128; }

// x rounded to f16, or NaN where that is not finite.
float f16_value(float x) {
    const float h = __half2float(__float2half_rn(x));
    return std::isfinite(h) ? h : std::nanf("");
}

// A group's scale for the step x >= 0 that its range needs: x rounded to f16, NaN where that is not finite. Below
// 2^-14, where f16 values are 2^-24 apart, it is rounded up: a smaller one would leave the group's largest weights out
// of reach of the codes, or be 0.
float f16_scale(float x) {
    const float h = f16_value(x);
    return h < x && x < 0x1p-14f ? h + 0x1p-24f : h;
}

// Whether x is a finite f16 value: 11 significant bits from 2^15 down to multiples of 2^-24.
bool is_f16(float x) {
    uint32_t u;
    std::memcpy(&u, &x, 4);
    const int e = static_cast<int>((u >> 23) & 255) - 127;
    if ((u << 1) == 0) return true;
    if (e > 15 || e < -24) return false;
    const int dropped = e < -14 ? 13 + (-14 - e) : 13;
    return (u & ((1u << dropped) - 1)) == 0;
}

void free_q4(Q4Weights* q) {
    if (!q) return;
    if (q->codes) cudaFree(q->codes);
    if (q->scales) cudaFree(q->scales);
    if (q->zeros) cudaFree(q->zeros);
    delete q;
}

// Host data on the device for the time of an upload.
struct Staged {
    void* p = nullptr;
    ~Staged() {
        if (p) cudaFree(p);
    }
    cudaError_t from(const void* src, size_t bytes) {
        const cudaError_t e = cudaMalloc(&p, bytes);
        return e != cudaSuccess ? e : cudaMemcpy(p, src, bytes, cudaMemcpyHostToDevice);
    }
};

// Workspaces come in stream order from the context's own pool: calls on several streams and captured graphs
// each have their own, and a graph keeps its own while it lives. The pool is made with the first weights, so
// that a product can be a capture's first call.
int make_pool(Ctx* ctx) {
    if (ctx->pool) return TELMO_OK;
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = ctx->device;
    if (int rc = ctx->cuda(cudaMemPoolCreate(&ctx->pool, &props), "memory pool")) return rc;
    uint64_t keep = UINT64_MAX;  // what a call gave back stays for the next
    return ctx->cuda(cudaMemPoolSetAttribute(ctx->pool, cudaMemPoolAttrReleaseThreshold, &keep), "memory pool");
}

int upload_q4(Ctx* ctx, size_t n, size_t k, size_t group, const uint8_t* codes, const float* scales,
              const uint8_t* zeros, Weights* w) {
    const size_t groups = (k + group - 1) / group, rows = (n + 127) / 128 * 128, chunks = (k + 127) / 128;
    for (size_t i = 0; i < n * groups; ++i)
        if (!is_f16(scales[i]))
            return ctx->fail(TELMO_ERR_ARGUMENT,
                             "telmo_weights_upload_q4: scale %zu (%g) is not a finite f16 value", i,
                             static_cast<double>(scales[i]));
    if (zeros)
        for (size_t i = 0; i < n * groups; ++i)
            if (zeros[i] > 15)
                return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_weights_upload_q4: zero point %zu (%d) is above 15", i,
                                 static_cast<int>(zeros[i]));
    if (int rc = make_pool(ctx)) return rc;
    Q4Weights* q = new Q4Weights();
    w->q4 = q;
    w->dev.n = q->n = static_cast<int>(n);
    w->dev.k = q->k = static_cast<int>(k);
    q->group = static_cast<int>(group);
    q->chunks = static_cast<int>(chunks);
    const size_t entries = rows * chunks * (128 / group);
    Staged hc, hs, hz;
    if (int rc = ctx->cuda(cudaMalloc(&q->codes, rows * chunks * 64), "weights")) return rc;
    if (int rc = ctx->cuda(cudaMalloc(&q->scales, entries * sizeof(__half)), "weights")) return rc;
    if (int rc = ctx->cuda(hc.from(codes, n * ((k + 1) / 2)), "weights")) return rc;
    if (int rc = ctx->cuda(hs.from(scales, n * groups * sizeof(float)), "weights")) return rc;
    if (zeros) {
        if (int rc = ctx->cuda(cudaMalloc(&q->zeros, entries), "weights")) return rc;
        if (int rc = ctx->cuda(hz.from(zeros, n * groups), "weights")) return rc;
    }
    if (int rc = ctx->cuda(q4_repack(static_cast<const uint8_t*>(hc.p), static_cast<const float*>(hs.p),
                                     static_cast<const uint8_t*>(hz.p), *q, nullptr),
                           "weights"))
        return rc;
    // The layout is complete before the caller can use it on any stream.
    return ctx->cuda(cudaStreamSynchronize(nullptr), "weights");
}

int q4_type(int dtype) {
    return dtype == TELMO_DTYPE_F32 ? kQ4F32 : dtype == TELMO_DTYPE_BF16 ? kQ4BF16 : dtype == TELMO_DTYPE_F16 ? kQ4F16 : -1;
}

}  // namespace

namespace telmo {

void free_q4_weights(Weights* w) {
    free_q4(w->q4);
    w->q4 = nullptr;
}

int linear_q4(Ctx* ctx, const void* a, int a_dtype, size_t lda, size_t m, const Weights* w, const float* bias, int act,
              float scale, int accumulate, void* out, int c_dtype, size_t ldc, cudaStream_t stream) {
    if (!w->q4) return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: the weights are not 4-bit weights");
    if (m == 0) return TELMO_OK;
    const int at = q4_type(a_dtype), ct = q4_type(c_dtype);
    const size_t n = static_cast<size_t>(w->q4->n), k = static_cast<size_t>(w->q4->k);
    if (at < 0) return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: unknown activation dtype %d", a_dtype);
    if (ct < 0) return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: unknown output dtype %d", c_dtype);
    if (!a || lda < k || m > (1u << 29) || lda > (size_t(1) << 40))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: a is NULL, lda %zu < k %zu or too many rows (%zu)", lda,
                         k, m);
    if (!out || ldc < n || ldc > (size_t(1) << 40))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: c is NULL or ldc %zu is below n %zu", ldc, n);
    if (act < TELMO_ACT_NONE || act > TELMO_ACT_SILU) return ctx->fail(TELMO_ERR_ARGUMENT, "unknown act %d", act);
    const size_t as = at == kQ4F32 ? 4 : 2, cs = ct == kQ4F32 ? 4 : 2;
    const auto misaligned = [](const void* p, uintptr_t b) { return reinterpret_cast<uintptr_t>(p) % b != 0; };
    if (misaligned(a, as) || misaligned(out, cs) || misaligned(bias, 4))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: a, c or bias is not aligned to its elements");
    const Span c_span{out, ldc * cs, n * cs, m};
    if (overlap(Span{a, lda * as, k * as, m}, c_span))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: a and c overlap");
    // One row may be written over its bias: the thread that reads a value writes its output.
    if (!(m == 1 && out == bias && ct == kQ4F32) && overlap(Span{bias, 0, n * sizeof(float), 1}, c_span))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_linear_q4: bias and c overlap");
    DeviceScope scope;
    if (int rc = scope.enter(ctx)) return rc;
    Q4Args g;
    g.w = w->q4;
    g.a = a;
    g.a_type = at;
    g.lda = static_cast<int64_t>(lda);
    g.m = static_cast<int>(m);
    g.bias = bias;
    g.act = act;
    g.scale = scale;
    g.accumulate = accumulate;
    g.c = out;
    g.c_type = ct;
    g.ldc = static_cast<int64_t>(ldc);
    g.sms = ctx->sms;
    g.error = ctx->error_word;
    if (q4_vec_fits(g)) return ctx->cuda(q4_linear_vec(g, stream), "telmo_linear_q4");
    // Row kernels for few rows, tcgen05 tiles beyond: bf16 4096 -> 4096, 8 rows 8.2 us against 12.1, 24 rows 10.8
    // against 12.4, 32 rows 11.0 against 12.4; 4096 -> 8192, 32 rows 17.1 against 18.4. f32 rows come in two planes
    // there and take as many instructions as twice the rows: 16 rows 11.6 against 13.9, 4096 -> 8192 with 16 rows
    // 17.7 against 20.9, with 24 23.2 against 21.2.
    const bool rows = m <= (at == kQ4F32 ? 16 : 32);
    const auto product = [&](const Q4Planes* planes) {
        return rows ? q4_linear_rows(g, planes, stream) : q4_linear_gemm(g, planes, stream);
    };
    if (!(rows ? q4_rows_planes(g) : q4_gemm_planes(g))) return ctx->cuda(product(nullptr), "telmo_linear_q4");
    void* ws = nullptr;
    if (int rc = ctx->cuda(cudaMallocFromPoolAsync(&ws, q4_planes_bytes(g), ctx->pool, stream),
                           "telmo_linear_q4: workspace"))
        return rc;
    Q4Planes planes;
    cudaError_t e = q4_make_planes(g, ws, &planes, stream);
    if (e == cudaSuccess) e = product(&planes);
    const cudaError_t f = cudaFreeAsync(ws, stream);
    return ctx->cuda(e != cudaSuccess ? e : f, "telmo_linear_q4");
}

}  // namespace telmo

extern "C" int telmo_encode_q4(const float* rows, size_t n, size_t k, size_t group, uint8_t* codes, float* scales,
                               uint8_t* zeros) {
    if (!rows || !codes || !scales || n == 0 || k == 0 || !group_ok(group)) return TELMO_ERR_ARGUMENT;
    const size_t groups = (k + group - 1) / group, row_bytes = (k + 1) / 2;
    std::memset(codes, 0, n * row_bytes);
    for (size_t o = 0; o < n; ++o) {
        for (size_t g = 0; g < groups; ++g) {
            const size_t i0 = g * group, i1 = std::min(k, i0 + group);
            float lo = 0.0f, hi = 0.0f;
            for (size_t i = i0; i < i1; ++i) {
                const float x = rows[o * k + i];
                if (!std::isfinite(x)) return TELMO_ERR_ARGUMENT;
                lo = std::min(lo, x);
                hi = std::max(hi, x);
            }
            // Without zero points codes stand for -8..7: the step is the larger of what the
            // group's extremes need. With them the range is [lo, hi], 0 included, in 15 steps.
            const float d = f16_scale(zeros ? hi / 15.0f - lo / 15.0f : std::max(hi / 7.0f, -lo / 8.0f));
            if (std::isnan(d)) return TELMO_ERR_ARGUMENT;
            const float id = d != 0.0f ? 1.0f / d : 0.0f;
            const float z = zeros ? std::fmin(std::fmax(std::round(-lo * id), 0.0f), 15.0f) : 8.0f;
            for (size_t i = i0; i < i1; ++i) {
                const float q = std::fmin(std::fmax(std::round(rows[o * k + i] * id) + z, 0.0f), 15.0f);
                codes[o * row_bytes + i / 2] |= static_cast<uint8_t>(static_cast<int>(q) << (4 * (i & 1)));
            }
            scales[o * groups + g] = d;
            if (zeros) zeros[o * groups + g] = static_cast<uint8_t>(z);
        }
    }
    return TELMO_OK;
}

extern "C" int telmo_weights_upload_q4(telmo_ctx* c, size_t n, size_t k, size_t group, const uint8_t* codes,
                                       const float* scales, const uint8_t* zeros, telmo_weights** out) {
    Ctx* ctx = as_ctx(c);
    if (!ctx || !out) return TELMO_ERR_ARGUMENT;
    *out = nullptr;
    if (n == 0 || k == 0 || n > (1u << 30) || k > (1u << 30))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_weights_upload_q4: bad sizes n=%zu k=%zu", n, k);
    if (!group_ok(group))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_weights_upload_q4: groups of 32, 64 or 128 inputs, not %zu", group);
    if (!codes || !scales) return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_weights_upload_q4: null data");
    DeviceScope scope;
    if (int rc = scope.enter(ctx)) return rc;
    auto* w = new (std::nothrow) Weights();
    if (!w) return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_weights_upload_q4: out of host memory");
    w->ctx = ctx;
    int rc;
    try {
        rc = upload_q4(ctx, n, k, group, codes, scales, zeros, w);
    } catch (const std::bad_alloc&) {
        rc = ctx->fail(TELMO_ERR_ARGUMENT, "telmo_weights_upload_q4: out of host memory");
    }
    if (rc) {
        free_q4_weights(w);
        delete w;
        return rc;
    }
    *out = reinterpret_cast<telmo_weights*>(w);
    return TELMO_OK;
}

extern "C" int telmo_linear_q4(telmo_ctx* c, const void* a, int a_dtype, size_t lda, size_t m, const telmo_weights* wp,
                               const float* bias, int act, float scale, int accumulate, void* out, int c_dtype,
                               size_t ldc, void* stream) {
    Ctx* ctx = as_ctx(c);
    auto* w = reinterpret_cast<const Weights*>(wp);
    if (!ctx || !w) return TELMO_ERR_ARGUMENT;
    if (w->ctx != ctx) return ctx->fail(TELMO_ERR_ARGUMENT, "the weights belong to another context");
    return linear_q4(ctx, a, a_dtype, lda, m, w, bias, act, scale, accumulate, out, c_dtype, ldc,
                     static_cast<cudaStream_t>(stream));
}
