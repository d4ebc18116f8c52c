// logits.cu -- logits under a decoder's rules, and the best tokens of each row.
//
// For row r and token v with n(v) occurrences among the row's tokens so far, the value is
//   x = l                                    the logit, in f32
//   n > 0:  x = x > 0 ? x / theta : x theta  repetition penalty
//           x = x - f n, then x - p          frequency and presence penalties
//   x = x + b(v)                             the sum of the biases listed for v
//   x = -inf                                 where the grammar state does not allow v
// each step rounded to f32 on its own, so that a caller's own f32 steps choose the same tokens.
// `constrain` stores x in the logits' type; `choose` keeps the k best x of a row, ties to the lowest
// token, and their log-probabilities x - log sum_v e^x, and stores nothing else.
//
// Both read the logits once and are bound by that (constrain writes them once more). A block takes
// tiles of 8192 tokens: it loads its logits, counts the row's tokens so far that fall into the tile
// in shared memory (integer atomics: the counts do not depend on their order), adds the listed
// biases (one warp, in list order, so that sums do not depend on timing), and sets a bit for
// every token so touched; eight tokens whose bits are clear skip the rules. Every block of a row
// reads the whole list of tokens (from L2), which is what a larger tile would save and shared
// memory limits. For `choose` the blocks of a row form a cluster of up to eight and meet through
// distributed shared memory: no workspace, no counters, one launch.
#include "../../include/telmo_b200.h"
#include "api_internal.h"
#include "kernels.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <climits>
#include <cmath>

namespace telmo {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 8192;                        // tokens per tile
constexpr int kPerThread = kTile / 8 / kThreads;   // groups of eight tokens a thread has in a tile
constexpr int kMaxK = 8;
constexpr float kLowest = -3.402823466e38f;

struct RuleParams {
    const void* logits;
    int64_t ld;
    int rows, vocab;
    const int32_t* history;
    int64_t history_ld;
    int n_history;
    const int32_t* history_len;
    const float *repetition, *frequency, *presence;
    const int32_t* bias_ids;
    const float* bias;
    int64_t bias_ld;
    int n_bias;
    const uint32_t* allowed;
    int64_t allowed_ld;
    int n_states;
    const int32_t* state;
    void* out;
    int64_t out_ld;
    int32_t* ids;
    float* logprobs;
    int k;
    int slices;  // blocks per row
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight values as they lie in memory.
template <typename T>
struct alignas(16) Eight {
    T v[8];
};

// A row's k best values so far, best first. Values arrive in the order of their tokens, so an
// equal value stays behind.
template <int K>
struct Best {
    float x[K];
    int id[K];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            x[i] = -INFINITY;
            id[i] = INT_MAX;
        }
    }
    // (v, token) goes before entry i where v is larger, or equal with a lower token.
    __device__ __forceinline__ void insert(float v, int token) {
#pragma unroll
        for (int i = K - 1; i >= 0; --i) {
            const bool here = v > x[i] || (v == x[i] && token < id[i]);
            const bool above = i > 0 && (v > x[i - 1] || (v == x[i - 1] && token < id[i - 1]));
            if (above) {
                x[i] = x[i - 1];
                id[i] = id[i - 1];
            } else if (here) {
                x[i] = v;
                id[i] = token;
            }
        }
    }
    __device__ __forceinline__ void drop_first() {
#pragma unroll
        for (int i = 0; i + 1 < K; ++i) {
            x[i] = x[i + 1];
            id[i] = id[i + 1];
        }
        x[K - 1] = -INFINITY;
        id[K - 1] = INT_MAX;
    }
};

// An unsigned number in the order of the floats (no NaN; -0 counts as 0).
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// The k best of the warp's lanes' lists: lane i ends with the i-th.
template <int K>
__device__ __forceinline__ void warp_best(Best<K>& mine, float& x, int& id) {
    const int lane = threadIdx.x % 32;
    x = -INFINITY;
    id = INT_MAX;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const uint32_t key = ordered(mine.x[0]);
        const uint32_t top = __reduce_max_sync(0xffffffffu, key);
        const int first = __reduce_min_sync(0xffffffffu, key == top ? mine.id[0] : INT_MAX);
        const bool owner = key == top && mine.id[0] == first;
        const unsigned owners = __ballot_sync(0xffffffffu, owner);
        const float v = __shfl_sync(0xffffffffu, mine.x[0], __ffs(owners) - 1);
        if (lane == i) {
            x = v;
            id = first;
        }
        if (owner) mine.drop_first();  // several own it only where nothing is left
    }
}

__device__ __forceinline__ float exp_of(float d) { return ex2_approx(d * 1.44269504f); }

// Running maximum and sum of e^(x - maximum).
struct MaxSum {
    float m = kLowest, s = 0.0f;
    __device__ __forceinline__ void merge(float m2, float s2) {
        const float top = fmaxf(m, m2);
        s = s * exp_of(m - top) + s2 * exp_of(m2 - top);
        m = top;
    }
};

__device__ __forceinline__ uint32_t ld_cluster_u32(const void* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}

// T: the logits' type. K: 0 stores every value (constrain), else the tokens kept per row. Blocks
// (x: slice of the row, y: row) take the row's tiles in turn.
template <typename T, int K>
__global__ void __launch_bounds__(kThreads) logits_kernel(const RuleParams p) {
    constexpr int kBest = K ? K : 1;
    extern __shared__ __align__(16) uint8_t smem[];
    const int row = blockIdx.y, slice = blockIdx.x;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const bool counting = p.history != nullptr, biasing = p.n_bias > 0;
    uint32_t* touched = reinterpret_cast<uint32_t*>(smem);  // one bit per token of the tile
    uint32_t* count = touched + kTile / 32;
    float* bias = reinterpret_cast<float*>(count + (counting ? kTile : 0));

    const T* in = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.ld;
    T* out = K ? nullptr : static_cast<T*>(p.out) + static_cast<int64_t>(row) * p.out_ld;
    // Tiles are cut where the row's addresses are multiples of 16 bytes: place e of the cut row is
    // token e - shift.
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
    const bool same_cut = !K && static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T)) == shift;
    const int places = p.vocab + shift;
    const int tiles = (places + kTile - 1) / kTile;

    int said = 0;
    float theta = 1.0f, freq = 0.0f, pres = 0.0f;
    if (counting) {
        said = __ldg(p.history_len + row);
        said = max(0, min(said, p.n_history));
        if (p.repetition) theta = __ldg(p.repetition + row);
        if (p.frequency) freq = __ldg(p.frequency + row);
        if (p.presence) pres = __ldg(p.presence + row);
    }
    const uint32_t* mask = nullptr;
    bool none = false;
    if (p.allowed) {
        const int st = p.state ? __ldg(p.state + row) : row;
        none = st >= p.n_states;
        if (st >= 0 && !none) mask = p.allowed + static_cast<int64_t>(st) * p.allowed_ld;
    }

    Best<kBest> best;
    best.clear();
    MaxSum total;

    for (int tile = slice; tile < tiles; tile += p.slices) {
        const int e0 = tile * kTile;
        Eight<T> raw[kPerThread];
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int e = e0 + (i * kThreads + tid) * 8;
            if (e >= shift && e + 8 <= places) {
                const int4* src = reinterpret_cast<const int4*>(in + (e - shift));
                int4* dst = reinterpret_cast<int4*>(&raw[i]);
#pragma unroll
                for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) dst[j] = src[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    raw[i].v[j] = e + j >= shift && e + j < places ? in[e + j - shift] : from_f32<T>(0.0f);
            }
        }
        if (counting || biasing) {
            __syncthreads();  // the previous tile has been read
            const int words = kTile / 32 + (counting ? kTile : 0) + (biasing ? kTile : 0);
            for (int i = tid; i < words / 4; i += kThreads)
                reinterpret_cast<uint4*>(touched)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            const int v0 = e0 - shift;  // the token at the tile's first place (negative before the row)
            if (counting) {
                const int32_t* h = p.history + static_cast<int64_t>(row) * p.history_ld;
                for (int i = tid; i < said; i += kThreads) {
                    const int v = __ldg(h + i);
                    if (v >= 0 && v < p.vocab && v >= v0 && v - v0 < kTile) {
                        atomicAdd(count + (v - v0), 1u);
                        atomicOr(touched + (v - v0) / 32, 1u << ((v - v0) % 32));
                    }
                }
            }
            if (biasing && warp == kWarps - 1) {
                const int32_t* ids = p.bias_ids + static_cast<int64_t>(row) * p.bias_ld;
                const float* values = p.bias + static_cast<int64_t>(row) * p.bias_ld;
                for (int base = 0; base < p.n_bias; base += 32) {
                    int v = -1;
                    float b = 0.0f;
                    if (base + lane < p.n_bias) {
                        v = __ldg(ids + base + lane);
                        b = __ldg(values + base + lane);
                    }
                    const bool here = v >= 0 && v < p.vocab && v >= v0 && v - v0 < kTile;
                    // The lowest lane of each token adds its lanes' values in lane order.
                    unsigned same = __match_any_sync(0xffffffffu, here ? v : -1);
                    const bool leader = here && __ffs(same) - 1 == lane;
                    float sum = leader ? bias[v - v0] : 0.0f;
                    while (__any_sync(0xffffffffu, leader && same)) {
                        const int from = same ? __ffs(same) - 1 : lane;
                        const float add = __shfl_sync(0xffffffffu, b, from);
                        if (leader && same) sum += add;
                        same &= same - 1;
                    }
                    if (leader) {
                        bias[v - v0] = sum;
                        atomicOr(touched + (v - v0) / 32, 1u << ((v - v0) % 32));
                    }
                    __syncwarp();
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int at = (i * kThreads + tid) * 8;  // place within the tile
            const int e = e0 + at, v = e - shift;     // place in the row, token
            if (e >= places) continue;
            // Bit j: token v + j exists and is allowed.
            uint32_t ok = 0xffu;
            if (v < 0) ok = (0xffu << -v) & 0xffu;
            if (v + 8 > p.vocab) ok &= 0xffu >> (v + 8 - p.vocab);
            const uint32_t inside = ok;
            if (none) ok = 0;
            if (mask) {
                uint32_t bits;
                if (v < 0) {
                    bits = __ldg(mask) << -v;
                } else {
                    const uint32_t w0 = __ldg(mask + v / 32);
                    const bool next = v % 32 > 24 && (v / 32 + 1) * 32 < p.vocab;
                    const uint32_t w1 = next ? __ldg(mask + v / 32 + 1) : 0u;
                    bits = __funnelshift_r(w0, w1, v % 32);
                }
                ok &= bits;
            }
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = to_f32(raw[i].v[j]);
            if (counting || biasing) {
                const uint32_t hit = (touched[at / 32] >> (at % 32)) & 0xffu;
                if (hit) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (!((hit >> j) & 1)) continue;
                        if (counting) {
                            const uint32_t c = count[at + j];
                            if (c) {
                                x[j] = x[j] > 0.0f ? __fdiv_rn(x[j], theta) : __fmul_rn(x[j], theta);
                                x[j] = __fsub_rn(x[j], __fmul_rn(freq, static_cast<float>(c)));
                                x[j] = __fsub_rn(x[j], pres);
                            }
                        }
                        if (biasing) x[j] = __fadd_rn(x[j], bias[at + j]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!((ok >> j) & 1)) x[j] = -INFINITY;
            if (K == 0) {
                Eight<T> y;
#pragma unroll
                for (int j = 0; j < 8; ++j) y.v[j] = from_f32<T>(x[j]);
                if (same_cut && inside == 0xffu) {
                    int4* dst = reinterpret_cast<int4*>(out + v);
                    const int4* src = reinterpret_cast<const int4*>(&y);
#pragma unroll
                    for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) dst[j] = src[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if ((inside >> j) & 1) out[v + j] = y.v[j];
                }
            } else {
                float top = x[0];
#pragma unroll
                for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
                if (top > total.m) {
                    total.s *= exp_of(total.m - top);
                    total.m = top;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) total.s += exp_of(x[j] - total.m);
                if (top > best.x[kBest - 1]) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (x[j] > best.x[kBest - 1]) best.insert(x[j], v + j);
                }
            }
        }
    }

    if (K) {
        __shared__ float warp_x[kWarps][kBest];
        __shared__ int warp_id[kWarps][kBest];
        __shared__ float warp_m[kWarps], warp_s[kWarps];
        __shared__ float block_x[kBest], block_ms[2];
        __shared__ int block_id[kBest];
        float x;
        int id;
        warp_best<kBest>(best, x, id);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            const float m2 = __shfl_xor_sync(0xffffffffu, total.m, d), s2 = __shfl_xor_sync(0xffffffffu, total.s, d);
            total.merge(m2, s2);
        }
        if (lane < kBest) {
            warp_x[warp][lane] = x;
            warp_id[warp][lane] = id;
        }
        if (lane == 0) {
            warp_m[warp] = total.m;
            warp_s[warp] = total.s;
        }
        __syncthreads();
        if (warp == 0) {
            best.clear();
            for (int c = lane; c < kWarps * kBest; c += 32) best.insert(warp_x[c / kBest][c % kBest], warp_id[c / kBest][c % kBest]);
            warp_best<kBest>(best, x, id);
            total = MaxSum();
            if (lane < kWarps) {
                total.m = warp_m[lane];
                total.s = warp_s[lane];
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2) {
                const float m2 = __shfl_xor_sync(0xffffffffu, total.m, d);
                const float s2 = __shfl_xor_sync(0xffffffffu, total.s, d);
                total.merge(m2, s2);
            }
            if (p.slices > 1) {
                if (lane < kBest) {
                    block_x[lane] = x;
                    block_id[lane] = id;
                }
                if (lane == 0) {
                    block_ms[0] = total.m;
                    block_ms[1] = total.s;
                }
            }
        }
        if (p.slices > 1) {
            cluster_sync();
            if (slice == 0 && warp == 0) {
                best.clear();
                for (int c = lane; c < p.slices * kBest; c += 32)
                    best.insert(__uint_as_float(ld_cluster_u32(block_x + c % kBest, c / kBest)),
                                static_cast<int>(ld_cluster_u32(block_id + c % kBest, c / kBest)));
                warp_best<kBest>(best, x, id);
                total = MaxSum();
                if (lane < p.slices) {
                    total.m = __uint_as_float(ld_cluster_u32(block_ms, lane));
                    total.s = __uint_as_float(ld_cluster_u32(block_ms + 1, lane));
                }
#pragma unroll
                for (int d = 16; d > 0; d /= 2) {
                    const float m2 = __shfl_xor_sync(0xffffffffu, total.m, d);
                    const float s2 = __shfl_xor_sync(0xffffffffu, total.s, d);
                    total.merge(m2, s2);
                }
            }
            cluster_sync();  // the other blocks' shared memory has been read
        }
        if (slice == 0 && warp == 0 && lane < p.k) {
            const bool found = id != INT_MAX;
            const int64_t at = static_cast<int64_t>(row) * p.k + lane;
            p.ids[at] = found ? id : -1;
            if (p.logprobs) p.logprobs[at] = found ? (x - total.m) - logf(total.s) : -INFINITY;
        }
    }
}

template <typename T, int K>
cudaError_t launch(const RuleParams& p, cudaStream_t stream) {
    static DeviceOnce once;
    const size_t rules = (p.history ? kTile * 4 : 0) + (p.n_bias > 0 ? kTile * 4 : 0);
    const size_t bytes = rules ? rules + kTile / 8 : 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!once.done(dev)) {
        if ((e = cudaFuncSetAttribute(logits_kernel<T, K>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kTile * 8 + kTile / 8)) != cudaSuccess)
            return e;
        once.mark(dev);
    }
    // Rows beyond a grid's y range go in further launches.
    for (int r0 = 0; r0 < p.rows; r0 += 65535) {
        RuleParams q = p;
        q.rows = std::min(65535, p.rows - r0);
        const auto move = [&](auto*& ptr, int64_t elements) {
            if (ptr) ptr += elements;
        };
        q.logits = static_cast<const T*>(p.logits) + r0 * p.ld;
        if (p.out) q.out = static_cast<T*>(p.out) + r0 * p.out_ld;
        move(q.history, r0 * p.history_ld);
        move(q.history_len, r0);
        move(q.repetition, r0);
        move(q.frequency, r0);
        move(q.presence, r0);
        move(q.bias_ids, r0 * p.bias_ld);
        move(q.bias, r0 * p.bias_ld);
        if (p.state) {
            move(q.state, r0);
        } else if (p.allowed) {
            move(q.allowed, r0 * p.allowed_ld);
            q.n_states = std::max(0, p.n_states - r0);
        }
        move(q.ids, static_cast<int64_t>(r0) * p.k);
        move(q.logprobs, static_cast<int64_t>(r0) * p.k);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(p.slices, q.rows);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = bytes;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = p.slices;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = K && p.slices > 1 ? 1 : 0;
        if ((e = cudaLaunchKernelEx(&cfg, logits_kernel<T, K>, q)) != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <int K>
cudaError_t launch_type(const RuleParams& p, int dtype, cudaStream_t stream) {
    if (dtype == TELMO_DTYPE_F32) return launch<float, K>(p, stream);
    if (dtype == TELMO_DTYPE_BF16) return launch<__nv_bfloat16, K>(p, stream);
    return launch<__half, K>(p, stream);
}

// Checks what both entry points share and fills `p`.
int prepare(Ctx* ctx, const char* who, const void* logits, int dtype, size_t ld, size_t rows, size_t vocab,
            const telmo_logit_rules* rules, RuleParams* p) {
    const auto bad = [&](const char* what) { return ctx->fail(TELMO_ERR_ARGUMENT, "%s: %s", who, what); };
    if (dtype != TELMO_DTYPE_F32 && dtype != TELMO_DTYPE_BF16 && dtype != TELMO_DTYPE_F16) return bad("unknown dtype");
    const uintptr_t size = dtype == TELMO_DTYPE_F32 ? 4 : 2;
    const auto misaligned = [](const void* q, uintptr_t b) { return reinterpret_cast<uintptr_t>(q) % b != 0; };
    constexpr size_t kMost = size_t(1) << 40;
    if (!logits || misaligned(logits, size)) return bad("logits are NULL or not aligned to their elements");
    if (vocab == 0 || vocab > (1u << 30) || rows > (1u << 30) || ld < vocab || ld > kMost) return bad("bad sizes");
    *p = RuleParams();
    p->logits = logits;
    p->ld = static_cast<int64_t>(ld);
    p->rows = static_cast<int>(rows);
    p->vocab = static_cast<int>(vocab);
    if (!rules) return TELMO_OK;
    const telmo_logit_rules& r = *rules;
    if (misaligned(r.history, 4) || misaligned(r.history_len, 4) || misaligned(r.repetition, 4) ||
        misaligned(r.frequency, 4) || misaligned(r.presence, 4) || misaligned(r.bias_ids, 4) || misaligned(r.bias, 4) ||
        misaligned(r.allowed, 4) || misaligned(r.state, 4))
        return bad("a rule's array is not aligned to its elements");
    if (r.history) {
        if (!r.history_len) return bad("tokens so far without their lengths");
        if (r.n_history > (1u << 30) || r.history_ld < r.n_history || r.history_ld > kMost)
            return bad("bad sizes of the tokens so far");
        p->n_history = static_cast<int>(r.n_history);
        p->history = r.history;
        p->history_ld = static_cast<int64_t>(r.history_ld);
        p->history_len = r.history_len;
        p->repetition = r.repetition;
        p->frequency = r.frequency;
        p->presence = r.presence;
    } else if (r.repetition || r.frequency || r.presence) {
        return bad("penalties without the tokens so far");
    }
    if (r.n_bias) {
        if (!r.bias_ids || !r.bias || r.n_bias > (1u << 30) || r.bias_ld < r.n_bias || r.bias_ld > kMost)
            return bad("bad bias lists");
        p->bias_ids = r.bias_ids;
        p->bias = r.bias;
        p->bias_ld = static_cast<int64_t>(r.bias_ld);
        p->n_bias = static_cast<int>(r.n_bias);
    }
    if (r.allowed) {
        if (r.n_states == 0 || r.n_states > (1u << 30) || r.allowed_ld < (vocab + 31) / 32 || r.allowed_ld > kMost)
            return bad("bad masks");
        if (!r.state && r.n_states < rows) return bad("fewer masks than rows, and no states");
        p->allowed = r.allowed;
        p->allowed_ld = static_cast<int64_t>(r.allowed_ld);
        p->n_states = static_cast<int>(r.n_states);
        p->state = r.state;
    } else if (r.state) {
        return bad("states without masks");
    }
    return TELMO_OK;
}

}  // namespace

}  // namespace telmo

using namespace telmo;

extern "C" int telmo_logits_constrain(telmo_ctx* c, const void* logits, int dtype, size_t ld, size_t rows, size_t vocab,
                                      const telmo_logit_rules* rules, void* out, size_t out_ld, void* stream) {
    Ctx* ctx = as_ctx(c);
    if (!ctx) return TELMO_ERR_ARGUMENT;
    if (rows == 0) return TELMO_OK;
    RuleParams p;
    if (int rc = prepare(ctx, "telmo_logits_constrain", logits, dtype, ld, rows, vocab, rules, &p)) return rc;
    if (!out || reinterpret_cast<uintptr_t>(out) % (dtype == TELMO_DTYPE_F32 ? 4 : 2) || out_ld < vocab ||
        out_ld > (size_t(1) << 40))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_constrain: out is NULL or misaligned, or its rows are short");
    DeviceScope scope;
    if (int rc = scope.enter(ctx)) return rc;
    p.out = out;
    p.out_ld = static_cast<int64_t>(out_ld);
    p.slices = (p.vocab + 7 + kTile - 1) / kTile;
    return ctx->cuda(launch_type<0>(p, dtype, static_cast<cudaStream_t>(stream)), "telmo_logits_constrain");
}

extern "C" int telmo_logits_choose(telmo_ctx* c, const void* logits, int dtype, size_t ld, size_t rows, size_t vocab,
                                   const telmo_logit_rules* rules, size_t k, int32_t* ids, float* logprobs,
                                   void* stream) {
    Ctx* ctx = as_ctx(c);
    if (!ctx) return TELMO_ERR_ARGUMENT;
    if (rows == 0) return TELMO_OK;
    RuleParams p;
    if (int rc = prepare(ctx, "telmo_logits_choose", logits, dtype, ld, rows, vocab, rules, &p)) return rc;
    if (k == 0 || k > kMaxK)
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_choose: 1 to %d tokens a row, not %zu", kMaxK, k);
    if (!ids || reinterpret_cast<uintptr_t>(ids) % 4 || reinterpret_cast<uintptr_t>(logprobs) % 4)
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_choose: ids are NULL, or ids or logprobs misaligned");
    DeviceScope scope;
    if (int rc = scope.enter(ctx)) return rc;
    p.ids = ids;
    p.logprobs = logprobs;
    p.k = static_cast<int>(k);
    // Enough blocks for two per SM, and no block without a tile.
    const int tiles = (p.vocab + 7 + kTile - 1) / kTile;
    p.slices = 1;
    while (p.slices < 8 && p.slices < tiles && static_cast<int64_t>(p.slices) * p.rows < 2 * ctx->sms) p.slices *= 2;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = k == 1 ? launch_type<1>(p, dtype, s) : k == 2 ? launch_type<2>(p, dtype, s)
                        : k <= 4 ? launch_type<4>(p, dtype, s) : launch_type<8>(p, dtype, s);
    return ctx->cuda(e, "telmo_logits_choose");
}
