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
// every token so touched; eight tokens whose bits are clear skip the rules. Only the touched places of
// the counts and biases are cleared, and a block keeps the lists in registers from tile to tile.
//
// The k best are found by a bound: a token's key is its value's order and then its place, so no two are
// equal; tokens whose key is below the block's bound are passed over, others go to a buffer in
// shared memory. The bound starts as the k-th largest of the threads' best keys of the first tile (k
// threads have a key that large) and rises when the buffer has to be emptied. So nearly all tokens cost
// one comparison of a group's maximum; per-thread lists of the k best, of which some lane of a
// warp always has a new entry, took 250 us where this takes 60 (256 rows of 131072 f32 values, k = 8).
// The blocks of a row form a cluster of up to eight and meet through distributed shared memory: no
// workspace, no counters, one launch.
#include "../../include/telmo_b200.h"
#include "api_internal.h"
#include "kernels.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace telmo {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 8192;                        // tokens per tile
constexpr int kPerThread = kTile / 8 / kThreads;   // groups of eight tokens a thread has in a tile
constexpr int kMaxK = 8;
constexpr int kBuffer = 1024;                      // keys a block keeps before it raises its bound
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

// A token's place in the order of choice: the larger value first (-0 counts as 0), then the lower
// token. 0 for what is never chosen: a NaN, or -infinity.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t order = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return x > -INFINITY ? (static_cast<uint64_t>(order) << 32) | static_cast<uint32_t>(~token) : 0;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int token_of(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

__device__ __forceinline__ uint64_t warp_max(uint64_t key) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32) == hi ? static_cast<uint32_t>(key) : 0u);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The k largest of `count` keys in shared memory, lane i of the warp (which all calls it) getting the
// i-th, 0 where there are fewer: k rounds, each lane offering the largest of its own that is below
// the last round's.
__device__ __forceinline__ uint64_t warp_best(const uint64_t* keys, int count, int k) {
    const int lane = threadIdx.x % 32;
    uint64_t last = ~0ull, mine = 0;
    for (int i = 0; i < k; ++i) {
        uint64_t top = 0;
        for (int c = lane; c < count; c += 32) {
            const uint64_t v = keys[c];
            if (v < last && v > top) top = v;
        }
        last = warp_max(top);
        if (lane == i) mine = last;
        if (last == 0) break;
    }
    return mine;
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
__device__ __forceinline__ uint64_t ld_cluster_u64(const void* p, uint32_t rank) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}

// One step of the rules on a touched token's value.
__device__ __forceinline__ float penalised(float x, uint32_t n, float theta, float freq, float pres) {
    if (n == 0) return x;
    x = x > 0.0f ? __fdiv_rn(x, theta) : __fmul_rn(x, theta);
    return __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(n))), pres);
}

// The choosing side of a block.
struct Choice {
    uint64_t buffer[kBuffer];
    uint64_t firsts[kWarps * kMaxK];
    uint64_t bound, best[kMaxK];
    int buffered;
    float warp_m[kWarps], warp_s[kWarps], m, s;
};

// Puts the buffer's k best at its start; every thread calls it. The k-th is then a bound.
__device__ void empty_buffer(Choice& ch, int k) {
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const uint64_t key = warp_best(ch.buffer, ch.buffered, k);
        const int found = __popc(__ballot_sync(0xffffffffu, key != 0));
        const uint64_t kth = __shfl_sync(0xffffffffu, key, k - 1);
        __syncwarp();
        if (lane < found) ch.buffer[lane] = key;
        if (lane == 0) {
            ch.buffered = found;
            if (kth > ch.bound) ch.bound = kth;
        }
    }
    __syncthreads();
}

// Raises the bound to the k-th largest of the threads' best keys; every thread calls it.
__device__ void bound_by_threads(Choice& ch, uint64_t key, int k) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int i = 0; i < k; ++i) {
        const uint64_t top = warp_max(key);
        if (lane == 0) ch.firsts[warp * k + i] = top;
        if (key == top) key = 0;  // a key that is not 0 is one thread's alone
    }
    __syncthreads();
    if (warp == 0) {
        const uint64_t kth = __shfl_sync(0xffffffffu, warp_best(ch.firsts, kWarps * k, k), k - 1);
        if (lane == 0 && kth > ch.bound) ch.bound = kth;
    }
    __syncthreads();
}

// T: the logits' type. CHOOSE: the k best of each row, else every value. Blocks (x: slice of the
// row, y: row) take the row's tiles in turn.
template <typename T, bool CHOOSE>
__global__ void __launch_bounds__(kThreads) logits_kernel(const RuleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t touched[kTile / 32];  // one bit per token of the tile
    __shared__ typename std::conditional<CHOOSE, Choice, int>::type choice;
    const int row = blockIdx.y, slice = blockIdx.x;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const bool counting = p.history != nullptr, biasing = p.n_bias > 0, listing = counting || biasing;
    uint32_t* count = reinterpret_cast<uint32_t*>(smem);
    float* bias = reinterpret_cast<float*>(count + (counting ? kTile : 0));

    const T* in = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.ld;
    T* out = CHOOSE ? nullptr : static_cast<T*>(p.out) + static_cast<int64_t>(row) * p.out_ld;
    // Tiles are cut where the row's addresses are multiples of 16 bytes: place e of the cut row is
    // token e - shift.
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
    const bool same_cut = !CHOOSE && static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T)) == shift;
    const int places = p.vocab + shift;
    const int tiles = (places + kTile - 1) / kTile;

    // The row's lists: the first of the tokens so far in every thread's registers, the first of the
    // biases in those of the last warp.
    constexpr int kKept = 4;
    int said = 0, kept[kKept], bias_kept_id[kKept];
    float bias_kept[kKept];
    float theta = 1.0f, freq = 0.0f, pres = 0.0f;
    const int32_t* history = counting ? p.history + static_cast<int64_t>(row) * p.history_ld : nullptr;
    const int32_t* bias_ids = biasing ? p.bias_ids + static_cast<int64_t>(row) * p.bias_ld : nullptr;
    const float* bias_values = biasing ? p.bias + static_cast<int64_t>(row) * p.bias_ld : nullptr;
    if (counting) {
        said = max(0, min(__ldg(p.history_len + row), p.n_history));
        if (p.repetition) theta = __ldg(p.repetition + row);
        if (p.frequency) freq = __ldg(p.frequency + row);
        if (p.presence) pres = __ldg(p.presence + row);
#pragma unroll
        for (int i = 0; i < kKept; ++i) kept[i] = tid + i * kThreads < said ? __ldg(history + tid + i * kThreads) : -1;
    }
    const bool bias_warp = biasing && warp == kWarps - 1;
    if (bias_warp) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
            const bool there = lane + 32 * i < p.n_bias;
            bias_kept_id[i] = there ? __ldg(bias_ids + lane + 32 * i) : -1;
            bias_kept[i] = there ? __ldg(bias_values + lane + 32 * i) : 0.0f;
        }
    }
    // Calls f(token) for each of this thread's tokens so far, g(token, bias) for a lane's biases in list order.
    const auto each_said = [&](auto f) {
        if (!counting) return;
#pragma unroll
        for (int i = 0; i < kKept; ++i) f(kept[i]);
        for (int i = tid + kKept * kThreads; i < said; i += kThreads) f(__ldg(history + i));
    };
    const auto each_bias = [&](auto f) {
        if (!bias_warp) return;
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (32 * i < p.n_bias) f(bias_kept_id[i], bias_kept[i]);
        for (int base = 32 * kKept; base < p.n_bias; base += 32) {
            const bool there = base + lane < p.n_bias;
            f(there ? __ldg(bias_ids + base + lane) : -1, there ? __ldg(bias_values + base + lane) : 0.0f);
        }
    };

    const uint32_t* mask = nullptr;
    bool none = false;
    if (p.allowed) {
        const int st = p.state ? __ldg(p.state + row) : row;
        none = st >= p.n_states;
        if (st >= 0 && !none) mask = p.allowed + static_cast<int64_t>(st) * p.allowed_ld;
    }

    MaxSum total;
    if constexpr (CHOOSE) {
        if (tid == 0) {
            choice.bound = 0x007fffffffffffffull;  // the value -infinity: below what can be chosen
            choice.buffered = 0;
        }
    }

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
        const int v0 = e0 - shift;  // the token at the tile's first place (negative before the row)
        const auto in_tile = [&](int v) { return v >= 0 && v < p.vocab && v >= v0 && v - v0 < kTile; };
        if (listing) {
            __syncthreads();  // the previous tile has been read
            for (int i = tid; i < kTile / 32; i += kThreads) touched[i] = 0;
            const auto clear = [&](int v) {
                if (!in_tile(v)) return;
                if (counting) count[v - v0] = 0;
                if (biasing) bias[v - v0] = 0.0f;
            };
            each_said(clear);
            each_bias([&](int v, float) { clear(v); });
            __syncthreads();
            const auto touch = [&](int v) { atomicOr(touched + (v - v0) / 32, 1u << ((v - v0) % 32)); };
            each_said([&](int v) {
                if (!in_tile(v)) return;
                atomicAdd(count + (v - v0), 1u);
                touch(v);
            });
            each_bias([&](int v, float b) {
                // The lowest lane of each token adds its lanes' values in lane order.
                const bool here = in_tile(v);
                if (!__any_sync(0xffffffffu, here)) return;
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
                    touch(v);
                }
                __syncwarp();
            });
            __syncthreads();
        }
        float x[kPerThread][8];
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int at = (i * kThreads + tid) * 8;  // place within the tile
            const int e = e0 + at, v = e - shift;     // place in the row, token
            if (e >= places) {
                if (CHOOSE) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[i][j] = -INFINITY;
                }
                continue;
            }
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
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = to_f32(raw[i].v[j]);
            if (listing) {
                const uint32_t hit = (touched[at / 32] >> (at % 32)) & 0xffu;
                if (hit) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (!((hit >> j) & 1)) continue;
                        if (counting) x[i][j] = penalised(x[i][j], count[at + j], theta, freq, pres);
                        if (biasing) x[i][j] = __fadd_rn(x[i][j], bias[at + j]);
                    }
                }
            }
            if (ok != 0xffu) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!((ok >> j) & 1)) x[i][j] = -INFINITY;
            }
            if (!CHOOSE) {
                Eight<T> y;
#pragma unroll
                for (int j = 0; j < 8; ++j) y.v[j] = from_f32<T>(x[i][j]);
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
            }
        }
        if constexpr (CHOOSE) {
            float top = x[0][0];
#pragma unroll
            for (int j = 1; j < 8 * kPerThread; ++j) top = fmaxf(top, x[j / 8][j % 8]);
            if (top > total.m) {
                total.s *= exp_of(total.m - top);
                total.m = top;
            }
#pragma unroll
            for (int j = 0; j < 8 * kPerThread; ++j) total.s += exp_of(x[j / 8][j % 8] - total.m);
            // Keys that reach the bound go to the buffer; it is emptied, and the bound raised, where the
            // tile might not fit.
            const int first = e0 - shift + tid * 8;  // the token of x[0][0]
            const auto best_key = [&] {
                uint64_t key = 0;
#pragma unroll
                for (int j = 0; j < 8 * kPerThread; ++j) {
                    const uint64_t one = key_of(x[j / 8][j % 8], first + j / 8 * (kThreads * 8) + j % 8);
                    if (one > key) key = one;
                }
                return key;
            };
            if (tile == slice) __syncthreads();  // the bound has been set
            int have = 0;  // read before the meeting: behind it some thread may be adding already
            const auto hot_threads = [&] {
                const uint64_t bound = choice.bound;
                have = choice.buffered;
                const bool hot = top > -INFINITY && top >= value_of(bound | 0xffffffffu) && best_key() >= bound;
                return __syncthreads_count(hot);
            };
            int hot = hot_threads();
            if (hot > 0) {
                if (have + hot * 8 * kPerThread > kBuffer) {
                    empty_buffer(choice, p.k);
                    hot = hot_threads();
                    if (have + hot * 8 * kPerThread > kBuffer) {
                        bound_by_threads(choice, best_key(), p.k);
                    }
                }
                const uint64_t bound = choice.bound;
                if (top > -INFINITY && top >= value_of(bound | 0xffffffffu)) {
#pragma unroll
                    for (int j = 0; j < 8 * kPerThread; ++j) {
                        const uint64_t key = key_of(x[j / 8][j % 8], first + j / 8 * (kThreads * 8) + j % 8);
                        if (key >= bound) choice.buffer[atomicAdd(&choice.buffered, 1)] = key;
                    }
                }
                __syncthreads();  // the buffer's count is settled before it is read again
            }
        }
    }

    if constexpr (CHOOSE) {
        if (slice >= tiles) __syncthreads();  // a block without a tile: its buffer has been set
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            const float m2 = __shfl_xor_sync(0xffffffffu, total.m, d), s2 = __shfl_xor_sync(0xffffffffu, total.s, d);
            total.merge(m2, s2);
        }
        if (lane == 0) {
            choice.warp_m[warp] = total.m;
            choice.warp_s[warp] = total.s;
        }
        __syncthreads();
        uint64_t key = 0;
        const auto across = [&](bool there, float m, float s) {  // over the warp's lanes
            total = MaxSum();
            if (there) {
                total.m = m;
                total.s = s;
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2) {
                const float m2 = __shfl_xor_sync(0xffffffffu, total.m, d);
                const float s2 = __shfl_xor_sync(0xffffffffu, total.s, d);
                total.merge(m2, s2);
            }
        };
        if (warp == 0) {
            key = warp_best(choice.buffer, choice.buffered, p.k);
            across(lane < kWarps, choice.warp_m[lane % kWarps], choice.warp_s[lane % kWarps]);
            if (lane < p.k) choice.best[lane] = key;
            if (lane == 0) {
                choice.m = total.m;
                choice.s = total.s;
            }
        }
        if (p.slices > 1) {
            __syncwarp();
            cluster_sync();
            if (slice == 0 && warp == 0) {
                // At most 8 blocks of 8 keys: two a lane.
                for (int c = lane; c < p.slices * p.k; c += 32)
                    choice.firsts[c] = ld_cluster_u64(&choice.best[c % p.k], c / p.k);
                __syncwarp();
                key = warp_best(choice.firsts, p.slices * p.k, p.k);
                const uint32_t from = lane < p.slices ? lane : 0;
                across(lane < p.slices, __uint_as_float(ld_cluster_u32(&choice.m, from)),
                       __uint_as_float(ld_cluster_u32(&choice.s, from)));
            }
            __syncwarp();
            cluster_sync();  // the other blocks' shared memory has been read
        }
        if (slice == 0 && warp == 0 && lane < p.k) {
            const int64_t at = static_cast<int64_t>(row) * p.k + lane;
            p.ids[at] = key ? token_of(key) : -1;
            if (p.logprobs) p.logprobs[at] = key ? (value_of(key) - total.m) - logf(total.s) : -INFINITY;
        }
    }
}

template <typename T, bool CHOOSE>
cudaError_t launch(const RuleParams& p, cudaStream_t stream) {
    static DeviceOnce once;
    const size_t bytes = (p.history ? kTile * 4 : 0) + (p.n_bias > 0 ? kTile * 4 : 0);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!once.done(dev)) {
        if ((e = cudaFuncSetAttribute(logits_kernel<T, CHOOSE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kTile * 8)) != cudaSuccess)
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
        cfg.numAttrs = CHOOSE && p.slices > 1 ? 1 : 0;
        if ((e = cudaLaunchKernelEx(&cfg, logits_kernel<T, CHOOSE>, q)) != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <bool CHOOSE>
cudaError_t launch_type(const RuleParams& p, int dtype, cudaStream_t stream) {
    if (dtype == TELMO_DTYPE_F32) return launch<float, CHOOSE>(p, stream);
    if (dtype == TELMO_DTYPE_BF16) return launch<__nv_bfloat16, CHOOSE>(p, stream);
    return launch<__half, CHOOSE>(p, stream);
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
    // As many blocks as tiles, or several tiles a block (whose lists are read once) where six blocks per
    // SM stay.
    const int tiles = (p.vocab + 7 + kTile - 1) / kTile;
    p.slices = std::min<int64_t>(tiles, std::max<int64_t>(1, (6ll * ctx->sms + p.rows - 1) / p.rows));
    return ctx->cuda(launch_type<false>(p, dtype, static_cast<cudaStream_t>(stream)), "telmo_logits_constrain");
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
    // Clusters of up to eight blocks a row until there are six blocks per SM or a tile for each.
    const int tiles = (p.vocab + 7 + kTile - 1) / kTile;
    p.slices = 1;
    while (p.slices < 8 && p.slices < tiles && static_cast<int64_t>(p.slices) * p.rows < 6 * ctx->sms) p.slices *= 2;
    return ctx->cuda(launch_type<true>(p, dtype, static_cast<cudaStream_t>(stream)), "telmo_logits_choose");
}
