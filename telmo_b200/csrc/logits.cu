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
// Both read the logits once and are bound by that (constrain writes them once more), if few
// instructions go to each value: 6.5 TB/s leave an SM about ten a value of 16 bits. So the pass over the
// logits knows masks alone, and the listed tokens, few against the vocabulary, come after it, a token
// a thread:
//   constrain  copies allowed values and writes -infinity elsewhere, in the logits' own type; then
//              each listed token that is allowed is read again (in place or not, it is still the
//              logit), goes through the rules and is written.
//   choose     leaves listed tokens out by a bit map of the window; then they go through the rules and
//              join the others.
// A block walks over windows of 8192 to 65536 tokens: it sets a bit for each listed token's place, numbers
// the bits in order (a prefix sum over the words' counts), and counts by number in shared memory with
// integer atomics (the counts do not depend on their order); a token's biases add up in list order, the
// first ones an entry a round, further ones by one walk over the list. Tokens go to threads by number, so no sum
// depends on timing. Numbers beyond kNumbers come in further rounds over the lists. With the rules inside the
// pass over the logits some lane of a warp nearly always had a listed token and all paid: 92 us for 256 rows of
// 131072 bf16 values with 2000 tokens each, which take 50 us here (137 MB to read and write; the pass alone 24,
// with masks 31, with lists and no masks 44).
//
// The k best are found by a bound: a token's key is its value's order and then its place, so no two are
// equal; tokens whose key is below the block's bound are passed over, others go to a buffer in
// shared memory. The bound starts as the k-th largest of the warps' largest values of the first tile (k
// warps have a value that large) and rises when the buffer has to be emptied, so nearly all tokens cost
// one comparison of a thread's maximum. The blocks of a row form a cluster of up to eight and meet
// through distributed shared memory: no workspace, no counters, one launch.
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
constexpr int kMostWindow = 8 * kTile;             // tokens per window at most
constexpr int kNumbers = 2048;                     // listed tokens with a number
constexpr int kMaxK = 8;
// Rounds over a list of biases that give each token its next one, before a walk over the whole list adds the rest.
// (256 entries, each token twice, 64 rows: 7.8 us with two rounds, 10.2 with none; 4096 entries of 64 tokens: 91 us
// with two, 125 with sixteen, 233 with as many as there are entries of a token, which is quadratic.)
constexpr int kBiasRounds = 2;
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
    int window;  // tokens per window, a multiple of kTile
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
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int token) {
    return x > -INFINITY ? (static_cast<uint64_t>(order_of(x)) << 32) | static_cast<uint32_t>(~token) : 0;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int token_of(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

__device__ __forceinline__ uint64_t warp_max(uint64_t key) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
    const bool highest = static_cast<uint32_t>(key >> 32) == hi;
    const uint32_t lo = __reduce_max_sync(0xffffffffu, highest ? static_cast<uint32_t>(key) : 0u);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The k largest of `count` keys in shared memory, in order, into best (0 where there are fewer). Every
// thread calls it, with the keys written and synchronised; best is written behind the next meeting.
__device__ __forceinline__ void find_best(const uint64_t* keys, int count, int k, uint64_t* best) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t mine = keys[i];
        int larger = 0;
        for (int j = 0; j < count; ++j) larger += keys[j] > mine;
        if (larger < k) best[larger] = mine;
    }
}

// The product is rounded before the instruction: 2^-24 of |d| log2 e, relative to a term e^d that is the smaller the
// larger |d| is. With one thread's values added one after another, log-probabilities of a row of 49157 were seen off
// by 7.5e-8 (f32 sums in a tree: 1.2e-8), well within what f32 can tell of a value near -10.
__device__ __forceinline__ float exp_of(float d) { return ex2_approx(d * 1.44269504f); }

// The sum of e^x as e^m s with the running maximum m. (One fused multiply-add for x log2 e - m log2 e would
// save an instruction a value, but overflow at a type's lowest value.)
struct MaxSum {
    float m = kLowest, s = 0.0f;
    __device__ __forceinline__ void reach(float top) {
        if (top > m) {
            s *= exp_of(m - top);
            m = top;
        }
    }
    __device__ __forceinline__ void add(float x) { s += exp_of(x - m); }
    // The warp's lanes together, in every lane.
    __device__ __forceinline__ void join() {
        const uint32_t order = __reduce_max_sync(0xffffffffu, order_of(m));  // m is no NaN
        const float top = value_of(static_cast<uint64_t>(order) << 32);
        s *= exp_of(m - top);
        m = top;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
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
    uint32_t warp_top[kWarps];
    float warp_m[kWarps], warp_s[kWarps], m, s;
};

// Keeps the buffer's k best alone and makes the k-th the bound; every thread calls it.
__device__ void empty_buffer(Choice& ch, int k) {
    if (threadIdx.x < kMaxK) ch.best[threadIdx.x] = 0;
    __syncthreads();
    find_best(ch.buffer, ch.buffered, k, ch.best);
    __syncthreads();
    if (threadIdx.x < k) ch.buffer[threadIdx.x] = ch.best[threadIdx.x];
    if (threadIdx.x == 0) {
        ch.buffered = min(ch.buffered, k);
        if (ch.best[k - 1] > ch.bound) ch.bound = ch.best[k - 1];
    }
    __syncthreads();
}

// Raises the bound to the k-th largest of the threads' best keys; every thread calls it.
__device__ void bound_by_threads(Choice& ch, uint64_t key, int k) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x < kMaxK) ch.best[threadIdx.x] = 0;
    for (int i = 0; i < k; ++i) {
        const uint64_t top = warp_max(key);
        if (lane == 0) ch.firsts[warp * k + i] = top;
        if (key == top) key = 0;  // a key that is not 0 is one thread's alone
    }
    __syncthreads();
    // Keys of 0 have as many larger ones as there are others: at most the last of them is one of the k best.
    find_best(ch.firsts, kWarps * k, k, ch.best);
    __syncthreads();
    if (threadIdx.x == 0 && ch.best[k - 1] > ch.bound) ch.bound = ch.best[k - 1];
    __syncthreads();
}

// The first bound: the k-th largest of the warps' largest values. top: the thread's.
__device__ void bound_by_warps(Choice& ch, float top, int k) {
    const uint32_t order = __reduce_max_sync(0xffffffffu, order_of(top > -INFINITY ? top : -INFINITY));
    if (threadIdx.x % 32 == 0) ch.warp_top[threadIdx.x / 32] = order;
    __syncthreads();
    if (threadIdx.x < kWarps) {
        const uint32_t mine = ch.warp_top[threadIdx.x];
        int before = 0;  // larger ones, and equal ones of earlier warps
        for (int w = 0; w < kWarps; ++w)
            before += ch.warp_top[w] > mine || (ch.warp_top[w] == mine && w < static_cast<int>(threadIdx.x));
        const uint64_t bound = static_cast<uint64_t>(mine) << 32;
        if (before == k - 1 && bound > ch.bound) ch.bound = bound;
    }
    __syncthreads();
}

// Eight values of which those with a bit of `ok` clear become -infinity.
__device__ __forceinline__ void keep_allowed(Eight<float>& y, uint32_t ok) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (!((ok >> j) & 1)) y.v[j] = -INFINITY;
}
template <typename T>
__device__ __forceinline__ void keep_allowed(Eight<T>& y, uint32_t ok) {
    constexpr uint32_t kNone = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    uint32_t* w = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t two = (ok >> (2 * j)) & 3u, keep = ((two | (two << 15)) & 0x00010001u) * 0xffffu;
        w[j] = (w[j] & keep) | (kNone & ~keep);
    }
}

// T: the logits' type. CHOOSE: the k best of each row, else every value. Blocks (x: slice of the
// row, y: row) take the row's windows in turn.
template <typename T, bool CHOOSE>
__global__ void __launch_bounds__(kThreads, CHOOSE ? 2 : 3) logits_kernel(const RuleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t listed[kMostWindow / 32];      // a bit per place of the window
    __shared__ uint16_t before[kMostWindow / 32];      // bits in the words before
    __shared__ int warp_bits[kWarps];
    __shared__ typename std::conditional<CHOOSE, Choice, int>::type choice;
    const int row = blockIdx.y, slice = blockIdx.x;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const bool counting = p.history != nullptr, biasing = p.n_bias > 0, listing = counting || biasing;
    uint16_t* list = reinterpret_cast<uint16_t*>(smem);  // places by number
    uint32_t* count = reinterpret_cast<uint32_t*>(list + kNumbers);
    float* bias = reinterpret_cast<float*>(count + kNumbers);
    uint32_t* entry = reinterpret_cast<uint32_t*>(bias + kNumbers);  // the token's last entry added to its bias
    uint32_t* later = entry + kNumbers;                              // and the one behind it

    const T* in = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.ld;
    T* out = CHOOSE ? nullptr : static_cast<T*>(p.out) + static_cast<int64_t>(row) * p.out_ld;
    // Tiles are cut where the row's addresses are multiples of 16 bytes: place e of the cut row is
    // token e - shift.
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
    const bool same_cut = !CHOOSE && static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T)) == shift;
    const int places = p.vocab + shift;

    // The row's lists. What lies outside the vocabulary becomes kNowhere. A thread's first entries stay in
    // registers, on their way before the first meeting (256 rows of 131072: constrain 52.6 -> 49.7 us, choose 74 ->
    // 71.5); further ones are read again for each window, from L1 or L2: keeping them too cost the pass spills.
    constexpr int kNowhere = INT_MIN;
    int said = 0;
    float theta = 1.0f, freq = 0.0f, pres = 0.0f;
    // Made again where they are used, which is cheaper than three pointers kept through the pass.
    const auto history = [&] { return p.history + static_cast<int64_t>(row) * p.history_ld; };
    const auto bias_ids = [&] { return p.bias_ids + static_cast<int64_t>(row) * p.bias_ld; };
    const auto bias_values = [&] { return p.bias + static_cast<int64_t>(row) * p.bias_ld; };
    const auto token = [&](const int32_t* list_at) {
        const int v = __ldg(list_at);
        return v >= 0 && v < p.vocab ? v : kNowhere;
    };
    if (counting) {
        said = max(0, min(__ldg(p.history_len + row), p.n_history));
        if (p.repetition) theta = __ldg(p.repetition + row);
        if (p.frequency) freq = __ldg(p.frequency + row);
        if (p.presence) pres = __ldg(p.presence + row);
    }
    // Calls f(token) for each of this thread's tokens so far, f(token, bias, entry) for its biases.
    const int first_said = tid < said ? token(history() + tid) : kNowhere;
    const auto each_said = [&](auto f) {
        f(first_said);
#pragma unroll 4
        for (int i = tid + kThreads; i < said; i += kThreads) f(token(history() + i));
    };
    const int first_biased = biasing && tid < p.n_bias ? token(bias_ids() + tid) : kNowhere;
    const auto each_bias = [&](auto f) {
        if (!biasing) return;
        f(first_biased, tid < p.n_bias ? __ldg(bias_values() + tid) : 0.0f, tid);
        for (int i = tid + kThreads; i < p.n_bias; i += kThreads) f(token(bias_ids() + i), __ldg(bias_values() + i), i);
    };

    const uint32_t* mask = nullptr;
    bool none = false;
    if (p.allowed) {
        const int st = p.state ? __ldg(p.state + row) : row;
        none = st >= p.n_states;
        if (st >= 0 && !none) mask = p.allowed + static_cast<int64_t>(st) * p.allowed_ld;
    }

    MaxSum total;
    bool bounded = false;  // the bound comes from a tile
    int used = 0;          // no fewer than the buffer's keys
    if constexpr (CHOOSE) {
        if (tid == 0) {
            choice.bound = 0x007fffffffffffffull;  // the value -infinity: below what can be chosen
            choice.buffered = 0;
        }
    }
    // Up to kMost tokens of every thread: those that reach the bound go to the buffer, which is emptied, and
    // the bound raised, where they might not fit. top: the thread's largest value; each_token(f) calls
    // f(value, token). Every thread calls this.
    const auto offer = [&](float top, auto each_token, auto most) {
        if constexpr (CHOOSE) {
            constexpr int kMost = decltype(most)::value;
            if (!bounded) {
                bound_by_warps(choice, top, p.k);
                bounded = true;
            }
            const auto hot = [&] { return top > -INFINITY && top >= value_of(choice.bound); };
            int n = __syncthreads_count(hot());
            if (n == 0) return;
            if (used + n * kMost > kBuffer) {
                empty_buffer(choice, p.k);
                used = p.k;
                n = __syncthreads_count(hot());
                if (used + n * kMost > kBuffer) {
                    uint64_t best = 0;
                    each_token([&](float x, int v) {
                        const uint64_t key = key_of(x, v);
                        if (key > best) best = key;
                    });
                    bound_by_threads(choice, best, p.k);
                    n = p.k;  // threads with a key that large
                }
            }
            used += n * kMost;
            const uint64_t bound = choice.bound;
            if (hot())
                each_token([&](float x, int v) {
                    if (!(x >= value_of(bound))) return;
                    const uint64_t key = key_of(x, v);
                    if (key >= bound) choice.buffer[atomicAdd(&choice.buffered, 1)] = key;
                });
        }
    };

    // (Unsigned: one step behind 2^30 places still fits.)
    const unsigned window = p.window;
    for (unsigned begin = slice * window; begin < static_cast<unsigned>(places); begin += p.slices * window) {
        const int w_begin = begin;
        const int w0 = w_begin - shift;  // the token at the window's first place (negative before the row)
        const auto in_window = [&](int v) {
            return v >= 0 ? static_cast<unsigned>(v) - static_cast<unsigned>(w0) : ~0u;
        };
        const auto clear = [&](int n) {
            for (int i = tid; i < n; i += kThreads) {
                count[i] = 0;
                bias[i] = 0.0f;
                entry[i] = ~0u;
            }
        };
        // Sets the bits of the listed tokens' places, numbers them, and prepares the first kNumbers. Returns how
        // many there are.
        const auto give_numbers = [&]() -> int {
            const int own_words = (window / 32 + kThreads - 1) / kThreads;  // neighbouring ones that a thread numbers
            for (int i = tid; i < own_words * kThreads; i += kThreads) listed[i] = 0;
            __syncthreads();
            const auto give = [&](int v) {
                const unsigned at = in_window(v);
                if (at < window) atomicOr(listed + at / 32, 1u << (at % 32));
            };
            each_said(give);
            each_bias([&](int v, float, int) { give(v); });
            __syncthreads();
            int own = 0;
            for (int q = 0; q < own_words; ++q) own += __popc(listed[tid * own_words + q]);
            const auto scan = [&](int v) {  // over the warp, the lane's own included
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int up = __shfl_up_sync(0xffffffffu, v, d);
                    if (lane >= d) v += up;
                }
                return v;
            };
            const int upto = scan(own);
            if (lane == 31) warp_bits[warp] = upto;
            __syncthreads();
            const int warps_upto = scan(lane < kWarps ? warp_bits[lane] : 0);
            const int all = __shfl_sync(0xffffffffu, warps_upto, 31);
            int i = upto - own + (warp ? __shfl_sync(0xffffffffu, warps_upto, warp ? warp - 1 : 0) : 0);
            for (int q = 0; q < own_words; ++q) {
                const int word = tid * own_words + q;
                before[word] = static_cast<uint16_t>(i);
                for (uint32_t b = listed[word]; b; b &= b - 1, ++i)
                    if (i < kNumbers) list[i] = static_cast<uint16_t>(word * 32 + __ffs(b) - 1);
            }
            clear(min(all, kNumbers));
            __syncthreads();
            return all;
        };
        // The counts and biases of the n tokens numbered from n0 (and their places, if they are not the first). A
        // token's biases add up in list order.
        const auto add_up = [&](int n0, int n) {
            if (n0 > 0) {
                clear(n);
                for (unsigned word = tid; word < window / 32; word += kThreads) {
                    int i = before[word] - n0;
                    for (uint32_t b = i < n ? listed[word] : 0; b; b &= b - 1, ++i)
                        if (i >= 0 && i < n) list[i] = static_cast<uint16_t>(word * 32 + __ffs(b) - 1);
                }
                __syncthreads();
            }
            // A place's number counted from n0; kNumbers or more behind these.
            const auto number = [&](unsigned at) {
                return before[at / 32] + __popc(listed[at / 32] & ((1u << (at % 32)) - 1)) - static_cast<unsigned>(n0);
            };
            each_said([&](int v) {
                const unsigned at = in_window(v);
                if (at >= window) return;
                const unsigned i = number(at);
                if (i < kNumbers) atomicAdd(count + i, 1u);
            });
            if (!biasing) return;
            // Calls f(number, bias, entry, token) for this thread's biases of these tokens.
            const auto each_number = [&](auto f) {
                each_bias([&](int v, float b, int j) {
                    const unsigned at = in_window(v);
                    if (at >= window) return;
                    const unsigned i = number(at);
                    if (i < kNumbers) f(i, b, static_cast<uint32_t>(j), v);
                });
            };
            bool again = false;  // this thread has an entry of a token that has another
            each_number([&](unsigned i, float, uint32_t j, int) { again |= atomicMin(entry + i, j) != ~0u; });
            int more = __syncthreads_count(again);
            each_number([&](unsigned i, float b, uint32_t j, int) {
                if (entry[i] == j) bias[i] = b;
            });
            if (more == 0) return;
            __syncthreads();
            // Further entries: one of each token a round, while many threads find some, ...
            for (int round = 0; round < kBiasRounds && more > 2 * kWarps; ++round) {
                for (int i = tid; i < n; i += kThreads) later[i] = ~0u;
                __syncthreads();
                each_number([&](unsigned i, float, uint32_t j, int) {
                    if (j > entry[i]) atomicMin(later + i, j);
                });
                __syncthreads();
                bool added = false;
                each_number([&](unsigned i, float b, uint32_t j, int) {
                    if (later[i] != j) return;
                    bias[i] = __fadd_rn(bias[i], b);
                    entry[i] = j;
                    added = true;
                });
                more = __syncthreads_count(added);
            }
            if (more == 0) return;
            // ... then every warp walks over the list once, 32 entries at a time, and adds what is left of the tokens
            // whose number is its own modulo the warps: the lowest lane of a token takes its lanes' values in order.
            const auto id_at = [&](int j) { return j < p.n_bias ? __ldg(bias_ids() + j) : -1; };
            int next = id_at(lane);
            for (int j0 = 0; j0 < p.n_bias; j0 += 32) {
                const int j = j0 + lane, v = next;
                next = id_at(j + 32);
                const unsigned at = v < p.vocab ? in_window(v) : ~0u;
                unsigned i = kNumbers;
                if (at < window) i = min(i, number(at));
                const bool mine = i < kNumbers && i % kWarps == warp && static_cast<uint32_t>(j) > entry[i];
                if (!__any_sync(0xffffffffu, mine)) continue;
                const float b = mine ? __ldg(bias_values() + j) : 0.0f;
                const unsigned lanes = __match_any_sync(0xffffffffu, mine ? i : kNumbers + lane);
                const bool lowest = mine && lane == __ffs(lanes) - 1;
                unsigned todo = lowest ? lanes : 0u;
                float sum = lowest ? bias[i] : 0.0f;
                for (unsigned most = __reduce_max_sync(0xffffffffu, __popc(todo)); most; --most) {
                    const float x = __shfl_sync(0xffffffffu, b, todo ? __ffs(todo) - 1 : lane);
                    if (todo) sum = __fadd_rn(sum, x);
                    todo &= todo - 1;
                }
                if (lowest) bias[i] = sum;
                __syncwarp();
            }
        };
        int numbers = 0;
        if (listing) {
            __syncthreads();  // the previous window is done with
            numbers = give_numbers();
        } else if (CHOOSE && !bounded) {
            __syncthreads();  // the bound has been set
        }

        // ---- the logits ----------------------------------------------------------------------------
        for (int e0 = w_begin; e0 < min(places, w_begin + static_cast<int>(window)); e0 += kTile) {
            const int v0 = e0 - shift;
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
            float x[CHOOSE ? kPerThread : 1][8];
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int e = e0 + (i * kThreads + tid) * 8, v = e - shift;  // place in the row, token
                // Bit j: token v + j exists and is allowed.
                uint32_t inside = 0xffu;
                if (v < 0) inside = (0xffu << -v) & 0xffu;
                if (v + 8 > p.vocab) inside = e < places ? inside & (0xffu >> (v + 8 - p.vocab)) : 0u;
                uint32_t ok = none ? 0u : inside;
                if (mask && inside) {
                    uint32_t bits;
                    if (v < 0) {
                        bits = __ldg(mask) << -v;
                    } else {
                        const uint32_t m0 = __ldg(mask + v / 32);
                        const bool next = v % 32 > 24 && (v / 32 + 1) * 32 < p.vocab;
                        const uint32_t m1 = next ? __ldg(mask + v / 32 + 1) : 0u;
                        bits = __funnelshift_r(m0, m1, v % 32);
                    }
                    ok &= bits;
                }
                if (CHOOSE) {
                    if (listing) ok &= ~(listed[(e - w_begin) / 32] >> (e % 32));
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[CHOOSE ? i : 0][j] = (ok >> j) & 1 ? to_f32(raw[i].v[j]) : -INFINITY;
                } else if (inside) {
                    if (ok != 0xffu) keep_allowed(raw[i], ok);
                    if (same_cut && inside == 0xffu) {
                        int4* dst = reinterpret_cast<int4*>(out + v);
                        const int4* src = reinterpret_cast<const int4*>(&raw[i]);
#pragma unroll
                        for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) dst[j] = src[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if ((inside >> j) & 1) out[v + j] = raw[i].v[j];
                    }
                }
            }
            if constexpr (CHOOSE) {
                float top = x[0][0];
#pragma unroll
                for (int j = 1; j < 8 * kPerThread; ++j) top = fmaxf(top, x[j / 8][j % 8]);
                total.reach(top);
#pragma unroll
                for (int j = 0; j < 8 * kPerThread; ++j) total.add(x[j / 8][j % 8]);
                offer(
                    top,
                    [&](auto f) {
#pragma unroll
                        for (int j = 0; j < 8 * kPerThread; ++j)
                            f(x[j / 8][j % 8], v0 + (j / 8 * kThreads + tid) * 8 + j % 8);
                    },
                    std::integral_constant<int, 8 * kPerThread>());
            }
        }

        // ---- the listed tokens, as many at once as there are numbers -----------------------------------
        for (int n0 = 0; n0 < numbers; n0 += kNumbers) {
            __syncthreads();  // the logits have been written (constrain), the previous ones are done with
            const int n = min(numbers - n0, kNumbers);
            add_up(n0, n);
            __syncthreads();
            float top = -INFINITY;
            for (int i = tid; i < n; i += kThreads) {
                const int v = w0 + list[i];
                const uint32_t bits = mask ? __ldg(mask + v / 32) : ~0u;
                float x = to_f32(in[v]);
                x = penalised(x, count[i], theta, freq, pres);
                if (biasing) x = __fadd_rn(x, bias[i]);
                const bool ok = !none && ((bits >> (v % 32)) & 1);
                if (CHOOSE) {
                    x = ok ? x : -INFINITY;
                    bias[i] = x;
                    top = fmaxf(top, x);
                } else if (ok) {
                    out[v] = from_f32<T>(x);
                }
            }
            if constexpr (CHOOSE) {
                total.reach(top);
                for (int i = tid; i < n; i += kThreads) total.add(bias[i]);
                offer(
                    top,
                    [&](auto f) {
                        for (int i = tid; i < n; i += kThreads) f(bias[i], w0 + list[i]);
                    },
                    std::integral_constant<int, kNumbers / kThreads>());
            }
        }
    }

    if constexpr (CHOOSE) {
        if (tid < kMaxK) choice.best[tid] = 0;
        __syncthreads();  // the buffer is complete; a block without a window has set it
        total.join();
        if (lane == 0) {
            choice.warp_m[warp] = total.m;
            choice.warp_s[warp] = total.s;
        }
        __syncthreads();
        find_best(choice.buffer, choice.buffered, p.k, choice.best);
        const auto across = [&](bool there, float m, float s) {  // over the warp's lanes
            total = MaxSum();
            if (there) {
                total.m = m;
                total.s = s;
            }
            total.join();
        };
        if (warp == 0) {
            across(lane < kWarps, choice.warp_m[lane % kWarps], choice.warp_s[lane % kWarps]);
            if (lane == 0) {
                choice.m = total.m;
                choice.s = total.s;
            }
        }
        __syncthreads();
        uint64_t key = lane < p.k ? choice.best[lane] : 0;
        if (p.slices > 1) {
            __syncwarp();
            cluster_sync();
            if (slice == 0 && warp == 0) {
                // At most 8 blocks of 8 keys, two a lane: each key's place is the number of larger ones.
                const int all = p.slices * p.k;
                for (int c = lane; c < all; c += 32) choice.firsts[c] = ld_cluster_u64(&choice.best[c % p.k], c / p.k);
                __syncwarp();
                if (lane < p.k) choice.buffer[lane] = 0;
                __syncwarp();
                for (int c = lane; c < all; c += 32) {
                    int larger = 0;
                    for (int j = 0; j < all; ++j) larger += choice.firsts[j] > choice.firsts[c];
                    if (larger < p.k) choice.buffer[larger] = choice.firsts[c];
                }
                __syncwarp();
                key = lane < p.k ? choice.buffer[lane] : 0;
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
    constexpr size_t kLists = kNumbers * 18;
    const size_t bytes = p.history || p.n_bias > 0 ? kLists : 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!once.done(dev)) {
        if ((e = cudaFuncSetAttribute(logits_kernel<T, CHOOSE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(kLists))) != cudaSuccess)
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

// Places of a row, some of whose rows may start up to seven values behind a 16-byte boundary.
int most_places(const RuleParams& p, size_t size) {
    const bool aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld * size % 16 == 0;
    return p.vocab + (aligned ? 0 : 7);
}
int ceil_div(int64_t a, int b) { return static_cast<int>((a + b - 1) / b); }

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
        if (!r.bias_ids || !r.bias || r.n_bias > (1u << 20) || r.bias_ld < r.n_bias || r.bias_ld > kMost)
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

// Calls f with the memory of each of the rules' arrays. Masks are one row: any row may read any.
template <typename F>
bool any_rule(const RuleParams& p, F f) {
    const size_t rows = static_cast<size_t>(p.rows), word = 4;
    const auto table = [&](const void* q, int64_t ld, int entries) {
        return f(Span{q, static_cast<size_t>(ld) * word, static_cast<size_t>(entries) * word, rows});
    };
    const auto vector = [&](const void* q) { return f(Span{q, word, word, rows}); };
    const size_t masks = p.allowed ? ((p.n_states - size_t(1)) * p.allowed_ld + (p.vocab + size_t(31)) / 32) * word : 0;
    return table(p.history, p.history_ld, p.n_history) || table(p.bias_ids, p.bias_ld, p.n_bias) ||
           table(p.bias, p.bias_ld, p.n_bias) || vector(p.history_len) || vector(p.repetition) || vector(p.frequency) ||
           vector(p.presence) || vector(p.state) || f(Span{p.allowed, 0, masks, 1});
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
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_constrain: out is NULL or misaligned, or its rows short");
    const size_t size = dtype == TELMO_DTYPE_F32 ? 4 : 2;
    const Span written{out, out_ld * size, vocab * size, rows};
    if (!(out == logits && (out_ld == ld || rows == 1)) && overlap(Span{logits, ld * size, vocab * size, rows}, written))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_constrain: out overlaps the logits and is not the logits");
    if (any_rule(p, [&](const Span& s) { return overlap(s, written); }))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_constrain: out overlaps a rule's array");
    DeviceScope scope;
    if (int rc = scope.enter(ctx)) return rc;
    p.out = out;
    p.out_ld = static_cast<int64_t>(out_ld);
    const int places = most_places(p, size);
    // A block's lists cost about as much as a tile, so windows are four tiles long, and shorter where the blocks
    // still fit on the SMs at once (three on each). 256 rows of 131072: 49 us at four tiles, 55 at two, 53 at
    // eight; 32 rows: 8.2 us at two tiles, 11.4 at one; 148 rows of 32000: 9.4 at two, 13.7 at one.
    p.window = 4 * kTile;
    const auto blocks = [&](int window) { return static_cast<int64_t>(ceil_div(places, window)) * p.rows; };
    while (p.window > kTile && blocks(p.window / 2) <= 3 * ctx->sms) p.window /= 2;
    p.slices = ceil_div(places, p.window);
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
    // A row's tokens are written once the row has been read, so they may lie among its own inputs (the next place of
    // its tokens so far, say), but not among other rows'.
    const size_t size = dtype == TELMO_DTYPE_F32 ? 4 : 2;
    const Span to_ids{ids, k * 4, k * 4, rows}, to_logprobs{logprobs, k * 4, k * 4, rows};
    const auto read_elsewhere = [&](const Span& s) {
        return overlaps_other_rows(s, to_ids) || overlaps_other_rows(s, to_logprobs);
    };
    if (overlap(to_ids, to_logprobs) || read_elsewhere(Span{logits, ld * size, vocab * size, rows}) ||
        any_rule(p, read_elsewhere))
        return ctx->fail(TELMO_ERR_ARGUMENT, "telmo_logits_choose: ids or logprobs overlap each other or another row's inputs");
    DeviceScope scope;
    if (int rc = scope.enter(ctx)) return rc;
    p.ids = ids;
    p.logprobs = logprobs;
    p.k = static_cast<int>(k);
    const int places = most_places(p, size);
    // A cluster of up to eight blocks a row: the number that takes the least time, if the SMs hold two blocks
    // each, a block's lists, first bound and end cost as much as two tiles, and a cluster's meetings too. 256 rows of 131072: 72 us on one
    // block a row, 78 on two; 300 rows: 75 on eight, 82 on one.
    const auto cost = [&](int slices) {
        return static_cast<int64_t>(ceil_div(static_cast<int64_t>(slices) * p.rows, 2 * ctx->sms)) *
                   (ceil_div(places, slices) + 2 * kTile) +
               (slices > 1 ? 2 * kTile : 0);
    };
    p.slices = 1;
    for (int s = 2; s <= 8; s *= 2)
        if (cost(s) < cost(p.slices)) p.slices = s;
    p.window = std::min(kMostWindow, ceil_div(ceil_div(places, p.slices), kTile) * kTile);
    p.slices = std::min(p.slices, ceil_div(places, p.window));
    return ctx->cuda(launch_type<true>(p, dtype, static_cast<cudaStream_t>(stream)), "telmo_logits_choose");
}
