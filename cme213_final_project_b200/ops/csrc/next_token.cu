// From logits to the next token, in one pass over a row:
//     x = logits (32 bits);   token in the history: x > 0 ? x / repetition : x * repetition;   generated before, c times:
//     x - frequency c, then - presence;   x + bias;   x / temperature (where that is > 0);   not allowed: -inf
//     token = argmax of x (+ noise, where temperature > 0), the lowest index of equals;   logprob = x[token] - logsumexp(x)
// Every step is one rounded operation, in this order, so that equal values stay equal and the lowest index decides.
//
// What bounds it: the bytes of a row (logits, noise, processed); with few rows, the chain of loads and barriers before them.  Most tokens
// need the division and the mask only.  Those of the history or with a bias are marked, one bit each in shared memory, and left out of the
// pass (done inside it, a marked token costs its warp 100 instructions); afterwards a thread each does all steps of them.  The number of marks before a token is its place among the records (count, bias, token): 12 KB of marks and numbers and as many
// records as entries for 50304 tokens, where counts by token take 200 KB, or have to be made and cleared 8192 at a time.
// A row belongs to a cluster of 1 to 8 CTAs, each with a slice of the vocabulary; maxima, sums and picks are joined in the first one's
// shared memory.
// 64 rows of 65 tokens 5.4 us; 64 of 50304, bf16, 1024 tokens of history and 64 biases each 13.6 us; 1024 of 50304 in fp32 with noise and the
// processed logits 127 to 130 us, 4.8 TB/s (calls one after the other; replayed as a graph 4.9, 13.6 and 125).
#include "common.h"
#include "token_desc.h"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_CLUSTER = 8;
constexpr size_t MAX_SMEM = 160 * 1024;    // of marks and records
constexpr size_t MAX_RING = 65 * 1024;     // of the loads under way

// Running softmax statistics and the pick of some tokens.
struct Pick {
    float m, s;              // maximum of x and sum of exp(x - m)
    float y, x;              // the pick's value with noise, and without
    int at;                  // its index; INT_MAX: none
};
__device__ __forceinline__ Pick nothing() { return Pick{-INFINITY, 0.f, -INFINITY, -INFINITY, INT_MAX}; }
// A NaN is picked before all numbers, as by torch's argmax.
__device__ __forceinline__ bool above(float y, int at, float best, int best_at) {
    if (y != y || best != best) return y != y && (best == best || at < best_at);
    return y > best || (y == best && at < best_at);
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * LOG2E); }
__device__ __forceinline__ Pick join(const Pick& a, const Pick& b) {
    Pick r;
    r.m = fmaxf(a.m, b.m);
    const float use = r.m == -INFINITY ? 0.f : r.m;
    // (a part without anything has no sum; its factor exp(-inf) is 0 too, and a NaN sum stays one)
    r.s = a.s * exp_of(a.m - use) + b.s * exp_of(b.m - use);
    const bool second = above(b.y, b.at, a.y, a.at);
    r.y = second ? b.y : a.y;
    r.x = second ? b.x : a.x;
    r.at = second ? b.at : a.at;
    return r;
}
__device__ __forceinline__ Pick shfl_xor(const Pick& p, int o) {
    Pick r;
    r.m = __shfl_xor_sync(0xffffffffu, p.m, o);
    r.s = __shfl_xor_sync(0xffffffffu, p.s, o);
    r.y = __shfl_xor_sync(0xffffffffu, p.y, o);
    r.x = __shfl_xor_sync(0xffffffffu, p.x, o);
    r.at = __shfl_xor_sync(0xffffffffu, p.at, o);
    return r;
}

constexpr int KEPT = 4;          // entries of a history that a thread keeps in registers
constexpr int STAGES = 4;        // of a thread's ring of loads

// Eight tokens of a thread: bf16 sixteen bytes in a row, fp32 twice sixteen bytes, a warp's width apart.
template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8, PIECES = 1;
    typedef uint4 Raw;
    static __device__ __forceinline__ void unpack(const Raw* r, float* f) { unpack8(r[0], f); }
    static __device__ __forceinline__ Raw pack(const float* f, int) { return pack8(f); }
};
template <> struct Vec<float> {
    static constexpr int N = 4, PIECES = 2;
    typedef float4 Raw;
    static __device__ __forceinline__ void unpack(const Raw* r, float* f) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { f[4 * i] = r[i].x; f[4 * i + 1] = r[i].y; f[4 * i + 2] = r[i].z; f[4 * i + 3] = r[i].w; }
    }
    static __device__ __forceinline__ Raw pack(const float* f, int i) { return make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]); }
};
// The largest of three: a NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// The largest of the warp (the first a NaN if one is).
__device__ __forceinline__ float warp_max_nan(float x) {
    float y;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_max_num(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float y;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// x / t, correctly rounded, for many x: with r = 1 / t correctly rounded and a quotient q that is off by one last place at the most, q + (x - q t) r
// rounds to the right one (Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990), if t's
// digits are not all ones and nothing under- or overflows; other x and t take the division itself.
struct Divisor {
    float t, r;
    bool fine;
    __device__ __forceinline__ explicit Divisor(float v) : t(v), r(1.f / v) {
        fine = v > 0x1p-60f && v < 0x1p60f && (__float_as_uint(v) & 0x7fffffu) != 0x7fffffu;
    }
    __device__ __forceinline__ void apply8(float* x) const {
        const F32x2 r2 = f2_splat(r), t2 = f2_splat(-t);
        float q[8];
        // smallest and largest magnitude; a NaN shows in the largest
        float low = fabsf(x[0]), high = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            low = min3(low, fabsf(x[e]), fabsf(x[e + 1]));
            high = max3_nan(high, fabsf(x[e]), fabsf(x[e + 1]));
            const F32x2 v = f2_pack(x[e], x[e + 1]);
            F32x2 d = f2_mul(v, r2);
            d = f2_fma(f2_fma(d, t2, v), r2, d);
            d = f2_fma(f2_fma(d, t2, v), r2, d);
            f2_unpack(d, q[e], q[e + 1]);
        }
        if (fine && low > 0x1p-60f && high < 0x1p60f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = q[e];
        } else {
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {                  // (one division in the code; the registers are moved round)
                const float d = __fdiv_rn(x[0], t);
#pragma unroll
                for (int k = 0; k < 7; ++k) x[k] = x[k + 1];
                x[7] = d;
            }
        }
    }
};

__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// VECTOR: logits, processed and noise have their 16-byte boundaries at the same elements of a row.
// STEPS: a CTA takes its tokens in `steps` slices one after the other, where the marks and records of all of them would not fit.
template <typename T, bool VECTOR, bool STEPS>
__global__ void __launch_bounds__(256, 4) next_token_kernel(const CmeToken p, int cluster, int steps, int slice, int words, int records, bool biased) {
    // [words + 1] marks, [words] marks in the words before, then for each mark [records]: times generated (bit 31: in the history), last bias
    // + 1, index in the slice
    extern __shared__ __align__(16) unsigned dyn[];
    __shared__ Pick parts[8], mine;
    __shared__ int scan[8], total;
    constexpr int N = VECTOR ? Vec<T>::N : 1, PIECES = Vec<T>::PIECES;
    const int rank = blockIdx.x % cluster, row = blockIdx.x / cluster, tid = threadIdx.x, threads = blockDim.x;
    const int lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    unsigned* const marks = dyn;
    int* const before = reinterpret_cast<int*>(marks + words + 1);
    int* const count = before + words;
    int* const bias = count + records;
    int* const which = bias + records;
    pdl_wait();
    // What does not depend on one another is on its way together: the row's numbers, its history, its first logits.
    const float rep = p.repetition ? p.repetition[row] : 1.f, pres = p.presence ? p.presence[row] : 0.f;
    const float freq = p.frequency ? p.frequency[row] : 0.f, temp = p.temperature ? p.temperature[row] : 1.f;
    const int told = p.history ? max(0, min(p.lengths[row], p.history_len)) : 0, given = p.history && p.prompts ? p.prompts[row] : 0;
    const int* hist = p.history + row * p.history_ld;
    int kept[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
        const int j = tid + k * threads;
        kept[k] = p.history && j < p.history_len ? hist[j] : -1;
    }
    const T* src = static_cast<const T*>(p.logits) + row * p.logits_ld;
    T* dst = p.processed ? static_cast<T*>(p.processed) + (long long)row * p.vocab : nullptr;
    const float* noise = p.noise && temp > 0.f ? p.noise + (long long)row * p.vocab : nullptr;
    const unsigned* allowed = p.allowed ? reinterpret_cast<const unsigned*>(p.allowed) + row * p.allowed_ld : nullptr;
    const int all_words = (p.vocab + 31) >> 5;

    const bool divides = temp > 0.f && p.temperature;
    const Divisor by(divides ? temp : 1.f);
    // A warp shares its maximum and the value to beat, so that few groups change them (a new largest of k groups comes once in k; with values
    // of a lane's own, some lane of 32 has one in most groups).  The loops over tokens go up, so that a tie leaves the lower index.
    Pick best = nothing();
    float to_beat = -INFINITY;
    // Values x of n tokens and the same with noise, y; -inf: not to be looked at.  Whole warps; token(e): its index; `any_order`: a tie may be won.
    auto take = [&](const float* x, const float* y, auto number, auto&& token, bool any_order) {
        constexpr int n = decltype(number)::value;
        float mx = x[0], top = y[0];
        if constexpr (n > 1) {
#pragma unroll
            for (int e = 0; e < n; e += 2) { mx = max3(mx, x[e], x[e + 1]); top = max3_nan(top, y[e], y[e + 1]); }
        }
        if (__any_sync(0xffffffffu, mx > best.m || !(top < to_beat || (top == to_beat && !any_order)))) {      // a NaN too
            mx = warp_max_num(mx);
            if (mx > best.m) {
                best.s *= exp_of(best.m - mx);             // (nothing yet: exp(-inf) = 0)
                best.m = mx;
            }
            if (__any_sync(0xffffffffu, top != top)) {     // a NaN, of a logit or of noise that is not finite (which counts only where x does)
#pragma unroll
                for (int e = 0; e < n; ++e) {
                    if (x[e] != -INFINITY && y[e] != -INFINITY && above(y[e], token(e), best.y, best.at)) {
                        best.y = y[e];
                        best.x = x[e];
                        best.at = token(e);
                    }
                }
            } else if (top > best.y || (any_order && top == best.y && top != -INFINITY)) {
                int at = token(n - 1);
                float xv = x[n - 1];
#pragma unroll
                for (int e = n - 2; e >= 0; --e) if (y[e] == top) { at = token(e); xv = x[e]; }
                if (top > best.y || at < best.at) { best.y = top; best.x = xv; best.at = at; }
            }
            to_beat = warp_max_nan(best.y);
        }
        const float use = best.m == -INFINITY ? 0.f : best.m;
        if constexpr (n == 1) {
            best.s += exp_of(x[0] - use);
        } else {
            const F32x2 shift = f2_splat(-use), scale = f2_splat(LOG2E);
            F32x2 sum = f2_splat(0.f);
#pragma unroll
            for (int e = 0; e < n; e += 2) {
                float a, b;
                f2_unpack(f2_mul(f2_add(f2_pack(x[e], x[e + 1]), shift), scale), a, b);
                sum = f2_add(sum, f2_pack(exp2_of(a), exp2_of(b)));
            }
            float a, b;
            f2_unpack(sum, a, b);
            best.s += a + b;
        }
    };
    auto not_allowed = [&](int v, int n) -> unsigned {     // bits [v, v + n), n <= 8
        if (!allowed) return 0;
        const int w = v >> 5;
        unsigned b = __ldg(allowed + w) >> (v & 31);
        if ((v & 31) + n > 32 && w + 1 < all_words) b |= __ldg(allowed + w + 1) << (32 - (v & 31));
        return ~b & ((1u << n) - 1u);
    };

    // slices of the CTA's tokens, in their order
    for (int step = 0; step < (STEPS ? steps : 1); ++step) {
        if (STEPS && step) __syncthreads();                // the last slice's marks and records are done with
        const int v0 = min(p.vocab, (STEPS ? rank * steps + step : rank) * slice), v1 = min(p.vocab, v0 + slice);
        // the first element on a 16-byte boundary, then groups, then what is left; marks of a group are whole bits of one byte
        const int head = VECTOR ? (int)((N - (row * p.logits_ld + v0) % N) % N) : v1 - v0;
        const int a0 = min(v1, v0 + head), groups = VECTOR ? (v1 - a0) / N : 0;      // (of sixteen bytes)
        const int origin = VECTOR ? v0 + head - N : v0;        // of the marks
        // f(index from the origin on, was it generated) for the entries of the history, f(index from the origin on, entry) for those of the biases
        auto for_history = [&](auto&& f) {
#pragma unroll
            for (int k = 0; k < KEPT; ++k) {
                const int j = tid + k * threads;
                if (j < told && kept[k] >= v0 && kept[k] < v1) f(kept[k] - origin, j >= given);
            }
            for (int j = tid + KEPT * threads; j < told; j += threads) {
                const int id = hist[j];
                if (id >= v0 && id < v1) f(id - origin, j >= given);
            }
        };
        auto for_biases = [&](auto&& f) {
            if (!biased) return;
            const int* ids = p.bias_ids + (long long)row * p.biases;
            for (int j = tid; j < p.biases; j += threads) {
                const int id = ids[j];
                if (id >= v0 && id < v1) f(id - origin, j);
            }
        };
        typedef typename Vec<T>::Raw Raw;
        const int stride = threads * PIECES, first = warp * 32 * PIECES + lane;      // a thread's groups: first, + 32 ..., a stride further ...
        // A thread's loads travel through a ring of its own in shared memory, STAGES - 1 turns ahead: with one turn ahead in registers, 64 bytes a
        // thread are on their way, and 1024 rows of 50304 in fp32 run at 3.9 TB/s.
        uint4* const ring = reinterpret_cast<uint4*>(dyn + (words ? (2 * words + 1 + 3 * records + 3) / 4 * 4 : 0)) + tid;
        const int pieces = PIECES + (p.noise ? 2 : 0);         // of 16 bytes, a turn
        auto fetch = [&](int turn) {
            if constexpr (VECTOR) {
                uint4* to = ring + turn % STAGES * pieces * threads;
#pragma unroll
                for (int k = 0; k < PIECES; ++k) {
                    const int j = first + turn * stride + k * 32;
                    if (j < groups) {
                        copy16(to + k * threads, src + a0 + j * N);
                        if (noise) {
#pragma unroll
                            for (int e = 0; e < N / 4; ++e) copy16(to + (PIECES + k * (N / 4) + e) * threads, noise + a0 + j * N + e * 4);
                        }
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        };
#pragma unroll
        for (int t = 0; t < STAGES - 1; ++t) fetch(t);
        float early = 0.f, early_noise = 0.f;                  // one by one, a thread's first token
        if (!VECTOR && v0 + tid < v1) {
            early = to_f32<T>(src[v0 + tid]);
            if (noise) early_noise = noise[v0 + tid];
        }
        auto place = [&](int l) { return before[l >> 5] + __popc(marks[l >> 5] & ((1u << (l & 31)) - 1u)); };
        if (words) {
            for (int i = tid; i <= words; i += threads) marks[i] = 0;
            for (int i = tid; i < 2 * records; i += threads) count[i] = 0;
            __syncthreads();
            for_history([&](int l, bool) { atomicOr(&marks[l >> 5], 1u << (l & 31)); });
            for_biases([&](int l, int) { atomicOr(&marks[l >> 5], 1u << (l & 31)); });
            __syncthreads();
            // marks before each word: a thread's own words, then the threads before it
            const int each = (words + threads - 1) / threads, w0 = min(words, tid * each), w1 = min(words, w0 + each);
            int sum = 0;
            for (int w = w0; w < w1; ++w) sum += __popc(marks[w]);
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            if (lane == 31) scan[warp] = upto;
            __syncthreads();
            int at = upto - sum;
            for (int w = 0; w < warp; ++w) at += scan[w];
            if (tid == threads - 1) total = at + sum;
            for (int w = w0; w < w1; ++w) { before[w] = at; at += __popc(marks[w]); }
            __syncthreads();
            // whole numbers: any order of the additions gives the same
            for_history([&](int l, bool made) {
                const int at = place(l);
                which[at] = l;
                atomicOr(&count[at], (int)0x80000000);
                if (made) atomicAdd(&count[at], 1);
            });
            for_biases([&](int l, int j) {
                const int at = place(l);
                which[at] = l;
                atomicMax(&bias[at], j + 1);
            });
        }
        // tokens [from, to) one by one, whole warps
        auto singles = [&](int from, int to) {
            for (int b = from + warp * 32; b < to; b += threads) {
                const int v = b + lane;
                float x = -INFINITY, g = 0.f;
                if (v < to) {
                    x = !VECTOR && v == v0 + tid ? early : to_f32<T>(src[v]);
                    if (noise) g = !VECTOR && v == v0 + tid ? early_noise : noise[v];
                    if (divides) x = __fdiv_rn(x, temp);
                    const int l = v - origin;
                    if (not_allowed(v, 1) || (words && (marks[l >> 5] >> (l & 31)) & 1)) x = -INFINITY;
                    if (dst) dst[v] = from_f32<T>(x);
                }
                const float y = noise ? __fadd_rn(x, g) : x;
                take(&x, &y, std::integral_constant<int, 1>{}, [&](int) { return v; }, false);
            }
        };
        singles(v0, a0);
        if constexpr (VECTOR) {
            const uint8_t* bytes = reinterpret_cast<const uint8_t*>(marks);
            auto eight = [&](int i, const Raw* r, const float4* g) {       // groups i (and i + 32)
                float x[8];
                Vec<T>::unpack(r, x);
                if (divides) by.apply8(x);
#pragma unroll
                for (int k = 0; k < PIECES; ++k) {
                    const int j = i + k * 32;
                    unsigned no = 0xff;
                    if (j < groups) {
                        no = allowed ? not_allowed(a0 + j * N, N) : 0;
                        if (words) no |= N == 8 ? bytes[j + 1] : bytes[(j + 1) >> 1] >> ((j + 1) & 1) * 4;
                    }
                    if (no & ((1u << N) - 1u)) {
#pragma unroll
                        for (int e = 0; e < N; ++e) if ((no >> e) & 1) x[k * N + e] = -INFINITY;
                    }
                    if (dst && j < groups) __stcs(reinterpret_cast<Raw*>(dst + a0) + j, Vec<T>::pack(x, k));
                }
                auto token = [&](int e) { return a0 + (i + e / N * 32) * N + e % N; };
                if (noise) {
                    const float* f = reinterpret_cast<const float*>(g);
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; e += 2) f2_unpack(f2_add(f2_pack(x[e], x[e + 1]), f2_pack(f[e], f[e + 1])), y[e], y[e + 1]);
                    take(x, y, std::integral_constant<int, 8>{}, token, false);
                } else {
                    take(x, x, std::integral_constant<int, 8>{}, token, false);
                }
            };
            for (int turn = 0, i = first; i - lane < groups; ++turn, i += stride) {
                fetch(turn + STAGES - 1);
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
                const uint4* from = ring + turn % STAGES * pieces * threads;
                Raw r[PIECES];
                float4 g[2];
#pragma unroll
                for (int k = 0; k < PIECES; ++k) r[k] = *reinterpret_cast<const Raw*>(from + k * threads);
                if (noise) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) g[k] = *reinterpret_cast<const float4*>(from + (PIECES + k) * threads);
                }
                eight(i, r, g);
            }
            singles(a0 + groups * N, v1);
        }
        if (words) {
            __syncthreads();                                   // the counts are made; what the pass wrote for marked tokens is overwritten
            for (int b = warp * 32; b < total; b += threads) {
                const int i = b + lane;
                int v = 0;
                float x = -INFINITY, g = 0.f;
                if (i < total) {
                    const int c = count[i], made = c & 0x7fffffff, j = bias[i] - 1;
                    v = origin + which[i];
                    x = to_f32<T>(src[v]);
                    if (noise) g = noise[v];
                    if (c < 0) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                    if (made) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)made)), pres);
                    if (j >= 0) x = __fadd_rn(x, p.bias_values[(long long)row * p.biases + j]);
                    if (divides) x = __fdiv_rn(x, temp);
                    if (not_allowed(v, 1)) x = -INFINITY;
                    if (dst) dst[v] = from_f32<T>(x);
                }
                const float y = noise ? __fadd_rn(x, g) : x;
                take(&x, &y, std::integral_constant<int, 1>{}, [&](int) { return v; }, true);
            }
        }
    }
    // (earlier, CTAs of the next kernel would crowd on the SMs that are done first: 1024 rows of 50304 183 us)
    pdl_release();
    // ---------------- joins ----------------
#pragma unroll
    for (int o = 16; o; o >>= 1) best = join(best, shfl_xor(best, o));
    if (lane == 0) parts[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = lane < warps ? parts[lane] : nothing();
#pragma unroll
        for (int o = 4; o; o >>= 1) best = join(best, shfl_xor(best, o));
        if (lane == 0) mine = best;
    }
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0 && warp == 0) {
            best = lane < cluster ? *cl.map_shared_rank(&mine, lane) : nothing();
#pragma unroll
            for (int o = 4; o; o >>= 1) best = join(best, shfl_xor(best, o));
        }
        cl.sync();
    }
    if (rank == 0 && tid == 0) {
        const bool none = best.at == INT_MAX;
        p.token[row] = none ? -1 : best.at;
        p.logprob[row] = none ? -INFINITY : best.x - best.m - logf(best.s);
    }
}

}  // namespace

CME_API int cme_next_token(const CmeToken* p, void* stream) {
    CME_REQUIRE(p->dtype == CME_F32 || p->dtype == CME_BF16, CME_ERR_UNSUPPORTED, "next token: unsupported dtype");
    CME_REQUIRE(p->rows >= 0 && p->vocab > 0 && p->logits_ld >= p->vocab && p->history_len >= 0 && p->biases >= 0, CME_ERR_SHAPE,
                "next token: bad sizes");
    CME_REQUIRE(!p->history || p->lengths, CME_ERR_SHAPE, "next token: a history needs its lengths");
    if (p->rows == 0) return CME_OK;
    int sms, rc;
    if ((rc = cme_num_sms(&sms))) return rc;
    const bool biased = p->bias_ids && p->biases, marks = biased || (p->history && p->history_len);
    const int n = p->dtype == CME_F32 ? 4 : 8;
    auto al16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    const bool aligned = al16(p->logits) && al16(p->processed) && al16(p->noise) && p->logits_ld % n == p->vocab % n;
    int slice, words, records, threads;
    bool vector;
    size_t tables, smem;
    auto lay_out = [&](int slices) {
        slice = (cme_cdiv(p->vocab, slices) + 31) / 32 * 32;
        words = marks ? slice / 32 + 1 : 0;                // (marks start up to eight tokens before the slice)
        records = marks ? (int)std::min((long long)slice, (long long)(p->history ? p->history_len : 0) + (biased ? p->biases : 0)) : 0;
        tables = smem = marks ? ((size_t)2 * words + 1 + 3 * (size_t)records) * 4 : 0;
        // In groups of sixteen bytes, where there is more than a turn or two of them and rows of logits start at the same place between
        // 16-byte boundaries as rows of noise and of the processed logits
        vector = slice >= 1024 && aligned;
        threads = slice <= 1024 ? 128 : 256;
        static_assert(STAGES * 256 * 16 * 4 + 16 <= MAX_RING, "ring");
        if (vector) smem = (smem + 15) / 16 * 16 + (size_t)STAGES * threads * 16 * ((p->dtype == CME_F32 ? 2 : 1) + (p->noise ? 2 : 0));
    };
    // As many CTAs as run at a time, with no fewer than 2048 tokens each: a second turn costs as much as a row's length (us, one CTA / two for
    // a row: 319 rows of 6186 10.7 / 18.0, 200 of 50304 in fp32, two / four 28.0 / 34.5).  Smaller slices where a CTA's records would not fit, and
    // from eight CTAs on several for each: a token of a slice has a record at the most, so that some number of them does.
    int cluster = MAX_CLUSTER, steps = 1;
    for (; cluster > 1; cluster /= 2) {
        lay_out(cluster);
        if (p->vocab / cluster >= 2048 && (long long)p->rows * cluster <= (long long)sms * std::min<size_t>(4, 227 * 1024 / (smem + 1024))) break;
    }
    for (lay_out(cluster); tables > MAX_SMEM; lay_out(cluster * steps)) (cluster < MAX_CLUSTER ? cluster : steps) *= 2;
    CME_REQUIRE((long long)p->rows * cluster < (1ll << 31), CME_ERR_LIMIT, "next token: too many rows");
    auto of = [&](auto several) {
        constexpr bool S = decltype(several)::value;
        return p->dtype == CME_F32 ? (vector ? next_token_kernel<float, true, S> : next_token_kernel<float, false, S>)
                                   : (vector ? next_token_kernel<__nv_bfloat16, true, S> : next_token_kernel<__nv_bfloat16, false, S>);
    };
    auto* kernel = steps > 1 ? of(std::true_type{}) : of(std::false_type{});
    static bool attr[2][2][2][CME_MAX_DEVICES] = {};      // function attributes are per device
    int dev = 0;
    CME_CUDA(cudaGetDevice(&dev));
    if (bool& set = attr[steps > 1][p->dtype == CME_F32][vector][dev % CME_MAX_DEVICES]; !set) {
        CME_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(MAX_SMEM + MAX_RING)));
        set = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p->rows * cluster));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CME_CUDA(cudaLaunchKernelEx(&cfg, kernel, *p, cluster, steps, slice, words, records, biased));
    CME_LAUNCH_CHECK();
    return CME_OK;
}
