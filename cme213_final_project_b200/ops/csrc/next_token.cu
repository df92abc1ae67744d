// From logits to the next token, in one pass over a row:
//     x = logits (32 bits);   token in the history: x > 0 ? x / repetition : x * repetition;   generated before, c times:
//     x - frequency c, then - presence;   x + bias;   x / temperature (where that is > 0);   not allowed: -inf
//     token = argmax of x (+ noise, where temperature > 0), the lowest index of equals;   logprob = x[token] - logsumexp(x)
// Every step is one rounded operation, in this order, so that equal values stay equal and the lowest index decides.
//
// What bounds it: the bytes of a row (logits, noise, processed).  Only tokens of the history or with a bias need more than the division
// and the mask.  A bitmap of the vocabulary in shared memory marks them, and the number of marks before one is its place among
// the records (count, bias), of which there are as many as marked tokens: 6 KB of marks for 50304 tokens and one byte of them to look at
// for eight logits, where counts for the whole vocabulary would take 200 KB to clear and read.
// A row belongs to a cluster of 1 to 8 CTAs, each with a slice of the vocabulary; maxima, sums and picks are joined in the first one's
// shared memory.
#include "common.h"
#include "token_desc.h"

#include <algorithm>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_CLUSTER = 8;

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
__device__ __forceinline__ float exp_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * LOG2E));
    return y;
}
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

// The marked tokens of a slice and their records, in shared memory.
struct Marks {
    unsigned* bits;          // [words + 1]
    int* before;             // [words] marks in the words before
    int* count;              // [marks] times generated; bit 31: in the history
    int* bias;               // [marks] last entry of the biases, or -1
    __device__ __forceinline__ int place(int local) const {
        return before[local >> 5] + __popc(bits[local >> 5] & ((1u << (local & 31)) - 1u));
    }
};

// Entries of the history that are tokens of [v0, v1); f(local index, was it generated).
template <typename F> __device__ __forceinline__ void for_history(const CmeToken& p, int row, int v0, int v1, F&& f) {
    if (!p.history) return;
    const int n = max(0, min(p.lengths[row], p.history_len)), given = p.prompts ? p.prompts[row] : 0;
    const int* h = p.history + row * p.history_ld;
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        const int id = h[j];
        if (id >= v0 && id < v1) f(id - v0, j >= given);
    }
}
template <typename F> __device__ __forceinline__ void for_biases(const CmeToken& p, int row, int v0, int v1, F&& f) {
    if (!p.bias_ids) return;
    const int* ids = p.bias_ids + (long long)row * p.biases;
    for (int j = threadIdx.x; j < p.biases; j += blockDim.x) {
        const int id = ids[j];
        if (id >= v0 && id < v1) f(id - v0, j);
    }
}

template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* f) { unpack8(__ldcs(reinterpret_cast<const uint4*>(p)), f); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) { __stcs(reinterpret_cast<uint4*>(p), pack8(f)); }
};
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float* p, float* f) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
    static __device__ __forceinline__ void store(float* p, const float* f) {
        __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
    }
};

// VECTOR: logits, processed and noise have their 16-byte boundaries at the same elements of a row.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) next_token_kernel(const CmeToken p, int cluster, int slice, int words, int records) {
    extern __shared__ __align__(16) unsigned dyn[];
    __shared__ Pick parts[8], mine;
    __shared__ int scan[8], total;
    constexpr int N = VECTOR ? Vec<T>::N : 1;
    const int rank = blockIdx.x % cluster, row = blockIdx.x / cluster;
    const int v0 = min(p.vocab, rank * slice), v1 = min(p.vocab, v0 + slice);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    Marks k;
    k.bits = dyn;
    k.before = reinterpret_cast<int*>(dyn + words + 1);
    k.count = k.before + words;
    k.bias = k.count + records;
    pdl_release();
    pdl_wait();
    // ---------------- marks and records ----------------
    if (words) {
        for (int i = threadIdx.x; i <= words; i += blockDim.x) k.bits[i] = 0;
        __syncthreads();
        for_history(p, row, v0, v1, [&](int v, bool) { atomicOr(&k.bits[v >> 5], 1u << (v & 31)); });
        for_biases(p, row, v0, v1, [&](int v, int) { atomicOr(&k.bits[v >> 5], 1u << (v & 31)); });
        __syncthreads();
        // marks before each word: a thread's own words, then the threads before it
        const int each = (words + blockDim.x - 1) / blockDim.x, w0 = min(words, (int)threadIdx.x * each), w1 = min(words, w0 + each);
        int sum = 0;
        for (int w = w0; w < w1; ++w) sum += __popc(k.bits[w]);
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
        if (threadIdx.x == blockDim.x - 1) total = at + sum;
        for (int w = w0; w < w1; ++w) { k.before[w] = at; at += __popc(k.bits[w]); }
        __syncthreads();
        for (int i = threadIdx.x; i < total; i += blockDim.x) { k.count[i] = 0; k.bias[i] = -1; }
        __syncthreads();
        // whole numbers: any order of the additions gives the same
        for_history(p, row, v0, v1, [&](int v, bool made) {
            int* c = &k.count[k.place(v)];
            atomicOr(c, (int)0x80000000);
            if (made) atomicAdd(c, 1);
        });
        for_biases(p, row, v0, v1, [&](int v, int j) { atomicMax(&k.bias[k.place(v)], j); });
        __syncthreads();
    }
    // ---------------- the row ----------------
    const float rep = p.repetition ? p.repetition[row] : 1.f, pres = p.presence ? p.presence[row] : 0.f;
    const float freq = p.frequency ? p.frequency[row] : 0.f, temp = p.temperature ? p.temperature[row] : 1.f;
    const bool warm = temp > 0.f;
    const T* src = static_cast<const T*>(p.logits) + row * p.logits_ld;
    T* dst = p.processed ? static_cast<T*>(p.processed) + (long long)row * p.vocab : nullptr;
    const float* noise = p.noise && warm ? p.noise + (long long)row * p.vocab : nullptr;
    const unsigned* allowed = p.allowed ? reinterpret_cast<const unsigned*>(p.allowed) + row * p.allowed_ld : nullptr;
    Pick best = nothing();
    // bits [v, v + n) of a row of words, n <= 8
    const int all_words = (p.vocab + 31) >> 5;
    auto allowed_bits = [&](int v, int n) {
        const int w = v >> 5;
        unsigned b = __ldg(allowed + w) >> (v & 31);
        if ((v & 31) + n > 32 && w + 1 < all_words) b |= __ldg(allowed + w + 1) << (32 - (v & 31));
        return b;
    };
    auto group = [&](int v, float* x, const float* g, auto count) {
        constexpr int n = decltype(count)::value;
        if (words) {
            const int local = v - v0;
            unsigned marked = __funnelshift_r(k.bits[local >> 5], k.bits[(local >> 5) + 1], local & 31) & ((1u << n) - 1u);
            while (marked) {
                const int i = __ffs(marked) - 1;
                marked &= marked - 1;
                const int at = k.place(local + i);
                const int c = k.count[at], j = k.bias[at];
                float t = 0.f;
#pragma unroll
                for (int e = 0; e < n; ++e) if (e == i) t = x[e];      // (registers have no index)
                if (c < 0) t = t > 0.f ? __fdiv_rn(t, rep) : __fmul_rn(t, rep);
                const int made = c & 0x7fffffff;
                if (made) { t = __fsub_rn(t, __fmul_rn(freq, (float)made)); t = __fsub_rn(t, pres); }
                if (j >= 0) t = __fadd_rn(t, p.bias_values[(long long)row * p.biases + j]);
#pragma unroll
                for (int e = 0; e < n; ++e) if (e == i) x[e] = t;
            }
        }
        if (warm && p.temperature) {
#pragma unroll
            for (int e = 0; e < n; ++e) x[e] = __fdiv_rn(x[e], temp);
        }
        if (allowed) {
            const unsigned ok = allowed_bits(v, n);
#pragma unroll
            for (int e = 0; e < n; ++e) if (!((ok >> e) & 1)) x[e] = -INFINITY;
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < n; ++e) mx = fmaxf(mx, x[e]);
        if (mx > best.m) {
            best.s *= exp_of(best.m - mx);                 // (nothing yet: exp(-inf) = 0)
            best.m = mx;
        }
        const float use = best.m == -INFINITY ? 0.f : best.m;
#pragma unroll
        for (int e = 0; e < n; ++e) {
            best.s += exp_of(x[e] - use);
            const float y = g && x[e] != -INFINITY ? __fadd_rn(x[e], g[e]) : x[e];
            if (y > best.y || (y != y && best.y == best.y)) { best.y = y; best.x = x[e]; best.at = v + e; }
        }
    };
    auto single = [&](int v) {
        float x = to_f32<T>(src[v]);
        const float g = noise ? noise[v] : 0.f;
        group(v, &x, noise ? &g : nullptr, std::integral_constant<int, 1>{});
        if (dst) dst[v] = from_f32<T>(x);
    };
    if constexpr (VECTOR) {
        // the first element of the slice on a 16-byte boundary, then groups, then what is left
        const int head = (int)((N - (row * p.logits_ld + v0) % N) % N), a0 = min(v1, v0 + head), groups = (v1 - a0) / N;
        if ((int)threadIdx.x < a0 - v0) single(v0 + threadIdx.x);
        for (int i = threadIdx.x; i < groups; i += blockDim.x) {
            const int v = a0 + i * N;
            float x[N], g[N];
            Vec<T>::load(src + v, x);
            if (noise) {
#pragma unroll
                for (int e = 0; e < N; e += 4) Vec<float>::load(noise + v + e, g + e);
            }
            group(v, x, noise ? g : nullptr, std::integral_constant<int, N>{});
            if (dst) Vec<T>::store(dst + v, x);
        }
        if (a0 + groups * N + (int)threadIdx.x < v1) single(a0 + groups * N + threadIdx.x);
    } else {
        for (int v = v0 + threadIdx.x; v < v1; v += blockDim.x) single(v);
    }
    // ---------------- joins ----------------
#pragma unroll
    for (int o = 16; o; o >>= 1) best = join(best, shfl_xor(best, o));
    if (lane == 0) parts[warp] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < warps; ++w) best = join(best, parts[w]);
        mine = best;
    }
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0 && threadIdx.x == 0)
            for (int r = 1; r < cluster; ++r) best = join(best, *cl.map_shared_rank(&mine, r));
        cl.sync();
    }
    if (rank == 0 && threadIdx.x == 0) {
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
    // As many CTAs as keep the SMs busy, with no fewer than 2048 tokens each.
    int cluster = 1;
    while (cluster < MAX_CLUSTER && (long long)p->rows * cluster < 4ll * sms && p->vocab / (2 * cluster) >= 2048) cluster *= 2;
    const bool marks = (p->history && p->history_len) || (p->bias_ids && p->biases);
    int slice, words, records;
    size_t smem;
    for (;; cluster *= 2) {
        slice = (cme_cdiv(p->vocab, cluster) + 31) / 32 * 32;
        words = marks ? slice / 32 : 0;
        records = marks ? (int)std::min((long long)slice, (long long)(p->history ? p->history_len : 0) + (p->bias_ids ? p->biases : 0)) : 0;
        smem = marks ? ((size_t)2 * words + 1 + 2 * (size_t)records) * 4 : 0;
        if (smem <= 200 * 1024) break;
        CME_REQUIRE(cluster < MAX_CLUSTER, CME_ERR_LIMIT, "next token: a history of %d with a vocabulary of %d", p->history_len, p->vocab);
    }
    CME_REQUIRE((long long)p->rows * cluster < (1ll << 31), CME_ERR_LIMIT, "next token: too many rows");
    const int n = p->dtype == CME_F32 ? 4 : 8;
    auto al16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    // rows of logits start at the same place between 16-byte boundaries as rows of noise and of the processed logits
    const bool vector = al16(p->logits) && al16(p->processed) && al16(p->noise) && p->logits_ld % n == p->vocab % n;
    auto* kernel = p->dtype == CME_F32 ? (vector ? next_token_kernel<float, true> : next_token_kernel<float, false>)
                                       : (vector ? next_token_kernel<__nv_bfloat16, true> : next_token_kernel<__nv_bfloat16, false>);
    if (smem > 48 * 1024) CME_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p->rows * cluster));
    cfg.blockDim = dim3(slice <= 1024 ? 128 : 256);
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
    CME_CUDA(cudaLaunchKernelEx(&cfg, kernel, *p, cluster, slice, words, records));
    CME_LAUNCH_CHECK();
    return CME_OK;
}
