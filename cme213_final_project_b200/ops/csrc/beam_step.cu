// One step of a search with beams: of all continuations of a group's beams, the `width` best.
//
//     value(beam, token) = score[beam] + x[token] - log sum exp x;      a finished beam has one continuation, itself, with its score
//
// The order is that of the values as real numbers; equal ones: lower beam, lower token.  Within a beam that is the order of x, also where the values'
// 64 bits are the same.  Between beams
// it hangs on the log-sum-exps, whose 32-bit sums are off by some 2^-20; so every pair of different beams that decides something is held
// against a bound of that error, and where one is closer, the log-sum-exps of its beams are made anew in 64 bits, which decide.  Equal rows have equal
// ones then, too.
//
// Two launches: `scan` goes once over the logits, a CTA a slice of a row: sum of exponentials and the `width` largest; `merge`, a CTA a group,
// joins the slices and picks.  Up to 256 tokens (characters) a row is a warp's, in 64 bits, and one launch does both.
// In scan a thread keeps the sum and the largest of each few of its elements only, which costs no branch; the width-th largest of the best of those
// bounds what can be chosen from below, and the few groups that hold something above it are looked through again, a vector a thread.
// What bounds it: the bytes of the logits; 64 x 16 beams of 50304 in fp32, a fifth of which have ended: 53.9 us, of which the scan 42 at 4 TB/s (a third
// of a CTA's clocks are its start and its choice) and joining and choosing 9.  16 x 4 beams of 65 tokens 5.8 us.
//
// The bound of a log-sum-exp's error: an exponential's argument x - r is rounded twice and multiplied by a rounded log2 e, 2.5 * 2^-24 of |x - r|, which
// weighted by the softmax comes to 2.5 * 2^-24 (log vocab + RAISE) at the most (a reference r is one of the x, and none above r + RAISE
// goes by it; the mean distance from the largest x is at most log vocab, as the entropy is); the
// exponential itself is good to 2^-22; a term takes part in at most eight additions in 32 bits, 8 * 2^-24; the rest is added in 64 bits.
#include "common.h"
#include "beam_desc.h"

#include <algorithm>
#include <climits>
#include <cooperative_groups.h>
#include <type_traits>

namespace cg = cooperative_groups;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_WIDTH = 32, MAX_BEAMS = 32;
constexpr int SCAN = 256;                  // threads of a scan CTA
constexpr int AHEAD = 4;                   // vectors of a thread in a step
constexpr int SCANS = 4;                   // CTAs of an SM (six of two vectors ahead: the same time)
constexpr int STEP = SCAN * AHEAD;         // of a CTA
constexpr int CAP = 1024;                  // elements that reach the bound that a scan CTA can hold
constexpr int MERGE = 256;                 // threads of a merge CTA
constexpr int SURVIVORS = MAX_WIDTH * MAX_WIDTH;
constexpr int NEAR = 1024;                 // candidates that a merge CTA keeps in shared memory
constexpr int SMALL_VOCAB = 256;
constexpr float RAISE = 8.f;

struct Cand { float x; int token; };
// What a slice of a row comes to; behind it [width] candidates, best first.
struct Part {
    double sum;                            // of exp(x - ref)
    float ref;
    int count, pad[4];
};
static_assert(sizeof(Part) == 32 && sizeof(Cand) == 8, "layout of the scratch");

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// The largest of the warp; a NaN only if all are.
__device__ __forceinline__ float warp_most(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.x > b.x || (a.x == b.x && a.token < b.token); }

// A row's elements [v0, v1): sixteen bytes at a time from the first 16-byte boundary on, and the few before and behind.
template <typename T> struct Slice {
    static constexpr int N = 16 / (int)sizeof(T);
    const T* src;
    const unsigned* allowed;
    int v0, v1, a0, vectors;

    __device__ __forceinline__ Slice(const CmeBeams& p, int row, int from, int to) : v0(from), v1(to) {
        src = static_cast<const T*>(p.logits) + row * p.logits_ld;
        allowed = p.allowed ? reinterpret_cast<const unsigned*>(p.allowed) + row * p.allowed_ld : nullptr;
        const int off = (int)((reinterpret_cast<uintptr_t>(src + v0) / sizeof(T)) % N);
        a0 = min(v1, v0 + (off ? N - off : 0));
        vectors = (v1 - a0) / N;
    }
    __device__ __forceinline__ bool is_allowed(int t) const { return !allowed || (__ldg(allowed + (t >> 5)) >> (t & 31)) & 1; }
    __device__ __forceinline__ float at(int t) const { return is_allowed(t) ? to_f32<T>(src[t]) : -INFINITY; }
    __device__ __forceinline__ int token(int g) const { return a0 + g * N; }
    // Vector g; all -inf behind the last one.
    __device__ __forceinline__ uint4 load(int g) const {
        constexpr unsigned NONE = N == 8 ? 0xff80ff80u : 0xff800000u;
        uint4 v = make_uint4(NONE, NONE, NONE, NONE);
        if (g < vectors) v = *reinterpret_cast<const uint4*>(src + token(g));
        return v;
    }
    // Its elements, those that are not allowed as -inf.
    __device__ __forceinline__ void unpack(const uint4& v, int g, float* x) const {
        if constexpr (N == 8) unpack8(v, x);
        else { x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w); }
        if (allowed && g < vectors) {
            const int t = token(g), w = t >> 5, shift = t & 31;
            unsigned bits = __ldg(allowed + w) >> shift;
            if (shift + N > 32) bits |= __ldg(allowed + w + 1) << (32 - shift);      // (the last element's word)
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = bits >> e & 1 ? x[e] : -INFINITY;
        }
    }
    // The elements before and behind the vectors, fewer than 2 N: thread i's, or -inf and a token below 0.
    __device__ __forceinline__ float end(int i, int& t) const {
        const int head = a0 - v0, tail = token(vectors);
        t = i < head ? v0 + i : i < head + v1 - tail ? tail + i - head : -1;
        return t < 0 ? -INFINITY : at(t);
    }
};

// ------------------------------------------------------------------------------------------------------
// Scan
// ------------------------------------------------------------------------------------------------------
// The best behind the last one, over and over: where more elements than can be held are as large as the bound.
template <typename T> __device__ __noinline__ int scan_one_by_one(const CmeBeams& p, int row, int v0, int v1, Cand* list) {
    constexpr int WARPS = SCAN / 32;
    __shared__ Cand round_best[WARPS];
    const Slice<T> s(p, row, v0, v1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Cand last{INFINITY, -1};
    int found = 0;
    for (; found < p.width; ++found) {
        Cand best{-INFINITY, INT_MAX};
        for (int t = v0 + tid; t < v1; t += SCAN) {
            const Cand c{s.at(t), t};
            if (before(last, c) && before(c, best)) best = c;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const Cand c{__shfl_xor_sync(0xffffffffu, best.x, o), __shfl_xor_sync(0xffffffffu, best.token, o)};
            if (before(c, best)) best = c;
        }
        __syncthreads();
        if (lane == 0) round_best[warp] = best;
        __syncthreads();
        best = round_best[0];
        for (int w = 1; w < WARPS; ++w) if (before(round_best[w], best)) best = round_best[w];
        if (!(best.x > -INFINITY)) break;
        if (tid == 0) list[found] = best;
        last = best;
    }
    return found;
}

template <typename T>
__global__ void __launch_bounds__(SCAN, SCANS) beam_scan_kernel(const __grid_constant__ CmeBeams p, int slices, int slice, int resident) {
    constexpr int WARPS = SCAN / 32, N = Slice<T>::N, KEPT = 8;
    __shared__ float group_top[KEPT][SCAN];    // largest of a thread's vectors, `coarse` steps together
    __shared__ __align__(16) float tops[WARPS * 8];
    __shared__ float first_refs[WARPS], refs[WARPS];
    __shared__ double sums[WARPS];
    __shared__ Cand held[CAP];
    __shared__ int count;
    pdl_wait();
    const int row = blockIdx.x / slices, part = blockIdx.x - row * slices, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    char* out = static_cast<char*>(p.ws) + (long long)blockIdx.x * (sizeof(Part) + p.width * sizeof(Cand));
    Part* result = reinterpret_cast<Part*>(out);
    Cand* list = reinterpret_cast<Cand*>(result + 1);
    const int v0 = (int)min((long long)p.vocab, (long long)part * slice), v1 = (int)min((long long)p.vocab, (long long)v0 + slice);
    const Slice<T> s(p, row, v0, v1);
    uint4 raw[AHEAD];                          // the step's vectors; the next one's are on their way while it is reckoned
    auto fetch = [&](int it) {
        if ((it + 1) * STEP <= s.vectors) {
            const uint4* from = reinterpret_cast<const uint4*>(s.src + s.a0) + it * STEP + tid;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) raw[u] = from[u * SCAN];
        } else {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) raw[u] = s.load(it * STEP + u * SCAN + tid);
        }
    };
    fetch(0);
    int end_token;
    const float end = s.end(tid, end_token);
    if ((p.finished && p.finished[row]) || !finite(p.scores[row])) {         // nothing of the row counts
        if (tid == 0) *result = Part{0.0, 0.f, 0, {0, 0, 0, 0}};
        return;
    }
    // The sums' reference is the largest of the block's first elements; a thread that finds one larger by much takes that.
    float y[AHEAD][N], top = end;
    auto step_of = [&](int it) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) s.unpack(raw[u], it * STEP + u * SCAN + tid, y[u]);
    };
    step_of(0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int e = 0; e < N; e += 2) top = max3(top, y[u][e], y[u][e + 1]);
    top = warp_most(top);
    if (lane == 0) first_refs[warp] = top;
    if (tid == 0) count = 0;
    if (tid < WARPS * 8) tops[tid] = -INFINITY;
    __syncthreads();
    float ref = first_refs[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) ref = fmaxf(ref, first_refs[w]);
    double sum = 0.0;
    top = end;
    const int steps = (s.vectors + STEP - 1) / STEP, coarse = max(1, (steps + KEPT - 1) / KEPT);
    float group = -INFINITY;
    F32x2 shift = f2_splat(ref == -INFINITY ? 0.f : -ref);
    float limit = ref == -INFINITY ? ref : ref + RAISE;
    auto raise = [&](float m) {
        if (ref > -INFINITY) sum *= exp((double)ref - (double)m);             // (else it is 0, or NaN)
        ref = m;
        limit = ref + RAISE;
        shift = f2_splat(-ref);
    };
    const F32x2 scale = f2_splat(LOG2E);
    for (int it = 0, kept = 0, in = 0; it < steps; ++it) {
        step_of(it);
        fetch(it + 1);
        float m[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            m[u] = fmaxf(y[u][0], y[u][1]);
#pragma unroll
            for (int e = 2; e < N; e += 2) m[u] = max3(m[u], y[u][e], y[u][e + 1]);
        }
        const float most = fmaxf(max3(m[0], m[1], m[2]), m[3]);
        group = fmaxf(group, most);
        if (most > limit) raise(most);
        F32x2 acc[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                float a, b;
                f2_unpack(f2_mul(f2_add(f2_pack(y[u][e], y[u][e + 1]), shift), scale), a, b);
                const F32x2 t = f2_pack(ex2(a), ex2(b));
                acc[u] = e ? f2_add(acc[u], t) : t;
            }
        float a, b;
        f2_unpack(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), a, b);
        sum += (double)(a + b);
        if (++in == coarse || it + 1 == steps) {
            group_top[kept++][tid] = group;
            top = fmaxf(top, group);
            group = -INFINITY;
            in = 0;
        }
    }
    if (end_token >= 0) {
        if (end > limit) raise(end);
        sum += (double)ex2((end - (ref == -INFINITY ? 0.f : ref)) * LOG2E);
    }
    // The first two steps of the slice whose CTA comes when this one has gone are on their way to L2 while this one chooses (54.8 us without, 61 with
    // the whole slice from the start on).
    if (tid == 0 && blockIdx.x + resident < gridDim.x) {
        const int other = blockIdx.x + resident, other_row = other / slices, other_part = other - other_row * slices;
        if (!p.finished || !p.finished[other_row]) {
            const int from = (int)min((long long)p.vocab, (long long)other_part * slice);
            const Slice<T> o(p, other_row, from, (int)min((long long)p.vocab, (long long)from + slice));
            if (o.vectors > 0)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(o.src + o.a0), "r"(min(o.vectors, 2 * STEP) * 16) : "memory");
        }
    }
    // (a NaN or +inf among the logits makes the sum a NaN, by which the row is left out)
    // each warp's sum, and the largest 2 ceil(width / warps) of its threads' largest
    const float warp_ref = warp_most(ref);
    if (ref != warp_ref && ref > -INFINITY) sum *= exp((double)ref - (double)warp_ref);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) { sums[warp] = sum; refs[warp] = warp_ref; }
    const int per_warp = 2 * ((p.width + WARPS - 1) / WARPS), given = WARPS * per_warp;
    float left = top;
    for (int k = 0; k < per_warp; ++k) {
        const float m = warp_most(left);
        const int who = __ffs(__ballot_sync(0xffffffffu, left == m)) - 1;
        if (lane == 0) tops[warp * per_warp + k] = m;
        if (lane == who) left = -INFINITY;
    }
    __syncthreads();
    pdl_release();                             // (all but the choice is done: the next kernel's blocks may come)
    // The width-th largest of what the warps gave, the largest that `width` of them reach: so many elements are as large at least.  Every warp for itself.
    float bound = -INFINITY;
    for (int at = lane; at < given; at += 32) {
        const float v = tops[at];
        int reach = 0;
        for (int k = 0; k < given; k += 8) {
            const float4 a = *reinterpret_cast<const float4*>(tops + k), b = *reinterpret_cast<const float4*>(tops + k + 4);
            reach += (a.x >= v) + (a.y >= v) + (a.z >= v) + (a.w >= v) + (b.x >= v) + (b.y >= v) + (b.z >= v) + (b.w >= v);
        }
        if (reach >= p.width) bound = fmaxf(bound, v);
    }
    bound = warp_most(bound);
    auto offer = [&](float v, int t) {
        if (v >= bound && v > -INFINITY) {
            const int at = atomicAdd(&count, 1);
            if (at < CAP) held[at] = Cand{v, t};
        }
    };
    // The threads' groups that reach it, a thread's next one at a time.
    unsigned groups = 0;
    if (top >= bound && top > -INFINITY) {
        if (end_token >= 0) offer(end, end_token);
        for (int k = 0; k * coarse < steps; ++k) groups |= (unsigned)(group_top[k][tid] >= bound) << k;
    }
    while (groups) {
        const int k = __ffs(groups) - 1;
        groups &= groups - 1;
        for (int it = k * coarse; it < min(steps, (k + 1) * coarse); ++it) {
            fetch(it);
            step_of(it);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) offer(y[u][e], s.token(it * STEP + u * SCAN + tid) + e);
        }
    }
    __syncthreads();
    int n = count;
    if (n > CAP) {
        n = scan_one_by_one<T>(p, row, v0, v1, list);
    } else {
        for (int i = tid; i < n; i += SCAN) {
            const Cand c = held[i];
            int rank = 0;
#pragma unroll 4
            for (int k = 0; k < n; ++k) rank += before(held[k], c);
            if (rank < p.width) list[rank] = c;
        }
        n = min(n, p.width);
    }
    if (tid == 0) {
        float block_ref = refs[0];
        for (int w = 1; w < WARPS; ++w) block_ref = fmaxf(block_ref, refs[w]);
        double total = 0.0;
        for (int w = 0; w < WARPS; ++w)
            total += refs[w] == block_ref || refs[w] == -INFINITY ? sums[w] : sums[w] * exp((double)refs[w] - (double)block_ref);
        *result = Part{total, block_ref, n, {0, 0, 0, 0}};
    }
}

// ------------------------------------------------------------------------------------------------------
// Selection
// ------------------------------------------------------------------------------------------------------
struct Select {
    double value[SURVIVORS];
    int from[SURVIVORS], token[SURVIVORS]; // from: beam, list << 8, place in it << 16
    double lse[MAX_BEAMS], score[MAX_BEAMS];
    double slack;                          // twice the largest error of a log-sum-exp
    int counted;
    unsigned close;                        // beams of which a pair is too close
    double heads[MERGE];
    int last;                              // list of the bound
};

// Of `lists` lists, best first, those of lower beams first: list l is beam_of(l)'s, with count_of(l) candidates at(l, k).  All threads of the
// block; `width` outputs of the group.  False: some order is not certain; sel.close has the beams.
template <int THREADS, typename Beam, typename Count, typename At>
__device__ bool pick(Select& sel, const CmeBeams& p, int group, int lists, Beam&& beam_of, Count&& count_of, At&& at) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const double slack = sel.slack;
    auto value = [&](int l, int k) {
        const int b = beam_of(l);
        const Cand c = at(l, k);
        return c.token < 0 ? sel.score[b] : sel.score[b] + ((double)c.x - sel.lse[b]);
    };
    // Whether (v, b, x, t) comes before (u, c, y, s): value, beam, logit, token.
    auto ahead = [](double v, int b, float x, int t, double u, int c, float y, int s) {
        return v > u || (v == u && (b < c || (b == c && (x > y || (x == y && t < s)))));
    };
    // The width-th best of the lists' first ones bounds the choice from below (of a beam's lists those before have the lower tokens).  With slack 0 no
    // more than `width` lists are that good, so all that is chosen from fits.
    __syncthreads();
    if (tid == 0) { sel.counted = 0; sel.close = 0; sel.last = -1; }
    for (int l = tid; l < lists; l += THREADS) sel.heads[l] = count_of(l) ? value(l, 0) : -INFINITY;
    __syncthreads();
    if (lists > p.width) {
        for (int l = tid; l < lists; l += THREADS) {
            const double v = sel.heads[l];
            if (v == -INFINITY) continue;
            int above = 0, equal = 0;                      // (itself among them)
#pragma unroll 4
            for (int k = 0; k < lists; ++k) { above += sel.heads[k] > v; equal += sel.heads[k] == v; }
            for (int k = 0; equal > 1 && k < lists; ++k) above += sel.heads[k] == v && ahead(v, beam_of(k), at(k, 0).x, k, v, beam_of(l), at(l, 0).x, l);
            if (above == p.width - 1) sel.last = l;
        }
        __syncthreads();
    }
    const int last = sel.last, last_beam = last < 0 ? 0 : beam_of(last);
    const double bound = last < 0 ? -INFINITY : sel.heads[last] - slack;
    const Cand last_head = last < 0 || sel.heads[last] == -INFINITY ? Cand{0.f, 0} : at(last, 0);
    for (int l = warp; l < lists; l += THREADS / 32) {     // a warp a list
        const int k = lane;
        if (k >= count_of(l) || sel.heads[l] < bound) continue;
        const double v = value(l, k);
        const Cand own = at(l, k);
        if (v < bound || (v == bound && slack == 0.0 && ahead(v, last_beam, last_head.x, last_head.token, v, beam_of(l), own.x, own.token))) continue;
        const int c = atomicAdd(&sel.counted, 1);
        if (c < SURVIVORS) { sel.value[c] = v; sel.from[c] = beam_of(l) | l << 8 | k << 16; sel.token[c] = own.token; }
    }
    __syncthreads();
    const int n = sel.counted;
    if (n > SURVIVORS) {                   // many near one another
        if (tid == 0) sel.close = 0xffffffffu;
        __syncthreads();
        return false;
    }
    const int outs = p.width;
    constexpr int SHARE = 8;                               // lanes that hold one against the others
    for (int i0 = 0; i0 < n; i0 += THREADS / SHARE) {      // whole warps
        const int i = i0 + tid / SHARE;
        const bool in = i < n;
        const double v = in ? sel.value[i] : 0.0;
        const int from = in ? sel.from[i] : 0, b = from & 255, t = in ? sel.token[i] : 0;
        int rank = 0, equal = 0;
        unsigned near = 0;
#pragma unroll 4
        for (int k = tid % SHARE; k < n; k += SHARE) {
            const double u = sel.value[k];
            const int c = sel.from[k] & 255;
            rank += u > v || (u == v && c < b);
            equal += u == v && c == b && k != i;
            if (c != b && fabs(u - v) <= slack) near |= 1u << c;
        }
        for (int k = tid % SHARE; equal && k < n; k += SHARE)
            if (sel.value[k] == v && (sel.from[k] & 255) == b)
                rank += ahead(v, b, at(sel.from[k] >> 8 & 255, sel.from[k] >> 16).x, sel.token[k], v, b, at(from >> 8 & 255, from >> 16).x, t);
#pragma unroll
        for (int o = 1; o < SHARE; o <<= 1) {
            rank += __shfl_xor_sync(0xffffffffu, rank, o);
            near |= __shfl_xor_sync(0xffffffffu, near, o);
        }
        if (in && tid % SHARE == 0 && rank < outs) {
            if (near && slack > 0.0) atomicOr(&sel.close, near | 1u << b);
            const long long o = (long long)group * outs + rank;
            p.parents[o] = b;
            p.tokens[o] = t;
            p.out[o] = (float)v;
        }
    }
    for (int i = n + tid; i < outs; i += THREADS) {
        const long long o = (long long)group * outs + i;
        p.parents[o] = i % p.beams;
        p.tokens[o] = -1;
        p.out[o] = -INFINITY;
    }
    __syncthreads();
    return sel.close == 0;
}

// Sum of exp(x - top) over tokens [from, to) of a row in 64 bits, in an order that hangs on them only, whatever the row's place in memory: the whole block.
template <int THREADS, typename T> __device__ double exact_sum(const CmeBeams& p, int row, double top, int from, int to, double* scratch) {
    const Slice<T> s(p, row, from, to);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int CHAINS = 4;
    double part[CHAINS] = {};
    for (int t = from + tid; t < to; t += THREADS * CHAINS) {
        double x[CHAINS];
#pragma unroll
        for (int c = 0; c < CHAINS; ++c) x[c] = t + c * THREADS < to ? s.at(t + c * THREADS) : -INFINITY;
#pragma unroll
        for (int c = 0; c < CHAINS; ++c) part[c] += exp(x[c] - top);       // (exp(-inf) = 0)
    }
    double sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) scratch[warp] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) sum += scratch[w];
    return sum;
}

// The first CTA of a group's cluster joins and picks; the others are there for the sums in 64 bits, should they be needed (two rows of 50304 take one
// CTA 20 us; the bound of the error calls for some in one call of two with 64 groups of 16 beams).
template <typename T>
__global__ void __launch_bounds__(MERGE) beam_merge_kernel(const CmeBeams p, int slices, int size) {
    __shared__ Select sel;
    __shared__ double scratch[MERGE / 32];
    __shared__ int counts[MERGE];
    __shared__ Cand near_list[NEAR];           // all candidates, if there are no more
    __shared__ double sums[MERGE];
    __shared__ float refs[MERGE];
    __shared__ unsigned char over_s[MAX_BEAMS], beams_of[MERGE];
    __shared__ double top[MAX_BEAMS], exact[MAX_BEAMS];        // largest x of a row; this CTA's part of its sum in 64 bits
    pdl_wait();
    const int group = blockIdx.x / size, rank = blockIdx.x - group * size, tid = threadIdx.x, lists = p.beams * slices;
    const long long stride = sizeof(Part) + p.width * sizeof(Cand);
    auto part_at = [&](int l) -> const Part* {
        return reinterpret_cast<const Part*>(static_cast<const char*>(p.ws) + ((long long)group * p.beams * slices + l) * stride);
    };
    const bool close_by = lists * p.width <= NEAR;
    auto beam_of = [&](int l) { return (int)beams_of[l]; };
    auto count_of = [&](int l) { return counts[l]; };
    auto at = [&](int l, int k) {
        return over_s[beams_of[l]] ? Cand{0.f, -1} : close_by ? near_list[l * p.width + k] : reinterpret_cast<const Cand*>(part_at(l) + 1)[k];
    };
    if (rank == 0) {
        if (close_by) {
            for (int l = tid >> 5; l < lists; l += MERGE / 32)
                if ((tid & 31) < p.width)      // (behind the count there is nothing)
                    near_list[l * p.width + (tid & 31)] = reinterpret_cast<const Cand*>(part_at(l) + 1)[tid & 31];
        }
        for (int l = tid; l < lists; l += MERGE) {
            const Part part = *part_at(l);
            sums[l] = part.sum;
            refs[l] = part.ref;
            counts[l] = part.count;
            beams_of[l] = (unsigned char)(l / slices);
        }
        float score = 0.f;
        bool over = false;
        if (tid < p.beams) {
            const long long row = (long long)group * p.beams + tid;
            score = p.scores[row];
            over = p.finished && p.finished[row];
            over_s[tid] = over;
        }
        // twice the bound of a log-sum-exp's error (log vocab in 32 bits, hence a bit more)
        if (tid == 0) sel.slack = 2.0 * (3 * 0x1p-22 + 2.5 * 0x1p-24 * ((double)logf((float)p.vocab) + RAISE + 1e-3));
        __syncthreads();
        if (tid < p.beams) {
            const int l0 = tid * slices;
            float ref = -INFINITY;
            for (int l = l0; l < l0 + slices; ++l) ref = sums[l] > 0.0 ? fmaxf(ref, refs[l]) : ref;
            double sum = 0.0;
            for (int l = l0; l < l0 + slices; ++l) {
                if (sums[l] != sums[l]) sum = sums[l];
                else if (sums[l] > 0.0) sum += refs[l] == ref ? sums[l] : sums[l] * exp((double)refs[l] - (double)ref);
            }
            const double lse = ref + log(sum);
            const bool fine = finite(score) && (over || (sum > 0.0 && fabs(lse) < INFINITY));
            sel.score[tid] = fine ? (double)score : -INFINITY;
            sel.lse[tid] = fine && !over ? lse : 0.0;
            double most = -INFINITY;
            for (int l = l0; l < l0 + slices; ++l) {
                if (counts[l]) most = fmax(most, (double)reinterpret_cast<const Cand*>(part_at(l) + 1)->x);
                counts[l] = !fine ? 0 : over ? l == l0 : counts[l];
            }
            top[tid] = most;
        }
        __syncthreads();
        pick<MERGE>(sel, p, group, lists, beam_of, count_of, at);
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (size > 1) cluster.sync();
    const Select& first = *cluster.map_shared_rank(&sel, 0);
    const unsigned close = first.close;
    if (close) {
        const double* tops = cluster.map_shared_rank(top, 0);
        const int each = (p.vocab + size - 1) / size, from = min((long long)p.vocab, (long long)rank * each), to = min((long long)p.vocab, (long long)from + each);
        for (int b = 0; b < p.beams; ++b) {
            const long long row = (long long)group * p.beams + b;
            if (!(close >> b & 1) || first.score[b] == -INFINITY || (p.finished && p.finished[row])) continue;
            const double sum = exact_sum<MERGE, T>(p, (int)row, tops[b], from, to, scratch);
            if (tid == 0) exact[b] = sum;
        }
    }
    if (size > 1) cluster.sync();
    else __syncthreads();
    if (close == 0) return;
    if (rank == 0 && tid < p.beams && close >> tid & 1 && sel.score[tid] != -INFINITY && !over_s[tid]) {
        double sum = 0.0;
        for (int r = 0; r < size; ++r) sum += *cluster.map_shared_rank(exact + tid, r);
        sel.lse[tid] = top[tid] + log(sum);
    }
    if (size > 1) cluster.sync();              // (nobody's shared memory goes while it is read)
    if (rank) return;
    if (tid == 0) sel.slack = 0.0;
    __syncthreads();
    pick<MERGE>(sel, p, group, lists, beam_of, count_of, at);
}

// Few tokens: a warp a row, in 64 bits.
constexpr int SMALL = 256;
template <typename T>
__global__ void __launch_bounds__(SMALL) beam_small_kernel(const CmeBeams p) {
    constexpr int WARPS = SMALL / 32, EACH = SMALL_VOCAB / 32;
    __shared__ Select sel;
    __shared__ Cand best[MAX_BEAMS][MAX_WIDTH];
    __shared__ int counts[MAX_BEAMS];
    pdl_release();
    pdl_wait();
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sel.slack = 0.0;
    for (int b = warp; b < p.beams; b += WARPS) {
        const long long row = (long long)group * p.beams + b;
        const float score = p.scores[row];
        const bool over = p.finished && p.finished[row];
        const Slice<T> s(p, (int)row, 0, p.vocab);
        float x[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) x[e] = e * 32 + lane < p.vocab ? s.at(e * 32 + lane) : -INFINITY;
        float m = -INFINITY;
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) m = fmaxf(m, x[e]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll 1
        for (int e = 0; e * 32 < p.vocab; ++e) {
            const float v = e * 32 + lane < p.vocab ? s.at(e * 32 + lane) : -INFINITY;
            if (v != -INFINITY) sum += exp((double)v - (double)m);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double lse = (double)m + log(sum);
        const bool fine = finite(score) && (over || (sum > 0.0 && fabs(lse) < INFINITY));
        int n = 0;
        if (fine && over) {
            n = 1;
            if (lane == 0) best[b][0] = Cand{0.f, -1};
        } else if (fine) {
            for (; n < p.width; ++n) {
                Cand c{-INFINITY, INT_MAX};
#pragma unroll
                for (int e = 0; e < EACH; ++e) if (x[e] > c.x) c = Cand{x[e], e * 32 + lane};
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const Cand d{__shfl_xor_sync(0xffffffffu, c.x, o), __shfl_xor_sync(0xffffffffu, c.token, o)};
                    if (before(d, c)) c = d;
                }
                if (c.x == -INFINITY) break;
                if (lane == 0) best[b][n] = c;
#pragma unroll
                for (int e = 0; e < EACH; ++e) if (e * 32 + lane == c.token) x[e] = -INFINITY;
            }
        }
        if (lane == 0) {
            sel.score[b] = fine ? (double)score : -INFINITY;
            sel.lse[b] = fine && !over ? lse : 0.0;
            counts[b] = n;
        }
    }
    __syncthreads();
    pick<SMALL>(sel, p, group, p.beams, [](int l) { return l; }, [&](int l) { return counts[l]; }, [&](int l, int k) { return best[l][k]; });
}

// ------------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------------
int check(const CmeBeams* a) {
    CME_REQUIRE(a->dtype == CME_F32 || a->dtype == CME_BF16, CME_ERR_UNSUPPORTED, "beam step: unsupported dtype");
    CME_REQUIRE(a->groups >= 0 && a->vocab > 0, CME_ERR_SHAPE, "beam step: bad sizes");
    CME_REQUIRE(a->beams > 0 && a->beams <= MAX_BEAMS && a->width > 0 && a->width <= MAX_WIDTH, CME_ERR_LIMIT,
                "beam step: %d beams and a width of %d (1 to 32 of both)", a->beams, a->width);
    CME_REQUIRE((long long)a->groups * a->beams * 256 < (1ll << 31), CME_ERR_LIMIT, "beam step: too many rows");
    CME_REQUIRE(a->vocab <= 1 << 30, CME_ERR_LIMIT, "beam step: too many tokens");      // (indexes run up to a few thousand beyond)
    return CME_OK;
}
// Slices of a row.
int slices_of(const CmeBeams* a, int sms) {
    const long long rows = std::max(1ll, (long long)a->groups * a->beams);
    const long long wanted = (sms * 8ll + rows - 1) / rows, fit = MERGE / a->beams, by_size = std::max(1, a->vocab / 2048);
    return (int)std::max(1ll, std::min(std::min(wanted, by_size), std::min(fit, 32ll)));
}
template <typename T> int launch(const CmeBeams* a, int sms, cudaStream_t st) {
    if (a->vocab <= SMALL_VOCAB) {
        CME_CUDA(cme_launch_dependent(beam_small_kernel<T>, dim3(a->groups), dim3(SMALL), 0, st, *a));
        CME_LAUNCH_CHECK();
        return CME_OK;
    }
    const int slices = slices_of(a, sms), slice = cme_cdiv(cme_cdiv(a->vocab, slices), 8) * 8;
    CME_CUDA(cme_launch_dependent(beam_scan_kernel<T>, dim3(a->groups * a->beams * slices), dim3(SCAN), 0, st, *a, slices, slice, sms * SCANS));
    CME_LAUNCH_CHECK();
    int size = 8;                                         // of a group's cluster: as many as run at a time
    while (size > 1 && (long long)a->groups * size > sms * 4ll) size /= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a->groups * size);
    cfg.blockDim = dim3(MERGE);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = size;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    CME_CUDA(cudaLaunchKernelEx(&cfg, beam_merge_kernel<T>, *a, slices, size));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

}  // namespace

// Scratch of a call, in bytes.
CME_API int cme_beam_step_ws_bytes(const CmeBeams* a, long long* out) {
    int rc, sms;
    if ((rc = check(a)) || (rc = cme_num_sms(&sms))) return rc;
    *out = a->vocab <= SMALL_VOCAB ? 0 : (long long)a->groups * a->beams * slices_of(a, sms) * (long long)(sizeof(Part) + a->width * sizeof(Cand));
    return CME_OK;
}

CME_API int cme_beam_step(const CmeBeams* a, void* stream) {
    int sms;
    long long need;
    int rc = cme_beam_step_ws_bytes(a, &need);
    if (rc || (rc = cme_num_sms(&sms))) return rc;
    if (a->groups == 0) return CME_OK;
    CME_REQUIRE(need <= a->ws_bytes && (reinterpret_cast<uintptr_t>(a->ws) & 15) == 0, CME_ERR_SHAPE, "beam step: %lld bytes of scratch, %lld are needed",
                a->ws_bytes, need);
    return a->dtype == CME_F32 ? launch<float>(a, sms, (cudaStream_t)stream) : launch<__nv_bfloat16>(a, sms, (cudaStream_t)stream);
}
