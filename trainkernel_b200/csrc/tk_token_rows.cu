// Log-probabilities of tokens from rows of logits, the gradient of the logits, and the losses built on them.
//
// Mathematics.  For a row x of V logits and its token t, with m = max x and S = sum_j exp(x_j - m):
//     logprob = (x_t - m) - log S,     d logprob / d x_j = [j = t] - exp(x_j - m) / S.
// Every loss here is a function of the log-probabilities, so its gradient is a coefficient per row times that row.
// (m, S) pairs of parts of a row join associatively: M = max(m1, m2), S = S1 exp(m1 - M) + S2 exp(m2 - M), so one
// pass over the row gives both.  m is a logit that occurs, and never below the lowest finite FP32 number: -inf needs no
// special case.  All statistics, coefficients and sums are FP32 or wider; the only rounding to 16 bits is the gradient's,
// once, at its store.
#include "tk_ops_host.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace {

using tk_ops::check;
using tk_ops::count_launch;
using tk_ops::DeviceScope;
using tk_ops::fail;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kExtreme = 65536.f;                // beyond it the rounding of logit * log2(e) is no longer small (see Exponent)

// 2^x by the hardware's approximation (relative error about 2^-22).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two FP32 numbers in one 64-bit register, for the paired arithmetic instructions.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 both(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 16 bytes of logits.
template <typename T> struct Vector;
template <> struct Vector<float> {
    static constexpr int kCount = 4;
    static constexpr bool kSplit = false;          // whether gradients need exp2_split
    static constexpr bool kWide = true;            // whether finite logits reach beyond kExtreme
    static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[2]) {
        f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
        return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    }
    static __device__ __forceinline__ float top(const uint4& v) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static __device__ __forceinline__ float load(float x) { return x; }
    static __device__ __forceinline__ float store(float x) { return x; }
};
template <> struct Vector<__nv_bfloat16> {
    static constexpr int kCount = 8;
    static constexpr bool kSplit = false;
    static constexpr bool kWide = true;
    static __device__ __forceinline__ float2 two(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[4]) {
        f[0] = two(v.x);
        f[1] = two(v.y);
        f[2] = two(v.z);
        f[3] = two(v.w);
    }
    static __device__ __forceinline__ uint32_t word(float2 f) {
        const __nv_bfloat162 h = __float22bfloat162_rn(f);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) { return make_uint4(word(f[0]), word(f[1]), word(f[2]), word(f[3])); }
    static __device__ __forceinline__ float top(const uint4& v) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
        const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ float load(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 store(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Vector<__half> {
    static constexpr int kCount = 8;
    static constexpr bool kSplit = true;
    static constexpr bool kWide = false;
    static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[4]) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __half22float2(h[i]);
    }
    static __device__ __forceinline__ uint32_t word(float2 f) {
        const __half2 h = __float22half2_rn(f);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) { return make_uint4(word(f[0]), word(f[1]), word(f[2]), word(f[3])); }
    static __device__ __forceinline__ float top(const uint4& v) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
        const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ float load(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half store(float x) { return __float2half_rn(x); }
};

// x log2(e), rounded on its own (never contracted into a fused operation with what follows).
__device__ __forceinline__ float scaled(float x) {
    float y;
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(kLog2e));
    return y;
}

// The exponent of 2 that stands for exp(x - top): x log2(e) - rn(top log2(e)) in one fused operation.  The rounding of
// the subtrahend is the same for every logit of the row and for its target, so it cancels, as long as 2 to that rounding
// is an ordinary number: it is at most 2^-8 while |top| <= 2^16, which holds for all of FP16, and would reach 2^7 near 3e9,
// where every term of the sum is infinite or zero.  Beyond 2^16 (rows filled with a large negative number in place of
// -inf) the difference is taken first, which is exact to half a step and multiplied after.
struct Exponent {
    float top, base;
    bool extreme;
    __device__ __forceinline__ explicit Exponent(float t) : top(t), base(scaled(t)), extreme(fabsf(t) > kExtreme) {}
    __device__ __forceinline__ float operator()(float x) const { return extreme ? (x - top) * kLog2e : fmaf(x, kLog2e, -base); }
};

struct Stat {
    float top, sum;                        // sum of 2^Exponent(top)(x)
};

// The exponent of 2 that takes a sum relative to the top `from` to one relative to `to`.  A sum is relative to its top's
// rounded base, or, beyond kExtreme, to the product itself; what is subtracted is rounded as it was used.
__device__ __forceinline__ float shift(float from, const Exponent& to) {
    const bool far = fabsf(from) > kExtreme;
    if (to.extreme) return far ? (from - to.top) * kLog2e : fmaf(-to.top, kLog2e, scaled(from));
    return far ? fmaf(from, kLog2e, -to.base) : scaled(from) - to.base;
}

// The same statistics relative to a top that is as large or larger.
__device__ __forceinline__ Stat raised(Stat s, float top) { return {top, s.sum * exp2_fast(shift(s.top, Exponent(top)))}; }

// 2^(x log2(e) - base) with the exponent split at a whole number, so that its fraction keeps all of its bits: the rounding of
// an exponent near -12 alone costs 2^-21 of the value, more than one part in a hundred of half a step of FP16, and with small
// gradients, which FP16 holds in few bits, would tip several times as many of them to the other side as FP32's exp does.
// BF16's half step is eight times as wide and its gradients do without: of 917760 gradients of 768 x 1195 logits 23 to 85 lie
// on the other side of a border than in 64 bits, 18 to 84 with FP32's exp (six seeds).
__device__ __forceinline__ float exp2_split(float x, float base) {
    const float whole = fmaxf(fmaf(x, kLog2e, -base), -126.f) + 12582912.f;           // 1.5 2^23: rounded to a whole number
    const float n = whole - 12582912.f;
    return exp2_fast(fmaf(x, kLog2e, -(base + n))) * __int_as_float((__float_as_int(whole) << 23) + 0x3f800000);
}

// Adds N vectors of logits to a thread's statistics.
template <typename T, int N>
__device__ __forceinline__ void accumulate(Stat& s, const uint4 (&v)[N]) {
    constexpr int kPairs = Vector<T>::kCount / 2;
    float top = s.top;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, Vector<T>::top(v[i]));
    const Exponent e(top);
    // Both tops within kExtreme, or nothing added yet (or only what is nothing beside the new top): the short form of `raised`.
    const bool far = e.extreme || (Vector<T>::kWide && s.top < -kExtreme && s.top != kLowest);
    if (!far) {
        s.sum *= exp2_fast(scaled(s.top) - e.base);
        s.top = top;
        const Pair scale = pair(kLog2e, kLog2e), base = pair(-e.base, -e.base);
        Pair sum = pair(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float2 f[kPairs];
            Vector<T>::unpack(v[i], f);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const float2 x = both(fma2(pair(f[k].x, f[k].y), scale, base));
                sum = add2(sum, pair(exp2_fast(x.x), exp2_fast(x.y)));
            }
        }
        const float2 total = both(sum);
        s.sum += total.x + total.y;
    } else {
        s = raised(s, top);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float2 f[kPairs];
            Vector<T>::unpack(v[i], f);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) s.sum += exp2_fast(e(f[k].x)) + exp2_fast(e(f[k].y));
        }
    }
}

template <typename T>
__device__ __forceinline__ void accumulate_one(Stat& s, T value) {
    const float x = Vector<T>::load(value);
    if (x > s.top) s = raised(s, x);
    s.sum += exp2_fast(Exponent(s.top)(x));
}

enum Mode { kStats, kGrad, kBoth };            // log-probabilities / gradient from saved stats / both

enum Loss { kWeights, kPolicy };               // where kBoth takes the coefficient from, and what kStats adds

struct Args {
    tk_token_rows rows;
    tk_token_array coefficients;               // kGrad and kBoth with kWeights: FP32 [batch, length]
    tk_policy_terms policy;
    tk_token_grad grad;
    float* logprobs;
    float* stats;
    float* row_coefficients;                   // kPolicy: dense d loss / d logprob, or NULL
    bool in_phase;                             // every row of the gradient lies as its logits do within 16 bytes
    // kPolicy: workspace
    unsigned* counter;
    float* weights;                            // one per sequence
    float* terms;                              // one per row
    float* loss;
    int64_t first_rows;                        // rows whose blocks start at once; those behind them start when one has ended
    unsigned* clear;                           // a word block 0 zeroes for the kernel that follows, or NULL
};

__device__ __forceinline__ int64_t target_of(const tk_token_rows& r, int64_t b, int64_t t) {
    const int64_t at = b * r.targets.stride_batch + t * r.targets.stride_token;
    return r.target_bytes == 8 ? static_cast<const int64_t*>(r.targets.data)[at] : static_cast<const int32_t*>(r.targets.data)[at];
}

__device__ __forceinline__ bool counts(const tk_token_rows& r, int64_t b, int64_t t) {
    return !r.mask.data || static_cast<const unsigned char*>(r.mask.data)[b * r.mask.stride_batch + t * r.mask.stride_token];
}

__device__ __forceinline__ float at(const tk_token_array& a, int64_t b, int64_t t) {
    return static_cast<const float*>(a.data)[b * a.stride_batch + t * a.stride_token];
}

// The statistics of 32 lanes, in every lane: the largest top first, then the sums relative to it.
__device__ __forceinline__ Stat warp_join(Stat mine) {
    float top = mine.top;
#pragma unroll
    for (int step = 16; step; step >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, step));
    float sum = raised(mine, top).sum;
#pragma unroll
    for (int step = 16; step; step >>= 1) sum += __shfl_xor_sync(~0u, sum, step);
    return {top, sum};
}

template <int THREADS>
__device__ Stat block_join(Stat mine, Stat* shared) {
    mine = warp_join(mine);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (lane == 0) shared[warp] = mine;
    __syncthreads();
    return warp_join(lane < THREADS / 32 ? shared[lane] : Stat{kLowest, 0.f});
}

// The loss of one token and its slope in the log-probability.
__device__ __forceinline__ void policy_token(const tk_policy_terms& p, float old_logprob, float advantage, float ref_logprob, float logprob,
                                             float* term, float* slope) {
    const float ratio = expf(logprob - old_logprob);
    const float free = ratio * advantage;
    const float bound = fminf(fmaxf(ratio, 1.f - p.clip_low), 1.f + p.clip_high) * advantage;
    const bool clipped = free > bound;                    // false for NaN: it then stays in the result
    *term = clipped ? -bound : -free;
    *slope = clipped ? 0.f : -free;
    if (p.ref_logprobs.data) {
        const float away = ref_logprob - logprob, grown = expm1f(away);
        *term += p.kl_weight * (grown - away);
        *slope -= p.kl_weight * grown;
    }
}

__device__ __forceinline__ float not_a_number() { return __int_as_float(0x7fffffff); }

// A row's parts: elements before the first 16-byte boundary, whole vectors, elements behind the last.
struct Parts {
    int head, vectors, tail;
};
template <typename T>
__device__ __forceinline__ Parts parts_of(const T* x, int vocab) {
    constexpr int kCount = Vector<T>::kCount;
    int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T));
    head = head < vocab ? head : vocab;
    return {head, (vocab - head) / kCount, (vocab - head) % kCount};
}

// A block's share of a row: all of it, or, where a cluster of blocks splits the row, an equal run of its vectors, with
// the elements before and behind them in the first and the last block.
struct Share {
    int rank, size;
    __device__ __forceinline__ int per(int vectors) const { return (vectors + size - 1) / size; }
    __device__ __forceinline__ int begin(int vectors) const { return min(rank * per(vectors), vectors); }
    __device__ __forceinline__ int end(int vectors) const { return min(rank * per(vectors) + per(vectors), vectors); }
    __device__ __forceinline__ bool first() const { return rank == 0; }
    __device__ __forceinline__ bool last() const { return rank == size - 1; }
};

// A load with an L2 policy, and the policy that keeps a line because it is read again soon.
__device__ __forceinline__ uint4 load_hint(const uint4* p, unsigned long long policy) {
    uint4 v;
    asm volatile("ld.global.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy));
    return v;
}
__device__ __forceinline__ unsigned long long keep_policy() {
    unsigned long long policy;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}

constexpr int kAhead = 4;                      // vectors a thread has in flight

// Asks L2 for the vectors of a thread's next turn before it loads those of this one: registers for a second set in flight
// would cost resident blocks.  Policy loss of 8000 x 32000 BF16 logits with gradient, in the block shape it had then: 198 ->
// 179 us; two or three turns ahead 186 and 190.  The statistics alone, whose blocks only read, do without: asking ahead
// takes 113 us instead of 110 at that size and 338 instead of 349 at 8192 x 128256.
template <int THREADS>
__device__ __forceinline__ void prefetch_turn(const uint4* body, int i, int end) {
    if (threadIdx.x % 8) return;                           // one request for every 128 bytes
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int next = i + (kAhead + k) * THREADS;
        if (next < end) asm volatile("prefetch.global.L2 [%0];" ::"l"(body + next));
    }
}

// Statistics of a row, or of a block's share of it.  The first `kept` vectors of a whole row also go to shared memory, where
// the thread that read them finds them again; of the rest L2 is asked to keep what is read `again`.
template <typename T, int THREADS>
__device__ __forceinline__ Stat row_stat(const T* x, int vocab, const Share share, uint4* kept_at, int kept, bool again) {
    const Parts p = parts_of(x, vocab);
    const uint4* body = reinterpret_cast<const uint4*>(x + p.head);
    Stat s{kLowest, 0.f};
    const int end = share.end(p.vectors);
    int i = share.begin(p.vectors) + threadIdx.x;
    const int first = min(kept, p.vectors);
    for (; i + (kAhead - 1) * THREADS < first; i += kAhead * THREADS) {
        prefetch_turn<THREADS>(body, i, end);
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = __ldcs(body + i + k * THREADS);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) kept_at[i + k * THREADS] = v[k];
        accumulate<T, kAhead>(s, v);
    }
    for (; i < first; i += THREADS) {
        const uint4 v[1] = {__ldcs(body + i)};
        kept_at[i] = v[0];
        accumulate<T, 1>(s, v);
    }
    const unsigned long long policy = keep_policy();
    for (; i + (kAhead - 1) * THREADS < end; i += kAhead * THREADS) {
        if (again) prefetch_turn<THREADS>(body, i, end);
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = again ? load_hint(body + i + k * THREADS, policy) : __ldcg(body + i + k * THREADS);
        accumulate<T, kAhead>(s, v);
    }
    for (; i < end; i += THREADS) {
        const uint4 v[1] = {__ldcg(body + i)};
        accumulate<T, 1>(s, v);
    }
    if (share.first() && threadIdx.x < p.head) accumulate_one(s, x[threadIdx.x]);
    if (share.last() && threadIdx.x < p.tail) accumulate_one(s, x[vocab - p.tail + threadIdx.x]);
    return s;
}

// coefficient * (delta - p) for every logit of a row; `factor` = -coefficient / sum.
template <typename T, int THREADS>
__device__ __forceinline__ void row_grad(T* out, const T* x, int vocab, const Share share, int target, const Exponent e, float factor, float coefficient, bool in_phase,
                                         const uint4* kept_at, int kept) {
    const auto one = [&](int j) {
        const float logit = Vector<T>::load(x[j]);
        float value = (Vector<T>::kSplit && !e.extreme ? exp2_split(logit, e.base) : exp2_fast(e(logit))) * factor;
        if (j == target) value += coefficient;
        out[j] = Vector<T>::store(value);
    };
    if (!in_phase || e.extreme) {
        for (int64_t j = threadIdx.x + share.rank * THREADS; j < vocab; j += THREADS * share.size) one(static_cast<int>(j));
        return;
    }
    constexpr int kCount = Vector<T>::kCount, kPairs = kCount / 2;
    const Parts p = parts_of(x, vocab);
    const uint4* body = reinterpret_cast<const uint4*>(x + p.head);
    uint4* to = reinterpret_cast<uint4*>(out + p.head);
    const int special = target >= p.head ? (target - p.head) / kCount : -1, place = (target - p.head) % kCount;
    const Pair scale = pair(kLog2e, kLog2e), base = pair(-e.base, -e.base), by = pair(factor, factor);
    const auto vector = [&](int i, const uint4& v) {
        float2 f[kPairs];
        Vector<T>::unpack(v, f);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            if (Vector<T>::kSplit) {
                f[k] = both(mul2(pair(exp2_split(f[k].x, e.base), exp2_split(f[k].y, e.base)), by));
            } else {
                const float2 y = both(fma2(pair(f[k].x, f[k].y), scale, base));
                f[k] = both(mul2(pair(exp2_fast(y.x), exp2_fast(y.y)), by));
            }
        }
        if (i == special) {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                if (place == 2 * k) f[k].x += coefficient;
                if (place == 2 * k + 1) f[k].y += coefficient;
            }
        }
        __stcs(to + i, Vector<T>::pack(f));
    };
    // From the row's end, which was read last and is near, to the part kept in shared memory.
    const int end = share.end(p.vectors), first = kept ? min(kept, p.vectors) : share.begin(p.vectors), left = (end - first) % (kAhead * THREADS);
    for (int i = end - kAhead * THREADS + threadIdx.x; i >= first + left; i -= kAhead * THREADS) {
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = __ldcs(body + i + k * THREADS);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) vector(i + k * THREADS, v[k]);
    }
    for (int i = first + threadIdx.x; i < first + left; i += THREADS) vector(i, __ldcs(body + i));
    if (kept)
        for (int i = threadIdx.x; i < first; i += THREADS) vector(i, kept_at[i]);
    if (share.first() && threadIdx.x < p.head) one(threadIdx.x);
    if (share.last() && threadIdx.x < p.tail) one(vocab - p.tail + threadIdx.x);
}

template <typename T, int THREADS>
__device__ __forceinline__ void row_zero(T* out, int vocab, const Share share) {
    const Parts p = parts_of(out, vocab);
    uint4* to = reinterpret_cast<uint4*>(out + p.head);
    for (int i = share.begin(p.vectors) + threadIdx.x; i < share.end(p.vectors); i += THREADS) __stcs(to + i, make_uint4(0, 0, 0, 0));
    if (share.first() && threadIdx.x < p.head) out[threadIdx.x] = Vector<T>::store(0.f);
    if (share.last() && threadIdx.x < p.tail) out[vocab - p.tail + threadIdx.x] = Vector<T>::store(0.f);
}

// Kernels that follow another one of the same call are launched while it still runs and wait here for its results.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float row_logprob(Stat stat, float value) {
    const Exponent e(stat.top);
    return e.extreme ? (value - stat.top) - logf(stat.sum) : (e(value) - log2f(stat.sum)) * kLn2;
}

// The sum of all rows' terms in an order that does not depend on which block forms it.
template <int THREADS>
__device__ __forceinline__ void sum_terms(const float* terms, int64_t rows, float* loss) {
    __shared__ double parts[32];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += THREADS) sum += __ldcg(terms + i);
#pragma unroll
    for (int step = 16; step; step >>= 1) sum += __shfl_xor_sync(~0u, sum, step);
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int i = 0; i < THREADS / 32; ++i) sum += parts[i];
        *loss = static_cast<float>(sum);
    }
}

constexpr int kMostShares = 8;                 // blocks of a cluster

// A block may write to another's shared memory once that one has started, so all of them report at their start.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }

// The statistics of all blocks of a cluster, in every thread: each block writes its own into every block's shared memory.
__device__ __forceinline__ Stat cluster_join(Stat mine, const Share share, float2* parts) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");          // for cluster_started
    if (threadIdx.x < share.size) {
        uint32_t to;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(parts + share.rank))), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to), "l"(pair(mine.top, mine.sum)) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int lane = threadIdx.x % 32;
    const float2 part = lane < share.size ? parts[lane] : make_float2(kLowest, 0.f);
    return warp_join({part.x, part.y});
}

// One block per row, or, with SPLIT, one cluster of blocks per row.  Memory bounds the statistics alone; with the gradient a
// block waits for its join between the passes, which only the other blocks of the multiprocessor fill, and every logit
// takes two exponentials (72 % of their unit's cycles at 4000 x 32000 BF16, 63 % at 1024 x 128256).  launch_type has the block shapes and their times.
template <typename T, Mode MODE, Loss LOSS, int THREADS, int BLOCKS, bool SPLIT>
__global__ void __launch_bounds__(THREADS, BLOCKS) token_rows_kernel(const __grid_constant__ Args a, const int kept) {
    extern __shared__ uint4 kept_at[];
    __shared__ Stat shared[32];
    __shared__ float shared_coefficient;
    __shared__ bool shared_last;
    __shared__ float2 shared_parts[SPLIT ? kMostShares : 1];
    const tk_token_rows& r = a.rows;
    Share share{0, 1};
    if (SPLIT) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(share.rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(share.size));
    }
    const int64_t row = blockIdx.x / static_cast<unsigned>(share.size), b = row / r.length, t = row % r.length;
    const T* x = static_cast<const T*>(r.logits) + b * r.stride_batch + t * r.stride_token;
    T* out = static_cast<T*>(a.grad.data) + b * a.grad.stride_batch + t * a.grad.stride_token;
    const bool keep = counts(r, b, t);
    const int vocab = static_cast<int>(r.vocab);
    if (SPLIT && MODE != kGrad && keep) cluster_started();               // the row is the cluster's: all of its blocks or none
    Stat stat{kLowest, 0.f};
    int target = -1;
    if (a.clear && blockIdx.x == 0 && threadIdx.x == 0) *a.clear = 0;
    if (keep) {
        const int64_t wanted = target_of(r, b, t);
        target = wanted >= 0 && wanted < vocab ? static_cast<int>(wanted) : -1;
    }
    // What the row's result needs besides its statistics is asked for before them, so that it has arrived behind them.
    float value = not_a_number(), old_logprob = 0.f, advantage = 0.f, ref_logprob = 0.f, weight = 0.f;
    if (MODE != kGrad && keep && threadIdx.x == 0) {
        if (target >= 0) value = Vector<T>::load(x[target]);
        if (LOSS == kPolicy) {
            old_logprob = at(a.policy.old_logprobs, b, t);
            advantage = at(a.policy.advantages, b, t);
            if (a.policy.ref_logprobs.data) ref_logprob = at(a.policy.ref_logprobs, b, t);
            // The first blocks start beside the kernel that computes the weights and ask for theirs behind the statistics.
            // When a later one starts it has ended, and the wait costs nothing.
            if (row >= a.first_rows) {
                wait_for_previous();
                weight = a.weights[b];
            }
        }
    }
    if (MODE == kGrad) wait_for_previous();
    if (MODE != kStats && LOSS != kPolicy && keep) weight = at(a.coefficients, b, t);
    if (MODE != kGrad && keep) {
        stat = block_join<THREADS>(row_stat<T, THREADS>(x, vocab, share, kept_at, kept, MODE == kBoth), shared);
        if (SPLIT) stat = cluster_join(stat, share, shared_parts);
    }
    if (MODE != kGrad && threadIdx.x == 0) {
        const float logprob = keep ? row_logprob(stat, value) : 0.f;
        if (share.first() && a.logprobs) a.logprobs[row] = logprob;
        if (share.first() && a.stats) {
            a.stats[2 * row] = stat.top;
            a.stats[2 * row + 1] = stat.sum;
        }
        if (LOSS == kPolicy) {
            float term = 0.f, slope = 0.f;
            if (row < a.first_rows || !keep) wait_for_previous();              // for the counter too
            if (keep) {
                if (row < a.first_rows) weight = a.weights[b];
                policy_token(a.policy, old_logprob, advantage, ref_logprob, logprob, &term, &slope);
                term *= weight;
                slope *= weight;
            }
            if (share.first()) {
                a.terms[row] = term;
                if (a.row_coefficients) a.row_coefficients[row] = slope;
            }
            shared_coefficient = slope;
        }
    }
    if (MODE != kStats) {
        if (keep) {
            float coefficient = a.grad.scale_at ? a.grad.scale * *a.grad.scale_at : a.grad.scale;
            if (LOSS == kPolicy) {
                __syncthreads();
                coefficient *= shared_coefficient;
            } else {
                coefficient *= weight;
            }
            if (MODE == kGrad) stat = {a.stats[2 * row], a.stats[2 * row + 1]};
            const float factor = target >= 0 ? -coefficient / stat.sum : not_a_number();
            row_grad<T, THREADS>(out, x, vocab, share, target, Exponent(stat.top), factor, coefficient, a.in_phase, kept_at, kept);
        } else {
            row_zero<T, THREADS>(out, vocab, share);
        }
    }
    if (MODE != kGrad && LOSS == kPolicy && a.counter && share.first()) {
        // The block that finishes last adds the terms of all rows.
        if (threadIdx.x == 0) {
            __threadfence();
            shared_last = atomicAdd(a.counter, 1u) == gridDim.x / share.size - 1;
            __threadfence();
        }
        __syncthreads();
        if (shared_last) sum_terms<THREADS>(a.terms, r.batch * r.length, a.loss);
    }
}

__global__ void __launch_bounds__(1024) policy_sum_kernel(const float* terms, int64_t rows, float* loss) {
    wait_for_previous();
    sum_terms<1024>(terms, rows, loss);
}

// What one counted token of every sequence weighs in the loss, from the mask alone, and the finish counter at zero.
__global__ void __launch_bounds__(1024) policy_weights_kernel(tk_token_rows r, int average, unsigned* counter, float* weights) {
    __shared__ long long shared_total;
    let_next_start();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        shared_total = 0;
        *counter = 0;
    }
    __syncthreads();
    for (int64_t b = warp; b < r.batch; b += 32) {
        int64_t count = 0;
        for (int64_t t = lane; t < r.length; t += 32) count += counts(r, b, t);
#pragma unroll
        for (int step = 16; step; step >>= 1) count += __shfl_xor_sync(~0u, count, step);
        if (lane == 0) {
            if (average == TK_AVERAGE_SEQUENCES) weights[b] = 1.f / (static_cast<float>(count > 0 ? count : 1) * static_cast<float>(r.batch));
            else atomicAdd(reinterpret_cast<unsigned long long*>(&shared_total), static_cast<unsigned long long>(count));
        }
    }
    if (average == TK_AVERAGE_SEQUENCES) return;
    __syncthreads();
    const float weight = 1.f / static_cast<float>(shared_total > 0 ? shared_total : 1);
    for (int64_t b = threadIdx.x; b < r.batch; b += 1024) weights[b] = weight;
}

// One block per pair: both sums of log-probabilities, the pair's loss and slope; the last block averages the losses.
__global__ void __launch_bounds__(256) preference_pairs_kernel(int64_t pairs, int64_t length, const float* logprobs, const float* reference,
                                                               int64_t reference_stride, float beta, float smoothing, float* sums,
                                                               float* coefficients, unsigned* counter, float* terms, float* loss) {
    __shared__ double parts[2][8];
    __shared__ bool shared_last;
    wait_for_previous();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t pair = blockIdx.x;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        double sum = 0.0;
        const float* from = logprobs + (pair + side * pairs) * length;
        for (int64_t t = threadIdx.x; t < length; t += 256) sum += from[t];
#pragma unroll
        for (int step = 16; step; step >>= 1) sum += __shfl_xor_sync(~0u, sum, step);
        if (lane == 0) parts[side][warp] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double both[2];
        for (int side = 0; side < 2; ++side) {
            both[side] = 0.0;
            for (int i = 0; i < 8; ++i) both[side] += parts[side][i];
            sums[pair + side * pairs] = static_cast<float>(both[side]);
        }
        // The differences cancel: they are formed from the FP64 sums.
        const float z = static_cast<float>(beta * ((both[0] - reference[pair * reference_stride])
                                                   - (both[1] - reference[(pair + pairs) * reference_stride])));
        const float tail = log1pf(expf(-fabsf(z)));
        // A weight of 0 drops its term: z is infinite where one sequence has a token of probability 0.
        const float term = (smoothing < 1.f ? (1.f - smoothing) * (fmaxf(-z, 0.f) + tail) : 0.f) + (smoothing > 0.f ? smoothing * (fmaxf(z, 0.f) + tail) : 0.f);
        const float up = 1.f / (1.f + expf(-z)), down = 1.f / (1.f + expf(z));
        const float slope = beta / static_cast<float>(pairs) * (smoothing * up - (1.f - smoothing) * down);
        // fmaxf drops NaN; a pair that has one must show it
        terms[pair] = z != z ? z : term;
        coefficients[pair] = slope;
        coefficients[pair + pairs] = -slope;
        __threadfence();
        shared_last = atomicAdd(counter, 1u) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    if (!shared_last) return;
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < pairs; i += 256) sum += __ldcg(terms + i);
#pragma unroll
    for (int step = 16; step; step >>= 1) sum += __shfl_xor_sync(~0u, sum, step);
    if (lane == 0) parts[0][warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int i = 0; i < 8; ++i) sum += parts[0][i];
        *loss = static_cast<float>(sum / static_cast<double>(pairs));
    }
}

// `early`: the kernel may start while the previous one of this call runs; it waits for it itself.
template <typename... A>
int launch_clusters(void (*kernel)(A...), int64_t grid, int cluster, int threads, size_t shared, bool early, cudaStream_t stream, A... arguments) {
    cudaLaunchAttribute attributes[2] = {};
    int count = 0;
    if (early) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = static_cast<unsigned>(cluster);
        attributes[count].val.clusterDim.y = attributes[count].val.clusterDim.z = 1;
        ++count;
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = static_cast<unsigned>(count);
    count_launch();
    return check(cudaLaunchKernelEx(&config, kernel, arguments...), "launching a token kernel");
}

template <typename... A>
int launch(void (*kernel)(A...), int64_t grid, int threads, size_t shared, bool early, cudaStream_t stream, A... arguments) {
    return launch_clusters(kernel, grid, 1, threads, shared, early, stream, arguments...);
}

constexpr int kKeptVectors = 2 * kAhead * 640;             // 80 KB

// How many threads share a row, and so how many rows are in flight.  More, smaller blocks hide one another's joins until
// registers run out: a policy loss of 16384 x 8000 BF16 logits with gradient takes 104 us with 18 blocks of 96 threads on an
// SM, 115 with 24 of 64, 120 with 16 of 128, 151 with 8 of 256; 8000 rows of 62 KB take 174 us with 6 blocks of 256 threads,
// 178 with 5, 183 with 4, 190 with 8 of 192, 199 with 3 of 512.  (The form with given weights holds more across its loops
// and spills in these shapes: 110 and 189 us.)  For long rows the second read has to find the row in L2, so few rows may be
// in flight: 4096 rows of 250 KB take 366 us with 2 blocks of 640 threads that keep the first 80 KB of their row in shared
// memory; before L2 was asked ahead 394, 417 without keeping, 444 with 3 blocks of 512.  The statistics alone take 110 us of
// 8000 x 32000 and 349 of 8192 x 128256 BF16 logits with 3 blocks of 512 threads; 6 of 256 take 89 and 323, 8 of 256 88 and 314.
// Short rows that all run at once get more threads each (256 x 1000 FP32 with gradient, captured: 6.7 us with 256 threads;
// when it was 7.0, 7.2 with 128 and 8.7 with 96).
template <typename T, Mode MODE, Loss LOSS>
int launch_type(const Args& given, int device, bool early, cudaStream_t stream) {
    Args a = given;
    const int64_t bytes = a.rows.vocab * static_cast<int64_t>(sizeof(T)), grid = a.rows.batch * a.rows.length;
    // Fewer rows than multiprocessors: clusters of blocks split them, as long as a block has 8 KB to read.
    const int sms = tk_ops::sm_count(device);
    int shares = 1;
    while (shares < kMostShares && grid * shares * 2 <= sms && bytes / (shares * 2) >= 8 * 1024) shares *= 2;
    if (shares > 1) {
        a.first_rows = grid;
        return launch_clusters(token_rows_kernel<T, MODE, LOSS, 256, 2, true>, grid * shares, shares, 256, 0, early, stream, a, 0);
    }
    // With `blocks` of them resident on a multiprocessor.
    const auto rows = [&](auto kernel, int threads, int blocks, int kept) {
        a.first_rows = static_cast<int64_t>(blocks) * sms;
        return launch(kernel, grid, threads, static_cast<size_t>(kept) * 16, early, stream, a, kept);
    };
    if (bytes <= 16 * 1024 && grid > 4 * sms) return rows(token_rows_kernel<T, MODE, LOSS, 96, 18, false>, 96, 18, 0);
    if constexpr (MODE != kBoth) {
        if (bytes > 16 * 1024) return rows(token_rows_kernel<T, MODE, LOSS, 512, 3, false>, 512, 3, 0);
    } else if (bytes > 80 * 1024 && a.in_phase) {
        auto kernel = token_rows_kernel<T, MODE, LOSS, 640, 2, false>;
        static std::atomic<bool> sized[64];
        if (device >= 64 || !sized[device].load(std::memory_order_relaxed)) {
            if (int code = check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeptVectors * 16), "sizing shared memory")) return code;
            if (device < 64) sized[device].store(true, std::memory_order_relaxed);
        }
        return rows(kernel, 640, 2, kKeptVectors);
    }
    return rows(token_rows_kernel<T, MODE, LOSS, 256, 6, false>, 256, 6, 0);
}

template <Mode MODE, Loss LOSS>
int launch_rows(const Args& a, int device, bool early, cudaStream_t stream) {
    switch (a.rows.dtype) {
        case TK_F32: return launch_type<float, MODE, LOSS>(a, device, early, stream);
        case TK_F16: return launch_type<__half, MODE, LOSS>(a, device, early, stream);
        default: return launch_type<__nv_bfloat16, MODE, LOSS>(a, device, early, stream);
    }
}

int check_rows(const tk_token_rows* r, const char* who) {
    if (!r || !r->logits || !r->targets.data || r->batch < 1 || r->length < 1 || r->vocab < 1 || r->batch > 0x7fffffff / r->length
        || r->vocab > 0x7ffffff0 || r->dtype < TK_F32 || r->dtype > TK_BF16 || (r->target_bytes != 4 && r->target_bytes != 8))
        return fail(TK_E_ARGUMENT, "trainkernel: invalid rows passed to %s", who);
    return 0;
}

Args arguments(const tk_token_rows* rows, const tk_token_grad* grad) {
    Args a{};
    a.rows = *rows;
    if (grad && grad->data) {
        a.grad = *grad;
        const int64_t bytes = rows->dtype == TK_F32 ? 4 : 2;
        const auto apart = [&](int64_t x, int64_t y) { return (x - y) * bytes % 16 != 0; };
        a.in_phase = (reinterpret_cast<uintptr_t>(rows->logits) - reinterpret_cast<uintptr_t>(grad->data)) % 16 == 0
                     && (rows->batch == 1 || !apart(rows->stride_batch, grad->stride_batch))
                     && (rows->length == 1 || !apart(rows->stride_token, grad->stride_token));
    }
    return a;
}

size_t padded(size_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

extern "C" int tk_token_logprobs(const tk_token_rows* rows, float* logprobs, float* stats, int device, void* stream) {
    if (int code = check_rows(rows, "tk_token_logprobs")) return code;
    DeviceScope scope(device);
    if (scope.status) return scope.status;
    Args a = arguments(rows, nullptr);
    a.logprobs = logprobs;
    a.stats = stats;
    return launch_rows<kStats, kWeights>(a, device, false, static_cast<cudaStream_t>(stream));
}

extern "C" int tk_token_logprobs_and_grad(const tk_token_rows* rows, const tk_token_array* weights, float* logprobs,
                                          const tk_token_grad* grad, int device, void* stream) {
    if (int code = check_rows(rows, "tk_token_logprobs_and_grad")) return code;
    if (!weights || !weights->data || !logprobs || !grad || !grad->data)
        return fail(TK_E_ARGUMENT, "trainkernel: invalid argument to tk_token_logprobs_and_grad");
    DeviceScope scope(device);
    if (scope.status) return scope.status;
    Args a = arguments(rows, grad);
    a.coefficients = *weights;
    a.logprobs = logprobs;
    return launch_rows<kBoth, kWeights>(a, device, false, static_cast<cudaStream_t>(stream));
}

extern "C" int tk_token_logits_grad(const tk_token_rows* rows, const tk_token_array* coefficients, const float* stats,
                                    const tk_token_grad* grad, int device, void* stream) {
    if (int code = check_rows(rows, "tk_token_logits_grad")) return code;
    if (!coefficients || !coefficients->data || !stats || !grad || !grad->data)
        return fail(TK_E_ARGUMENT, "trainkernel: invalid argument to tk_token_logits_grad");
    DeviceScope scope(device);
    if (scope.status) return scope.status;
    Args a = arguments(rows, grad);
    a.coefficients = *coefficients;
    a.stats = const_cast<float*>(stats);
    return launch_rows<kGrad, kWeights>(a, device, false, static_cast<cudaStream_t>(stream));
}

extern "C" size_t tk_policy_workspace_bytes(int64_t batch, int64_t length) {
    if (batch < 1 || length < 1) return 0;
    return 16 + padded(4 * static_cast<size_t>(batch)) + padded(4 * static_cast<size_t>(batch) * static_cast<size_t>(length));
}

extern "C" int tk_policy_loss(const tk_token_rows* rows, const tk_policy_terms* terms, float* loss, float* logprobs, float* stats,
                              float* coefficients, const tk_token_grad* grad, void* workspace, int device, void* stream) {
    if (int code = check_rows(rows, "tk_policy_loss")) return code;
    if (!terms || !terms->old_logprobs.data || !terms->advantages.data || !loss || !logprobs || !workspace
        || (terms->average != TK_AVERAGE_TOKENS && terms->average != TK_AVERAGE_SEQUENCES))
        return fail(TK_E_ARGUMENT, "trainkernel: invalid argument to tk_policy_loss");
    DeviceScope scope(device);
    if (scope.status) return scope.status;
    Args a = arguments(rows, grad);
    a.policy = *terms;
    if (terms->kl_weight == 0.f) a.policy.ref_logprobs.data = nullptr;      // no term: 0 times an exponential that overflows is not 0
    a.logprobs = logprobs;
    a.stats = stats;
    a.row_coefficients = coefficients;
    a.loss = loss;
    char* at = static_cast<char*>(workspace);
    a.counter = reinterpret_cast<unsigned*>(at);
    a.weights = reinterpret_cast<float*>(at + 16);
    a.terms = reinterpret_cast<float*>(at + 16 + padded(4 * static_cast<size_t>(rows->batch)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (int code = launch(policy_weights_kernel, 1, 1024, 0, false, s, *rows, static_cast<int>(terms->average), a.counter, a.weights)) return code;
    // A few rows: their last block adds the terms, which saves a launch.  Many rows: every block would wait for its
    // answer from the counter, and a launch of its own is cheaper.
    const int64_t count = rows->batch * rows->length;
    const bool apart = count > 1024;
    if (apart) a.counter = nullptr;
    if (int code = a.grad.data ? launch_rows<kBoth, kPolicy>(a, device, true, s) : launch_rows<kStats, kPolicy>(a, device, true, s)) return code;
    if (!apart) return 0;
    return launch(policy_sum_kernel, 1, 1024, 0, true, s, static_cast<const float*>(a.terms), count, loss);
}

extern "C" size_t tk_preference_workspace_bytes(int64_t batch, int64_t length) {
    if (batch < 1 || length < 1) return 0;
    return 16 + padded(4 * static_cast<size_t>(batch)) + padded(4 * static_cast<size_t>(batch) * static_cast<size_t>(length));
}

extern "C" int tk_preference_loss(const tk_token_rows* rows, const float* reference, int64_t reference_stride, float beta,
                                  float label_smoothing, float* loss, float* sums, float* stats, float* coefficients,
                                  const tk_token_grad* grad, void* workspace, int device, void* stream) {
    if (int code = check_rows(rows, "tk_preference_loss")) return code;
    if (!reference || !loss || !sums || !stats || !coefficients || !workspace || rows->batch % 2)
        return fail(TK_E_ARGUMENT, "trainkernel: invalid argument to tk_preference_loss");
    DeviceScope scope(device);
    if (scope.status) return scope.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    char* at = static_cast<char*>(workspace);
    unsigned* counter = reinterpret_cast<unsigned*>(at);
    float* terms = reinterpret_cast<float*>(at + 16);
    float* logprobs = reinterpret_cast<float*>(at + 16 + padded(4 * static_cast<size_t>(rows->batch)));
    Args a = arguments(rows, nullptr);
    a.logprobs = logprobs;
    a.stats = stats;
    a.clear = counter;
    if (int code = launch_rows<kStats, kWeights>(a, device, false, s)) return code;
    const int64_t pairs = rows->batch / 2;
    if (int code = launch(preference_pairs_kernel, pairs, 256, 0, true, s, pairs, rows->length, static_cast<const float*>(logprobs), reference,
                          reference_stride, beta, label_smoothing, sums, coefficients, counter, terms, loss)) return code;
    if (!grad || !grad->data) return 0;
    Args g = arguments(rows, grad);
    g.stats = stats;
    g.coefficients = {coefficients, 1, 0};
    return launch_rows<kGrad, kWeights>(g, device, true, s);
}
