// AdamW over many tensors in one launch, moments in 32 or in 8 bits.
//
// Mathematics, per element, with t steps taken including this one:
//     m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2,
//     p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps).
// In 8 bits a block of 256 elements shares one FP32 scale per moment, m is held as e4m3 times its scale, and of v the
// square root, which needs half the exponent range.  Rounding to nearest would stop both moments: with b2 = 0.999 a root
// moves by at most 0.05 % a step towards zero, and the nearest e4m3 number is up to 6 % away, so the code would never
// change.  Both are rounded up with the probability of the part that is cut (the expected value is the unrounded one); the
// 16 random bits come from a hash of the element's place and the step, so a run repeats exactly.  A root above zero is
// never rounded to zero, which would divide by eps alone.  The update itself uses the unrounded moments.  The products and
// sums of the moments, their scales and the scaled values are rounded one by one (no fused multiply-add): which way a value
// on a border is rounded then follows from the formulas alone, in whatever form they are compiled.
#include "tk_ops_host.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

namespace {

using tk_ops::check;
using tk_ops::count_launch;
using tk_ops::DeviceScope;
using tk_ops::fail;

constexpr int kThreads = 256;
constexpr int kPerThread = 8;
constexpr int kChunk = kThreads * kPerThread;     // elements one block updates at a time: 8 scale blocks, one per warp
constexpr int kFew = 64, kMany = 768;             // tensors in one launch's parameter block (at most 32,764 bytes)
constexpr float kE4m3Max = 448.f;
constexpr float kSmallest = 7.888609052e-31f;      // 2^-100: a block whose largest value is below it is held as zeros (448 / value stays finite)

struct Item {
    void* param;
    const void* grad;
    int64_t offset, count;
    int32_t first_chunk;
    float weight_decay;
};

template <int CAPACITY>
struct Args {
    tk_adamw_state state;
    const float *lr_at, *scale_at;
    double log_beta1, log_beta2;
    float lr, beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
    uint32_t seed;
    int32_t count, chunks, last;
    Item items[CAPACITY];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// A 32-bit mixing function of two multiplications (xor-shift-multiply, constants from C. Wellons' published search for
// low-bias hashes, https://nullprogram.com/blog/2018/07/31/).
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ (x >> 16);
}

// Two FP32 numbers in one 64-bit register: the paired instructions round each exactly as the single ones do.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// Hardware approximation, 1 ulp; the divisor is at least eps, which the entry point keeps among the normal numbers.
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float least(float a, float b) {   // NaN if either is
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Eight values on one of the two e4m3 numbers around each: the larger one when the cut part exceeds its 16 random bits.
// From 2^-6 up an e4m3 number is an FP32 number without its last 20 bits, so adding the random bits above the last four
// and cutting does it, whatever the sign (a value two units in the last place above 448 still ends on 448: the sum
// carries only from sixteen on).  Below, they are multiples of 2^-9; that form is needed by few warps (a value 3e-5 of its
// block's largest), so the warp asks once whether anybody needs it.  NaN takes it and stays NaN.  ROOT: a value
// that stands for a number above zero (`above`) is not rounded to zero.
template <bool ROOT>
__device__ __forceinline__ void round8(float (&x)[8], const uint32_t (&random)[8], const float (&above)[8]) {
    float smallest = kE4m3Max;
#pragma unroll
    for (int i = 0; i < 8; ++i) smallest = least(smallest, fabsf(x[i]));
    const bool any_small = __any_sync(~0u, !(smallest >= 0.015625f));
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t dither = ROOT ? random[i] >> 16 : random[i] & 0xffffu;
        q[i] = __uint_as_float((__float_as_uint(x[i]) + (dither << 4)) & 0xfff00000u);
    }
    if (any_small) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t dither = ROOT ? random[i] >> 16 : random[i] & 0xffffu;
            const float a = least(fabsf(x[i]), kE4m3Max), part = __uint_as_float(0x3f800000u | (dither << 7)) - 1.f;    // dither / 2^16
            float whole = __fadd_rd(fmaf(a, 512.f, part), 8388608.f) - 8388608.f;                                       // rounded down: at most 9
            if (ROOT && above[i] > 0.f && whole < 1.f) whole = 1.f;
            if (!(a >= 0.015625f)) q[i] = copysignf(whole * (1.f / 512.f), x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = q[i];
}

template <typename T> __device__ __forceinline__ void load8(float (&to)[8], const T* from, int64_t left, bool wide) {
    if (wide && left >= 8) {
        constexpr int kVectors = 8 * sizeof(T) / 16;
        union { uint4 vector[kVectors]; T element[8]; } u;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) u.vector[i] = __ldcs(reinterpret_cast<const uint4*>(from) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = to_float(u.element[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = i < left ? to_float(from[i]) : 0.f;
    }
}

template <typename T> __device__ __forceinline__ void store8(T* to, const float (&from)[8], int64_t left, bool wide) {
    if (wide && left >= 8) {
        constexpr int kVectors = 8 * sizeof(T) / 16;
        union { uint4 vector[kVectors]; T element[8]; } u;
#pragma unroll
        for (int i = 0; i < 8; ++i) u.element[i] = from_float<T>(from[i]);
#pragma unroll
        for (int i = 0; i < kVectors; ++i) __stcs(reinterpret_cast<uint4*>(to) + i, u.vector[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) to[i] = from_float<T>(from[i]);
    }
}

__device__ __forceinline__ void decode8(float (&to)[8], uint2 codes, float scale) {
    const Pair scales = pair(scale, scale);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t two = (i < 4 ? codes.x : codes.y) >> (8 * (i % 4));
        const __half2_raw halves = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
        const float2 values = __half22float2(__half2(halves));
        split(mul2(pair(values.x, values.y), scales), to[i], to[i + 1]);
    }
}

__device__ __forceinline__ uint2 encode8(const float (&from)[8]) {
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(from[i], from[i + 1]), __NV_SATFINITE, __NV_E4M3);
        word[i / 4] |= two << (8 * (i % 4));
    }
    return make_uint2(word[0], word[1]);
}

// The largest of 32 non-negative numbers: their bit patterns have their order.
__device__ __forceinline__ float warp_max(float x) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(x))); }

struct Numbers {
    Pair beta1, beta2, rest1, rest2, scale, spread, eps, pace;
    uint32_t salt;
};

// One thread's eight elements: FULL when they, and the whole block of 256 around them, lie inside the tensor and on
// 16-byte boundaries.  Otherwise lanes behind the tensor's end stay in the warp for the block maximum, with zeros.
template <typename P, typename G, int BITS, bool FULL>
__device__ __forceinline__ void update8(const tk_adamw_state& state, const Item& item, const Numbers& n, float decay, int64_t at, int64_t left) {
    const int64_t flat = item.offset + at;
    P* param = static_cast<P*>(item.param) + at;
    const G* grad = static_cast<const G*>(item.grad) + at;
    const bool wide_param = FULL || reinterpret_cast<uintptr_t>(item.param) % 16 == 0;
    const bool wide_grad = FULL || reinterpret_cast<uintptr_t>(item.grad) % 16 == 0;
    const int64_t inside = FULL ? 8 : left;
    const bool in_block = FULL || left + (threadIdx.x % 32) * kPerThread > 0;
    float p[8], g[8], m[8] = {}, v[8] = {};
    float mean_scale = 0.f, root_scale = 0.f;
    uint2 mean_codes = make_uint2(0, 0), root_codes = make_uint2(0, 0);
    const int64_t block = flat / TK_ADAMW_BLOCK;
    if (BITS == 8) {
        if (in_block) {
            mean_scale = state.mean_scale[block];
            root_scale = state.root_scale[block];
            mean_codes = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(state.mean) + flat));
            root_codes = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(state.square) + flat));
        }
    } else if (FULL || left > 0) {
        // the flat state is padded to whole blocks, so it is always read and written whole
        load8<float>(m, static_cast<const float*>(state.mean) + flat, 8, true);
        load8<float>(v, static_cast<const float*>(state.square) + flat, 8, true);
    }
    load8<P>(p, param, inside, wide_param);
    load8<G>(g, grad, inside, wide_grad);
    if (BITS == 8) {
        decode8(m, mean_codes, mean_scale);
        decode8(v, root_codes, root_scale);
    }
    float top_mean = 0.f, top_root = 0.f;
    const Pair decays = pair(decay, decay);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const Pair gradient = mul2(pair(g[i], g[i + 1]), n.scale);
        Pair square = pair(v[i], v[i + 1]);
        if (BITS == 8) square = mul2(square, square);
        float a, b, c, d;
        const Pair kept1 = mul2(n.beta1, pair(m[i], m[i + 1])), new1 = mul2(n.rest1, gradient);
        const Pair kept2 = mul2(n.beta2, square), new2 = mul2(mul2(n.rest2, gradient), gradient);
        split(kept1, a, b);
        split(new1, c, d);
        m[i] = __fadd_rn(a, c);                              // single additions: paired ones are fused with the products
        m[i + 1] = __fadd_rn(b, d);
        split(kept2, a, b);
        split(new2, c, d);
        v[i] = __fadd_rn(a, c);
        v[i + 1] = __fadd_rn(b, d);
        const Pair mean = pair(m[i], m[i + 1]);
        a = sqrtf(v[i]);
        b = sqrtf(v[i + 1]);
        split(fma2(pair(a, b), n.spread, n.eps), c, d);
        // p decay - pace m / (sqrt(v) spread + eps); n.pace is negative
        const Pair change = mul2(mul2(n.pace, mean), pair(reciprocal(c), reciprocal(d)));
        split(fma2(pair(p[i], p[i + 1]), decays, change), p[i], p[i + 1]);
        if (BITS == 8) {
            v[i] = a;
            v[i + 1] = b;
            if (FULL || i < inside) top_mean = fmaxf(top_mean, fabsf(m[i])), top_root = fmaxf(top_root, a);
            if (FULL || i + 1 < inside) top_mean = fmaxf(top_mean, fabsf(m[i + 1])), top_root = fmaxf(top_root, b);
        }
    }
    store8<P>(param, p, inside, wide_param);
    if (BITS == 8) {
        top_mean = warp_max(top_mean);
        top_root = warp_max(top_root);
        const float mean_factor = top_mean >= kSmallest ? __fmul_rn(__frcp_rn(top_mean), kE4m3Max) : 0.f;
        const float root_factor = top_root >= kSmallest ? __fmul_rn(__frcp_rn(top_root), kE4m3Max) : 0.f;
        const Pair mean_factors = pair(mean_factor, mean_factor), root_factors = pair(root_factor, root_factor);
        uint32_t random[8];
        float root[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) random[i] = mix(static_cast<uint32_t>(flat) ^ n.salt ^ i);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            split(mul2(pair(m[i], m[i + 1]), mean_factors), m[i], m[i + 1]);
            split(mul2(pair(v[i], v[i + 1]), root_factors), root[i], root[i + 1]);
        }
        round8<false>(m, random, v);
        round8<true>(root, random, v);
        if (!FULL) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= inside) m[i] = root[i] = 0.f;
        }
        if (in_block) {
            __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(state.mean) + flat), encode8(m));
            __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(state.square) + flat), encode8(root));
            if (threadIdx.x % 32 == 0) {
                state.mean_scale[block] = top_mean >= kSmallest ? __fmul_rn(top_mean, 1.f / kE4m3Max) : 0.f;
                state.root_scale[block] = top_root >= kSmallest ? __fmul_rn(top_root, 1.f / kE4m3Max) : 0.f;
            }
        }
    } else if (FULL || left > 0) {
        if (!FULL) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= inside) m[i] = v[i] = 0.f;
        }
        store8<float>(static_cast<float*>(state.mean) + flat, m, 8, true);
        store8<float>(static_cast<float*>(state.square) + flat, v, 8, true);
    }
}

template <typename P, typename G, int BITS, int CAPACITY>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ Args<CAPACITY> a) {
    const float scale = a.scale_at ? *a.scale_at : 1.f;
    if (!(fabsf(scale) <= 3.402823466e38f)) return;                    // not finite: this step does not happen
    const int64_t step = a.state.steps[blockIdx.x] + 1;
    const float lr = a.lr_at ? *a.lr_at : a.lr;
    // 1 - b^t without cancellation
    const float left1 = -expm1f(static_cast<float>(static_cast<double>(step) * a.log_beta1));
    const float left2 = -expm1f(static_cast<float>(static_cast<double>(step) * a.log_beta2));
    const float pace = lr / left1, spread = 1.f / sqrtf(left2);
    Numbers n;
    n.beta1 = pair(a.beta1, a.beta1);
    n.beta2 = pair(a.beta2, a.beta2);
    n.rest1 = pair(a.one_minus_beta1, a.one_minus_beta1);
    n.rest2 = pair(a.one_minus_beta2, a.one_minus_beta2);
    n.scale = pair(scale, scale);
    n.spread = pair(spread, spread);
    n.eps = pair(a.eps, a.eps);
    n.pace = pair(-pace, -pace);
    n.salt = mix(static_cast<uint32_t>(step) + a.seed * 0x9e3779b9u);

    // Chunks are dealt out one by one, so that blocks that run together touch neighbouring memory (contiguous runs per
    // block took 135 us where this takes 113 us: 33.5M elements, 8-bit moments, FP32 gradients).
    const int begin = blockIdx.x;
    int low = 0, high = a.count - 1;
    while (low < high) {
        const int middle = (low + high + 1) / 2;
        if (a.items[middle].first_chunk <= begin) low = middle;
        else high = middle - 1;
    }
    int which = low;
    for (int chunk = begin; chunk < a.chunks; chunk += gridDim.x) {
        while (which + 1 < a.count && a.items[which + 1].first_chunk <= chunk) ++which;
        const Item& item = a.items[which];
        const int64_t at = static_cast<int64_t>(chunk - item.first_chunk) * kChunk + threadIdx.x * kPerThread;
        const int64_t left = item.count - at;
        const float decay = 1.f - lr * item.weight_decay;
        const bool whole = item.count - static_cast<int64_t>(chunk - item.first_chunk) * kChunk >= kChunk
                           && (reinterpret_cast<uintptr_t>(item.param) | reinterpret_cast<uintptr_t>(item.grad)) % 16 == 0;
        if (whole) update8<P, G, BITS, true>(a.state, item, n, decay, at, left);
        else update8<P, G, BITS, false>(a.state, item, n, decay, at, left);
    }
    // Only this block reads the counters it advances, so no block can see another's new value.
    if (a.last)
        for (int i = blockIdx.x + gridDim.x * threadIdx.x; i < TK_ADAMW_COUNTERS; i += gridDim.x * kThreads) {
            if (i == blockIdx.x) continue;
            a.state.steps[i] = step;
        }
    __syncthreads();
    if (a.last && threadIdx.x == 0) a.state.steps[blockIdx.x] = step;
}

template <typename P, typename G, int BITS, int CAPACITY>
int launch(const tk_adamw_tensor* tensors, int count, const tk_adamw_state* state, const tk_adamw_options* o, int last, int device, cudaStream_t stream) {
    Args<CAPACITY> a;
    a.state = *state;
    a.lr_at = o->lr_at;
    a.scale_at = o->scale_at;
    a.log_beta1 = log(o->beta1);
    a.log_beta2 = log(o->beta2);
    a.lr = static_cast<float>(o->lr);
    a.beta1 = static_cast<float>(o->beta1);
    a.beta2 = static_cast<float>(o->beta2);
    a.one_minus_beta1 = static_cast<float>(1.0 - o->beta1);
    a.one_minus_beta2 = static_cast<float>(1.0 - o->beta2);
    a.eps = static_cast<float>(o->eps);
    a.seed = o->seed;
    a.count = count;
    a.last = last;
    int64_t chunks = 0;
    for (int i = 0; i < count; ++i) {
        a.items[i] = {tensors[i].param, tensors[i].grad, tensors[i].offset, tensors[i].count, static_cast<int32_t>(chunks), tensors[i].weight_decay};
        chunks += (tensors[i].count + kChunk - 1) / kChunk;
        if (chunks > 0x7fffffff) return fail(TK_E_ARGUMENT, "trainkernel: too many elements in one tk_adamw_update");
    }
    a.chunks = static_cast<int32_t>(chunks);
    // 32-bit moments are bound by memory: as many blocks as there are counters, so that the hardware evens out what they take
    // (33.5M elements: 170 us with one wave of 592 blocks, 164 with two, 157 with three, 148 with six).  8-bit moments
    // are bound by arithmetic, a block's start-up counts, and whole waves of four chunks or more a block are best (8.4M
    // elements: 24.7 us with one wave, 28.3 with a block per chunk, 30.4 with 1.2 waves; 33.5M: 101 with 2.3, 93 with seven).
    int64_t grid = chunks;
    const int64_t wave = 4 * static_cast<int64_t>(tk_ops::sm_count(device));
    if (BITS == 8 && wave > 0) {
        const int64_t waves = chunks / (4 * wave);
        grid = wave * (waves < 1 ? 1 : waves > 6 ? 6 : waves);
        if (grid > chunks) grid = chunks;
    }
    if (grid > TK_ADAMW_COUNTERS) grid = TK_ADAMW_COUNTERS;
    if (grid > chunks) grid = chunks;
    if (grid < 1) grid = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    count_launch();
    return check(cudaLaunchKernelEx(&config, adamw_kernel<P, G, BITS, CAPACITY>, a), "launching the AdamW kernel");
}

template <typename P, typename G, int BITS>
int launch_all(const tk_adamw_tensor* tensors, int count, const tk_adamw_state* state, const tk_adamw_options* o, int last, int device, cudaStream_t stream) {
    while (count > kMany) {
        if (int code = launch<P, G, BITS, kMany>(tensors, kMany, state, o, 0, device, stream)) return code;
        tensors += kMany;
        count -= kMany;
    }
    return count > kFew ? launch<P, G, BITS, kMany>(tensors, count, state, o, last, device, stream)
                        : launch<P, G, BITS, kFew>(tensors, count, state, o, last, device, stream);
}

template <typename P, typename G>
int by_bits(const tk_adamw_tensor* t, int n, const tk_adamw_state* s, const tk_adamw_options* o, int last, int device, cudaStream_t stream) {
    return o->bits == 8 ? launch_all<P, G, 8>(t, n, s, o, last, device, stream) : launch_all<P, G, 32>(t, n, s, o, last, device, stream);
}

template <typename P>
int by_grad(int dtype, const tk_adamw_tensor* t, int n, const tk_adamw_state* s, const tk_adamw_options* o, int last, int device, cudaStream_t stream) {
    switch (dtype) {
        case TK_F32: return by_bits<P, float>(t, n, s, o, last, device, stream);
        case TK_F16: return by_bits<P, __half>(t, n, s, o, last, device, stream);
        default: return by_bits<P, __nv_bfloat16>(t, n, s, o, last, device, stream);
    }
}

}  // namespace

extern "C" int tk_adamw_update(const tk_adamw_tensor* tensors, int count, int param_dtype, int grad_dtype, const tk_adamw_state* state,
                               const tk_adamw_options* options, int last, int device, void* stream) {
    if (!tensors || count < 1 || !state || !options || !state->mean || !state->square || !state->steps || param_dtype < TK_F32
        || param_dtype > TK_BF16 || grad_dtype < TK_F32 || grad_dtype > TK_BF16 || (options->bits != 8 && options->bits != 32)
        || (options->bits == 8 && (!state->mean_scale || !state->root_scale)) || !(options->beta1 >= 0 && options->beta1 < 1)
        || !(options->beta2 >= 0 && options->beta2 < 1) || !(options->eps >= 1e-30))
        return fail(TK_E_ARGUMENT, "trainkernel: invalid argument to tk_adamw_update");
    for (int i = 0; i < count; ++i)
        if (tensors[i].count < 0 || tensors[i].offset < 0 || tensors[i].offset % TK_ADAMW_BLOCK
            || (tensors[i].count && (!tensors[i].param || !tensors[i].grad)))
            return fail(TK_E_ARGUMENT, "trainkernel: invalid tensor %d passed to tk_adamw_update", i);
    DeviceScope scope(device);
    if (scope.status) return scope.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (param_dtype) {
        case TK_F32: return by_grad<float>(grad_dtype, tensors, count, state, options, last, device, s);
        case TK_F16: return by_grad<__half>(grad_dtype, tensors, count, state, options, last, device, s);
        default: return by_grad<__nv_bfloat16>(grad_dtype, tensors, count, state, options, last, device, s);
    }
}
