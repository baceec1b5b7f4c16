// Log-probabilities of tokens from rows of logits, the gradient of the logits, and the losses built on them.
//
// Mathematics.  For a row x of V logits and its token t, with m = max x and S = sum_j exp(x_j - m):
//     logprob = (x_t - m) - log S,     d logprob / d x_j = [j = t] - exp(x_j - m) / S.
// Every loss here is a function of the log-probabilities, so its gradient is a coefficient per row times that row.
// (m, S) pairs of parts of a row join associatively: M = max(m1, m2), S = S1 exp(m1 - M) + S2 exp(m2 - M), so one
// pass over the row gives both.  m is kept as a logit that occurs (never below the lowest finite FP32 number) and
// subtracted before anything is scaled: logits of the type's lowest value and -inf then need no special case, and
// the differences near the maximum are exact.  All statistics, coefficients and sums are FP32 or wider; the only
// rounding to 16 bits is the gradient's, once, at its store.
#include "tk_ops_host.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace {

using tk_ops::check;
using tk_ops::count_launch;
using tk_ops::DeviceScope;
using tk_ops::fail;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
constexpr int kThreads = 512;

// 2^x by the hardware's approximation (relative error about 2^-22).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

struct Stat {
    float top, sum;
};

__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float top = fmaxf(a.top, b.top);
    return {top, a.sum * exp2_fast((a.top - top) * kLog2e) + b.sum * exp2_fast((b.top - top) * kLog2e)};
}

enum Mode { kStats, kGrad, kBoth };            // log-probabilities / gradient from saved stats / both
enum Loss { kWeights, kPolicy };               // where kBoth takes the coefficient from, and what kStats adds

struct Args {
    tk_token_rows rows;
    tk_token_array coefficients;               // kGrad and kBoth with kWeights: FP32 [batch, length]
    tk_policy_terms policy;
    float* logprobs;
    float* stats;
    float* row_coefficients;                   // kPolicy: dense d loss / d logprob, or NULL
    void* grad;
    const float* scale_at;
    float scale;
    // kPolicy: workspace
    unsigned* counter;
    float* weights;                            // one per sequence
    float* terms;                              // one per row
    float* loss;
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

__device__ Stat block_join(Stat mine, Stat* shared) {
#pragma unroll
    for (int step = 16; step; step >>= 1)
        mine = join(mine, {__shfl_xor_sync(~0u, mine.top, step), __shfl_xor_sync(~0u, mine.sum, step)});
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (lane == 0) shared[warp] = mine;
    __syncthreads();
    mine = lane < kThreads / 32 ? shared[lane] : Stat{kLowest, 0.f};
#pragma unroll
    for (int step = 16; step; step >>= 1)
        mine = join(mine, {__shfl_xor_sync(~0u, mine.top, step), __shfl_xor_sync(~0u, mine.sum, step)});
    return mine;
}

// The loss of one token and its slope in the log-probability.
__device__ __forceinline__ void policy_token(const tk_policy_terms& p, int64_t b, int64_t t, float logprob, float* term, float* slope) {
    const float advantage = at(p.advantages, b, t);
    const float ratio = expf(logprob - at(p.old_logprobs, b, t));
    const float free = ratio * advantage;
    const float bound = fminf(fmaxf(ratio, 1.f - p.clip_low), 1.f + p.clip_high) * advantage;
    const bool clipped = free > bound;                    // false for NaN: it then stays in the result
    *term = clipped ? -bound : -free;
    *slope = clipped ? 0.f : -free;
    if (p.ref_logprobs.data) {
        const float away = at(p.ref_logprobs, b, t) - logprob, grown = expm1f(away);
        *term += p.kl_weight * (grown - away);
        *slope -= p.kl_weight * grown;
    }
}

template <typename T, Mode MODE, Loss LOSS>
__global__ void __launch_bounds__(kThreads) token_rows_kernel(const __grid_constant__ Args a) {
    __shared__ Stat shared[32];
    __shared__ float shared_coefficient;
    __shared__ bool shared_last;
    const tk_token_rows& r = a.rows;
    const int64_t row = blockIdx.x, b = row / r.length, t = row % r.length;
    const T* x = static_cast<const T*>(r.logits) + b * r.stride_batch + t * r.stride_token;
    T* out = static_cast<T*>(a.grad) + row * r.vocab;
    const bool keep = counts(r, b, t);
    const int64_t vocab = r.vocab;
    float coefficient = 0.f, scale = 0.f;
    Stat stat{kLowest, 0.f};
    int64_t target = -1;
    if (a.clear && row == 0 && threadIdx.x == 0) *a.clear = 0;
    if (keep) target = target_of(r, b, t);
    if (MODE != kGrad && keep) {
        for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
            const float value = to_float(x[j]);
            if (value > stat.top) {
                stat.sum *= exp2_fast((stat.top - value) * kLog2e);
                stat.top = value;
            }
            stat.sum += exp2_fast((value - stat.top) * kLog2e);
        }
        stat = block_join(stat, shared);
    }
    if (MODE != kGrad && threadIdx.x == 0) {
        float logprob = 0.f;
        if (keep) logprob = target >= 0 && target < vocab ? to_float(x[target]) - stat.top - logf(stat.sum) : __int_as_float(0x7fffffff);
        if (a.logprobs) a.logprobs[row] = logprob;
        if (a.stats) {
            a.stats[2 * row] = stat.top;
            a.stats[2 * row + 1] = stat.sum;
        }
        if (LOSS == kPolicy) {
            float term = 0.f, slope = 0.f;
            if (keep) {
                policy_token(a.policy, b, t, logprob, &term, &slope);
                const float weight = a.weights[b];
                term *= weight;
                slope *= weight;
            }
            a.terms[row] = term;
            if (a.row_coefficients) a.row_coefficients[row] = slope;
            shared_coefficient = slope;
        }
    }
    if (MODE != kStats) {
        if (keep) {
            scale = a.scale_at ? a.scale * *a.scale_at : a.scale;
            if (LOSS == kPolicy) {
                __syncthreads();
                coefficient = shared_coefficient * scale;
            } else {
                coefficient = at(a.coefficients, b, t) * scale;
            }
            if (MODE == kGrad) stat = {a.stats[2 * row], a.stats[2 * row + 1]};
            const bool known = target >= 0 && target < vocab;
            const float factor = known ? -coefficient / stat.sum : __int_as_float(0x7fffffff);
            for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
                float value = exp2_fast((to_float(x[j]) - stat.top) * kLog2e) * factor;
                if (j == target) value += coefficient;
                out[j] = from_float<T>(value);
            }
        } else {
            for (int64_t j = threadIdx.x; j < vocab; j += kThreads) out[j] = from_float<T>(0.f);
        }
    }
    if (MODE != kGrad && LOSS == kPolicy) {
        // The block that finishes last adds the terms of all rows, in an order that does not depend on who that is.
        if (threadIdx.x == 0) {
            __threadfence();
            shared_last = atomicAdd(a.counter, 1u) == gridDim.x - 1;
            __threadfence();
        }
        __syncthreads();
        if (shared_last) {
            __shared__ double parts[kThreads];
            double sum = 0.0;
            const int64_t rows = r.batch * r.length;
            for (int64_t i = threadIdx.x; i < rows; i += kThreads) sum += __ldcg(a.terms + i);
            parts[threadIdx.x] = sum;
            __syncthreads();
            for (int step = kThreads / 2; step; step >>= 1) {
                if (threadIdx.x < step) parts[threadIdx.x] += parts[threadIdx.x + step];
                __syncthreads();
            }
            if (threadIdx.x == 0) *a.loss = static_cast<float>(parts[0]);
        }
    }
}

// What one counted token of every sequence weighs in the loss, from the mask alone, and the finish counter at zero.
__global__ void __launch_bounds__(1024) policy_weights_kernel(tk_token_rows r, int average, unsigned* counter, float* weights) {
    __shared__ long long shared_total;
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
        const float term = (1.f - smoothing) * (fmaxf(-z, 0.f) + tail) + smoothing * (fmaxf(z, 0.f) + tail);
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

template <Mode MODE, Loss LOSS>
int launch_rows(const Args& a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.rows.batch * a.rows.length);
    switch (a.rows.dtype) {
        case TK_F32: token_rows_kernel<float, MODE, LOSS><<<grid, kThreads, 0, stream>>>(a); break;
        case TK_F16: token_rows_kernel<__half, MODE, LOSS><<<grid, kThreads, 0, stream>>>(a); break;
        default: token_rows_kernel<__nv_bfloat16, MODE, LOSS><<<grid, kThreads, 0, stream>>>(a); break;
    }
    count_launch();
    return check(cudaGetLastError(), "launching the token kernel");
}

int check_rows(const tk_token_rows* r, const char* who) {
    if (!r || !r->logits || !r->targets.data || r->batch < 1 || r->length < 1 || r->vocab < 1 || r->batch > 0x7fffffff / r->length
        || r->vocab > 0x7fffffff || r->dtype < TK_F32 || r->dtype > TK_BF16 || (r->target_bytes != 4 && r->target_bytes != 8))
        return fail(TK_E_ARGUMENT, "trainkernel: invalid rows passed to %s", who);
    return 0;
}

Args arguments(const tk_token_rows* rows, const tk_token_grad* grad) {
    Args a{};
    a.rows = *rows;
    a.scale = 1.f;
    if (grad) {
        a.grad = grad->data;
        a.scale_at = grad->scale_at;
        a.scale = grad->scale;
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
    return launch_rows<kStats, kWeights>(a, static_cast<cudaStream_t>(stream));
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
    return launch_rows<kBoth, kWeights>(a, static_cast<cudaStream_t>(stream));
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
    return launch_rows<kGrad, kWeights>(a, static_cast<cudaStream_t>(stream));
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
    a.logprobs = logprobs;
    a.stats = stats;
    a.row_coefficients = coefficients;
    a.loss = loss;
    char* at = static_cast<char*>(workspace);
    a.counter = reinterpret_cast<unsigned*>(at);
    a.weights = reinterpret_cast<float*>(at + 16);
    a.terms = reinterpret_cast<float*>(at + 16 + padded(4 * static_cast<size_t>(rows->batch)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    policy_weights_kernel<<<1, 1024, 0, s>>>(*rows, terms->average, a.counter, a.weights);
    count_launch();
    if (int code = check(cudaGetLastError(), "launching the weight kernel")) return code;
    return a.grad ? launch_rows<kBoth, kPolicy>(a, s) : launch_rows<kStats, kPolicy>(a, s);
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
    if (int code = launch_rows<kStats, kWeights>(a, s)) return code;
    const int64_t pairs = rows->batch / 2;
    preference_pairs_kernel<<<static_cast<unsigned>(pairs), 256, 0, s>>>(pairs, rows->length, logprobs, reference, reference_stride, beta,
                                                                         label_smoothing, sums, coefficients, counter, terms, loss);
    count_launch();
    if (int code = check(cudaGetLastError(), "launching the pair kernel")) return code;
    if (!grad || !grad->data) return 0;
    Args g = arguments(rows, grad);
    g.stats = stats;
    g.coefficients = {coefficients, 1, 0};
    return launch_rows<kGrad, kWeights>(g, s);
}
