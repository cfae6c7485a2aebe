// Log probabilities of given tokens, the entropy and the most likely
// alternatives of rows of logits. With M = max x, c the number of logits equal
// to M, S = sum over the others of e^(x - M) and A = sum of e^(x - M) (M - x):
//   log p_t = (x_t - M) - log(c + S),   H = log(c + S) + A / (c + S).
// S leaves the largest logits out, so that log(1 + S) keeps its digits where one
// token is nearly certain; every term of H is positive.
#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

__device__ __forceinline__ float logit(const float *x, size_t i) { return x[i]; }
__device__ __forceinline__ float logit(const uint16_t *x, size_t i) { return bf16_f32(x[i]); }

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// One block a row: the maximum, the sums, then `top` times the best logit after
// the last one (larger, or equal with a larger id).
template <class T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T *x, size_t vocab, size_t stride,
                                                            const uint32_t *tokens, int top, float *logprobs,
                                                            float *entropy, uint32_t *ids, float *tops) {
    __shared__ float red[kWaves];
    __shared__ double red64[3][kWaves];
    __shared__ unsigned long long best[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    x += row * stride;
    float m = -INFINITY;
    for (size_t i = tid; i < vocab; i += kThreads) m = fmaxf(m, logit(x, i));
    m = wave_max(m);
    if (lane == 0) red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float ref = m == -INFINITY ? 0.f : m;
    double c = 0, S = 0, A = 0;
    for (size_t i = tid; i < vocab; i += kThreads) {
        const float d = logit(x, i) - ref, e = expf(d);
        if (d == 0.f) c += 1;
        else S += e;
        if (!(e == 0.f)) A -= (double)e * d;  // a NaN reaches both sums
    }
    c = wave_sum_f64(c);
    S = wave_sum_f64(S);
    A = wave_sum_f64(A);
    if (lane == 0) {
        red64[0][wave] = c;
        red64[1][wave] = S;
        red64[2][wave] = A;
    }
    __syncthreads();
    c = S = A = 0;
    for (int w = 0; w < kWaves; ++w) {
        c += red64[0][w];
        S += red64[1][w];
        A += red64[2][w];
    }
    const bool empty = m == -INFINITY && S == 0;
    const double logsum = c == 1 ? log1p(S) : log(c + S);
    auto logprob = [&](float v) { return empty ? -INFINITY : (float)((double)v - (double)m - logsum); };
    if (tid == 0) {
        if (logprobs) {
            const uint32_t t = tokens[row];
            logprobs[row] = t < vocab ? logprob(logit(x, t)) : NAN;
        }
        if (entropy) entropy[row] = empty ? 0.f : (float)(logsum + A / (c + S));
    }
    // Keys: the value in order, then the id descending.
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; ++k) {
        unsigned long long b = 0;
        for (size_t i = tid; i < vocab; i += kThreads) {
            float v = logit(x, i) + 0.f;  // -0 and 0 are equal
            if (v != v) v = -INFINITY;
            const uint32_t u = __float_as_uint(v), o = u & 0x80000000u ? ~u : u | 0x80000000u;
            const unsigned long long key = ((unsigned long long)o << 32) | (0xFFFFFFFFu - (uint32_t)i);
            if (key < last && key > b) b = key;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) b = max(b, (unsigned long long)__shfl_xor(b, off, 64));
        __syncthreads();
        if (lane == 0) best[wave] = b;
        __syncthreads();
        last = max(max(best[0], best[1]), max(best[2], best[3]));
        if (tid == 0) {
            const uint32_t id = 0xFFFFFFFFu - (uint32_t)last;
            ids[row * top + k] = id;
            tops[row * top + k] = logprob(logit(x, id));
        }
    }
}

}  // namespace

int launch_logprobs(const LogprobJob &j, hipStream_t s) {
    const dim3 grid((unsigned)j.rows);
    if (j.f32)
        hipLaunchKernelGGL((logprobs_kernel<float>), grid, dim3(kThreads), 0, s, (const float *)j.x, j.vocab, j.stride,
                           j.tokens, j.top, j.logprobs, j.entropy, j.ids, j.tops);
    else
        hipLaunchKernelGGL((logprobs_kernel<uint16_t>), grid, dim3(kThreads), 0, s, (const uint16_t *)j.x, j.vocab,
                           j.stride, j.tokens, j.top, j.logprobs, j.entropy, j.ids, j.tops);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace chip
