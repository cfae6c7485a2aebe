// Log probabilities of given tokens, the entropy and the most likely
// alternatives of rows of logits. With M = max x, c the number of logits equal
// to M, S = sum over the others of e^(x - M) and A = sum of e^(x - M) (M - x):
//   log p_t = (x_t - M) - log(c + S),   H = log(c + S) + A / (c + S).
// S leaves the largest logits out, so that log(1 + S) keeps its digits where one
// token is nearly certain; every term of H is positive.
//
// One pass over the logits. A row is cut into segments, a block each
// (logprobs_kernel); a block walks its segment in chunks that sit in registers,
// each thread with its own running maximum and sums (f32 over a chunk's at most
// 32 logits, in 64 bits from chunk to chunk), the block with the best `top`
// logits so far. A logit joins those only if it is larger than the last of them
// (ids rise, so an equal one loses), which is rare after the first chunk. Few
// rows have many segments, joined by logprobs_join_kernel; many rows have one
// each and are done in one launch.
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kCap = 512;       // candidates a block holds beside its best
constexpr int kMaxSegs = 128;   // two a lane of the join's waves
constexpr float kLog2e = 1.44269504088896340736f;

// A row's sums over a part of it: the maximum, the logits equal to it, the sum
// over the others, the sum of the entropy's terms.
struct Sums {
    double S, A;
    float m;
    int c;
};

struct LogprobArgs {
    const void *x;
    const uint32_t *tokens;
    float *logprobs, *entropy;
    uint32_t *ids;
    float *tops;
    size_t stride;
    unsigned vocab, seg;  // logits of a row, of a segment
    int top, segs;
    Sums *sums;       // [row][segment]
    uint64_t *picks;  // [row][segment][top]: keys
};

// Alternatives are ordered by their keys: the value's bits in order, then the
// id from the largest. -0 counts as 0 and NaN as -inf. 0 is no logit's key.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const float v = x == x ? x + 0.f : -INFINITY;
    const uint32_t u = __float_as_uint(v), o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t key_id(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {  // wave_sum's steps
    v += dpp_f64<kDppXor1>(v);
    v += dpp_f64<kDppXor2>(v);
    v += dpp_f64<kDppHalfMirror>(v);
    v += dpp_f64<kDppMirror>(v);
    return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}

// Sums about their own maximum -> about the larger m. Without a finite logit
// (-inf) they are 0, or NaN, which stays.
__device__ __forceinline__ void raise(Sums &s, float m) {
    if (s.m == m) return;
    const float d = s.m - m;
    const double f = s.m == -INFINITY ? 0.0 : (double)__builtin_amdgcn_exp2f(d * kLog2e), w = s.c + s.S;
    s.A = f == 0.0 ? 0.0 * w : f * (s.A - (double)d * w);
    s.S = f * w;
    s.c = 0;
    s.m = m;
}

// The wave's sums about m, the largest maximum.
__device__ __forceinline__ Sums wave_join(Sums s, float m) {
    raise(s, m);
    Sums t;
    t.m = m;
    t.S = wave_sum_f64(s.S);
    t.A = wave_sum_f64(s.A);
    t.c = (int)wave_sum((float)s.c);  // at most the few ties of threads: below 2^24 a lane
    return t;
}

// A row's results from its sums, alternatives from their keys (any LDS or
// global array), by the threads of a block.
struct Result {
    double m, logsum;
    bool empty;
    __device__ Result(const Sums &s) : m(s.m), logsum(log1p((double)(s.c - 1) + s.S)), empty(s.m == -INFINITY && s.S == 0) {}
    __device__ float logprob(float x) const { return empty ? -INFINITY : (float)((double)x - m - logsum); }
};
template <class T>
__device__ __forceinline__ void store_row(const LogprobArgs &a, const T *x, size_t row, const Sums &s, const uint64_t *best) {
    const int tid = threadIdx.x;
    const Result r(s);
    if (tid == 0 && a.logprobs) {
        const uint32_t t = a.tokens[row];
        float v = NAN;
        if (t < a.vocab) {
            if constexpr (sizeof(T) == 4) v = r.logprob(x[t]);
            else v = r.logprob(bf16_f32(x[t]));
        }
        a.logprobs[row] = v;
    }
    if (tid == 0 && a.entropy) a.entropy[row] = r.empty ? 0.f : (float)(r.logsum + s.A / ((double)s.c + s.S));
    if (tid < a.top) {
        const uint64_t k = best[tid];
        a.ids[row * a.top + tid] = key_id(k);
        a.tops[row * a.top + tid] = r.logprob(key_value(k));
    }
}

// The best `top` keys that a block has seen, in order, and candidates behind
// them. Every function is called by the whole block.
constexpr int kRoom = kMaxTop + kCap;  // keys held; up to kMaxTop ties go behind them
struct Best {
    uint64_t key[kRoom + kMaxTop + 8];
    float wave_value[kWaves];
    uint64_t wave_key[kWaves];
    int ties[kWaves];
    int count;  // keys held, the best among them
};

// Sorts the keys held and keeps the first `top`: each thread ranks its keys
// among all of them, eight reads in flight.
template <int R>
__device__ __forceinline__ void best_rank(Best &b, int top, int n) {
    const int tid = threadIdx.x;
    uint64_t mine[R];
    int rank[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        mine[i] = tid + kThreads * i < n ? b.key[tid + kThreads * i] : ~0ull;
        rank[i] = 0;
    }
    if (tid < 8) b.key[n + tid] = 0;  // above no key
    __syncthreads();
    if (R > 1 || tid < (n + 63) / 64 * 64)
        for (int j = 0; j < n; j += 8) {
            uint64_t k[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) k[q] = b.key[j + q];
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int i = 0; i < R; ++i) rank[i] += k[q] > mine[i];
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (tid + kThreads * i < n && rank[i] < top) b.key[rank[i]] = mine[i];
    if (tid == 0) b.count = min(n, top);
    __syncthreads();
}
__device__ __forceinline__ void best_prune(Best &b, int top) {
    constexpr int R = (kRoom + kMaxTop + kThreads - 1) / kThreads;
    const int n = b.count;
    if (n <= kThreads) best_rank<1>(b, top, n);
    else best_rank<R>(b, top, n);
}

// What the best are taken from, 16 bytes of logits a thread and vector or a
// pick; equal ones' ids rise with (vector, thread, place in it). Read again
// from memory: the registers that hold a chunk would not do for both.
template <class T>
struct Logits {
    static constexpr int VE = 16 / sizeof(T);
    const T *from;
    unsigned e0, head, end, last_load;
    int vectors;
    struct Vec {
        u32x4 w;
        unsigned e;
    };
    __device__ Vec load(int v) const {
        const unsigned e = e0 + (kThreads * v + threadIdx.x) * VE;
        return Vec{*(const u32x4 *)(from + min(e, last_load)), e};
    }
    __device__ bool ok(const Vec &v, int q) const { return v.e + q >= head && v.e + q < end; }
    __device__ uint32_t id(const Vec &v, int q) const { return v.e + q - head; }
    __device__ float value(const Vec &v, int q) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(v.w[q]);
        else return q & 1 ? bf16_hi(v.w[q >> 1]) : bf16_lo(v.w[q >> 1]);
    }
};
struct Picks {
    static constexpr int VE = 1;
    const uint64_t *key;
    int n, vectors;
    typedef uint64_t Vec;
    __device__ Vec load(int v) const {
        const int e = kThreads * v + (int)threadIdx.x;
        return e < n ? key[e] : 0;
    }
    __device__ bool ok(Vec v, int) const { return v != 0; }
    __device__ uint32_t id(Vec v, int) const { return key_id(v); }
    __device__ float value(Vec v, int) const { return key_value(v); }
};

__device__ __forceinline__ void best_settle(Best &b, int top, bool &full, float &last) {
    best_prune(b, top);
    full = b.count == top;
    last = full ? key_value(b.key[top - 1]) : -INFINITY;
}

// Takes a chunk of which any number may belong to the best: those above `last`
// while `full`, all otherwise. `most`: the thread's largest value of it.
template <class Src>
__device__ __forceinline__ void best_refill(Best &b, int top, bool &full, float &last, const Src &src, float most) {
    constexpr int VE = Src::VE;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int held = b.count;
    // At least `top` logits reach the smallest of the waves' (top / 4) largest
    // thread maxima. (Ranked by their ordered bits, the lowest six the lane's, so
    // that every lane has a rank of its own.)
    {
        most = most == most ? most : -INFINITY;  // (a signalling NaN came last)
        const uint32_t u = __float_as_uint(most), o = u & 0x80000000u ? ~u : u | 0x80000000u;
        const uint32_t mine = (o & ~63u) | lane;
        int rank = 0;
#pragma unroll 16
        for (int j = 0; j < 64; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, j) > mine;
        const float least = -wave_max(rank < (top + kWaves - 1) / kWaves ? -most : -INFINITY);
        if (lane == 0) b.wave_value[wave] = least;
    }
    __syncthreads();
    const float from = fminf(fminf(b.wave_value[0], b.wave_value[1]), fminf(b.wave_value[2], b.wave_value[3]));
    auto open = [&](float v) { return !full || v > last; };
    // Every open logit from `from` on (`above`: only larger ones); the count may
    // pass the room.
    auto append = [&](bool above) {
        for (int v = 0; v < src.vectors; ++v) {
            const auto w = src.load(v);
#pragma unroll
            for (int q = 0; q < VE; ++q) {
                const float x = src.value(w, q);
                if (src.ok(w, q) && open(x) && (above ? x > from : !(x < from))) {
                    const int at = atomicAdd(&b.count, 1);
                    if (at < kRoom) b.key[at] = key_of(x, src.id(w, q));
                }
            }
        }
        __syncthreads();
    };
    auto back = [&]() {
        __syncthreads();
        if (tid == 0) b.count = held;
        __syncthreads();
    };
    append(false);
    if (b.count > kRoom) {
        // Ties (a mask's, most likely): the larger ones, and the first `top` of those
        // equal to `from`.
        back();
        append(true);
        const int larger = b.count;
        if (larger <= kRoom) {
            auto tie = [&](const typename Src::Vec &w, int q) {
                const float x = src.value(w, q);
                return src.ok(w, q) && open(x) && !(x < from) && !(x > from);
            };
            int base = 0;
            for (int v = 0; v < src.vectors && base < top; ++v) {
                const auto w = src.load(v);
                int n = 0, before = 0;
#pragma unroll
                for (int q = 0; q < VE; ++q) {
                    const uint64_t m = __ballot(tie(w, q));
                    n += __builtin_popcountll(m);
                    before += __builtin_popcountll(m & ((1ull << lane) - 1));
                }
                if (lane == 0) b.ties[wave] = n;
                __syncthreads();
                int at = base + before;
                for (int x = 0; x < kWaves; ++x) {
                    if (x < wave) at += b.ties[x];
                    base += b.ties[x];
                }
#pragma unroll
                for (int q = 0; q < VE; ++q)
                    if (tie(w, q)) {
                        if (at < top) b.key[larger + at] = key_of(src.value(w, q), src.id(w, q));
                        ++at;
                    }
                __syncthreads();
            }
            if (tid == 0) b.count = larger + min(base, top);
            __syncthreads();
        } else {
            // Logits that rise with their ids: the best open one after the last, `top` times.
            back();
            uint64_t prev = ~0ull;
            for (int r = 0; r < top; ++r) {
                uint64_t k = 0;
                for (int v = 0; v < src.vectors; ++v) {
                    const auto w = src.load(v);
#pragma unroll
                    for (int q = 0; q < VE; ++q) {
                        const float x = src.value(w, q);
                        const uint64_t c = src.ok(w, q) && open(x) ? key_of(x, src.id(w, q)) : 0;
                        if (c < prev && c > k) k = c;
                    }
                }
#pragma unroll
                for (int off = 32; off > 0; off >>= 1) {
                    const uint64_t c = (uint64_t)__shfl_xor((unsigned long long)k, off, 64);
                    k = c > k ? c : k;
                }
                __syncthreads();
                if (lane == 0) b.wave_key[wave] = k;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWaves; ++w) k = max(k, b.wave_key[w]);
                if (k == 0) break;  // no more (the same in every thread)
                if (tid == 0) b.key[b.count++] = k;
                prev = k;
            }
            __syncthreads();
        }
    }
    best_settle(b, top, full, last);
}

// One segment of a row, kThreads * PER logits at a time.
template <class T, int PER>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobArgs a) {
    constexpr int VE = 16 / sizeof(T), NV = PER / VE;  // logits of a 16-byte load, loads of a thread
    constexpr unsigned CHUNK = kThreads * PER;
    __shared__ Best best;
    __shared__ Sums part[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x / (unsigned)a.segs;
    const unsigned seg = blockIdx.x % (unsigned)a.segs;
    const T *x_row = (const T *)a.x + row * a.stride;
    // 16-byte loads from the row's last boundary on: logit e of them has id
    // e - head. A load holds at least one logit of the row.
    const unsigned head = (unsigned)((uintptr_t)x_row & 15) / sizeof(T), all = head + a.vocab;
    const T *from = x_row - head;
    const unsigned begin = seg * a.seg, end = min(begin + a.seg, all), last_load = (all - 1) / VE * VE;
    u32x4 raw[NV];
    auto load = [&](unsigned e0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) raw[v] = *(const u32x4 *)(from + min(e0 + (kThreads * v + tid) * VE, last_load));
    };
    load(begin);
    if (tid == 0) best.count = 0;
    __syncthreads();
    Sums s{0.0, 0.0, -INFINITY, 0};
    bool full = false;
    float last = -INFINITY;
    for (unsigned e0 = begin; e0 < end; e0 += CHUNK) {
        float x[PER];
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    x[4 * v + i] = __uint_as_float(raw[v][i]);
                } else {
                    x[8 * v + 2 * i] = bf16_lo(raw[v][i]);
                    x[8 * v + 2 * i + 1] = bf16_hi(raw[v][i]);
                }
            }
        if (e0 + CHUNK < end) load(e0 + CHUNK);
        auto at = [&](int i) { return e0 + (kThreads * (i / VE) + tid) * VE + i % VE; };
        auto ok = [&](int i) { return at(i) >= head && at(i) < end; };
        const bool whole = e0 >= head && e0 + CHUNK <= end;
        if (!whole)
#pragma unroll
            for (int i = 0; i < PER; ++i) x[i] = ok(i) ? x[i] : -INFINITY;
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i) most = fmaxf(most, x[i]);
        raise(s, fmaxf(s.m, most));
        const float m = s.m == -INFINITY ? 0.f : s.m;
        float S = 0.f, A = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float d = x[i] - m, e = __builtin_amdgcn_exp2f(d * kLog2e), o = d == 0.f ? 0.f : e;
            s.c += d == 0.f;
            S += o;
            A = fmaf(o, -fmaxf(d, -150.f), A);  // 0 from -150 on, -inf too
        }
        s.S += S;
        s.A += A;
        if (a.top && __syncthreads_or(!full || most > last)) {
            const Logits<T> src{from, e0, head, end, last_load, (int)((min(end - e0, CHUNK) + kThreads * VE - 1) / (kThreads * VE))};
            if (full) {  // few: straight from the registers
                const int held = best.count;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (x[i] > last) {  // (never a logit that is not ok: -inf)
                        const int k = atomicAdd(&best.count, 1);
                        if (k < kRoom) best.key[k] = key_of(x[i], at(i) - head);
                    }
                __syncthreads();
                const int n = best.count;
                if (n <= kRoom) {
                    if (n >= a.top + 64) best_settle(best, a.top, full, last);
                    continue;
                }
                __syncthreads();
                if (tid == 0) best.count = held;
                __syncthreads();
                best_settle(best, a.top, full, last);
            }
            best_refill(best, a.top, full, last, src, most);
        }
    }
    // The block's sums.
    const float wm = wave_max(s.m);
    const Sums t = wave_join(s, wm);
    if (lane == 0) part[wave] = t;
    __syncthreads();
    Sums all_waves = part[0];
    float m = all_waves.m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, part[w].m);
    raise(all_waves, m);
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        Sums u = part[w];
        raise(u, m);
        all_waves.S += u.S;
        all_waves.A += u.A;
        all_waves.c += u.c;
    }
    if (a.top && best.count > a.top) {  // candidates left
        __syncthreads();
        best_prune(best, a.top);
    }
    if (a.segs == 1) {
        store_row(a, x_row, row, all_waves, best.key);
        return;
    }
    const size_t at = row * a.segs + seg;
    if (tid == 0) a.sums[at] = all_waves;
    if (tid < a.top) a.picks[at * a.top + tid] = tid < best.count ? best.key[tid] : 0;
}

// The segments of a row.
template <class T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobArgs a) {
    __shared__ Best best;
    const int tid = threadIdx.x, lane = tid & 63;
    const size_t row = blockIdx.x;
    Sums s{0.0, 0.0, -INFINITY, 0}, s2 = s;
    if (lane < a.segs) s = a.sums[row * a.segs + lane];
    if (lane + 64 < a.segs) s2 = a.sums[row * a.segs + lane + 64];
    const int n = a.segs * a.top;
    const Picks src{a.picks + row * n, n, (n + kThreads - 1) / kThreads};
    float most = -INFINITY;
    for (int v = 0; v < src.vectors; ++v) {
        const uint64_t k = src.load(v);
        most = fmaxf(most, k ? key_value(k) : -INFINITY);
    }
    if (tid == 0) best.count = 0;
    __syncthreads();
    const float m = wave_max(fmaxf(s.m, s2.m));
    s = wave_join(s, m);
    s2 = wave_join(s2, m);
    s.S += s2.S;
    s.A += s2.A;
    s.c += s2.c;
    if (a.top) {
        bool full = false;
        float last = -INFINITY;
        best_refill(best, a.top, full, last, src, most);
    }
    store_row(a, (const T *)a.x + row * a.stride, row, s, best.key);
}

// Segments of a row: enough for two blocks a CU, of at least a small chunk.
int logprob_segs(size_t rows, size_t vocab) {
    const size_t want = 2 * (size_t)std::max(device_cus(), 1) / rows, most = (vocab + 2039) / 2040;
    return (int)std::max<size_t>(std::min({want, most, (size_t)kMaxSegs}), 1);
}

template <class T>
int launch_logprobs_t(const LogprobJob &j, LogprobArgs &a, hipStream_t s) {
    const size_t blocks = j.rows * (size_t)a.segs;
    if (blocks > (size_t)INT32_MAX) return fail("HIP backend: logprobs grid out of range.");
    if (a.seg <= (unsigned)(8 * kThreads))
        hipLaunchKernelGGL((logprobs_kernel<T, 8>), dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((logprobs_kernel<T, 32>), dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
    CHIP_CHECK(hipGetLastError());
    if (a.segs == 1) return 0;
    hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3((unsigned)j.rows), dim3(kThreads), 0, s, a);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace

size_t logprobs_workspace_bytes(size_t rows, size_t vocab, int top) {
    const size_t segs = (size_t)logprob_segs(rows, vocab);
    return segs == 1 ? 0 : rows * segs * (sizeof(Sums) + (size_t)top * sizeof(uint64_t));
}

int launch_logprobs(const LogprobJob &j, hipStream_t s) {
    if (!j.x || j.rows == 0 || j.vocab == 0 || j.vocab > (size_t)INT32_MAX - 64 || j.stride < j.vocab || j.top < 0 ||
        j.top > kMaxTop || (size_t)j.top > j.vocab)
        return fail("HIP backend: logprobs shape out of range.");
    LogprobArgs a{};
    a.x = j.x;
    a.tokens = j.tokens;
    a.logprobs = j.logprobs;
    a.entropy = j.entropy;
    a.ids = j.ids;
    a.tops = j.tops;
    a.stride = j.stride;
    a.vocab = (unsigned)j.vocab;
    a.top = j.top;
    a.segs = logprob_segs(j.rows, j.vocab);
    // Up to seven logits of another row or of padding come before the row's first.
    a.seg = ((unsigned)j.vocab + 7 + (unsigned)a.segs - 1) / (unsigned)a.segs;
    a.seg = (a.seg + 7) / 8 * 8;
    if (a.segs > 1) {
        if (!j.ws || j.ws_bytes < logprobs_workspace_bytes(j.rows, j.vocab, j.top))
            return fail("HIP backend: logprobs workspace too small.");
        a.sums = (Sums *)j.ws;
        a.picks = (uint64_t *)(a.sums + j.rows * (size_t)a.segs);
    }
    return j.f32 ? launch_logprobs_t<float>(j, a, s) : launch_logprobs_t<uint16_t>(j, a, s);
}

}  // namespace chip
