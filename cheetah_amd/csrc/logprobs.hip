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
// 16 logits, in 64 bits from chunk to chunk), the block with the best `top`
// logits so far. A logit joins those only if it is larger than the last of them
// (ids rise, so an equal one loses), which is rare after the first chunk. Many
// rows have one segment each; few rows have many, whose results go through memory
// to the row's last block, which joins them in the same launch.
//
// Bound: 512 f32 rows of 151936 (311 MB) with one alternative take 57.4 us, 5.42
// TB/s, above a large copy's rate (5.16, read and write); BF16 rows 0.79 of the time
// (the exponentials then count: 16 of them a thread and chunk). Fewer rows are bound
// by the steps before and behind the loop, each a memory or LDS round trip: of 64
// rows' 20.1 us with 20 alternatives the loop ends at 13, the segment's sums and
// picks are in memory and counted at 14.6, read by the last block at 15.3, ranked at
// 17.5. As two launches these 64 rows took 3 us more, one row the same. A release
// fence in place of the write-through stores (it writes the whole L2 back) made
// them 29.6 for 20.4 then.
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kCap = 512;       // candidates a block holds beside its best
constexpr int kMaxSegs = 128;   // two a lane of the join's waves
constexpr float kLog2e = 1.44269504088896340736f;

// Block barrier that waits on LDS traffic only: the next chunk's loads stay in
// flight across it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A row's sums over a part of it: the maximum, the logits equal to it, the sum
// over the others, the sum of the entropy's terms.
struct Sums {
    double S, A;
    float m;
    int c;
};

// Words that blocks of one launch hand on. An agent-scope access goes past the
// caches of its own XCD, so that a block anywhere reads what is there.
__device__ __forceinline__ void agent_store(uint64_t *p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t agent_load(const uint64_t *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
constexpr int kCountStride = 32;  // a row's count has a cache line of its own
constexpr int kSumWords = sizeof(Sums) / sizeof(uint64_t);
__device__ __forceinline__ Sums agent_load(const Sums *p) {
    uint64_t w[kSumWords];
#pragma unroll
    for (int i = 0; i < kSumWords; ++i) w[i] = agent_load((const uint64_t *)p + i);
    Sums s;
    __builtin_memcpy(&s, w, sizeof(s));
    return s;
}

struct LogprobArgs {
    const void *x;
    const uint32_t *tokens;
    float *logprobs, *entropy;
    uint32_t *ids;
    float *tops;
    size_t stride;
    unsigned vocab, seg;  // logits of a row, of a segment
    int top, segs;
    Sums *sums;         // [row][segment]
    uint64_t *picks;    // [row][segment][top]: keys, 0 for none
    uint32_t *arrived;  // [row][kCountStride]: segments done, 0 between launches
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

// The given token's logit, in the first thread; NaN where there is none. Read at
// a block's start, its two round trips to memory pass beside the first chunk's.
template <class T>
__device__ __forceinline__ float token_logit(const LogprobArgs &a, const T *x, size_t row) {
    if (!a.logprobs || threadIdx.x) return NAN;
    const uint32_t t = a.tokens[row];
    if (t >= a.vocab) return NAN;
    if constexpr (sizeof(T) == 4) return x[t];
    else return bf16_f32(x[t]);
}

// A row's results from its sums, alternatives from their keys, by the threads of
// a block.
struct Result {
    double m, logsum;
    bool empty;
    __device__ Result(const Sums &s) : m(s.m), logsum(log1p((double)(s.c - 1) + s.S)), empty(s.m == -INFINITY && s.S == 0) {}
    __device__ float logprob(float x) const { return empty ? -INFINITY : (float)((double)x - m - logsum); }
};
__device__ __forceinline__ void store_row(const LogprobArgs &a, size_t row, float token, const Sums &s, const uint64_t *best) {
    const int tid = threadIdx.x;
    const Result r(s);
    if (tid == 0 && a.logprobs) a.logprobs[row] = token == token ? r.logprob(token) : NAN;
    if (tid == 0 && a.entropy) a.entropy[row] = r.empty ? 0.f : (float)(r.logsum + s.A / ((double)s.c + s.S));
    if (tid < a.top) {
        const uint64_t k = best[tid];
        a.ids[row * a.top + tid] = key_id(k);
        a.tops[row * a.top + tid] = r.logprob(key_value(k));
    }
}

// The best `top` keys that a block has seen, in order, and candidates behind
// them. Logits of -inf (and NaN) are never among them: fill_masked adds the first
// of those at the end where others are fewer than `top`. Every function is called
// by the whole block and ends with its results visible.
constexpr int kRoom = kMaxTop + kCap;
struct Best {
    uint64_t key[kRoom + 8];
    uint16_t above[kWaves][kRoom];
    float wave_value[kWaves];
    int hist[256], wave_total[kWaves], found[3];
    int count;  // keys held, the best among them; past kRoom: some had no room
};

// n places for the wave's keys (the same n in its lanes, all of which call).
__device__ __forceinline__ int best_take(Best &b, int n) {
    int k = 0;
    if ((threadIdx.x & 63) == 0) k = atomicAdd(&b.count, n);
    return __builtin_amdgcn_readfirstlane(k);
}
// How many of the lanes in m are below this one.
__device__ __forceinline__ int lanes_below(uint64_t m) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// Sorts the keys held and keeps the first `top`. Every wave takes all the keys, R a
// lane, and a quarter of them to compare with, eight reads in flight; a key's rank
// is the sum of the waves' counts of larger ones. (A thread with a key of its own
// and all the others to compare: 160 keys 2.2 us, so 1.5.)
template <int R>
__device__ __forceinline__ void best_rank(Best &b, int top, int n) {
    constexpr int OWN = (64 * R + kThreads - 1) / kThreads;  // keys whose ranks a thread adds up
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = (n + 8 * kWaves - 1) / (8 * kWaves) * 8, j0 = min(wave * part, n), j1 = min(j0 + part, n);
    uint64_t mine[R], own[OWN];
    int rank[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        mine[i] = lane + 64 * i < n ? b.key[lane + 64 * i] : ~0ull;
        rank[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) own[i] = tid + kThreads * i < n ? b.key[tid + kThreads * i] : 0;
    if (tid < 8) b.key[n + tid] = 0;  // above no key
    lds_barrier();
    for (int j = j0; j < j1; j += 8) {
        uint64_t k[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) k[q] = b.key[j + q];
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int i = 0; i < R; ++i) rank[i] += k[q] > mine[i];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) b.above[wave][lane + 64 * i] = (uint16_t)rank[i];
    lds_barrier();
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        const int at = tid + kThreads * i;
        if (at >= n) break;
        int r = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) r += b.above[w][at];
        if (r < top) b.key[r] = own[i];
    }
    if (tid == 0) b.count = min(n, top);
    lds_barrier();
}

// Prunes to the best `top`, says above what a logit would join them and how many
// are held (the count itself may grow again before every wave has read it).
__device__ __forceinline__ int best_settle(Best &b, int top, float &last) {
    const int n = b.count;
    if (n <= 128) best_rank<2>(b, top, n);
    else if (n <= 256) best_rank<4>(b, top, n);
    else best_rank<kRoom / 64>(b, top, n);
    last = n < top ? -INFINITY : key_value(b.key[top - 1]);
    return min(n, top);
}

// A value that at least `top` of the logits reach whose thread maxima are `most`.
// Up to eight: the smallest of the four waves' or eight half waves' maxima. More:
// the smallest of the waves' (top / 4) largest, ranked by their ordered bits, the
// lowest six the lane's, so that every lane has a rank of its own: 64 steps, but
// fewer candidates than smaller groups would leave (5 rows with 1 alternative 9.9
// us by ranks, 8.6 by maxima; 16 rows with 20 alternatives 17.5 by ranks, 19.6 by
// the maxima of eight lanes).
__device__ __forceinline__ float best_bound(Best &b, int top, float most) {
    const int lane = threadIdx.x & 63;
    most = most == most ? most + 0.f : -INFINITY;  // (NaN: a signalling one came last)
    float least;
    if (top <= 2 * kWaves) {
        float g = fmaxf(most, dpp_mov<kDppXor1>(most));
        g = fmaxf(g, dpp_mov<kDppXor2>(g));
        g = fmaxf(g, dpp_mov<kDppHalfMirror>(g));
        g = fmaxf(g, dpp_mov<kDppMirror>(g));  // of 16 lanes
        const float lo = fmaxf(lane_read(g, 0), lane_read(g, 16)), hi = fmaxf(lane_read(g, 32), lane_read(g, 48));
        least = top <= kWaves ? fmaxf(lo, hi) : fminf(lo, hi);
    } else {
        const uint32_t u = __float_as_uint(most), o = u & 0x80000000u ? ~u : u | 0x80000000u, mine = (o & ~63u) | lane;
        int rank = 0;
#pragma unroll 16
        for (int j = 0; j < 64; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, j) > mine;
        least = -wave_max(rank < (top + kWaves - 1) / kWaves ? -most : -INFINITY);
    }
    if (lane == 0) b.wave_value[threadIdx.x >> 6] = least;
    lds_barrier();
    return fminf(fminf(b.wave_value[0], b.wave_value[1]), fminf(b.wave_value[2], b.wave_value[3]));
}

// The largest value below v.
__device__ __forceinline__ float just_below(float v) {
    if (v == 0.f) return __uint_as_float(0x80000001u);
    const uint32_t u = __float_as_uint(v);
    return v == -INFINITY ? v : __uint_as_float(v > 0.f ? u - 1 : u + 1);
}

// Logits, 16 bytes a thread and vector, or segments' picks, as keys read from
// memory: 0 where there is none, or none above `last`.
template <class T>
struct Logits {
    static constexpr int VE = 16 / sizeof(T);
    const T *from;
    unsigned e0, head, end, last_load;
    float last;
    int vectors;
    struct Vec {
        u32x4 w;
        unsigned e;
    };
    __device__ Vec load(int v) const {
        const unsigned e = e0 + (kThreads * v + threadIdx.x) * VE;
        return Vec{*(const u32x4 *)(from + min(e, last_load)), e};
    }
    __device__ uint64_t key(const Vec &v, int q) const {
        float x;
        if constexpr (sizeof(T) == 4) x = __uint_as_float(v.w[q]);
        else x = q & 1 ? bf16_hi(v.w[q >> 1]) : bf16_lo(v.w[q >> 1]);
        return v.e + q >= head && v.e + q < end && x > last ? key_of(x, v.e + q - head) : 0;
    }
};
struct Picks {
    static constexpr int VE = 1;
    const uint64_t *picks;
    int segs, top, vectors;
    typedef uint64_t Vec;
    // In the order of their ranks, so that a thread's largest is of its own segment.
    __device__ Vec load(int v) const {
        const int e = kThreads * v + (int)threadIdx.x;
        return e < segs * top ? agent_load(picks + (e % segs * top + e / segs)) : 0;
    }
    __device__ uint64_t key(Vec v, int) const { return v; }
};

// Takes the keys of which there are too many for a bound to tell apart (ties):
// the `top`-th largest by its digits, eight bits at a time, until those from it on
// have room. Keys are unique, so that they do in the end.
template <class Src>
__device__ __forceinline__ void best_select(Best &b, int top, const Src &src) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, room = kRoom - b.count;
    uint64_t prefix = 0, from = 0;
    int need = top, taken = 0;
    for (int shift = 56;; shift -= 8) {
        lds_barrier();
        b.hist[tid] = 0;
        lds_barrier();
        for (int v = 0; v < src.vectors; ++v) {
            const auto w = src.load(v);
#pragma unroll
            for (int q = 0; q < Src::VE; ++q) {
                const uint64_t k = src.key(w, q);
                const bool in = k && (shift == 56 || k >> (shift + 8) == prefix);
                const int digit = (int)(k >> shift) & 255;
                const uint64_t m = __ballot(in);
                if (!m) continue;
                const int first = __builtin_amdgcn_readlane(digit, __builtin_ctzll(m));
                if (__ballot(in && digit != first) == 0) {  // one bin, as ties have
                    if (lane == 0) atomicAdd(&b.hist[first], __builtin_popcountll(m));
                } else if (in) {
                    atomicAdd(&b.hist[digit], 1);
                }
            }
        }
        lds_barrier();
        // Keys with this thread's digit or a larger one.
        const int h = b.hist[tid];
        int sum = h;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int other = __shfl_down(sum, off, 64);
            if (lane + off < 64) sum += other;
        }
        if (lane == 0) b.wave_total[wave] = sum;
        lds_barrier();
        for (int w = wave + 1; w < kWaves; ++w) sum += b.wave_total[w];
        if (sum >= need && sum - h < need) {
            b.found[0] = tid;
            b.found[1] = sum - h;
            b.found[2] = h;
        }
        lds_barrier();
        prefix = prefix << 8 | (uint64_t)b.found[0];
        taken += b.found[1];
        need -= b.found[1];
        from = prefix << shift;
        if (taken + b.found[2] <= room || shift == 0) break;
    }
    for (int v = 0; v < src.vectors; ++v) {
        const auto w = src.load(v);
#pragma unroll
        for (int q = 0; q < Src::VE; ++q) {
            const uint64_t k = src.key(w, q);
            if (k && k >= from) b.key[atomicAdd(&b.count, 1)] = k;
        }
    }
    lds_barrier();
}

// The first of the row's logits without a probability, up to `top` alternatives.
template <class T>
__device__ __forceinline__ void fill_masked(Best &b, int top, const T *x, unsigned vocab) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int at = b.count;  // (no more change it)
    for (unsigned i0 = 0; at < top && i0 < vocab; i0 += kThreads) {
        const unsigned i = i0 + tid;
        bool masked = false;
        if (i < vocab) {
            if constexpr (sizeof(T) == 4) masked = !(x[i] > -INFINITY);
            else masked = !(bf16_f32(x[i]) > -INFINITY);
        }
        const uint64_t m = __ballot(masked);
        lds_barrier();
        if (lane == 0) b.wave_total[wave] = __builtin_popcountll(m);
        lds_barrier();
        int mine = at + __builtin_popcountll(m & ((1ull << lane) - 1));
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) mine += b.wave_total[w];
            at += b.wave_total[w];
        }
        if (masked && mine < top) b.key[mine] = key_of(-INFINITY, i);
    }
    lds_barrier();
}

// The segments of a row, by the block that was the last to end one.
template <class T>
__device__ __forceinline__ void join_row(const LogprobArgs &a, Best &best, const T *x_row, size_t row, float token) {
    const int tid = threadIdx.x, lane = tid & 63;
    Sums s{0.0, 0.0, -INFINITY, 0}, s2 = s;
    if (lane < a.segs) s = agent_load(a.sums + row * a.segs + lane);
    if (lane + 64 < a.segs) s2 = agent_load(a.sums + row * a.segs + lane + 64);
    const int n = a.segs * a.top;
    const Picks src{a.picks + row * n, a.segs, a.top, (n + kThreads - 1) / kThreads};
    constexpr int HELD = 4;  // picks a thread keeps from the first look at them
    uint64_t picks[HELD];
#pragma unroll
    for (int v = 0; v < HELD; ++v) picks[v] = src.load(v);
    float most = -INFINITY;
#pragma unroll
    for (int v = 0; v < HELD; ++v) most = fmaxf(most, picks[v] ? key_value(picks[v]) : -INFINITY);
    for (int v = HELD; v < src.vectors; ++v) {
        const uint64_t k = src.load(v);
        most = fmaxf(most, k ? key_value(k) : -INFINITY);
    }
    if (tid == 0) best.count = 0;
    lds_barrier();
    const float m = wave_max(fmaxf(s.m, s2.m));
    if (a.segs > 64) {
        raise(s, m);
        raise(s2, m);
        s.S += s2.S;
        s.A += s2.A;
        s.c += s2.c;
    }
    s = wave_join(s, m);
    if (a.top) {
        const float from = n <= kThreads ? -INFINITY : best_bound(best, a.top, most);
        auto append = [&](uint64_t k) {
            const uint64_t m = __ballot(k && key_value(k) >= from);
            if (!m) return;
            const int place = best_take(best, __builtin_popcountll(m)) + lanes_below(m);
            if (k && key_value(k) >= from && place < kRoom) best.key[place] = k;
        };
#pragma unroll
        for (int v = 0; v < HELD; ++v) append(picks[v]);
        for (int v = HELD; v < src.vectors; ++v) append(src.load(v));
        lds_barrier();
        const bool many = best.count > kRoom;
        lds_barrier();
        if (many) {
            if (tid == 0) best.count = 0;
            lds_barrier();
            best_select(best, a.top, src);
        }
        float last;
        if (best_settle(best, a.top, last) < a.top) fill_masked(best, a.top, x_row, a.vocab);
    }
    store_row(a, row, token, s, best.key);
}

// One segment of a row, kThreads * PER logits at a time.
template <class T, int PER>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobArgs a) {
    constexpr int VE = 16 / sizeof(T), NV = PER / VE;  // logits of a 16-byte load, loads of a thread
    constexpr unsigned CHUNK = kThreads * PER;
    __shared__ Best best;
    __shared__ Sums part[kWaves];
    __shared__ bool last_here;
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
    const float token = token_logit(a, x_row, row);
    if (tid == 0) best.count = 0;
    lds_barrier();
    Sums s{0.0, 0.0, -INFINITY, 0};
    // A logit above `last` may be among the best. Waves hand theirs over as they
    // go; the block looks at them after 1, 2, 4, 8, .. chunks, between which as many
    // more as `top` are to be expected, and takes the chunks since (from `since`)
    // again where they had no room. (A look every fourth chunk, kept where 64 had
    // come: 512 rows of 151936 with one alternative 59.9 us, so 57.5; BF16 53.9, so
    // 45.5; f32 with 64 78.0, so 72.3.)
    float last = -INFINITY;
    unsigned since = begin;
    int held = 0, chunk = 0, look = 0;
    for (unsigned e0 = begin; e0 < end; e0 += CHUNK, ++chunk) {
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
        if (e0 < head || e0 + CHUNK > end)
#pragma unroll
            for (int i = 0; i < PER; ++i) x[i] = at(i) >= head && at(i) < end ? x[i] : -INFINITY;
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
        if (!a.top) continue;
        float above = last;
        if (chunk == 0) above = just_below(best_bound(best, a.top, most));  // all of them would be too many
        if (__any(most > above)) {
            // A wave's candidates in one run of places: logit by logit, lane by lane.
            int n = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) n += __builtin_popcountll(__ballot(x[i] > above));
            int k = best_take(best, n);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint64_t m = __ballot(x[i] > above);
                if (!m) continue;
                const int place = k + lanes_below(m);
                if (x[i] > above && place < kRoom) best.key[place] = key_of(x[i], at(i) - head);
                k += __builtin_popcountll(m);
            }
        }
        if (chunk == look || e0 + CHUNK >= end) {
            look = 2 * chunk + 1;
            lds_barrier();
            const int n = best.count;
            lds_barrier();  // the same in every wave, before one goes on
            if (n > kRoom) {
                // Ties, or logits that rise with their ids.
                if (tid == 0) best.count = held;
                lds_barrier();
                const unsigned upto = min(end, e0 + CHUNK);
                const Logits<T> src{from, since, head, upto, last_load, last, (int)((upto - since + kThreads * VE - 1) / (kThreads * VE))};
                best_select(best, a.top, src);
            }
            if (n > held || e0 + CHUNK >= end) {
                held = best_settle(best, a.top, last);
                since = e0 + CHUNK;
            }
        }
    }
    // The block's sums.
    const float wm = wave_max(s.m);
    const Sums t = wave_join(s, wm);
    if (lane == 0) part[wave] = t;
    lds_barrier();
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
    if (a.segs == 1) {
        if (held < a.top) fill_masked(best, a.top, x_row, a.vocab);
        store_row(a, row, token, all_waves, best.key);
        return;
    }
    // The first wave leaves the segment's results and counts it; the row's last
    // block joins them, in the segments' order whichever it is.
    const size_t at = row * a.segs + seg;
    if (wave == 0) {
        uint64_t w[kSumWords];
        __builtin_memcpy(w, &all_waves, sizeof(all_waves));
#pragma unroll
        for (int i = 0; i < kSumWords; ++i)
            if (tid == i) agent_store((uint64_t *)(a.sums + at) + i, w[i]);
        if (tid < a.top) agent_store(a.picks + at * a.top + tid, tid < held ? best.key[tid] : 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // they are there before the count says so
        if (tid == 0) {
            uint32_t *count = a.arrived + row * kCountStride;
            last_here = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)a.segs - 1;
            if (last_here) *count = 0;
        }
    }
    lds_barrier();
    if (!last_here) return;
    join_row(a, best, x_row, row, token);
}


// Segments of a row: enough for two blocks a CU, of at least a small chunk.
int logprob_segs(size_t rows, size_t vocab) {
    const size_t want = 2 * (size_t)std::max(device_cus(), 1) / rows, most = (vocab + 2039) / 2040;
    return (int)std::max<size_t>(std::min({want, most, (size_t)kMaxSegs}), 1);
}

// A launch has fewer than 2^32 threads: rows past that (in one segment each) take
// another.
constexpr size_t kLaunchRows = UINT32_MAX / kThreads;
template <class T>
int launch_logprobs_t(const LogprobJob &j, LogprobArgs &a, hipStream_t s) {
    for (size_t left = j.rows; left;) {
        const size_t rows = std::min(left, kLaunchRows / (size_t)a.segs), top = (size_t)a.top;
        const dim3 grid((unsigned)(rows * (size_t)a.segs));
        if (a.seg <= (unsigned)(8 * kThreads))
            hipLaunchKernelGGL((logprobs_kernel<T, 8>), grid, dim3(kThreads), 0, s, a);
        else
            hipLaunchKernelGGL((logprobs_kernel<T, 16>), grid, dim3(kThreads), 0, s, a);
        CHIP_CHECK(hipGetLastError());
        if (!(left -= rows)) break;
        a.x = (const T *)a.x + rows * a.stride;
        if (a.tokens) a.tokens += rows;
        if (a.logprobs) a.logprobs += rows;
        if (a.entropy) a.entropy += rows;
        if (top) {
            a.ids += rows * top;
            a.tops += rows * top;
        }
    }
    return 0;
}

}  // namespace

// The rows' counts at a workspace's start (rows in segments are at most half the
// blocks of two a CU).
constexpr size_t kCountBytes = 1024 * kCountStride * sizeof(uint32_t);

int logprobs_workspace_clear(void *ws, hipStream_t s) {
    CHIP_CHECK(hipMemsetAsync(ws, 0, kCountBytes, s));
    return 0;
}

size_t logprobs_workspace_bytes(size_t rows, size_t vocab, int top) {
    const size_t segs = (size_t)logprob_segs(rows, vocab);
    return segs == 1 ? 0 : kCountBytes + rows * segs * (sizeof(Sums) + (size_t)top * sizeof(uint64_t));
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
        if (j.rows > kCountBytes / (kCountStride * sizeof(uint32_t))) return fail("HIP backend: logprobs grid out of range.");
        a.arrived = (uint32_t *)j.ws;
        a.sums = (Sums *)((uint8_t *)j.ws + kCountBytes);
        a.picks = (uint64_t *)(a.sums + j.rows * (size_t)a.segs);
    }
    return j.f32 ? launch_logprobs_t<float>(j, a, s) : launch_logprobs_t<uint16_t>(j, a, s);
}

}  // namespace chip
