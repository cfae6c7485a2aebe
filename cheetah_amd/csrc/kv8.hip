// An 8-bit paged K/V cache: rows quantised as they are written, read back, and
// causal attention over all of it or over a sliding window and a few first
// positions.
//
// A block is 32 consecutive positions of one KV head, K and V apart: E4M3 codes
// c (sign, 4 bits of exponent, 3 of fraction, no infinities) and one scale 2^e,
// kept as the byte e + 127. A cached value is c 2^e. e is the least with
// |x| <= 448 2^e for the block's values when they were written, so nothing
// saturates; it lies in [kScaleLeast, kScaleMost], where every product c 2^e is a
// normal f32 and an exact BF16. A floating code under one scale keeps small
// channels next to large ones (keys have a few large channels), which whole
// numbers do not; a power of two can grow without rounding the block's codes
// twice, but for those that become subnormal (they move by at most 2^-10 of the
// new scale).
//
// Codes lie in the order in which the 32-wide matrix instructions take them:
//   K block [head_dim / 32][32 positions][32 dims],  V block [head_dim][32 positions],
// so that a lane's operand is 16 consecutive bytes of a 1 KB piece, and a wave's
// load one piece.
#include <algorithm>
#include <atomic>

#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = kKv8Block;
constexpr int kScaleLeast = -117, kScaleMost = 119;

// Block barrier that waits for LDS only: loads stay in flight across it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 2^e, e in [-126, 127].
__device__ __forceinline__ float two_to(int e) { return __int_as_float((e + 127) << 23); }

// Where a block's codes and its scale lie.
struct BlockAt {
    size_t codes, scale;
};
__device__ __forceinline__ BlockAt block_at(const Kv8Geom &g, int page, int sub, int head, int hd) {
    const size_t i = ((size_t)page * g.kv_heads + head) * (g.page_size / kBlock) + sub;
    return BlockAt{i * kBlock * hd, i};
}

// Four codes' values (without the scale).
__device__ __forceinline__ f32x4 code_values(uint32_t w) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f32x4{a[0], a[1], b[0], b[1]};
}
// Four values as codes: to nearest, ties to an even fraction; an infinity or a
// NaN is the NaN code. (A value past 448 is one past 448 2^kScaleMost.)
__device__ __forceinline__ uint32_t codes_of(f32x4 x, float inv) {
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = fabsf(x[i]) < INFINITY ? __builtin_amdgcn_fmed3f(x[i] * inv, -448.f, 448.f) : NAN;
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
// Codes under a scale 2^-down of what they had.
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float factor) {
    const f32x4 v = code_values(w) * factor;
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
    return (uint32_t)r;
}

// The exponent of a block whose largest finite magnitude is `most`.
__device__ __forceinline__ int exponent_for(float most) {
    const uint32_t u = __float_as_uint(most);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);  // 448 = 1.75 * 2^8
    return min(max(e, kScaleLeast), kScaleMost);
}

// ---------------------------------------------------------------------------
// Append: a block of threads per (KV head, K or V, run of blocks: 64 positions at
// head_dim 128, 128 at 64). A thread takes 8 dims of 4 positions; the largest
// magnitude of a block gives its scale; V codes are turned four by four bytes on
// their way into LDS and leave it a dim a thread. Rows of the block that were there
// before are rounded again where the scale grows.
// ---------------------------------------------------------------------------
template <int HD>
constexpr int kRun = kThreads / HD;      // blocks of positions a block of threads
constexpr int kTurnRow = kBlock + 2;     // a V dim's bytes in LDS, with its share of 16 for 8 dims
__device__ __forceinline__ int turn_at(int d) { return d * kBlock + d / 8 * 16; }

// Bytes i of four words as words.
__device__ __forceinline__ void turn4(const uint32_t (&w)[4], uint32_t (&t)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    t[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    t[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    t[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    t[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

struct AppendArgs {
    const void *x[2];  // K, V rows
    long stride, head_stride;
    uint8_t *codes[2], *scales[2];
    Kv8Geom g;
    int offset, rows;  // (positions are below 2^31, block bounds behind the last too)
};

template <class T, bool VEC>
__device__ __forceinline__ void load8(const T *p, f32x4 (&v)[2]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) v[i / 4][i % 4] = p[i];
            else v[i / 4][i % 4] = bf16_f32(p[i]);
        }
    } else if constexpr (sizeof(T) == 4) {
        v[0] = *(const f32x4 *)p;
        v[1] = *(const f32x4 *)(p + 4);
    } else {
        const u32x4 w = *(const u32x4 *)p;
        v[0] = f32x4{bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
        v[1] = f32x4{bf16_lo(w[2]), bf16_hi(w[2]), bf16_lo(w[3]), bf16_hi(w[3])};
    }
}

template <int HD, class T, bool VEC>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(AppendArgs a) {
    __shared__ float s_max[kThreads / 64];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[kRun<HD>][HD * kTurnRow];
    const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
    const int mine = tid / HD, u = tid % HD;
    const int d = u % (HD / 8) * 8, p = u / (HD / 8) * 4;
    const int first = (a.offset / kBlock + (int)blockIdx.x * kRun<HD> + mine) * kBlock;  // the block's first position
    const int keep = max(a.offset - first, 0);                                           // its earlier rows
    const int stop = max(min(a.offset + a.rows - first, kBlock), 0);                     // new rows end here
    const bool any = stop > keep;  // (a wave's threads share a block)
    const T *x = (const T *)(which ? a.x[1] : a.x[0]) + (first - a.offset) * a.stride + head * a.head_stride;
    f32x4 v[4][2];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i][0] = v[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p + i >= keep && p + i < stop) load8<T, VEC>(x + (long)(p + i) * a.stride + d, v[i]);
    }
    uint8_t *codes = nullptr, *scale = nullptr;
    int e_old = kScaleLeast;
    if (any) {
        const uint32_t page = (uint32_t)first / (uint32_t)a.g.page_size;
        const BlockAt at = block_at(a.g, a.g.page_table[page], (first - (int)page * a.g.page_size) / kBlock, head, HD);
        codes = (which ? a.codes[1] : a.codes[0]) + at.codes;
        scale = (which ? a.scales[1] : a.scales[0]) + at.scale;
        if (keep) e_old = min(max((int)*scale - 127, kScaleLeast), kScaleMost);
    }
    // V's codes that stay, on their way with the scale.
    const bool whole = keep == 0 && stop == kBlock;
    u32x4 *const v_to = (u32x4 *)(codes + u * kBlock);  // dim u's 32 positions
    u32x4 stay[2] = {};
    if (which && any && !whole) stay[0] = v_to[0], stay[1] = v_to[1];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float m = fabsf(v[i][k / 4][k % 4]);
            most = fmaxf(most, m < INFINITY ? m : 0.f);
        }
    most = wave_max(most);
    if constexpr (HD > 64) {  // two waves a block
        if ((tid & 63) == 0) s_max[tid >> 6] = most;
        __syncthreads();
        most = fmaxf(s_max[2 * mine], s_max[2 * mine + 1]);
    }
    const int e = max(exponent_for(most), e_old);
    const float inv = two_to(-e), grown = two_to(max(e_old - e, -126));
    if (any && u == 0) *scale = (uint8_t)(e + 127);
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = codes_of(v[i][0], inv), hi[i] = codes_of(v[i][1], inv);
    if (!which) {
        if (!any) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint2 *to = (uint2 *)(codes + d / 32 * (kBlock * 32) + (p + i) * 32 + d % 32);
            if (p + i >= keep && p + i < stop) {
                *to = make_uint2(lo[i], hi[i]);
            } else if (p + i < keep && e > e_old) {
                const uint2 o = *to;
                *to = make_uint2(rescaled(o.x, grown), rescaled(o.y, grown));
            }
        }
        return;
    }
    uint32_t tl[4], th[4];
    turn4(lo, tl);
    turn4(hi, th);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        *(uint32_t *)(s_v[mine] + turn_at(d + i) + p) = tl[i];
        *(uint32_t *)(s_v[mine] + turn_at(d + 4 + i) + p) = th[i];
    }
    __syncthreads();
    if (!any) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        u32x4 w = *(const u32x4 *)(s_v[mine] + turn_at(u) + 16 * j);
        if (!whole) {
            const u32x4 o = stay[j];
            auto below = [](int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; };  // the first n bytes
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = 16 * j + 4 * k;
                const uint32_t old = below(keep - at), fresh = below(stop - at) & ~old;
                const uint32_t kept = e > e_old ? rescaled(o[k], grown) : o[k];
                w[k] = (w[k] & fresh) | (kept & old) | (o[k] & ~(fresh | old));
            }
        }
        v_to[j] = w;
    }
}

// ---------------------------------------------------------------------------
// A decode step's row: RoPE on its query and key heads, its K and V quantised into
// the position that the device holds; a thread an element, HD of them a head. The
// bits of a rotation by launch_rope_append and an append, which took 3.5 us a layer
// more. Bound by its round trips: position, page, scale.
// ---------------------------------------------------------------------------
struct RopeArgs {
    const float *qkv;  // [q | k | v]
    float *q;
    Kv8Cache kv;
    int q_heads, rotary_dim;
    const float *cos, *sin;  // [position][rotary_dim / 2]
    const int32_t *pos_dev;
};

template <int HD>
__global__ __launch_bounds__(kThreads) void kv8_rope_append_kernel(RopeArgs a) {
    __shared__ float s_max[kThreads / 64];
    const int tid = threadIdx.x, d = tid % HD, kvh = a.kv.g.kv_heads;
    const int head = (int)blockIdx.x * (kThreads / HD) + tid / HD;  // q, then k, then v heads
    const bool there = head < a.q_heads + 2 * kvh, v = head >= a.q_heads + kvh;
    const float *src = a.qkv + (size_t)(there ? head : 0) * HD;
    const int pos = *a.pos_dev, keep = pos % kBlock, half = a.rotary_dim / 2;
    const float *cr = a.cos + (size_t)pos * half, *sr = a.sin + (size_t)pos * half;
    const float x = v ? src[d] : rope_elem(src, d, half, a.rotary_dim, cr, sr);
    float most = fabsf(x);
    most = wave_max(most < INFINITY ? most : 0.f);
    if constexpr (HD > 64) {  // two waves a head
        if ((tid & 63) == 0) s_max[tid >> 6] = most;
        __syncthreads();
        most = fmaxf(s_max[tid / HD * 2], s_max[tid / HD * 2 + 1]);
    }
    uint8_t *codes = nullptr, *scale = nullptr;
    int e_old = kScaleLeast;
    const bool writes = there && head >= a.q_heads;
    if (there && !writes) a.q[(size_t)head * HD + d] = x;
    if (writes) {
        const int page = a.kv.g.page_table[pos / a.kv.g.page_size];
        const BlockAt at = block_at(a.kv.g, page, pos % a.kv.g.page_size / kBlock, (head - a.q_heads) % kvh, HD);
        codes = (v ? a.kv.v : a.kv.k) + at.codes;
        scale = (v ? a.kv.v_scales : a.kv.k_scales) + at.scale;
        if (keep) e_old = min(max((int)*scale - 127, kScaleLeast), kScaleMost);
    }
    if constexpr (HD > 64) __syncthreads();  // both waves have the scale before one writes it
    if (!writes) return;
    const int e = max(exponent_for(most), e_old);
    const uint32_t code = codes_of(f32x4{x, 0.f, 0.f, 0.f}, two_to(-e)) & 0xFFu;
    if (d == 0) *scale = (uint8_t)(e + 127);
    if (e > e_old && keep) {  // earlier rows: 32 bytes a thread, of K a position's, of V a dim's
        const float grown = two_to(max(e_old - e, -126));
        u32x4 *to = (u32x4 *)(codes + d * kBlock);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const u32x4 o = to[j];
            u32x4 w = o;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int n = v ? min(max(keep - (16 * j + 4 * k), 0), 4) : d % kBlock < keep ? 4 : 0;  // bytes of them
                const uint32_t old = n == 4 ? ~0u : (1u << (8 * n)) - 1;
                w[k] = (rescaled(o[k], grown) & old) | (o[k] & ~old);
                if (v && (keep - 16 * j) / 4 == k && keep / 16 == j)
                    w[k] = (w[k] & ~(0xFFu << (8 * (keep % 4)))) | code << (8 * (keep % 4));
            }
            if (v || d % kBlock < keep) to[j] = w;
        }
        if (v) return;
    }
    codes[v ? d * kBlock + keep : d / 32 * (kBlock * 32) + keep * 32 + d % 32] = (uint8_t)code;
}

// ---------------------------------------------------------------------------
// Read: threads and their values as in the append. 32,768 positions of 4 KV heads
// of 128 as BF16 (100 MB): 16.3 us, 6.2 TB/s (21.9 with a byte at a time from LDS and
// stores that pass through the caches).
// ---------------------------------------------------------------------------
struct ReadArgs {
    const uint8_t *codes[2], *scales[2];
    Kv8Geom g;
    int begin, n;
    void *out[2];
};

__device__ __forceinline__ void store8(float *p, f32x4 a, f32x4 b) {
    __builtin_nontemporal_store(a, (f32x4 *)p);
    __builtin_nontemporal_store(b, (f32x4 *)(p + 4));
}
__device__ __forceinline__ void store8(uint16_t *p, f32x4 a, f32x4 b) {  // exact: the low halves are 0
    auto high = [](float x, float y) {
        return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    };
    const u32x4 w = u32x4{high(a[0], a[1]), high(a[2], a[3]), high(b[0], b[1]), high(b[2], b[3])};
    __builtin_nontemporal_store(w, (u32x4 *)p);
}

template <int HD, class T>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(ReadArgs a) {
    constexpr int RB = kRun<HD>;
    __shared__ __attribute__((aligned(16))) uint8_t s_v[RB][HD * kTurnRow];
    const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
    const int first = a.begin / kBlock, last = (a.begin + a.n - 1) / kBlock;
    const int mine = tid / HD;  // of the run's blocks
    const int blk = min(first + (int)blockIdx.x * RB + mine, last);
    const uint32_t per = (uint32_t)a.g.page_size / kBlock, page = (uint32_t)blk / per;
    const BlockAt at = block_at(a.g, a.g.page_table[page], blk - (int)(page * per), head, HD);
    const uint8_t *codes = (which ? a.codes[1] : a.codes[0]) + at.codes;
    const float scale = two_to((int)(which ? a.scales[1] : a.scales[0])[at.scale] - 127);
    const int u = tid % HD, d = u % (HD / 8) * 8, p = u / (HD / 8) * 4;
    uint32_t lo[4], hi[4];  // dims d .. d + 3 and d + 4 .. d + 7 of positions p ..
    if (!which) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint2 w = *(const uint2 *)(codes + d / 32 * (kBlock * 32) + (p + i) * 32 + d % 32);
            lo[i] = w.x, hi[i] = w.y;
        }
    } else {
        const u32x4 x = *(const u32x4 *)(codes + u * kBlock), y = *(const u32x4 *)(codes + u * kBlock + 16);
        uint8_t *to = s_v[mine] + turn_at(u);
        *(u32x4 *)to = x;
        *(u32x4 *)(to + 16) = y;
        __syncthreads();
        uint32_t x4[4], y4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t *from = s_v[mine] + turn_at(d + i) + p;
            x4[i] = *(const uint32_t *)from;
            y4[i] = *(const uint32_t *)(from + 4 * kBlock);
        }
        turn4(x4, lo);
        turn4(y4, hi);
    }
    if (first + (int)blockIdx.x * RB + mine > last) return;
    T *out = (T *)(which ? a.out[1] : a.out[0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = blk * kBlock + p + i - a.begin;
        if (row < 0 || row >= a.n) continue;
        store8(out + (size_t)row * a.g.kv_heads * HD + (size_t)head * HD + d, code_values(lo[i]) * scale,
               code_values(hi[i]) * scale);
    }
}

// ---------------------------------------------------------------------------
// Attention: row i is at position offset + i and sees the positions p <= offset +
// i that are above offset + i - window (all with window 0) or below sinks.
// ---------------------------------------------------------------------------
struct Kv8AttnArgs {
    const float *q;
    const uint8_t *k, *v, *k_scales, *v_scales;
    Kv8Geom g;
    int q_heads, rows, offset, window, sinks;
    uint32_t over_group;  // ceil(2^32 / G) for G > 1 query heads per KV head
    float *out;
    float *part;  // [row][head][split][HD]: weighted sums
    float2 *ml;   // [row][head][split]: reference (log2 units), weight sum
    const int32_t *pos_dev;     // offset's word on the device (null: offset)
    uint16_t *out_hi, *out_lo;  // BF16 halves of out (null: not written); out may then be null
};

__device__ __forceinline__ int first_pos(const Kv8AttnArgs &a) { return a.pos_dev ? *a.pos_dev : a.offset; }

// N consecutive outputs from element i on, and their BF16 halves where asked for.
template <int N>
__device__ __forceinline__ void store_out(const Kv8AttnArgs &a, size_t i, const float (&v)[N]) {
    if (a.out) {
        if constexpr (N == 4) *(f32x4 *)(a.out + i) = f32x4{v[0], v[1], v[2], v[3]};
        else if constexpr (N == 2) *(float2 *)(a.out + i) = make_float2(v[0], v[1]);
        else a.out[i] = v[0];
    }
    if (!a.out_hi) return;
    uint16_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const __bf16 hb = (__bf16)v[k];
        h[k] = __builtin_bit_cast(uint16_t, hb);
        l[k] = __builtin_bit_cast(uint16_t, (__bf16)(v[k] - (float)hb));
    }
    if constexpr (N == 4) {
        *(uint2 *)(a.out_hi + i) = make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
        *(uint2 *)(a.out_lo + i) = make_uint2((uint32_t)l[0] | (uint32_t)l[1] << 16, (uint32_t)l[2] | (uint32_t)l[3] << 16);
    } else if constexpr (N == 2) {
        *(uint32_t *)(a.out_hi + i) = (uint32_t)h[0] | (uint32_t)h[1] << 16;
        *(uint32_t *)(a.out_lo + i) = (uint32_t)l[0] | (uint32_t)l[1] << 16;
    } else {
        a.out_hi[i] = h[0];
        a.out_lo[i] = l[0];
    }
}

// The first position of the window of a row at `pos` (0 without one).
__device__ __forceinline__ int window_start(const Kv8AttnArgs &a, int pos) {
    return a.window ? max(pos + 1 - a.window, 0) : 0;
}

// One row and head in plain f32 products, a wave: the maximum and the weight sum,
// then the values under finished weights, so that finite values average to a
// finite output and an infinity or a NaN in a value that the row sees shows. A
// call, so that it takes no registers of the loops it is behind, and one that gets
// the kernel's arguments where they are, so that it needs no stack (kernels with
// one start some 5 us later).
typedef const __attribute__((address_space(4))) Kv8AttnArgs *Kv8KernArgs;
__device__ __forceinline__ Kv8KernArgs kernel_args() { return (Kv8KernArgs)__builtin_amdgcn_kernarg_segment_ptr(); }
template <int HD>
__device__ __attribute__((noinline)) void plain_row(Kv8KernArgs args, int row, int head) {
    const Kv8AttnArgs a = *(const Kv8AttnArgs *)args;
    constexpr int C = HD / 32;
    const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
    const int g = head / (a.q_heads / a.g.kv_heads), pos = first_pos(a) + row;
    const int lo = window_start(a, pos), sinks = a.window ? min(a.sinks, lo) : 0;
    const float sl2 = (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f;
    const float *q = a.q + ((size_t)row * a.q_heads + head) * HD + 16 * half;
    float m = -INFINITY, l = 0.f, o[C];
#pragma unroll
    for (int u = 0; u < C; ++u) o[u] = 0.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
        for (int b = 0; b <= pos / kBlock; ++b) {
            if (b * kBlock >= sinks && (b + 1) * kBlock <= lo) b = lo / kBlock;
            const int page = a.g.page_table[(size_t)b * kBlock / a.g.page_size];
            const BlockAt at = block_at(a.g, page, b % (a.g.page_size / kBlock), g, HD);
            // (Scaled values, not codes: those over large queries could pass the range.)
            const float k_scale = two_to((int)a.k_scales[at.scale] - 127);
            float dot = 0.f;
#pragma unroll 1
            for (int c = 0; c < C; ++c) {
                const uint32_t *w = (const uint32_t *)(a.k + at.codes + c * (kBlock * 32) + n * 32 + 16 * half);
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                    const f32x4 k = code_values(w[i]) * k_scale, x = *(const f32x4 *)(q + 32 * c + 4 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dot = fmaf(k[e], x[e], dot);
                }
            }
            dot += __shfl_xor(dot, 32, 64);
            const int p = b * kBlock + n;
            const bool seen = p <= pos && (p >= lo || p < sinks);
            const float s = seen ? dot * sl2 : -INFINITY;
            if (pass == 0) {
                const float mn = fmaxf(m, wave_max(s));
                const float w = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
                l = (m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f(m - mn)) + 0.5f * wave_sum(w);  // both halves hold it
                m = mn;
            } else {
                const float w = seen ? __builtin_amdgcn_exp2f(s - m) / l : 0.f;
                const float scale = two_to((int)a.v_scales[at.scale] - 127);
#pragma unroll 1
                for (int j = 16 * half; j < 16 * half + 16; j += 4) {
                    float wj[4];
                    bool there[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int pj = b * kBlock + j + e;
                        wj[e] = __shfl(w, j + e, 64);
                        there[e] = pj <= pos && (pj >= lo || pj < sinks);
                    }
#pragma unroll
                    for (int u = 0; u < C; ++u) {
                        const f32x4 x = code_values(*(const uint32_t *)(a.v + at.codes + (32 * u + n) * kBlock + j)) * scale;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[u] = there[e] ? fmaf(wj[e], x[e], o[u]) : o[u];
                    }
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < C; ++u) {
        const float v[1] = {o[u] + __shfl_xor(o[u], 32, 64)};
        if (half == 0) store_out<1>(a, ((size_t)row * a.q_heads + head) * HD + 32 * u + n, v);
    }
}

// The blocks of positions that a range of rows sees, in order: the first `sink`
// ones, then blocks from `first` on, `count` in all.
struct Reach {
    int sink, first, count;
    __device__ int block(int i) const { return i < sink ? i : first + i - sink; }
};
__host__ __device__ __forceinline__ Reach reach_of(int pos_lo, int pos_hi, int window, int sinks) {
    const int lo = window && pos_lo + 1 > window ? pos_lo + 1 - window : 0;
    Reach r;
    r.sink = ((sinks < lo ? sinks : lo) + kBlock - 1) / kBlock;
    r.first = lo / kBlock > r.sink ? lo / kBlock : r.sink;
    r.count = r.sink + pos_hi / kBlock + 1 - r.first;
    return r;
}

// ---------------------------------------------------------------------------
// On the matrix cores: v_mfma_f32_32x32x16_f16 over 32 "M rows" (query row x head
// of the KV group) a wave and blocks of 32 positions,
//   S^T = K Q^T     A = K: lane (n, h) takes the 16 dims 32 c + 16 h .. of position
//                   kpos(n); B = the queries, in registers.
//   O^T += V^T P^T  A = V^T: lane (n, h) takes positions 16 h .. + 15 of dim
//                   32 u + n; B = the probabilities: with that kpos lane (m, h)
//                   holds those of its row at positions 16 h .. + 15, where the
//                   first product leaves them.
// Codes are exact F16 numbers. Queries are two F16 parts, 22 bits of a row's largest
// (a power of two of each row's own fills F16's range). Probabilities are two parts as
// well; a long tail behind one large weight (a sink, whose value may be 0) is made of
// weights far below F16's normal numbers, so the low part carries 2^11 and meets V times
// 2^-11: 22 bits for a weight of 2^-21 of the largest that a wave has seen and more, for
// smaller ones 2^-44 of it. (Low parts without a factor lose weights below 2^-25: 3 % of
// the time of 512 rows on 4,096, 73.5 against 75.9 us, for outputs 1e-4 off.) A K scale
// multiplies the scores, a V scale comes with the conversion, relative
// to one that the running sums carry (a power of two, changed without rounding).
//
// Blocks of 8 waves, one a CU: WR of them hold 32 M rows each, the other 8 / WR - 1
// times as many take other blocks of positions (so that a short call fills its CUs
// without a second launch); two waves a SIMD of 220 to 256 registers. One row wave:
// K and V go from memory into registers, no wave waits for another. More: direct
// copies fill three tiles of LDS, a barrier a tile. (Few rows have a kernel of their
// own, kv8_few_kernel.)
//
// Bound: with many rows vector and matrix instructions, which hardly overlap (512 rows
// on 4,096, 32 / 8 heads of 128: 76.9 us, vector instructions in 55 % of the SIMDs'
// cycles, matrix ones in 46 %; queries in and outputs out take 12); with few round
// trips.
// ---------------------------------------------------------------------------
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ int kpos(int n) { return 16 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3); }

// Four codes times 2^k as F16, and eight.
__device__ __forceinline__ uint2 codes_f16x4(uint32_t w, float scale) {
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true)));
}
__device__ __forceinline__ f16x8 operand(uint2 a, uint2 b) {
    return __builtin_bit_cast(f16x8, u32x4{a.x, a.y, b.x, b.y});
}
__device__ __forceinline__ f16x8 codes_f16(uint32_t a, uint32_t b, float scale) {
    return operand(codes_f16x4(a, scale), codes_f16x4(b, scale));
}
// The larger of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Two values' F16 parts: the first 11 bits of each (cut off, so that the subtraction
// takes no conversion back) and the rest, rounded. Below F16's normal numbers both
// round at 2^-25.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo) {
    const float ha = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u), hb = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
    hi = __builtin_bit_cast(uint32_t, f16x2{(_Float16)ha, (_Float16)hb});
    lo = __builtin_bit_cast(uint32_t, f16x2{(_Float16)(a - ha), (_Float16)(b - hb)});
}

// Two weights' F16 parts: the first 11 bits of each, and the rest times 2^11, which
// meets V times 2^-11 (kLow): a weight below F16's normal numbers keeps its bits
// down to 2^-35. Rounded once, by at most 2^-36 or 2^-23 of it.
constexpr float kLowUp = 0x1p11f;
constexpr _Float16 kLow = (_Float16)0x1p-11f;
__device__ __forceinline__ void split_weights(float a, float b, uint32_t &hi, uint32_t &lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, f16x2{(_Float16)fmaf((float)h[0], -kLowUp, a * kLowUp),
                                            (_Float16)fmaf((float)h[1], -kLowUp, b * kLowUp)});
}
// Weights are taken against a reference kLift powers of two below the largest score,
// raised when a score passes it by more than kLift + kRaise: 2^14 at most (F16 ends
// at 2^16), 2^8 at least for the largest key of a wave. (Of a key 2^-25 of it 2^-17 is
// left, 18 bits.) The factor is in weights and sums alike and drops out in the quotient.
constexpr float kLift = 8.0f, kRaise = 6.0f;

// A block's weights, added up, onto the sum of all: compensated, so that a long tail
// behind one large weight is not lost to it (N weights of 2^-26 of it are N 2^-26 of
// the sum, each below its last bit). Four instructions a block.
struct WeightSum {
    float sum = 0.f, over = 0.f;  // the true sum is sum - over
    __device__ __forceinline__ void add(float x) {
        const float y = x - over, t = sum + y;
        over = (t - sum) - y;
        sum = t;
    }
    __device__ __forceinline__ void scale(float f) { sum *= f, over *= f; }
};

// A wave's output sums are in units of 2^e; V's codes meet them under 2^(e_v - e), which
// is exact in F16 for differences of -down .. 7. Past these the sums move to the block's
// unit, a power of two away, without rounding. Where units have come to lie more than
// 2^kFar apart, the rows are computed again (a NaN weight sum): weights are right to
// 2^-44 of the largest alone, which is not enough for a value 2^44 times as large, and
// sums could end behind the type's range, in one step or in several. A block of zeros
// takes any unit, and sums that are 0 have none.
constexpr int kFar = 20;
struct ValueUnit {
    int e = 0, least = 0, most = 0;
    // The factor of a block's codes; `codes` and `sums` return the bits of all that a lane
    // holds of either, `move` multiplies the sums by 2^n.
    template <class Codes, class Sums, class Move>
    __device__ __forceinline__ float factor(int e_v, bool first, int down, WeightSum &l, Codes codes, Sums sums, Move move) {
        if (first) e = least = most = e_v;
        if (e_v - e > 7 || e_v - e < -down) {
            if (!__any(codes() & 0x7F7F7F7Fu)) return 1.f;
            if (!__any(sums() << 1)) least = most = e_v;
            least = min(least, e_v), most = max(most, e_v);
            if (most - least > kFar) l.sum = NAN;
            move(e - e_v);
            e = e_v;
        }
        return two_to(e_v - e);
    }
};

// Which of the positions base .. base + 15 lie at or below `last` and at or above
// `first` or below `sinks`, a bit each.
__device__ __forceinline__ uint32_t seen_bits(int base, int last, int first, int sinks) {
    auto below = [](int n) { return 0xFFFFu >> (16 - min(max(n, 0), 16)); };  // the first n
    return below(last - base + 1) & (~below(first - base) | below(sinks - base));
}

// The factors of a row's waves in the sum of their outputs, from words of each
// (reference, weight sum, unit), `stride` apart; returned: what the sum is multiplied
// with, 1 / (weight sum), or with `ml` (a split's word) 1. A wave that saw nothing
// counts nothing; a NaN sum shows. (The quotient comes last: with the least unit a
// factor divided by a large sum would be no normal number.)
template <int N>
__device__ __forceinline__ float wave_factors(const f32x4 *words, int stride, float (&f)[N], bool one, float2 *ml) {
    f32x4 word[N];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        word[k] = words[k * stride];
        top = fmaxf(top, word[k][0]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float m = word[k][0], w = m == -INFINITY && word[k][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - top);
        sum += w != 0.f || word[k][1] != word[k][1] ? w * word[k][1] : 0.f;
        f[k] = w * word[k][2];
    }
    if (ml) *ml = make_float2(top, sum);
    return one ? 1.0f / sum : 1.f;
}

constexpr int kWaves = 8;
template <int HD>
constexpr int kRowPad = HD + 4;  // floats of a row of outputs in LDS
constexpr size_t kStage = 96 * 1024;   // LDS of three tiles
template <int HD>
constexpr int kQRow = HD * 4 + 16;     // bytes of a query row's parts in LDS: high, low, padding
// A block's LDS: tiles, then the waves' sums in their place; query rows on their way
// to the operands (of one row wave behind the sums, else in the third tile's place
// and behind it); a word of each wave and row (reference, weight sum, the sums' unit);
// the query rows' exponents; rows to compute again.
template <int HD, int WR>
constexpr size_t kQueriesAt = WR == 1 ? kWaves * 32 * kRowPad<HD> * 4 : kStage / 3 * 2;
template <int HD, int WR>
constexpr size_t kWordsAt = std::max({WR == 1 ? (size_t)0 : kStage, (size_t)(kWaves * 32 * kRowPad<HD> * 4),
                                      kQueriesAt<HD, WR> + 32 * WR * kQRow<HD>});
template <int HD, int WR>
constexpr size_t kv8_attn_lds_bytes() { return kWordsAt<HD, WR> + kWaves * 32 * 16 + 32 * WR * 4 + 16; }

template <int HD, int WR>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void kv8_attn_kernel(Kv8AttnArgs a, int S) {
    constexpr int WK = kWaves / WR, C = HD / 32;
    constexpr bool DIRECT = WR == 1;    // no other wave reads this wave's blocks
    constexpr int PIECES = 2 * C / WR;  // of a block, copied by a wave (1 KB each)
    constexpr int BB = kBlock * HD;     // bytes of a block of K or V
    constexpr int NB = DIRECT ? 1 : (int)kStage / (3 * WK * 2 * BB);  // a key wave's blocks of a tile
    extern __shared__ __attribute__((aligned(256))) uint8_t smem[];
    f32x4 *words = (f32x4 *)(smem + kWordsAt<HD, WR>);
    int *sq_exp = (int *)(words + kWaves * 32);
    int *odd = sq_exp + 32 * WR;  // a row wave's rows to compute again
    auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int lane = threadIdx.x & 63;
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int wr = wave % WR, wk = wave / WR;
    const int n = lane & 31, half = lane >> 5;
    // Division by G: exact below 2^29 (the launch refuses more rows).
    const int G = a.q_heads / a.g.kv_heads, M = a.rows * G, RB = (M + 32 * WR - 1) / (32 * WR);
    auto over_g = [&](int x) { return G == 1 ? x : (int)__umulhi((uint32_t)x, a.over_group); };
    // Blocks b, b + 8, .. run on one XCD: each takes a run of (KV head, split, row
    // block), so that few of them read a cache's block. Rows that see the most and
    // the fewest positions alternate.
    const int total = RB * S * a.g.kv_heads, run = (total + 7) / 8;
    const int work = (int)blockIdx.x % 8 * run + (int)blockIdx.x / 8;
    if (work >= total) return;
    const int pair = work / RB, turn = work % RB, rb = uniform(turn & 1 ? turn / 2 : RB - 1 - turn / 2);
    const int g = uniform(pair % a.g.kv_heads), split = uniform(pair / a.g.kv_heads);
    const int m0 = rb * 32 * WR, m = m0 + wr * 32 + n;
    const bool rvalid = m < M;
    const int offset = uniform(first_pos(a)), pos = offset + (rvalid ? over_g(m) : 0), lo = window_start(a, pos);
    // Rows of the block and of the wave.
    const int pos_lo = uniform(offset + over_g(m0)), pos_hi = uniform(offset + over_g(min(M, m0 + 32 * WR) - 1));
    const int wave_lo = uniform(offset + over_g(min(m0 + wr * 32, M - 1)));
    const int wave_hi = uniform(offset + over_g(min(M, m0 + wr * 32 + 32) - 1));
    const int seen_lo = window_start(a, pos_lo), wave_first = window_start(a, wave_hi);
    const Reach reach = reach_of(pos_lo, pos_hi, a.window, a.sinks);
    const int each = reach.count / S, extra = reach.count % S;
    const int begin = uniform(split * each + min(split, extra)), end = uniform(begin + each + (split < extra));
    const int steps = (end - begin + WK - 1) / WK;  // of the longest key wave
    const int mine = max(end - begin - wk + WK - 1, 0) / WK;

    // Where this wave's next 64 blocks lie and their scales, a lane each.
    int held_at = 0;
    uint32_t held_k = 0, held_v = 0;
    auto look_up = [&](int i0) {
        const int i = min(i0 + lane, max(mine - 1, 0));
        const int b = reach.block(min(begin + wk + i * WK, reach.count - 1));
        const int per = a.g.page_size / kBlock;
        const int page = a.g.page_table[b / per];
        held_at = (page * a.g.kv_heads + g) * per + b % per;
    };
    auto look_up_scales = [&]() {
        held_k = a.k_scales[held_at];
        held_v = a.v_scales[held_at];
    };
    // Waited for here, not at every use.
    auto landed = [&]() { asm volatile("" : "+v"(held_k), "+v"(held_v)); };
    auto at_of = [&](int i) { return (size_t)(uint32_t)__builtin_amdgcn_readlane(held_at, i & 63); };

    const int koff = kpos(n) * 32 + 16 * half, voff = n * kBlock + 16 * half;
    u32x4 kr[C], vr[C];
    auto load_k = [&](size_t at) {
#pragma unroll
        for (int c = 0; c < C; ++c) kr[c] = *(const u32x4 *)(a.k + at * BB + 1024 * c + koff);
    };
    auto load_v = [&](size_t at) {
#pragma unroll
        for (int c = 0; c < C; ++c) vr[c] = *(const u32x4 *)(a.v + at * BB + 1024 * c + voff);
    };
    // A block's pieces to LDS, each lane's own 16 bytes at 16 lane: [K pieces | V pieces].
    auto copy = [&](size_t at, int i) {
        uint8_t *to = smem + (i % (3 * NB) * WK + wk) * 2 * BB;
        const __amdgpu_buffer_rsrc_t rk =
            __builtin_amdgcn_make_buffer_rsrc((void *)(a.k + at * BB), (short)0, BB, 0x00020000);
        const __amdgpu_buffer_rsrc_t rv =
            __builtin_amdgcn_make_buffer_rsrc((void *)(a.v + at * BB), (short)0, BB, 0x00020000);
#pragma unroll
        for (int j = 0; j < PIECES / 2; ++j) {
            const int c = wr * (PIECES / 2) + j;
            buf_to_lds<16>(rk, to + 1024 * c, koff, 1024 * c);
            buf_to_lds<16>(rv, to + BB + 1024 * c, voff, 1024 * c);
        }
        if constexpr (PIECES == 1) {  // K by the first half of the waves, V by the others
            const int c = wr % C;
            if (wr < C) buf_to_lds<16>(rk, to + 1024 * c, koff, 1024 * c);
            else buf_to_lds<16>(rv, to + BB + 1024 * c, voff, 1024 * c);
        }
    };

    // The start: page entries, queries, the first blocks and their scales, every load
    // in flight before the first is waited for. Queries come in whole rows, times
    // log2(e) / sqrt(HD) and by a power of two of each row's own to 2^14 .. 2^15, and
    // reach the matrix operands by way of LDS (from memory an operand is 16 bytes of
    // each of 32 rows a load: 4 us for the eight waves).
    look_up(0);
    uint8_t *sq = smem + kQueriesAt<HD, WR>;
    constexpr int LPR = HD / 4, RPI = 64 / LPR, QI = 4 * WR / RPI;  // lanes a row, rows a load, loads a wave
    {
        f32x4 raw[QI];
#pragma unroll
        for (int j = 0; j < QI; ++j) {
            const int r = m0 + (wave * QI + j) * RPI + lane / LPR, rr = min(r, M - 1);
            raw[j] = *(const f32x4 *)(a.q + ((size_t)over_g(rr) * a.q_heads + g * G + rr - over_g(rr) * G) * HD + lane % LPR * 4);
        }
        __builtin_amdgcn_sched_barrier(0);
        look_up_scales();
        // (Counts known here, so that the queries are not waited for with the copies:
        // behind the last block it is copied again.)
        if constexpr (DIRECT) {
            load_k(at_of(0)), load_v(at_of(0));
        } else {
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) copy(at_of(max(min(i, mine - 1), 0)), i);
        }
        __builtin_amdgcn_sched_barrier(0);
        const float sl2 = (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f;
#pragma unroll
        for (int j = 0; j < QI; ++j) {
            const int r = (wave * QI + j) * RPI + lane / LPR;
            f32x4 v = raw[j] * (m0 + r < M ? sl2 : 0.f);
            float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
            for (int d = 1; d < LPR; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
            const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -112), 127) - 14;
            v *= two_to(-e);
            uint2 hi, lo;
            split_f16(v[0], v[1], hi.x, lo.x);
            split_f16(v[2], v[3], hi.y, lo.y);
            *(uint2 *)(sq + r * kQRow<HD> + lane % LPR * 8) = hi;
            *(uint2 *)(sq + r * kQRow<HD> + HD * 2 + lane % LPR * 8) = lo;
            if (lane % LPR == 0) sq_exp[r] = e;
        }
    }
    landed();
    lds_barrier();
    f16x8 qh[2 * C], ql[2 * C];
    const int q_exp = sq_exp[wr * 32 + n];
#pragma unroll
    for (int k = 0; k < 2 * C; ++k) {
        const uint8_t *from = sq + (wr * 32 + n) * kQRow<HD> + k / 2 * 64 + 32 * half + 16 * (k % 2);
        qh[k] = *(const f16x8 *)from;
        ql[k] = *(const f16x8 *)(from + HD * 2);
    }

    f32x16 o[C];
#pragma unroll
    for (int u = 0; u < C; ++u) o[u] = f32x16{};
    float m2 = -INFINITY;
    WeightSum l;
    ValueUnit unit;  // of o
    uint32_t now_k = held_k, now_v = held_v, next_k = 0, next_v = 0;  // (the next ones are looked up a tile ahead)
    auto lds_at = [&](int i) { return smem + (i % (3 * NB) * WK + wk) * 2 * BB + 16 * lane; };
    auto read_k = [&](int i) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int c = 0; c < C; ++c) kr[c] = *(const u32x4 *)(lds_at(i) + 1024 * c);
        }
    };
    auto read_v = [&](int i) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int u = 0; u < C; ++u) vr[u] = *(const u32x4 *)(lds_at(i) + BB + 1024 * u);
        }
    };
    auto scores = [&](f32x16 &s) {
        s = f32x16{};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const f16x8 k0 = codes_f16(kr[c][0], kr[c][1], 1.f), k1 = codes_f16(kr[c][2], kr[c][3], 1.f);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[2 * c], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[2 * c], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[2 * c + 1], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[2 * c + 1], s, 0, 0, 0);
        }
    };
    // Masks, where a row of the wave does not see all of block i.
    auto mask = [&](int i, f32x16 &s) {
        const int p0 = reach.block(begin + wk + i * WK) * kBlock;
        if (p0 + kBlock - 1 > wave_lo || (p0 < wave_first && p0 + kBlock > a.sinks)) {
            const uint32_t bits = seen_bits(p0 + 16 * half, pos, lo, a.sinks);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = bits >> r & 1 ? s[r] : -INFINITY;
        }
    };
    auto largest = [&](const f32x16 &s) {
        float t = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) t = fmaxf(t, s[r]);
        return max_halves(t);
    };
    auto scale_of = [&](int i) {  // of block i's scores
        return ldexpf(1.f, max(q_exp + (int)__builtin_amdgcn_readlane(now_k, i & 63) - 127, -126));
    };
    // The running sums are rescaled only where the reference is raised.
    auto raise_to = [&](float tmax) {
        const bool raise = tmax > m2 + (kLift + kRaise);
        if (__any(raise)) {
            const float mnew = raise ? tmax - kLift : m2;
            const float alpha = raise ? __builtin_amdgcn_exp2f(m2 - mnew) : 1.f;
            l.scale(alpha);
#pragma unroll
            for (int u = 0; u < C; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[u][r] *= alpha;
            m2 = mnew;
        }
    };
    f32x16 s;
    float fs = 0.f;
    auto reference = [&]() { return m2 == -INFINITY ? 0.f : m2; };
    // The factor of block i's codes, exact in F16 times 2^-11 too.
    auto value_scale = [&](int i) {
        return unit.factor(
            (int)__builtin_amdgcn_readlane(now_v, i & 63) - 127, i == 0, 4, l,
            [&]() {
                uint32_t codes = 0;
#pragma unroll
                for (int u = 0; u < C; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) codes |= vr[u][j];
                return codes;
            },
            [&]() {
                uint32_t sums = 0;
#pragma unroll
                for (int u = 0; u < C; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums |= __float_as_uint(o[u][r]);
                return sums;
            },
            [&](int n) {
#pragma unroll
                for (int u = 0; u < C; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[u][r] = ldexpf(o[u][r], n);
            });
    };
    // Positions that no row of the block sees may hold anything: zeros.
    auto clear_v = [&](int i) {
        const int p0 = reach.block(begin + wk + i * WK) * kBlock;
        if (p0 + kBlock - 1 > pos_hi || (p0 < seen_lo && p0 + kBlock > a.sinks)) {
            const uint32_t bits = seen_bits(p0 + 16 * half, pos_hi, seen_lo, a.sinks);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t bytes = ((bits >> (4 * j) & 15) * 0x204081u & 0x01010101u) * 0xFFu;
#pragma unroll
                for (int u = 0; u < C; ++u) vr[u][j] &= bytes;
            }
        }
    };
    // Probability r - 1 of a block from its score's exponential, in two F16 parts (a
    // pair at a time), and the exponential of score r, so that none is waited for.
    uint32_t ph[8], pl[8];
    float block_sum = 0.f;
    auto exponential = [&](int r, float mref, f32x16 &s) {
        if (r < 16) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], fs, -mref));
        if (r > 0) block_sum = r == 1 ? s[0] : block_sum + s[r - 1];
        if (r == 16) l.add(block_sum);
        if (r > 0 && r % 2 == 0) {
            split_weights(s[r - 2], s[r - 1], ph[r / 2 - 1], pl[r / 2 - 1]);
        }
    };
    auto part = [&](const uint32_t (&p)[8], int k) {
        return __builtin_bit_cast(f16x8, u32x4{p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3]});
    };
    if constexpr (DIRECT) {
        // No other wave waits for this one's blocks: the next block's loads are issued
        // as soon as the registers are free.
        for (int i = 0; i < mine; ++i) {
            if (i > 0 && (i & 63) == 0) now_k = held_k, now_v = held_v;
            if (((i + 1) & 63) == 0 && i + 1 < mine) look_up(i + 1), look_up_scales(), landed();
            const size_t at_next = at_of(i + 1);
            scores(s);
            if (i + 1 < mine) load_k(at_next);
            __builtin_amdgcn_sched_barrier(0);
            mask(i, s);
            fs = scale_of(i);
            raise_to(largest(s) * fs);
            const float mref = reference();
#pragma unroll
            for (int r = 0; r <= 16; ++r) exponential(r, mref, s);
            clear_v(i);
            const float vs = value_scale(i);
#pragma unroll
            for (int u = 0; u < C; ++u) {
                const f16x8 v0 = codes_f16(vr[u][0], vr[u][1], vs), v1 = codes_f16(vr[u][2], vr[u][3], vs);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, part(ph, 0), o[u], 0, 0, 0);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, part(ph, 1), o[u], 0, 0, 0);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0 * kLow, part(pl, 0), o[u], 0, 0, 0);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1 * kLow, part(pl, 1), o[u], 0, 0, 0);
            }
            if (i + 1 < mine) load_v(at_next);
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        // A block's exponentials are laid between the products of the next block's
        // scores, and the next maxima between its own V products: a wave's vector
        // instructions run while its matrix instructions do, and two waves of a SIMD that
        // do the same thing at the same time do not overlap. K and V are read from LDS
        // one phase before their use. Two steps a turn, so that scores change places
        // without moves (512 rows on 4,096 77.1 -> 75.9 us).
        // The first tile has landed (copies end in order; one block a tile: the second too).
        constexpr int LATER = NB == 1 ? 0 : NB * PIECES;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(LATER) : "memory");
        if (NB == 1 && mine > 2) copy(at_of(2), 2);
        if (mine > 0) {
            read_k(0);
            scores(s);
            mask(0, s);
            fs = scale_of(0);
            raise_to(largest(s) * fs);
            if (mine > 1) read_k(1);
        }
        constexpr int E = 4 / C;  // exponentials for a product
        auto step = [&](int i, f32x16 &s, f32x16 &t) {
            t = f32x16{};
            float vs = 0.f;
            if (i < mine) {
                read_v(i);
                const float mref = reference();
                uint2 k4[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) k4[q] = codes_f16x4(kr[0][q], 1.f);
                // (Behind the last block: scores of an earlier one, which nothing reads.)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const f16x8 k0 = operand(k4[0], k4[1]), k1 = operand(k4[2], k4[3]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        t = __builtin_amdgcn_mfma_f32_32x32x16_f16(q < 2 ? k0 : k1, q & 1 ? ql[2 * c + q / 2] : qh[2 * c + q / 2], t, 0,
                                                                   0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if (c + 1 < C) k4[q] = codes_f16x4(kr[c + 1][q], 1.f);
#pragma unroll
                        for (int x = 0; x < E; ++x) exponential((4 * c + q) * E + x, mref, s);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                exponential(16, mref, s);
            }
            // The tile of block i + 2: it has landed, and V of block i and all before is read
            // by all; the tile after it takes the place of the one before the last.
            const int ahead = i + 2 + NB;
            if ((i + 2) % NB == 0 && i + 2 < steps) {
                if ((ahead & 63) == 0 && ahead < mine) look_up(ahead), look_up_scales(), landed(), next_k = held_k, next_v = held_v;
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                for (int j = ahead; j < min(ahead + NB, mine); ++j) copy(at_of(j), j);
            }
            if (i >= mine) return;
            if (i + 2 < mine) read_k(i + 2);
            clear_v(i);
            vs = value_scale(i);
            if (i + 1 < mine) mask(i + 1, t);
            float tmax = t[0];
            uint2 v4[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v4[q] = codes_f16x4(vr[0][q], vs);
#pragma unroll
            for (int u = 0; u < C; ++u) {
                f16x8 v[2] = {operand(v4[0], v4[1]), operand(v4[2], v4[3])};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[q & 1], q < 2 ? part(ph, q) : part(pl, q - 2), o[u], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (q < 2) v[q] *= kLow;
                    if (u + 1 < C) v4[q] = codes_f16x4(vr[u + 1][q], vs);
#pragma unroll
                    for (int x = 0; x < E; ++x) tmax = fmaxf(tmax, t[(4 * u + q) * E + x]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (i + 1 < mine) {
                if (((i + 1) & 63) == 0) now_k = next_k, now_v = next_v;
                fs = scale_of(i + 1);
                raise_to(max_halves(tmax) * fs);
            }
        };
        f32x16 t;
        for (int i = 0; i < steps; i += 2) {
            step(i, s, t);
            if (i + 1 < steps) step(i + 1, t, s);
        }
    }
    // The key waves' parts meet in LDS. (In the tiles' place: their last reads are
    // done, and copies that nothing reads.)
    l.sum += __shfl_xor(l.sum, 32, 64);
    if constexpr (!DIRECT) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    const int held_rows = min(32 * WR, M - m0);
    if (rvalid) {
        float *so = (float *)smem + ((size_t)wave * 32 + n) * kRowPad<HD>;
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(f32x4 *)(so + 32 * u + 8 * q + 4 * half) =
                    f32x4{o[u][4 * q], o[u][4 * q + 1], o[u][4 * q + 2], o[u][4 * q + 3]};
        if (half == 0) words[wave * 32 + n] = f32x4{m2, l.sum, two_to(unit.e), 0.f};
    }
    if (threadIdx.x < WR) odd[threadIdx.x] = 0;
    __syncthreads();
    auto item_of = [&](int r) {  // row and head of the block's row r
        const int row = over_g(m0 + r);
        return (size_t)row * a.q_heads + g * G + (m0 + r - row * G);
    };
    auto factors = [&](int r, float (&f)[WK], bool to_part) {
        return wave_factors(words + r, WR * 32, f, S == 1, to_part ? a.ml + item_of(r) * S + split : nullptr);
    };
    // A few rows: every thread finds its row's factors, a barrier less (6.3 -> 5.9 us for
    // 333 rows of 14 / 2 heads of 64 on nothing). Many: a thread a row (1,000 windowed rows 42.7 -> 41.9).
    if constexpr (WR > 1) {
        const int r = (int)threadIdx.x;
        if (r < held_rows) {
            float f[WK];
            const float inv = factors(r, f, S > 1);
            words[r][1] = inv;
#pragma unroll
            for (int k = 0; k < WK; ++k) words[k * WR * 32 + r][0] = f[k];
        }
        __syncthreads();
    }
#pragma unroll WR
    for (int u = (int)threadIdx.x; u < held_rows * (HD / 4); u += 64 * kWaves) {  // 4 dims of a row
        const int r = u / (HD / 4), d = u % (HD / 4) * 4;
        float f[WK], inv, v[4] = {0.f, 0.f, 0.f, 0.f};
        if constexpr (WR == 1) inv = factors(r, f, S > 1 && d == 0);
        else inv = words[r][1];
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            const int at = k * WR * 32 + r;
            if constexpr (WR > 1) f[k] = words[at][0];
            const f32x4 p = *(const f32x4 *)((const float *)smem + (size_t)at * kRowPad<HD> + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(f[k], p[e], v[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= inv;
        const size_t item = item_of(r);
        if (S == 1) {
            store_out<4>(a, item * HD + d, v);
            if (!(fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY))
                atomicOr(&odd[r / 32], 1 << (r % 32));
        } else {
            *(f32x4 *)(a.part + (item * S + split) * HD + d) = f32x4{v[0], v[1], v[2], v[3]};
        }
    }
    if (S > 1) return;
    __syncthreads();
    for (int r = wave; r < held_rows; r += kWaves)
        if (uniform(odd[r / 32]) >> (r % 32) & 1)
            plain_row<HD>(kernel_args(), over_g(m0 + r), g * G + (m0 + r - over_g(m0 + r) * G));
}

// ---------------------------------------------------------------------------
// Few M rows: v_mfma_f32_16x16x32_f16 over blocks of R = 8 or 16 of them. The 16
// columns of 8 rows (a token's heads of a group) are their high parts and their low
// parts, so that one product takes both, a quarter of the 32-wide products' time; 16
// rows take two products.
//   S^T = K Q^T     two tiles of 16 positions; A = K: lane (n, q) takes 16 dims
//                   64 c + 16 q .. of position 8 (n / 4) + 4 t + n % 4 of tile t; of 8
//                   rows the columns' sum, n and n + 8, is the score.
//   O^T += V^T P^T  A = V^T: lane (n, q) takes positions 8 q .. + 7 of dim 16 u + n;
//                   lane (m, q) holds the probabilities of its row there.
// Blocks of 8 waves, every one with blocks of positions of its own, K and V from
// memory into registers. 1 on 576 (14 / 2 heads of 64) 5.5 us (6.3 with 32-wide
// products), 1 on 32,767 (28 / 4 of 128) 12.2 (12.9), under a window of 4,096 8.9 (9.5),
// 13 on 1,999 (32 / 8 of 128) 9.0 (11.0). Of 8 rows 16 waves 6.4 / 14.2 / 10.9, two
// blocks a CU 5.7 / 13.2 / 8.5, two blocks of positions in flight 5.8 / 13.5 / 9.2.
// Bound by round trips (page, K and V, the join) and the merge's launch.
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 8;
constexpr int kFew8 = -8, kFew16 = -16;  // a cut's rows in place of row waves
template <int HD, int R>
constexpr size_t kFewQueries = kFewWaves * R * kRowPad<HD> * 4;  // behind the waves' sums
template <int HD>
constexpr int kFewQRow = HD * 2 + 16;  // bytes of a row's part
template <int HD, int R>
constexpr size_t kFewWords = kFewQueries<HD, R> + 2 * R * kFewQRow<HD>;
template <int HD, int R>
constexpr size_t kFewLds = kFewWords<HD, R> + kFewWaves * R * 16 + R * 4 + 16;

// A lane's value and that of the lane 16 away, and of the four rows of 16 lanes.
template <class F>
__device__ __forceinline__ float over_quads(float x, F f) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

template <int HD, int R>
__global__ __launch_bounds__(64 * kFewWaves) void kv8_few_kernel(Kv8AttnArgs a, int S) {
    constexpr int W = kFewWaves, CC = HD / 64, U = HD / 16, BB = kBlock * HD;
    constexpr int P = R / 8;  // products for the two parts
    extern __shared__ __attribute__((aligned(256))) uint8_t smem[];
    uint8_t *sq = smem + kFewQueries<HD, R>;
    f32x4 *words = (f32x4 *)(smem + kFewWords<HD, R>);
    int *sq_exp = (int *)(words + W * R), *odd = sq_exp + R;
    auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int n = lane & 15, quad = lane >> 4, r = n % R;
    const int G = a.q_heads / a.g.kv_heads, M = a.rows * G, RB = (M + R - 1) / R;
    auto over_g = [&](int x) { return G == 1 ? x : (int)__umulhi((uint32_t)x, a.over_group); };
    const int total = RB * S * a.g.kv_heads, run = (total + 7) / 8;
    const int work = (int)blockIdx.x % 8 * run + (int)blockIdx.x / 8;
    if (work >= total) return;
    const int pair = work / RB, m0 = uniform(work % RB * R), rows = min(R, M - m0);  // of the block
    const int g = uniform(pair % a.g.kv_heads), split = uniform(pair / a.g.kv_heads);
    const int offset = uniform(first_pos(a));
    const int pos_lo = uniform(offset + over_g(m0)), pos_hi = uniform(offset + over_g(m0 + rows - 1));
    const int pos = r < rows ? offset + over_g(m0 + r) : pos_lo, lo = window_start(a, pos);
    const int seen_lo = window_start(a, pos_lo), all_first = window_start(a, pos_hi);
    const Reach reach = reach_of(pos_lo, pos_hi, a.window, a.sinks);
    const int each = reach.count / S, extra = reach.count % S;
    const int begin = uniform(split * each + min(split, extra)), end = uniform(begin + each + (split < extra));
    const int mine = max(end - begin - wave + W - 1, 0) / W;

    // Where this wave's next 64 blocks lie and their scales, a lane each.
    int held_at = 0;
    uint32_t held_k = 0, held_v = 0;
    auto look_up = [&](int i0) {
        const int b = reach.block(min(begin + wave + min(i0 + lane, max(mine - 1, 0)) * W, reach.count - 1));
        const int per = a.g.page_size / kBlock;
        const int page = a.g.page_table[b / per];
        held_at = (page * a.g.kv_heads + g) * per + b % per;
    };
    auto look_up_scales = [&]() {
        held_k = a.k_scales[held_at];
        held_v = a.v_scales[held_at];
    };
    auto landed = [&]() { asm volatile("" : "+v"(held_k), "+v"(held_v)); };
    auto at_of = [&](int i) { return (size_t)(uint32_t)__builtin_amdgcn_readlane(held_at, i & 63); };
    const int koff = quad / 2 * 1024 + (8 * (n / 4) + n % 4) * 32 + 16 * (quad % 2), voff = n * kBlock + 8 * quad;
    u32x4 kr[CC][2];
    uint2 vr[U];
    auto load_k = [&](size_t at) {
#pragma unroll
        for (int c = 0; c < CC; ++c)
#pragma unroll
            for (int t = 0; t < 2; ++t) kr[c][t] = *(const u32x4 *)(a.k + at * BB + 2048 * c + 128 * t + koff);
    };
    auto load_v = [&](size_t at) {
#pragma unroll
        for (int u = 0; u < U; ++u) vr[u] = *(const uint2 *)(a.v + at * BB + 16 * kBlock * u + voff);
    };

    // The start, as kv8_attn_kernel's: a wave loads 256 floats of the queries.
    look_up(0);
    constexpr int LPR = HD / 4, RPI = 64 / LPR;  // lanes a row, rows a load
    const int row = wave * RPI + lane / LPR;
    const bool queries = wave < R / RPI;
    f32x4 raw = {0.f, 0.f, 0.f, 0.f};
    if (queries) {
        const int rr = m0 + min(row, rows - 1);
        raw = *(const f32x4 *)(a.q + ((size_t)over_g(rr) * a.q_heads + g * G + rr - over_g(rr) * G) * HD + lane % LPR * 4);
    }
    __builtin_amdgcn_sched_barrier(0);
    look_up_scales();
    load_k(at_of(0)), load_v(at_of(0));
    __builtin_amdgcn_sched_barrier(0);
    if (queries) {
        const float sl2 = (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f;
        f32x4 v = raw * (row < rows ? sl2 : 0.f);
        float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
        const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -112), 127) - 14;
        v *= two_to(-e);
        uint2 hi, lw;
        split_f16(v[0], v[1], hi.x, lw.x);
        split_f16(v[2], v[3], hi.y, lw.y);
        *(uint2 *)(sq + row * kFewQRow<HD> + lane % LPR * 8) = hi;
        *(uint2 *)(sq + (R + row) * kFewQRow<HD> + lane % LPR * 8) = lw;
        if (lane % LPR == 0) sq_exp[row] = e;
    }
    if (threadIdx.x == 0) *odd = 0;
    landed();
    lds_barrier();
    f16x8 qo[P][CC][2];
    const int q_exp = sq_exp[r];
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
        for (int c = 0; c < CC; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                qo[j][c][i] = *(const f16x8 *)(sq + (j * R + n) * kFewQRow<HD> + 128 * c + 32 * quad + 16 * i);

    // A row's value from its columns: the high and the low part's, 8 away (row_ror:8).
    auto whole_row = [](float x) {
        if constexpr (P == 1) return x + dpp_mov<0x128>(x);
        else return x;
    };
    f32x4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m2 = -INFINITY;
    WeightSum l;
    ValueUnit unit;  // of o
    uint32_t now_k = held_k, now_v = held_v;
    for (int i = 0; i < mine; ++i) {
        if (i > 0 && (i & 63) == 0) now_k = held_k, now_v = held_v;
        if (((i + 1) & 63) == 0 && i + 1 < mine) look_up(i + 1), look_up_scales(), landed();
        const size_t at_next = at_of(i + 1);
        const int p0 = reach.block(begin + wave + i * W) * kBlock;
        f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < CC; ++c)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const u32x4 x = kr[c][t];
                const f16x8 x0 = codes_f16(x[0], x[1], 1.f), x1 = codes_f16(x[2], x[3], 1.f);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, qo[j][c][0], st[t], 0, 0, 0);
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, qo[j][c][1], st[t], 0, 0, 0);
                }
            }
        if (i + 1 < mine) load_k(at_next);
        __builtin_amdgcn_sched_barrier(0);
        float s[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = whole_row(st[k / 4][k % 4]);
        if (p0 + kBlock - 1 > pos_lo || (p0 < all_first && p0 + kBlock > a.sinks)) {
            const uint32_t bits = seen_bits(p0 + 8 * quad, pos, lo, a.sinks);
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k] = bits >> k & 1 ? s[k] : -INFINITY;
        }
        const float fs = ldexpf(1.f, max(q_exp + (int)__builtin_amdgcn_readlane(now_k, i & 63) - 127, -126));
        float tmax = s[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) tmax = fmaxf(tmax, s[k]);
        tmax = over_quads(tmax, [](float x, float y) { return fmaxf(x, y); }) * fs;
        if (__any(tmax > m2 + (kLift + kRaise))) {
            const bool raise = tmax > m2 + (kLift + kRaise);
            const float mnew = raise ? tmax - kLift : m2, alpha = raise ? __builtin_amdgcn_exp2f(m2 - mnew) : 1.f;
            l.scale(alpha);
#pragma unroll
            for (int u = 0; u < U; ++u) o[u] *= alpha;
            m2 = mnew;
        }
        const float mref = m2 == -INFINITY ? 0.f : m2;
        uint32_t p[P][4];
        float block_sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * k], fs, -mref)), y = __builtin_amdgcn_exp2f(fmaf(s[2 * k + 1], fs, -mref));
            block_sum += x;
            block_sum += y;
            uint32_t hi, lw;
            split_weights(x, y, hi, lw);
            p[0][k] = n < R ? hi : lw;
            if constexpr (P == 2) p[1][k] = lw;
        }
        l.add(block_sum);
        if (p0 + kBlock - 1 > pos_hi || (p0 < seen_lo && p0 + kBlock > a.sinks)) {
            // Positions that no row sees may hold anything: zeros.
            const uint32_t bits = seen_bits(p0 + 8 * quad, pos_hi, seen_lo, a.sinks);
            const uint32_t b0 = ((bits & 15) * 0x204081u & 0x01010101u) * 0xFFu, b1 = ((bits >> 4 & 15) * 0x204081u & 0x01010101u) * 0xFFu;
#pragma unroll
            for (int u = 0; u < U; ++u) vr[u].x &= b0, vr[u].y &= b1;
        }
        // (Of 8 rows the low parts' columns carry the 2^-11, not V.)
        const float vs = unit.factor(
            (int)__builtin_amdgcn_readlane(now_v, i & 63) - 127, i == 0, P == 1 ? 15 : 4, l,
            [&]() {
                uint32_t codes = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) codes |= vr[u].x | vr[u].y;
                return codes;
            },
            [&]() {
                uint32_t sums = 0;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) sums |= __float_as_uint(o[u][k]);
                return sums;
            },
            [&](int by) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[u][k] = ldexpf(o[u][k], by);
            });
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const f16x8 x = codes_f16(vr[u].x, vr[u].y, vs);
#pragma unroll
            for (int j = 0; j < P; ++j)
                o[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    j == 0 ? x : x * kLow, __builtin_bit_cast(f16x8, u32x4{p[j][0], p[j][1], p[j][2], p[j][3]}), o[u], 0, 0, 0);
        }
        if (i + 1 < mine) load_v(at_next);
        __builtin_amdgcn_sched_barrier(0);
    }
    // The waves' parts meet in LDS.
    l.sum = over_quads(l.sum, [](float x, float y) { return x + y; });
    float *so = (float *)smem + (size_t)(wave * R + r) * kRowPad<HD> + 4 * quad;
    const float column = n < R ? 1.f : 1.f / kLowUp;  // a low part's
#pragma unroll
    for (int u = 0; u < U; u += 3 - P) {  // (a row's two columns take turns to write)
        f32x4 v[3 - P];
#pragma unroll
        for (int i = 0; i < 3 - P; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = whole_row(o[u + i][k] * column);
        if (r < rows) *(f32x4 *)(so + 16 * (u + n / R)) = n < R ? v[0] : v[2 - P];
    }
    if (lane < R) words[wave * R + r] = f32x4{m2, l.sum, two_to(unit.e), 0.f};
    __syncthreads();
    for (int u = (int)threadIdx.x; u < rows * (HD / 4); u += 64 * W) {  // 4 dims of a row
        const int rr = u / (HD / 4), d = u % (HD / 4) * 4, at = over_g(m0 + rr);
        const size_t item = (size_t)at * a.q_heads + g * G + (m0 + rr - at * G);
        float f[W], v[4] = {0.f, 0.f, 0.f, 0.f};
        const float inv = wave_factors(words + rr, R, f, S == 1, S > 1 && d == 0 ? a.ml + item * S + split : nullptr);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const f32x4 x = *(const f32x4 *)((const float *)smem + (size_t)(k * R + rr) * kRowPad<HD> + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(f[k], x[e], v[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= inv;
        if (S == 1) {
            store_out<4>(a, item * HD + d, v);
            if (!(fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY))
                atomicOr(odd, 1 << rr);
        } else {
            *(f32x4 *)(a.part + (item * S + split) * HD + d) = f32x4{v[0], v[1], v[2], v[3]};
        }
    }
    if (S > 1) return;
    __syncthreads();
    for (int rr = wave; rr < rows; rr += W)
        if (uniform(*odd) >> rr & 1)
            plain_row<HD>(kernel_args(), over_g(m0 + rr), g * G + (m0 + rr - over_g(m0 + rr) * G));
}

// The splits of a row and head, joined by W waves (each takes every W-th); the
// values are on their way while the weights are found.
constexpr int kMaxSplits = 128;
template <int HD, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void kv8_merge_kernel(Kv8AttnArgs a, int S) {
    constexpr int D = HD / 64, I = W == 1 ? 4 : 1, B = W == 1 ? 8 : kMaxSplits / W;  // items a block, splits at once
    __shared__ float s_o[W == 1 ? 1 : W][HD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w0 = W == 1 ? 0 : wave;
    const long item = (long)blockIdx.x * I + (W == 1 ? wave : 0);
    if (item >= (long)a.rows * a.q_heads) return;  // (a wave's own where W is 1)
    const float2 *ml = a.ml + item * S;
    const float *part = a.part + item * S * HD + D * lane;
    float v[D], p[B][D];
#pragma unroll
    for (int d = 0; d < D; ++d) v[d] = 0.f;
    const float2 x = ml[min(lane, S - 1)], y = ml[min(lane + 64, S - 1)];
    auto load = [&](int s0) {
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const float *q = part + (size_t)min(s0 + b * W, S - 1) * HD;
            if constexpr (D == 2) {
                const float2 t = *(const float2 *)q;
                p[b][0] = t.x, p[b][D - 1] = t.y;
            } else {
                p[b][0] = *q;
            }
        }
    };
    load(w0);
    const float top = wave_max(fmaxf(x.x, y.x));
    // A split that saw nothing counts nothing; a NaN sum shows.
    const float wx = lane >= S || (x.x == -INFINITY && x.y == 0.f) ? 0.f : __builtin_amdgcn_exp2f(x.x - top);
    const float wy = lane + 64 >= S || (y.x == -INFINITY && y.y == 0.f) ? 0.f : __builtin_amdgcn_exp2f(y.x - top);
    const float sum = wave_sum((wx != 0.f || x.y != x.y ? wx * x.y : 0.f) + (wy != 0.f || y.y != y.y ? wy * y.y : 0.f));
    for (int s0 = w0; s0 < S; s0 += B * W) {
        if (s0 != w0) load(s0);
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int s = s0 + b * W;
            if (s >= S) break;
            // (A weight of 0 too: a NaN among its values shows. Empty splits hold zeros.)
            const float w = __shfl(s < 64 ? wx : wy, s & 63, 64);
#pragma unroll
            for (int d = 0; d < D; ++d) v[d] = fmaf(w, p[b][d], v[d]);
        }
    }
    const float inv = 1.0f / sum;
#pragma unroll
    for (int d = 0; d < D; ++d) v[d] *= inv;
    if constexpr (W > 1) {
#pragma unroll
        for (int d = 0; d < D; ++d) s_o[wave][D * lane + d] = v[d];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int k = 1; k < W; ++k)
#pragma unroll
            for (int d = 0; d < D; ++d) v[d] += s_o[k][D * lane + d];
    }
    bool fine = true;
#pragma unroll
    for (int d = 0; d < D; ++d) fine = fine && fabsf(v[d]) < INFINITY;
    store_out<D>(a, item * HD + D * lane, v);
    if (__any(!fine)) plain_row<HD>(kernel_args(), (int)(item / a.q_heads), (int)(item % a.q_heads));
}

template <int HD, int WR>
int launch_attn_blocks(const Kv8AttnArgs &a, int S, hipStream_t s) {
    constexpr size_t lds = kv8_attn_lds_bytes<HD, WR>();
    const long M = (long)a.rows * (a.q_heads / a.g.kv_heads), RB = (M + 32 * WR - 1) / (32 * WR);
    const long blocks = (RB * S * a.g.kv_heads + 7) / 8 * 8;
    hipLaunchKernelGGL((kv8_attn_kernel<HD, WR>), dim3((unsigned)blocks), dim3(64 * kWaves), lds, s, a, S);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

template <int HD, int R>
int launch_few(const Kv8AttnArgs &a, int S, hipStream_t s) {
    const long M = (long)a.rows * (a.q_heads / a.g.kv_heads);
    const long blocks = ((M + R - 1) / R * S * a.g.kv_heads + 7) / 8 * 8;
    hipLaunchKernelGGL((kv8_few_kernel<HD, R>), dim3((unsigned)blocks), dim3(64 * kFewWaves), (kFewLds<HD, R>), s, a, S);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

template <int HD>
int launch_attn(const Kv8AttnArgs &a, int wr, int S, hipStream_t s) {
    if (wr == kFew8) CHIP_TRY((launch_few<HD, 8>(a, S, s)));
    else if (wr == kFew16) CHIP_TRY((launch_few<HD, 16>(a, S, s)));
    else if (wr == 1) CHIP_TRY((launch_attn_blocks<HD, 1>(a, S, s)));
    else if (wr == 2) CHIP_TRY((launch_attn_blocks<HD, 2>(a, S, s)));
    else CHIP_TRY((launch_attn_blocks<HD, 4>(a, S, s)));
    if (S == 1) return 0;
    const long items = (long)a.rows * a.q_heads;
    if (S > 8) hipLaunchKernelGGL((kv8_merge_kernel<HD, 8>), dim3((unsigned)items), dim3(512), 0, s, a, S);
    else hipLaunchKernelGGL((kv8_merge_kernel<HD, 1>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, a, S);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

template <int HD, class T>
int launch_append(const Kv8AppendJob &j, const AppendArgs &a, bool vec, unsigned blocks, hipStream_t s) {
    const dim3 grid(blocks, j.kv.g.kv_heads, 2);
    if (vec) hipLaunchKernelGGL((kv8_append_kernel<HD, T, true>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((kv8_append_kernel<HD, T, false>), grid, dim3(kThreads), 0, s, a);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace

int launch_kv8_append(const Kv8AppendJob &j, hipStream_t s) {
    AppendArgs a;
    a.x[0] = j.k, a.x[1] = j.v;
    a.stride = (long)j.stride;
    a.head_stride = (long)(j.head_stride ? j.head_stride : (size_t)j.kv.g.head_dim);
    a.codes[0] = j.kv.k, a.codes[1] = j.kv.v, a.scales[0] = j.kv.k_scales, a.scales[1] = j.kv.v_scales;
    a.g = j.kv.g;
    a.offset = (int)j.offset;
    a.rows = (int)j.rows;
    const size_t run = kThreads / (size_t)j.kv.g.head_dim;
    const size_t blocks = ((j.offset + j.rows - 1) / kBlock - j.offset / kBlock + 1 + run - 1) / run;
    const size_t unit = j.f32 ? 4 : 2;
    const bool vec = ((uintptr_t)j.k | (uintptr_t)j.v | (j.stride * unit) | (a.head_stride * unit)) % 16 == 0;
    const unsigned n = (unsigned)blocks;
    if (j.kv.g.head_dim == 64)
        return j.f32 ? launch_append<64, float>(j, a, vec, n, s) : launch_append<64, uint16_t>(j, a, vec, n, s);
    return j.f32 ? launch_append<128, float>(j, a, vec, n, s) : launch_append<128, uint16_t>(j, a, vec, n, s);
}

int launch_kv8_rope_append(const float *qkv, float *q, int q_heads, const Kv8Cache &kv, const float *rope_cos,
                           const float *rope_sin, int rotary_dim, const int32_t *pos_dev, hipStream_t s) {
    if (rotary_dim <= 0 || rotary_dim > kv.g.head_dim || rotary_dim % 2)
        return fail("HIP backend: rotary_dim must be even and at most head_dim.");
    const RopeArgs a{qkv, q, kv, q_heads, rotary_dim, rope_cos, rope_sin, pos_dev};
    const int heads = kThreads / kv.g.head_dim;  // a block
    const dim3 grid((unsigned)((q_heads + 2 * kv.g.kv_heads + heads - 1) / heads));
    if (kv.g.head_dim == 64) hipLaunchKernelGGL((kv8_rope_append_kernel<64>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((kv8_rope_append_kernel<128>), grid, dim3(kThreads), 0, s, a);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

int launch_kv8_read(const Kv8Cache &kv, size_t begin, size_t n, bool f32, void *k_out, void *v_out, hipStream_t s) {
    ReadArgs a;
    a.codes[0] = kv.k, a.codes[1] = kv.v, a.scales[0] = kv.k_scales, a.scales[1] = kv.v_scales;
    a.g = kv.g;
    a.begin = (int)begin;
    a.n = (int)n;
    a.out[0] = k_out, a.out[1] = v_out;
    const size_t blocks = (begin + n - 1) / kBlock - begin / kBlock + 1, run = kThreads / (size_t)kv.g.head_dim;
    const dim3 grid((unsigned)((blocks + run - 1) / run), kv.g.kv_heads, 2), threads(kThreads);
    if (kv.g.head_dim == 64) {
        if (f32) hipLaunchKernelGGL((kv8_read_kernel<64, float>), grid, threads, 0, s, a);
        else hipLaunchKernelGGL((kv8_read_kernel<64, uint16_t>), grid, threads, 0, s, a);
    } else {
        if (f32) hipLaunchKernelGGL((kv8_read_kernel<128, float>), grid, threads, 0, s, a);
        else hipLaunchKernelGGL((kv8_read_kernel<128, uint16_t>), grid, threads, 0, s, a);
    }
    CHIP_CHECK(hipGetLastError());
    return 0;
}

// How a call is cut: rows a block (its waves split its keys in LDS) and splits of the
// keys (a block each, joined by a merge kernel). The cheapest by an estimate, in us:
// for a round of blocks, one a CU, its start and end and a step a block of positions
// of a wave; for splits a merge's launch and 4.5 TB/s for its partials. kv8_attn_kernel
// with one row wave reads K and V from the caches for every 32 rows, with four for
// 128: ties go to more. Rows of 32 / 8 heads of 128, 16-row blocks against its own:
// 64 on nothing 6.0 us, 12.2; 13 on 1,023 9.6, 10.6; 20 on 4,095 11.7, 15.4; 64 on
// 16,383 45.4, 42.5; 180 on 1,023 18.8, 14.4. 8-row blocks with and without splits: 1 on
// 767 7.6, 7.0; 1 on 2,047 7.8, 11.8.
struct Cut {
    int wr, splits;
};
static Cut cut_of(const Kv8AttnJob &j) {
    const size_t G = j.q_heads / j.kv.g.kv_heads, M = j.rows * G, kvh = j.kv.g.kv_heads, hd = j.kv.g.head_dim;
    const size_t cus = (size_t)std::max(device_cus(), 1), tiles = (M + 31) / 32;
    const int last = (int)(j.offset + j.rows - 1);
    Cut best{1, 1};
    double least = 0;
    auto consider = [&](int kind, size_t rows, size_t wk, double base, double step, double merge) {
        const size_t blocks = (M + rows - 1) / rows * kvh;
        const int first = std::max(last + 1 - (int)std::min<size_t>(j.rows, (rows + G - 1) / G + 1), 0);
        const size_t reach = (size_t)reach_of(first, last, (int)j.window, (int)j.sinks).count;
        const size_t most = std::max<size_t>(1, std::min<size_t>(kMaxSplits, std::min((reach + wk - 1) / wk, cus / blocks)));
        for (size_t S = 1; S <= most; S = S < most && S * 2 > most ? most : S * 2) {
            const double rounds = (double)((blocks * S + cus - 1) / cus), steps = (double)((reach + S * wk - 1) / (S * wk));
            double us = rounds * (base + steps * step);
            if (S > 1) us += merge + 2.0 * (double)(j.rows * j.q_heads * S * hd * 4) / 4.5e6;
            if (least == 0 || us < least) least = us, best = Cut{kind, (int)S};
        }
    };
    if (M <= 8) {
        consider(kFew8, 8, kFewWaves, 4.2, hd == 64 ? 0.7 : 0.95, 2.4);
        return best;
    }
    for (int wr = 4; wr >= 1; wr /= 2)
        if (wr == 1 || tiles > (size_t)wr / 2)  // (else row waves without rows)
            consider(wr, 32 * wr, kWaves / wr, 5.5, hd == 64 ? 0.9 : 1.7, 3);
    consider(kFew16, 16, kFewWaves, hd == 64 ? 3.8 : 4.7, hd == 64 ? 0.72 : 1, 3.1);
    return best;
}

int kv8_attention_splits(const Kv8AttnJob &j) { return cut_of(j).splits; }

size_t kv8_attention_part_floats(const Kv8AttnJob &j, int splits) {
    return splits <= 1 ? 0 : j.rows * (size_t)j.q_heads * splits * (j.kv.g.head_dim + 2);
}

// Partials of any call of a head size: its splits and row blocks are one block of at
// most 128 rows (query row x head) a CU, or one split.
size_t kv8_attention_part_most(int head_dim) { return (size_t)std::max(device_cus(), 1) * 128 * (head_dim + 2); }

template <int HD>
static int prepare() {
    static std::atomic<uint64_t> set[5];
    CHIP_TRY(allow_dynamic_lds((const void *)kv8_few_kernel<HD, 8>, kFewLds<HD, 8>, set[3]));
    CHIP_TRY(allow_dynamic_lds((const void *)kv8_few_kernel<HD, 16>, kFewLds<HD, 16>, set[4]));
    CHIP_TRY(allow_dynamic_lds((const void *)kv8_attn_kernel<HD, 1>, kv8_attn_lds_bytes<HD, 1>(), set[0]));
    CHIP_TRY(allow_dynamic_lds((const void *)kv8_attn_kernel<HD, 2>, kv8_attn_lds_bytes<HD, 2>(), set[1]));
    return allow_dynamic_lds((const void *)kv8_attn_kernel<HD, 4>, kv8_attn_lds_bytes<HD, 4>(), set[2]);
}
int kv8_attention_prepare(int head_dim) { return head_dim == 64 ? prepare<64>() : prepare<128>(); }

int launch_kv8_attention(const Kv8AttnJob &j, hipStream_t s) {
    CHIP_TRY(kv8_attention_prepare(j.kv.g.head_dim));
    if (!j.out && !(j.out_hi && j.out_lo)) return fail("HIP backend: 8-bit attention without an output.");
    if (j.pos_dev && j.rows != 1) return fail("HIP backend: a position on the device goes with one row.");
    const int S = std::max(1, j.splits), wr = cut_of(j).wr;
    if (S > kMaxSplits || j.part_floats < kv8_attention_part_floats(j, S))
        return fail("HIP backend: 8-bit attention partial buffer too small.");
    const size_t items = j.rows * (size_t)j.q_heads;
    if (items / j.kv.g.kv_heads >= (size_t)1 << 29 || items > (size_t)INT32_MAX) return fail("HIP backend: attention with too many rows.");
    Kv8AttnArgs a;
    a.q = j.q;
    a.k = j.kv.k, a.v = j.kv.v, a.k_scales = j.kv.k_scales, a.v_scales = j.kv.v_scales;
    a.g = j.kv.g;
    a.q_heads = j.q_heads;
    a.rows = (int)j.rows, a.offset = (int)j.offset, a.window = (int)j.window, a.sinks = (int)j.sinks;
    const uint64_t group = (uint64_t)(j.q_heads / j.kv.g.kv_heads);
    a.over_group = group > 1 ? (uint32_t)(((1ull << 32) + group - 1) / group) : 0;
    a.out = j.out;
    a.out_hi = j.out_hi, a.out_lo = j.out_lo;
    a.pos_dev = j.pos_dev;
    a.part = j.part;
    a.ml = (float2 *)(j.part + items * (size_t)S * j.kv.g.head_dim);
    return j.kv.g.head_dim == 64 ? launch_attn<64>(a, wr, S, s) : launch_attn<128>(a, wr, S, s);
}

}  // namespace chip
