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

#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = kKv8Block;
constexpr int kScaleLeast = -117, kScaleMost = 119;
constexpr uint32_t kNanCode = 0x7F;

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
    for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(x[i] * inv, -448.f), 448.f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    uint32_t r = (uint32_t)w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!(fabsf(x[i]) < INFINITY)) r = (r & ~(0xFFu << (8 * i))) | (kNanCode << (8 * i));
    return r;
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
// Append: a block of threads per (32 positions, KV head, K or V). Its rows come
// in 8 dims a thread, the largest magnitude of all of them gives the scale, V
// codes are turned in LDS. Rows of the block that were there before are rounded
// again where the scale grows.
// ---------------------------------------------------------------------------
struct AppendArgs {
    const void *x[2];  // K, V rows
    long stride;
    uint8_t *codes[2], *scales[2];
    Kv8Geom g;
    const int32_t *pos_dev;  // the first row's position, where set
    long offset;
    int rows;
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

// Bytes of a V dim's 32 codes in LDS, an odd number of words.
constexpr int kTurn = 36;

template <int HD, class T, bool VEC>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(AppendArgs a) {
    constexpr int U = kBlock * HD / 8 / kThreads;  // units of 8 values a thread
    __shared__ float s_max[kThreads / 64];
    __shared__ __attribute__((aligned(16))) uint8_t s_turn[HD * kTurn];
    const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
    const long offset = a.pos_dev ? (long)*a.pos_dev : a.offset;
    const long first = offset / kBlock * kBlock + (long)blockIdx.x * kBlock;  // the block's first position
    const int keep = (int)max(offset - first, 0l);                            // its earlier rows
    const int stop = (int)min(offset + a.rows - first, (long)kBlock);         // new rows end here
    if (stop <= keep) return;  // (a fixed grid may hold one block more than the rows reach)
    const int page = a.g.page_table[first / a.g.page_size];
    const BlockAt at = block_at(a.g, page, (int)(first % a.g.page_size) / kBlock, head, HD);
    uint8_t *codes = (which ? a.codes[1] : a.codes[0]) + at.codes;
    uint8_t *scale = (which ? a.scales[1] : a.scales[0]) + at.scale;
    const T *x = (const T *)(which ? a.x[1] : a.x[0]) + (first - offset) * a.stride + (size_t)head * HD;
    const int e_old = keep ? (int)*scale - 127 : kScaleLeast;

    f32x4 v[U][2];
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int u = tid + kThreads * k, p = u / (HD / 8), d = u % (HD / 8) * 8;
        const bool fresh = p >= keep && p < stop;
        if (fresh) load8<T, VEC>(x + (long)p * a.stride + d, v[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = fabsf(v[k][i / 4][i % 4]);
            most = fmaxf(most, fresh && m < INFINITY ? m : 0.f);
        }
    }
    most = wave_max(most);
    if ((tid & 63) == 0) s_max[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const int e = max(exponent_for(most), e_old);
    const float inv = two_to(-e), grown = two_to(max(e_old - e, -126));
    if (tid == 0) *scale = (uint8_t)(e + 127);

#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int u = tid + kThreads * k, p = u / (HD / 8), d = u % (HD / 8) * 8;
        const bool fresh = p >= keep && p < stop;
        const uint2 w = fresh ? make_uint2(codes_of(v[k][0], inv), codes_of(v[k][1], inv)) : make_uint2(0, 0);
        if (!which) {
            uint2 *to = (uint2 *)(codes + d / 32 * (kBlock * 32) + p * 32 + d % 32);
            if (fresh) {
                *to = w;
            } else if (p < keep && e > e_old) {
                const uint2 o = *to;
                *to = make_uint2(rescaled(o.x, grown), rescaled(o.y, grown));
            }
        } else if (fresh) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s_turn[(d + i) * kTurn + p] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
        }
    }
    if (!which) return;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k) {  // 8 positions of a dim
        const int u = tid + kThreads * k, d = u / (kBlock / 8), p = u % (kBlock / 8) * 8;
        if (p >= stop || (p + 8 <= keep && e == e_old)) continue;  // nothing changes
        uint2 *to = (uint2 *)(codes + d * kBlock + p);
        uint32_t w[2], o[2] = {0, 0};
        if (p < keep || p + 8 > stop) {
            const uint2 q = *to;
            o[0] = q.x, o[1] = q.y;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t n = *(const uint32_t *)&s_turn[d * kTurn + p + 4 * j], r = rescaled(o[j], grown);
            w[j] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pos = p + 4 * j + i;
                const uint32_t from = pos < keep ? (e > e_old ? r : o[j]) : pos < stop ? n : o[j];
                w[j] |= from & (0xFFu << (8 * i));
            }
        }
        *to = make_uint2(w[0], w[1]);
    }
}

// ---------------------------------------------------------------------------
// Read: a block of threads per (32 positions, KV head, K or V).
// ---------------------------------------------------------------------------
struct ReadArgs {
    const uint8_t *codes[2], *scales[2];
    Kv8Geom g;
    long begin;
    long n;
    void *out[2];
};

__device__ __forceinline__ void store8(float *p, f32x4 a, f32x4 b) {
    *(f32x4 *)p = a;
    *(f32x4 *)(p + 4) = b;
}
__device__ __forceinline__ void store8(uint16_t *p, f32x4 a, f32x4 b) {  // exact
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        w[i] = (uint32_t)f32_bf16_rne(a[2 * i]) | ((uint32_t)f32_bf16_rne(a[2 * i + 1]) << 16);
        w[2 + i] = (uint32_t)f32_bf16_rne(b[2 * i]) | ((uint32_t)f32_bf16_rne(b[2 * i + 1]) << 16);
    }
    *(u32x4 *)p = w;
}

template <int HD, class T>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(ReadArgs a) {
    constexpr int U = kBlock * HD / 8 / kThreads;
    __shared__ __attribute__((aligned(16))) uint8_t s_turn[HD * kTurn];
    const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
    const long first = a.begin / kBlock * kBlock + (long)blockIdx.x * kBlock;
    const int page = a.g.page_table[first / a.g.page_size];
    const BlockAt at = block_at(a.g, page, (int)(first % a.g.page_size) / kBlock, head, HD);
    const uint8_t *codes = (which ? a.codes[1] : a.codes[0]) + at.codes;
    const float scale = two_to((int)(which ? a.scales[1] : a.scales[0])[at.scale] - 127);
    T *out = (T *)(which ? a.out[1] : a.out[0]);
    if (which) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int u = tid + kThreads * k, d = u / (kBlock / 8), p = u % (kBlock / 8) * 8;
            const uint2 w = *(const uint2 *)(codes + d * kBlock + p);
            *(uint32_t *)&s_turn[d * kTurn + p] = w.x;
            *(uint32_t *)&s_turn[d * kTurn + p + 4] = w.y;
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int u = tid + kThreads * k, p = u / (HD / 8), d = u % (HD / 8) * 8;
        const long row = first + p - a.begin;
        if (row < 0 || row >= a.n) continue;
        uint2 w;
        if (!which) {
            w = *(const uint2 *)(codes + d / 32 * (kBlock * 32) + p * 32 + d % 32);
        } else {
            uint32_t b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = s_turn[(d + i) * kTurn + p];
            w = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
        }
        store8(out + (size_t)row * a.g.kv_heads * HD + (size_t)head * HD + d, code_values(w.x) * scale,
               code_values(w.y) * scale);
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
    float *out;
};

// The first position of the window of a row at `pos` (0 without one).
__device__ __forceinline__ int window_start(const Kv8AttnArgs &a, int pos) {
    return a.window ? max(pos + 1 - a.window, 0) : 0;
}

// One row and head in plain f32 products, a wave: the maximum and the weight sum,
// then the values under finished weights, so that finite values average to a
// finite output and an infinity or a NaN in a value that the row sees shows.
template <int HD>
__device__ void plain_row(const Kv8AttnArgs &a, int row, int head, float *out) {
    constexpr int C = HD / 32;
    const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
    const int g = head / (a.q_heads / a.g.kv_heads), pos = a.offset + row;
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
            float dot = 0.f;
#pragma unroll 1
            for (int c = 0; c < C; ++c) {
                const u32x4 w = *(const u32x4 *)(a.k + at.codes + c * (kBlock * 32) + n * 32 + 16 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 k = code_values(w[i]), x = *(const f32x4 *)(q + 32 * c + 4 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dot = fmaf(k[e], x[e], dot);
                }
            }
            dot += __shfl_xor(dot, 32, 64);
            const int p = b * kBlock + n;
            const bool seen = p <= pos && (p >= lo || p < sinks);
            const float s = seen ? dot * two_to((int)a.k_scales[at.scale] - 127) * sl2 : -INFINITY;
            if (pass == 0) {
                const float mn = fmaxf(m, wave_max(s));
                const float w = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
                l = (m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f(m - mn)) + 0.5f * wave_sum(w);  // both halves hold it
                m = mn;
            } else {
                const float w = seen ? __builtin_amdgcn_exp2f(s - m) / l : 0.f;
                const float scale = two_to((int)a.v_scales[at.scale] - 127);
#pragma unroll
                for (int u = 0; u < C; ++u) {
                    const u32x4 c = *(const u32x4 *)(a.v + at.codes + (32 * u + n) * kBlock + 16 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 x = code_values(c[i]) * scale;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = 16 * half + 4 * i + e;
                            const float wj = __shfl(w, j, 64);
                            const int pj = b * kBlock + j;
                            if (pj <= pos && (pj >= lo || pj < sinks)) o[u] = fmaf(wj, x[e], o[u]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < C; ++u) {
        const float v = o[u] + __shfl_xor(o[u], 32, 64);
        if (half == 0) out[32 * u + n] = v;
    }
}

template <int HD>
__global__ __launch_bounds__(kThreads) void kv8_attn_plain_kernel(Kv8AttnArgs a) {
    const long item = (long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (item >= (long)a.rows * a.q_heads) return;
    const int row = (int)(item / a.q_heads), head = (int)(item % a.q_heads);
    plain_row<HD>(a, row, head, a.out + (size_t)item * HD);
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
    a.codes[0] = j.kv.k, a.codes[1] = j.kv.v, a.scales[0] = j.kv.k_scales, a.scales[1] = j.kv.v_scales;
    a.g = j.kv.g;
    a.pos_dev = j.pos_dev;
    a.offset = (long)j.offset;
    a.rows = (int)j.rows;
    // With the position on the device a chunk may reach one block more.
    const size_t blocks = j.pos_dev ? (j.rows + kBlock - 2) / kBlock + 1
                                    : (j.offset + j.rows - 1) / kBlock - j.offset / kBlock + 1;
    const size_t unit = j.f32 ? 4 : 2;
    const bool vec = ((uintptr_t)j.k | (uintptr_t)j.v | (j.stride * unit)) % 16 == 0;
    const unsigned n = (unsigned)blocks;
    if (j.kv.g.head_dim == 64)
        return j.f32 ? launch_append<64, float>(j, a, vec, n, s) : launch_append<64, uint16_t>(j, a, vec, n, s);
    return j.f32 ? launch_append<128, float>(j, a, vec, n, s) : launch_append<128, uint16_t>(j, a, vec, n, s);
}

int launch_kv8_read(const Kv8Cache &kv, size_t begin, size_t n, bool f32, void *k_out, void *v_out, hipStream_t s) {
    ReadArgs a;
    a.codes[0] = kv.k, a.codes[1] = kv.v, a.scales[0] = kv.k_scales, a.scales[1] = kv.v_scales;
    a.g = kv.g;
    a.begin = (long)begin;
    a.n = (long)n;
    a.out[0] = k_out, a.out[1] = v_out;
    const dim3 grid((unsigned)((begin + n - 1) / kBlock - begin / kBlock + 1), kv.g.kv_heads, 2), threads(kThreads);
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

int launch_kv8_attention(const Kv8AttnJob &j, hipStream_t s) {
    Kv8AttnArgs a;
    a.q = j.q;
    a.k = j.kv.k, a.v = j.kv.v, a.k_scales = j.kv.k_scales, a.v_scales = j.kv.v_scales;
    a.g = j.kv.g;
    a.q_heads = j.q_heads;
    a.rows = (int)j.rows, a.offset = (int)j.offset, a.window = (int)j.window, a.sinks = (int)j.sinks;
    a.out = j.out;
    const dim3 grid((unsigned)((j.rows * j.q_heads + 3) / 4));
    if (j.kv.g.head_dim == 64) hipLaunchKernelGGL((kv8_attn_plain_kernel<64>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((kv8_attn_plain_kernel<128>), grid, dim3(kThreads), 0, s, a);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace chip
