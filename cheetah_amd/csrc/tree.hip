// Attention for a tree of drafted tokens over the paged KV cache, and the move
// of its accepted branch's K/V rows into place.
//
// Node i of n has its parent parents[i] < i (anything else: none, a root). Its
// K/V row sits at cache position offset + i. With the cached prefix [0, offset)
// every node sees its ancestors and itself:
//   out[i, h] = sum_p w_p v[p, h / G],  w = softmax_p(q[i, h] . k[p, h / G] / sqrt(head_dim))
// over p in [0, offset) and offset + a, a = i or an ancestor of i.
#include <algorithm>
#include <type_traits>

#include "attn_tiles.hpp"
#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256;

struct TreeArgs {
    const float *q;
    const void *k, *v;
    const int32_t *page_table;
    const int32_t *parents;
    float *part;
    float *out;
    uint16_t *out_hi, *out_lo;  // BF16 halves of out (null: not written)
    int page_size, kv_heads, q_heads, offset, n;
};

// Four outputs of a row at element i, and their BF16 halves where asked for.
__device__ __forceinline__ void store_out4(const TreeArgs &a, size_t i, f32x4 v) {
    if (a.out) *(f32x4 *)(a.out + i) = v;
    if (a.out_hi) {
        uint16_t h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const __bf16 hb = (__bf16)v[k];
            h[k] = __builtin_bit_cast(uint16_t, hb);
            l[k] = __builtin_bit_cast(uint16_t, (__bf16)(v[k] - (float)hb));
        }
        *(uint2 *)(a.out_hi + i) = make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
        *(uint2 *)(a.out_lo + i) = make_uint2((uint32_t)l[0] | ((uint32_t)l[1] << 16), (uint32_t)l[2] | ((uint32_t)l[3] << 16));
    }
}

// The ancestors of every node, themselves among them, as 256-bit words in LDS,
// by the whole block (thread i: node i). up[i] is the nearest ancestor that
// anc[i] does not hold yet, so each round doubles the length of the paths held:
// log2(depth) rounds, whatever the tree's shape.
constexpr int kAncWords = kMaxTreeNodes / 64;
struct TreeLds {
    uint64_t anc[kMaxTreeNodes][kAncWords];
    uint64_t sick[kAncWords];  // nodes with an infinity or NaN in V
    uint32_t odd[4];           // a row wave's rows to compute again
    int sick_prefix;           // an infinity or NaN in the prefix's V (f32)
    int16_t up[kMaxTreeNodes];
};
__device__ __forceinline__ void find_ancestors(const int32_t *parents, int n, TreeLds &t) {
    static_assert(kThreads == kMaxTreeNodes, "a thread per node");
    const int i = threadIdx.x;
    int p = i < n ? parents[i] : -1;
    if (p >= i) p = -1;
    uint64_t w[kAncWords];
#pragma unroll
    for (int k = 0; k < kAncWords; ++k) t.anc[i][k] = w[k] = i >> 6 == k ? 1ull << (i & 63) : 0;
    t.up[i] = (int16_t)(p < 0 ? -1 : p);
    if (i < kAncWords) t.sick[i] = 0;
    while (__syncthreads_or(p >= 0)) {
        if (p >= 0) {
#pragma unroll
            for (int k = 0; k < kAncWords; ++k) w[k] |= t.anc[p][k];
            p = t.up[p];
        } else {
            p = -1;
        }
        __syncthreads();  // every path is read before one grows
#pragma unroll
        for (int k = 0; k < kAncWords; ++k) t.anc[i][k] = w[k];
        t.up[i] = (int16_t)p;
    }
}

__device__ __forceinline__ float kv_value(const uint16_t *p) { return bf16_f32(*p); }
__device__ __forceinline__ float kv_value(const float *p) { return *p; }

// One row over positions [start, end) in plain f32 products, a wave per row and
// a lane per HD / 64 dims: the rare rows that the matrix cores' parts do not
// carry. They see an infinity or NaN in a tree node's V (or anywhere in an f32
// cache), which 0 x V would spread over the tile's rows, or their weight sum is
// NaN, where a score of -inf has to weigh nothing. A NaN sum ends the row.
template <int HD, class KT>
__device__ void plain_row(const TreeArgs &a, const TreeLds &t, int node, int head, int g, int start, int end, int S,
                          int split) {
    constexpr int D = HD / 64;
    const int lane = threadIdx.x & 63;
    const size_t row = ((size_t)node * a.q_heads + head) * HD;
    const float scale = (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f;
    float q[D], o[D], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) {
        q[d] = a.q[row + lane + 64 * d];
        o[d] = 0.f;
    }
#pragma unroll 1
    for (int p = start; p < end && l == l; ++p) {
        const int x = p - a.offset;
        if (x >= 0 && !(t.anc[node][x >> 6] >> (x & 63) & 1)) continue;
        const size_t at = (((size_t)a.page_table[p / a.page_size] * a.kv_heads + g) * a.page_size + p % a.page_size) * HD;
        float dot = 0.f;
#pragma unroll
        for (int d = 0; d < D; ++d) dot = fmaf(q[d], kv_value((const KT *)a.k + at + lane + 64 * d), dot);
        const float s = wave_sum(dot) * scale, mn = fmaxf(m, s);
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float w = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
        m = mn;
        l = l * alpha + w;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = fmaf(w, kv_value((const KT *)a.v + at + lane + 64 * d), o[d] * alpha);
    }
    float *part = a.part + (((size_t)node * a.q_heads + head) * S + split) * (HD + 2);
#pragma unroll
    for (int d = 0; d < D; ++d) {
        if (S > 1) {
            part[lane + 64 * d] = o[d];
        } else {
            const float v = o[d] / l;
            if (a.out) a.out[row + lane + 64 * d] = v;
            if (a.out_hi) {
                const __bf16 hb = (__bf16)v;
                a.out_hi[row + lane + 64 * d] = __builtin_bit_cast(uint16_t, hb);
                a.out_lo[row + lane + 64 * d] = __builtin_bit_cast(uint16_t, (__bf16)(v - (float)hb));
            }
        }
    }
    if (S > 1 && lane == 0) {
        part[HD] = l == l ? m : INFINITY;  // a NaN row: no split outweighs it
        part[HD + 1] = l;
    }
}

// ---------------------------------------------------------------------------
// On the matrix cores. The M = n G rows (node, head of the group) of a KV head
// are cut into waves of 32 and blocks of WR row waves; the 4 / WR key waves of
// a row wave take 32-position steps of the block's tiles in turn and are joined
// at the end. Per step, as attn_prefill_kernel's:
//   S^T = K Q^T     K rows from LDS, Q^T in registers
//   O^T += V^T P^T  V read transposed, P^T as the scores' registers lie
// Q (scaled by log2(e) / sqrt(HD)) and P are three BF16 parts each, all 24 bits
// of them. Over a BF16 cache K and V are exact: three products for one, as
// exact as f32 ones; with two parts the output would be 3.5e-6 off where f32
// products give 1e-6. An f32 cache's K and V are three parts too, and six of
// the nine part products are taken (attn_prefill_f32_kernel's).
//
// BF16 tiles of T positions go global to LDS, the next one while the current
// one computes; f32 tiles of 64 wait in registers and are split while staged.
//
// Splits are runs of `chunk` positions (whole tiles); merged by the attention
// merge. Blocks with the same (split, KV head) and other rows are 8 apart, on
// one XCD: they read the same tiles through its L2.
// ---------------------------------------------------------------------------
template <int WR, class KT>
constexpr int tree_tile() { return WR == 1 && sizeof(KT) == 2 ? 128 : 64; }
template <int HD, int WR, class KT>
constexpr size_t tree_tile_lds() {  // two BF16 tiles, or one of three parts
    return sizeof(KT) == 2 ? (size_t)4 * tree_tile<WR, KT>() * HD * 2 : (size_t)6 * 64 * HD * 2;
}
template <int HD, int WR, class KT>
constexpr size_t tree_lds_bytes() { return tree_tile_lds<HD, WR, KT>() + sizeof(TreeLds); }
// Blocks of a CU: what its LDS and registers let in.
template <int HD, int WR, class KT>
constexpr int tree_blocks_per_cu() { return HD == 128 && (WR == 1 || sizeof(KT) == 4) ? 1 : 2; }

template <int HD, int WR, class KT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(tree_blocks_per_cu<HD, WR, KT>())))
void tree_attn_kernel(TreeArgs a, int S, int chunk) {
    constexpr bool F32 = sizeof(KT) == 4;
    constexpr int WK = 4 / WR, T = tree_tile<WR, KT>(), STEPS = T / (32 * WK);
    constexpr int KSTEPS = HD / 16, UT = HD / 32;
    constexpr int CPR = HD / 8;       // 16-byte chunks per LDS row
    constexpr int HC = HD / 32;       // BF16: a wave's copies for 64 positions; f32: a thread's 8-dim units of a tile
    constexpr int PL = F32 ? 3 : 1;   // parts (planes) of K and V
    constexpr int TB = T * HD * 2;    // bytes of a tile's plane
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    uint8_t *ks = smem, *vs = smem + (F32 ? 3 : 2) * TB;
    TreeLds &tree = *(TreeLds *)(smem + tree_tile_lds<HD, WR, KT>());
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wr = wave % WR, wk = wave / WR;
    const int n = lane & 31, half = lane >> 5;
    const int G = a.q_heads / a.kv_heads, M = a.n * G, RB = (M + 32 * WR - 1) / (32 * WR);
    const int pair = (int)blockIdx.x / (8 * RB) * 8 + (int)blockIdx.x % 8, rb = (int)blockIdx.x / 8 % RB;
    if (pair >= S * a.kv_heads) return;
    const int g = pair % a.kv_heads, split = pair / a.kv_heads;
    const int m0 = rb * 32 * WR, m = m0 + wr * 32 + n;
    const bool rvalid = m < M;
    const int node = rvalid ? m / G : 0, head = g * G + (rvalid ? m % G : 0);
    const int start = split * chunk;
    const int end = min(start + chunk, a.offset + (min(M, m0 + 32 * WR) - 1) / G + 1);
    float *part = a.part + (((size_t)node * a.q_heads + head) * S + split) * (HD + 2);
    if (start >= end) {  // no row of the block reaches the split
        if (rvalid && wk == 0 && half == 0) part[HD] = -INFINITY;
        return;
    }
    const bool in_tree = end > a.offset;  // block-uniform
    const int last = (end - 1) / 64 * 64;  // the last 64 positions with a row in them
    auto page_of = [&](int p) {  // a scalar load, one tile ahead of its use
        return ((const __attribute__((address_space(4))) int32_t *)a.page_table)[p / a.page_size];
    };
    int page[T / 64];  // of the next tile to fetch
    auto next_pages = [&](int t0) {
#pragma unroll
        for (int x = 0; x < T / 64; ++x) page[x] = page_of(min(t0 + 64 * x, last));
    };

    // BF16 copies of a tile: copy c of a wave fills 1 KB, 64 / CPR rows, of the
    // block's 4 KB; K rows at krow_of, chunks swizzled (attn_prefill_kernel's).
    // Positions past the block's rows may hold stale bytes: masked, and V cleared.
    const int lr = wave * (64 / CPR) + lane / CPR;
    const int koff = krow_of(lr) * HD * 2 + 16 * ((lane % CPR) ^ (lr % CPR));
    const int voff = lr * HD * 2 + 16 * ((lane % CPR) ^ vseg<HD>(lr));
    // f32 units: 8 dims of position idx / CPR, in registers.
    f32x4 kr[F32 ? HC : 1][2], vr[F32 ? HC : 1][2];
    auto fetch = [&](int t0, int b) {
#pragma unroll
        for (int x = 0; x < T / 64; ++x) {
            const int p0 = t0 + 64 * x;
            if (p0 >= end) break;
            const size_t tile = (((size_t)page[x] * a.kv_heads + g) * a.page_size + p0 % a.page_size) * HD;
            if constexpr (F32) {
#pragma unroll
                for (int c = 0; c < HC; ++c) {
                    const int idx = (int)threadIdx.x + kThreads * c;
                    const float *kp = (const float *)a.k + tile + (size_t)idx * 8;
                    const float *vp = (const float *)a.v + tile + (size_t)idx * 8;
                    kr[c][0] = *(const f32x4 *)kp;
                    kr[c][1] = *(const f32x4 *)(kp + 4);
                    vr[c][0] = *(const f32x4 *)vp;
                    vr[c][1] = *(const f32x4 *)(vp + 4);
                }
            } else {
                const int at = b * TB + x * 64 * HD * 2 + wave * 1024;
                const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)((const uint16_t *)a.k + tile), (short)0, 64 * HD * 2, 0x00020000);
                const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)((const uint16_t *)a.v + tile), (short)0, 64 * HD * 2, 0x00020000);
#pragma unroll
                for (int c = 0; c < HC; ++c) buf_to_lds<16>(rk, ks + at + 4096 * c, koff, 4096 * c);
#pragma unroll
                for (int c = 0; c < HC; ++c) buf_to_lds<16>(rv, vs + at + 4096 * c, voff, 4096 * c);
            }
        }
    };
    // V rows past the block's rows become zeros (unwritten memory: a probability
    // of 0 does not clear a NaN), and so do those with an infinity or NaN (f32:
    // or a value that weights of up to 2^8 take past the largest number), whose
    // position is marked. BF16: in a landed tile that reaches the tree, a row by
    // the wave that copied it. f32: while a tile is staged.
    auto mark = [&](int p) {
        const int x = p - a.offset;
        if (x < 0) tree.sick_prefix = 1;
        else atomicOr((unsigned long long *)&tree.sick[x >> 6], 1ull << (x & 63));
    };
    auto clean_v = [&](int t0, int b) {
        for (int c = 0; c < HC * T / 64; ++c) {
            const int p = t0 + lr + 256 / CPR * c;
            if (p < a.offset) continue;
            u32x4 *at = (u32x4 *)(vs + b * TB + wave * 1024 + 4096 * c + 16 * lane);
            bool bad = p >= end;
            if (!bad) {
                const u32x4 w = *at;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    bad |= (w[i] & 0x7F800000u) == 0x7F800000u || (w[i] & 0x7F80u) == 0x7F80u;
                if (bad) mark(p);
            }
            if (bad) *at = u32x4{0u, 0u, 0u, 0u};
        }
    };
    auto stage = [&](int t0) {
#pragma unroll
        for (int c = 0; c < (F32 ? HC : 0); ++c) {
            const int idx = (int)threadIdx.x + kThreads * c, r = idx / CPR, ch = idx % CPR, kr_ = krow_of(r);
            const float kv[8] = {kr[c][0][0], kr[c][0][1], kr[c][0][2], kr[c][0][3],
                                 kr[c][1][0], kr[c][1][1], kr[c][1][2], kr[c][1][3]};
            float vv[8] = {vr[c][0][0], vr[c][0][1], vr[c][0][2], vr[c][0][3],
                           vr[c][1][0], vr[c][1][1], vr[c][1][2], vr[c][1][3]};
            bool fine = true;
#pragma unroll
            for (int i = 0; i < 8; ++i) fine = fine && fabsf(vv[i]) < 0x1p119f;
            const bool past = t0 + r >= end;
            if (!fine && !past) mark(t0 + r);
#pragma unroll
            for (int i = 0; i < 8; ++i) vv[i] = fine && !past ? vv[i] : 0.f;
            bf16x8 w[3];
            split3x8(kv, w);
#pragma unroll
            for (int k = 0; k < 3; ++k) *(bf16x8 *)(ks + k * TB + kr_ * HD * 2 + 16 * (ch ^ (kr_ % CPR))) = w[k];
            split3x8(vv, w);
#pragma unroll
            for (int k = 0; k < 3; ++k) *(bf16x8 *)(vs + k * TB + r * HD * 2 + 16 * (ch ^ vseg<HD>(r))) = w[k];
        }
    };

    next_pages(start);
    fetch(start, 0);
    next_pages(start + T);
    if (threadIdx.x < 4) tree.odd[threadIdx.x] = 0;
    if (threadIdx.x == 0) tree.sick_prefix = 0;
    if (in_tree) find_ancestors(a.parents, a.n, tree);

    bf16x8 q3[KSTEPS][3];
    {
        const float sl2 = (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f;
        const float *qp = a.q + ((size_t)node * a.q_heads + head) * HD + 8 * half;
        const float sq = rvalid ? sl2 : 0.f;  // rows without a query: their scores are not used
        f32x4 raw[KSTEPS][2];  // every load before the first use: one round trip
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
            raw[s][0] = *(const f32x4 *)(qp + 16 * s);
            raw[s][1] = *(const f32x4 *)(qp + 16 * s + 4);
        }
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
            const float v[8] = {raw[s][0][0] * sq, raw[s][0][1] * sq, raw[s][0][2] * sq, raw[s][0][3] * sq,
                                raw[s][1][0] * sq, raw[s][1][1] * sq, raw[s][1][2] * sq, raw[s][1][3] * sq};
            split3x8(v, q3[s]);
        }
    }
    // This lane's transposing V reads in a 16-position block: rows
    // 8 half + i / 4 (and + 4), dims 32 u + 16 ((lane / 16) % 2) + 4 (i % 4).
    const int vi = lane & 15, vrow = 8 * half + (vi >> 2);
    uint32_t vaddr[UT];
#pragma unroll
    for (int u = 0; u < UT; ++u) {
        const int c = (4 * u + 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1)) ^ vseg<HD>(vrow);
        vaddr[u] = (uint32_t)(uintptr_t)(vs + vrow * HD * 2 + 16 * c + 8 * (vi & 1));
    }

    f32x16 oacc[UT];
#pragma unroll
    for (int u = 0; u < UT; ++u) oacc[u] = f32x16{};
    float m2 = -INFINITY, l = 0.f;
    if constexpr (!F32) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (start + T > a.offset) clean_v(start, 0);
    }
    __syncthreads();
    int b = 0;
    for (int t0 = start; t0 < end; t0 += T) {
        const bool more = t0 + T < end;
        if constexpr (F32) {
            stage(t0);
            __syncthreads();
        }
        if (more) {
            fetch(t0 + T, b ^ 1);
            next_pages(t0 + 2 * T);
        }
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            const int p0 = 32 * (wk * STEPS + st);
            if (t0 + p0 >= end) break;
            uint32_t vad[UT];
#pragma unroll
            for (int u = 0; u < UT; ++u) vad[u] = vaddr[u] + b * TB + p0 * HD * 2;
            f32x16 sacc = f32x16{}, slow = f32x16{};
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) {
                const int r = p0 + n;
                const uint8_t *kp = ks + b * TB + r * HD * 2 + 16 * ((2 * s + half) ^ (r % CPR));
                bf16x8 ka[PL];
#pragma unroll
                for (int k = 0; k < PL; ++k) ka[k] = *(const bf16x8 *)(kp + k * TB);
                if constexpr (F32) {
                    slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[2], q3[s][0], slow, 0, 0, 0);
                    slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[1], q3[s][1], slow, 0, 0, 0);
                }
                slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[0], q3[s][2], slow, 0, 0, 0);
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[0], q3[s][0], sacc, 0, 0, 0);
                if constexpr (F32) slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[1], q3[s][0], slow, 0, 0, 0);
                slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[0], q3[s][1], slow, 0, 0, 0);
            }
            sacc += slow;
            // The step's V^T fragments, while the score products drain.
            bf16x8 va[F32 ? 1 : 2][PL][UT];
            if constexpr (!F32) {
                read_vt<HD, 0>(vad, va[0][0]);
                read_vt<HD, 16 * HD * 2>(vad, va[1][0]);
            }
            // Register r holds position 8 half + (r & 3) + (r & 4) + 2 (r & 8) of the step.
            const int x0 = t0 + p0 - a.offset;  // node of the step's first position
            if (x0 + 32 > 0) {
                uint64_t w;
                if (x0 >= 0) {
                    const int i = x0 >> 6, sh = x0 & 63;
                    w = tree.anc[node][i] >> sh;
                    if (sh > 32 && i + 1 < kAncWords) w |= tree.anc[node][i + 1] << (64 - sh);
                } else {
                    w = tree.anc[node][0] << -x0 | ((1ull << -x0) - 1);
                }
                const uint32_t bits = (uint32_t)w >> (8 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(bits >> ((r & 3) + (r & 4) + 2 * (r & 8)) & 1)) sacc[r] = -INFINITY;
            }
            float tmax = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, sacc[r]);
            tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
            // Exponentials against a maximum that is raised only by more than 8
            // (log2 units), so weights are at most 256 and rescaling is rare.
            const bool raise = tmax > m2 + 8.0f;
            if (__any(raise)) {
                const float mnew = raise ? tmax : m2;
                const float alpha = raise ? __builtin_amdgcn_exp2f(m2 - mnew) : 1.f;  // 0 from -inf
                l *= alpha;
#pragma unroll
                for (int u = 0; u < UT; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) oacc[u][r] *= alpha;
                m2 = mnew;
            }
            // A row that has seen no key yet keeps m2 = -inf; its weights are 0.
            const float mref = m2 == -INFINITY ? 0.f : m2;
            float tsum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float pv = __builtin_amdgcn_exp2f(sacc[r] - mref);
                sacc[r] = pv;
                tsum += pv;
            }
            tsum += __shfl_xor(tsum, 32, 64);
            l += tsum;
            auto mix = [&](auto block) {
                constexpr int s2 = decltype(block)::value;
                float pv[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) pv[j] = sacc[8 * s2 + j];
                bf16x8 p3[3];
                split3x8(pv, p3);
                auto product = [&](const bf16x8 (&v)[UT], const bf16x8 &p) {
#pragma unroll
                    for (int u = 0; u < UT; ++u)
                        oacc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[u], p, oacc[u], 0, 0, 0);
                };
                if constexpr (F32) {
                    auto &v = va[0];
                    read_vt<HD, s2 * 16 * HD * 2>(vad, v[0]);
                    read_vt<HD, TB + s2 * 16 * HD * 2>(vad, v[1]);
                    read_vt<HD, 2 * TB + s2 * 16 * HD * 2>(vad, v[2]);
                    product(v[2], p3[0]);
                    product(v[1], p3[1]);
                    product(v[0], p3[2]);
                    product(v[1], p3[0]);
                    product(v[0], p3[1]);
                    product(v[0], p3[0]);
                } else {
                    product(va[s2][0], p3[2]);
                    product(va[s2][0], p3[1]);
                    product(va[s2][0], p3[0]);
                }
            };
            mix(std::integral_constant<int, 0>{});
            mix(std::integral_constant<int, 1>{});
        }
        if constexpr (!F32) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (more && t0 + 2 * T > a.offset) clean_v(t0 + T, b ^ 1);
            b ^= 1;
        }
        __syncthreads();
    }

    // Key waves past the first leave their rows in the tiles' LDS (rows padded
    // by 16 bytes, off each other's banks), the first adds them up in order.
    if constexpr (WK > 1) {
        constexpr int LD = HD + 4;
        static_assert((size_t)(WK - 1) * WR * 32 * (LD + 2) * 4 <= tree_tile_lds<HD, WR, KT>(), "joined in the tiles' LDS");
        auto rows_of = [&](int w) { return (float *)smem + ((w - 1) * WR + wr) * 32 * (LD + 2); };
        if (wk > 0) {
            float *so = rows_of(wk);
#pragma unroll
            for (int u = 0; u < UT; ++u)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4 *)(so + n * LD + 32 * u + 8 * q + 4 * half) =
                        f32x4{oacc[u][4 * q], oacc[u][4 * q + 1], oacc[u][4 * q + 2], oacc[u][4 * q + 3]};
            if (half == 0) {
                so[32 * LD + 2 * n] = m2;
                so[32 * LD + 2 * n + 1] = l;
            }
        }
        __syncthreads();
        if (wk == 0) {
#pragma unroll
            for (int w = 1; w < WK; ++w) {
                const float *si = rows_of(w);
                const float mi = si[32 * LD + 2 * n], li = si[32 * LD + 2 * n + 1];
                const float mn = fmaxf(m2, mi);
                // A wave that saw no key (m = -inf) adds nothing.
                const float fa = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
                const float fb = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - mn);
                m2 = mn;
                l = fmaf(fb, li, l * fa);
#pragma unroll
                for (int u = 0; u < UT; ++u)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 v = *(const f32x4 *)(si + n * LD + 32 * u + 8 * q + 4 * half);
#pragma unroll
                        for (int e = 0; e < 4; ++e) oacc[u][4 * q + e] = fmaf(fb, v[e], oacc[u][4 * q + e] * fa);
                    }
            }
        }
    }
    if (wk == 0 && rvalid) {
        bool odd = l != l || (F32 && tree.sick_prefix);
        if (in_tree)
#pragma unroll
            for (int k = 0; k < kAncWords; ++k) odd |= (tree.anc[node][k] & tree.sick[k]) != 0;
        if (odd) {
            if (half == 0) atomicOr(&tree.odd[wr], 1u << n);
        } else if (S == 1) {
            const float inv = 1.0f / l;
            const size_t ob = ((size_t)node * a.q_heads + head) * HD;
#pragma unroll
            for (int u = 0; u < UT; ++u)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    store_out4(a, ob + 32 * u + 8 * q + 4 * half,
                               f32x4{oacc[u][4 * q] * inv, oacc[u][4 * q + 1] * inv, oacc[u][4 * q + 2] * inv,
                                     oacc[u][4 * q + 3] * inv});
        } else {
#pragma unroll
            for (int u = 0; u < UT; ++u)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4 *)(part + 32 * u + 8 * q + 4 * half) =
                        f32x4{oacc[u][4 * q], oacc[u][4 * q + 1], oacc[u][4 * q + 2], oacc[u][4 * q + 3]};
            if (half == 0) {
                part[HD] = m2;
                part[HD + 1] = l;
            }
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int r = wave; r < 32 * WR; r += 4)
        if (tree.odd[r >> 5] >> (r & 31) & 1) {
            const int i = (m0 + r) / G;
            plain_row<HD, KT>(a, tree, i, g * G + (m0 + r) % G, g, start, min(end, a.offset + i + 1), S, split);
        }
}

// The move of a branch, by value in the launch's arguments: no device copy of
// it to wait for.
struct CommitArgs {
    struct View {
        uint8_t *k, *v;
        const int32_t *page_table;
    } view[kCommitViews];
    uint8_t node[kMaxTreeNodes];
    int count, offset, page_size, kv_heads, row_bytes;
};
static_assert(sizeof(CommitArgs) <= 4096, "a launch's arguments");

// A thread owns one 16-byte column of one KV head's K or V rows in one view and
// moves it for the whole branch, in order. nodes[j] >= j and rises, so the row
// a move overwrites was the source of an earlier move or of none: each batch's
// rows are read before they are written, and a later batch's sources are past
// everything an earlier batch wrote.
__global__ __launch_bounds__(kThreads) void tree_commit_kernel(CommitArgs a, int views) {
    const int cols = a.row_bytes / 16;
    const int t = blockIdx.x * kThreads + threadIdx.x;
    const int c = t % cols, head = t / cols % a.kv_heads, which = t / cols / a.kv_heads;
    if (which >= 2 * views) return;
    const CommitArgs::View &w = a.view[which >> 1];
    uint8_t *pool = which & 1 ? w.v : w.k;
    auto at = [&](int node) {
        const int p = a.offset + node;
        return (u32x4 *)(pool + (((size_t)w.page_table[p / a.page_size] * a.kv_heads + head) * a.page_size +
                                 p % a.page_size) * a.row_bytes + 16 * c);
    };
    constexpr int B = 8;
    for (int j0 = 0; j0 < a.count; j0 += B) {
        u32x4 r[B];
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (j0 + j < a.count) r[j] = *at(a.node[j0 + j]);
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (j0 + j < a.count && a.node[j0 + j] != j0 + j) *at(j0 + j) = r[j];
    }
}

}  // namespace

namespace {

// Row waves of a block: as many as hold the rows, up to 4. An f32 tile has room
// for two key waves only.
int tree_row_waves(const TreeJob &j) {
    const int rows = (int)j.n * (j.q_heads / j.g.kv_heads);
    return rows <= 32 && !j.g.kv_f32 ? 1 : rows <= 64 ? 2 : 4;
}

template <int HD, int WR, class KT>
int launch_tree_blocks(const TreeArgs &a, int S, int chunk, hipStream_t s) {
    constexpr size_t lds = tree_lds_bytes<HD, WR, KT>();
    static std::atomic<uint64_t> lds_set{0};
    CHIP_TRY(allow_dynamic_lds((const void *)tree_attn_kernel<HD, WR, KT>, lds, lds_set));
    const int rb = (a.n * (a.q_heads / a.kv_heads) + 32 * WR - 1) / (32 * WR);
    const size_t blocks = ((size_t)S * a.kv_heads + 7) / 8 * 8 * (size_t)rb;
    if (blocks > (size_t)INT32_MAX) return fail("HIP backend: tree attention grid out of range.");
    hipLaunchKernelGGL((tree_attn_kernel<HD, WR, KT>), dim3((unsigned)blocks), dim3(kThreads), lds, s, a, S, chunk);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

template <int HD>
int launch_tree_h(const TreeJob &j, const TreeArgs &a, int S, int chunk, hipStream_t s) {
    const int wr = tree_row_waves(j);
    if (j.g.kv_f32)
        return wr == 2 ? launch_tree_blocks<HD, 2, float>(a, S, chunk, s) : launch_tree_blocks<HD, 4, float>(a, S, chunk, s);
    return wr == 1   ? launch_tree_blocks<HD, 1, uint16_t>(a, S, chunk, s)
           : wr == 2 ? launch_tree_blocks<HD, 2, uint16_t>(a, S, chunk, s)
                     : launch_tree_blocks<HD, 4, uint16_t>(a, S, chunk, s);
}

int tree_tile_of(const TreeJob &j) { return tree_row_waves(j) == 1 ? 128 : 64; }

}  // namespace

// Splits of the keys: as many as fill the chip with blocks, of whole tiles.
int tree_attention_splits(const TreeJob &j) {
    const int rows = (int)j.n * (j.q_heads / j.g.kv_heads), wr = tree_row_waves(j);
    const size_t tile = (size_t)tree_tile_of(j), tiles = (j.offset + j.n + tile - 1) / tile;
    const size_t per_cu = j.g.head_dim == 128 && (wr == 1 || j.g.kv_f32) ? 1 : 2;
    const size_t blocks = (size_t)((rows + 32 * wr - 1) / (32 * wr)) * (size_t)j.g.kv_heads;
    const size_t want = std::max<size_t>(per_cu * (size_t)std::max(device_cus(), 1) / blocks, 1);
    const size_t S = std::min({want, tiles, (size_t)attention_max_splits()}), each = (tiles + S - 1) / S;
    return (int)((tiles + each - 1) / each);
}

int launch_tree_attention(const TreeJob &j, hipStream_t s) {
    if (!j.q || (!j.out && !j.out_hi) || !j.out_hi != !j.out_lo || !j.k || !j.v || !j.g.page_table || !j.parents)
        return fail("HIP backend: tree attention is missing a buffer.");
    if (j.n == 0 || j.n > (size_t)kMaxTreeNodes || j.offset > (size_t)INT32_MAX - j.n)
        return fail("HIP backend: tree attention shape out of range.");
    int S = tree_attention_splits(j);
    const size_t split_floats = attention_part_floats(j.n, j.q_heads, 1, j.g.head_dim);
    if (S > 1) S = (int)std::min<size_t>((size_t)S, std::max<size_t>(j.part ? j.part_floats / split_floats : 1, 1));
    const size_t tile = (size_t)tree_tile_of(j), tiles = (j.offset + j.n + tile - 1) / tile, each = (tiles + S - 1) / S;
    S = (int)((tiles + each - 1) / each);
    TreeArgs a{};
    a.q = j.q;
    a.k = j.k;
    a.v = j.v;
    a.page_table = j.g.page_table;
    a.parents = j.parents;
    a.part = j.part;
    a.out = j.out;
    a.out_hi = j.out_hi;
    a.out_lo = j.out_lo;
    a.page_size = j.g.page_size;
    a.kv_heads = j.g.kv_heads;
    a.q_heads = j.q_heads;
    a.offset = (int)j.offset;
    a.n = (int)j.n;
    const int chunk = (int)(each * tile);
    if (j.g.head_dim == 64) CHIP_TRY(launch_tree_h<64>(j, a, S, chunk, s));
    else CHIP_TRY(launch_tree_h<128>(j, a, S, chunk, s));
    return launch_attention_merge(j.part, S, j.n, j.q_heads, j.g.head_dim, j.out, j.out_hi, j.out_lo, s);
}

int launch_tree_commit(const KvLayer *layers, const int32_t *const *page_tables, size_t views, const KvGeom &g,
                       size_t offset, const uint32_t *nodes, size_t count, hipStream_t s) {
    size_t first = 0;  // nodes already in place
    while (first < count && nodes[first] == first) ++first;
    if (first == count) return 0;
    CommitArgs a{};
    for (size_t j = 0; j < count; ++j) a.node[j] = (uint8_t)nodes[j];
    a.count = (int)count;
    a.offset = (int)offset;
    a.page_size = g.page_size;
    a.kv_heads = g.kv_heads;
    a.row_bytes = g.head_dim * (g.kv_f32 ? 4 : 2);
    for (size_t v0 = 0; v0 < views; v0 += kCommitViews) {
        const size_t n = std::min(views - v0, (size_t)kCommitViews);
        for (size_t i = 0; i < n; ++i)
            a.view[i] = {(uint8_t *)layers[v0 + i].k, (uint8_t *)layers[v0 + i].v, page_tables[v0 + i]};
        const size_t threads = 2 * n * (size_t)g.kv_heads * (size_t)(a.row_bytes / 16);
        hipLaunchKernelGGL(tree_commit_kernel, dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                           s, a, (int)n);
        CHIP_CHECK(hipGetLastError());
    }
    return 0;
}

}  // namespace chip
