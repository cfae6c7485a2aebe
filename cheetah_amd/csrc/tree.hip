// Attention for a tree of drafted tokens over the paged KV cache, and the move
// of its accepted branch's K/V rows into place.
//
// Node i of n has its parent parents[i] < i (anything else: none, a root). Its
// K/V row sits at cache position offset + i. With the cached prefix [0, offset)
// every node sees its ancestors and itself:
//   out[i, h] = sum_p w_p v[p, h / G],  w = softmax_p(q[i, h] . k[p, h / G] / sqrt(head_dim))
// over p in [0, offset) and offset + a, a = i or an ancestor of i.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "attn_tiles.hpp"
#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256;

// Block barrier that waits on LDS traffic only: loads stay in flight across it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct TreeArgs {
    const float *q;
    const void *k, *v;
    const int32_t *page_table;
    const int32_t *parents;
    float *part;  // [row][head][split][HD]: weighted sums
    float2 *ml;   // [row][head][split]: maximum (log2 units), weight sum
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
// log2(depth) rounds, whatever the tree's shape. The caller's next barrier
// makes them visible.
constexpr int kAncWords = kMaxTreeNodes / 64;
struct TreeLds {
    uint64_t anc[kMaxTreeNodes][kAncWords];
    uint64_t sick[kAncWords];  // nodes with an infinity or NaN in V
    uint32_t odd[4];           // a row wave's rows to compute again
    int32_t pages[64];         // the split's first page table entries
    int16_t up[kMaxTreeNodes];
};
__device__ __forceinline__ void find_ancestors(int p, int n, TreeLds &t) {  // p: parents[thread]
    const int i = threadIdx.x;  // nodes are the first kMaxTreeNodes threads
    if (i >= n || p >= i) p = -1;
    if (i < kAncWords) t.sick[i] = 0;
    if (n <= 64) {  // one wave, in registers
        if (i >= 64) return;
        uint64_t w = 1ull << i;
        while (__any(p >= 0)) {
            const int from = max(p, 0);
            const uint64_t up = (uint64_t)(uint32_t)__shfl((int)w, from, 64) |
                                (uint64_t)(uint32_t)__shfl((int)(w >> 32), from, 64) << 32;
            const int q = __shfl(p, from, 64);
            w = p >= 0 ? w | up : w;
            p = p >= 0 ? q : p;
        }
        t.anc[i][0] = w;
#pragma unroll
        for (int k = 1; k < kAncWords; ++k) t.anc[i][k] = 0;
        return;
    }
    uint64_t w[kAncWords];
    const bool mine = i < kMaxTreeNodes;
    if (mine) {
#pragma unroll
        for (int k = 0; k < kAncWords; ++k) t.anc[i][k] = w[k] = i >> 6 == k ? 1ull << (i & 63) : 0;
        t.up[i] = (int16_t)max(p, -1);
    }
    while (__syncthreads_or(p >= 0)) {
        if (p >= 0) {
#pragma unroll
            for (int k = 0; k < kAncWords; ++k) w[k] |= t.anc[p][k];
            p = t.up[p];
        }
        __syncthreads();  // every path is read before one grows
        if (mine) {
#pragma unroll
            for (int k = 0; k < kAncWords; ++k) t.anc[i][k] = w[k];
            t.up[i] = (int16_t)max(p, -1);
        }
    }
}

__device__ __forceinline__ float kv_value(const uint16_t *p) { return bf16_f32(*p); }
__device__ __forceinline__ float kv_value(const float *p) { return *p; }

// One row over positions [start, end) in plain f32 products, a wave per row and
// a lane per HD / 64 dims: the rare rows that the matrix cores' parts do not
// carry. They see an infinity or NaN in a tree node's V, which 0 x V would spread
// over the tile's rows and which is cleared there; or an output is not finite,
// where a weight's part of 0 has met an infinity in the prefix, or weights of up to
// 2^8 have taken a sum of large values past the largest number; or their weight sum
// is NaN, where a score of -inf has to weigh nothing. A NaN sum ends the row. Where
// a sum overflows with weights of at most 1 too, it is taken again of V / 2^32 (it
// has fewer than 2^32 keys): the average itself is no larger than V. A key takes a
// wave some 0.4 us: an infinity that 256 nodes see on 4,097 (28 / 4 heads of 128)
// makes 6.9 ms of 52 us, a NaN key (the row ends there) 74 us.
template <int HD, class KT>
__device__ void plain_row(const TreeArgs &a, const TreeLds &t, int node, int head, int g, int start, int end, int S,
                          int split) {
    constexpr int D = HD / 64;
    const int lane = threadIdx.x & 63;
    const size_t row = ((size_t)node * a.q_heads + head) * HD;
    const float scale = (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f;
    float q[D], o[D], seen[D], m, l;  // seen: NaN with an infinity or NaN in a key's V
#pragma unroll
    for (int d = 0; d < D; ++d) q[d] = a.q[row + lane + 64 * d];
    int shift = 0;  // V / 2^shift
    for (;;) {
        const float vs = shift ? 0x1p-32f : 1.f;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = seen[d] = 0.f;
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
            for (int d = 0; d < D; ++d) {
                const float v = kv_value((const KT *)a.v + at + lane + 64 * d);
                o[d] = fmaf(w, v * vs, o[d] * alpha);
                seen[d] = fmaf(v, 0.f, seen[d]);
            }
        }
        bool over = false;
#pragma unroll
        for (int d = 0; d < D; ++d) over |= seen[d] == 0.f && o[d] * 0.f != 0.f;
        if (shift || l != l || !__any(over)) break;
        shift = 32;
    }
    const size_t at = ((size_t)node * a.q_heads + head) * S + split;
#pragma unroll
    for (int d = 0; d < D; ++d) {
        if (S > 1) {
            a.part[at * HD + lane + 64 * d] = o[d];
        } else {
            const float v = o[d] / l * (shift ? 0x1p32f : 1.f);
            if (a.out) a.out[row + lane + 64 * d] = v;
            if (a.out_hi) {
                const __bf16 hb = (__bf16)v;
                a.out_hi[row + lane + 64 * d] = __builtin_bit_cast(uint16_t, hb);
                a.out_lo[row + lane + 64 * d] = __builtin_bit_cast(uint16_t, (__bf16)(v - (float)hb));
            }
        }
    }
    // A NaN row: no split outweighs it. A scaled one: its sums are 2^-32 of theirs,
    // about a maximum 2^32 higher. Scores of -inf only: not a split without a key.
    if (S > 1 && lane == 0)
        a.ml[at] = make_float2(l == l ? fmaxf(m + (float)shift, -FLT_MAX) : INFINITY, shift ? l * 0x1p-32f : l);
}

// Eight values as three BF16 parts, each the top 8 bits of what the ones before
// leave: all 24 bits of a value (no roundings: 11 instructions a pair where
// split3x8's rounded parts take 16).
__device__ __forceinline__ void cut3x8(const float (&v)[8], bf16x8 (&out)[3]) {
    u32x4 w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t x[2], y[2], z[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            x[k] = __float_as_uint(v[2 * i + k]);
            const float r = v[2 * i + k] - __uint_as_float(x[k] & 0xFFFF0000u);
            y[k] = __float_as_uint(r);
            z[k] = __float_as_uint(r - __uint_as_float(y[k] & 0xFFFF0000u));
        }
        w[0][i] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
        w[1][i] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302u);
        w[2][i] = __builtin_amdgcn_perm(z[1], z[0], 0x07060302u);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) out[k] = __builtin_bit_cast(bf16x8, w[k]);
}

// A value that is to be there at this point, in vector or in accumulation registers.
__device__ __forceinline__ void pin_v(bf16x8 &x) {
    u32x4 w = __builtin_bit_cast(u32x4, x);
    asm volatile("" : "+v"(w));
    x = __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ void pin_a(bf16x8 &x) {
    u32x4 w = __builtin_bit_cast(u32x4, x);
    asm volatile("" : "+a"(w));
    x = __builtin_bit_cast(bf16x8, w);
}

// read_vt of two blocks of 16 positions, OFF and OFF + 16 rows, in one wait.
template <int HD>
__device__ __forceinline__ void read_vt2(const uint32_t (&addr)[HD / 32], bf16x8 (&v0)[HD / 32], bf16x8 (&v1)[HD / 32]) {
    s16x4_t r[2][HD / 32][2];
    if constexpr (HD == 128) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%20\n\t"
            "ds_read_b64_tr_b16 %2, %17\n\tds_read_b64_tr_b16 %3, %17 offset:%20\n\t"
            "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:%20\n\t"
            "ds_read_b64_tr_b16 %6, %19\n\tds_read_b64_tr_b16 %7, %19 offset:%20\n\t"
            "ds_read_b64_tr_b16 %8, %16 offset:%21\n\tds_read_b64_tr_b16 %9, %16 offset:%22\n\t"
            "ds_read_b64_tr_b16 %10, %17 offset:%21\n\tds_read_b64_tr_b16 %11, %17 offset:%22\n\t"
            "ds_read_b64_tr_b16 %12, %18 offset:%21\n\tds_read_b64_tr_b16 %13, %18 offset:%22\n\t"
            "ds_read_b64_tr_b16 %14, %19 offset:%21\n\tds_read_b64_tr_b16 %15, %19 offset:%22\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0][0][0]), "=&v"(r[0][0][1]), "=&v"(r[0][1][0]), "=&v"(r[0][1][1]), "=&v"(r[0][2][0]),
              "=&v"(r[0][2][1]), "=&v"(r[0][3][0]), "=&v"(r[0][3][1]), "=&v"(r[1][0][0]), "=&v"(r[1][0][1]),
              "=&v"(r[1][1][0]), "=&v"(r[1][1][1]), "=&v"(r[1][2][0]), "=&v"(r[1][2][1]), "=&v"(r[1][3][0]),
              "=&v"(r[1][3][1])
            : "v"(addr[0]), "v"(addr[1]), "v"(addr[2]), "v"(addr[3]), "i"(4 * HD * 2), "i"(16 * HD * 2), "i"(20 * HD * 2)
            : "memory");
    } else {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
            "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%10\n\t"
            "ds_read_b64_tr_b16 %4, %8 offset:%11\n\tds_read_b64_tr_b16 %5, %8 offset:%12\n\t"
            "ds_read_b64_tr_b16 %6, %9 offset:%11\n\tds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0][0][0]), "=&v"(r[0][0][1]), "=&v"(r[0][1][0]), "=&v"(r[0][1][1]), "=&v"(r[1][0][0]),
              "=&v"(r[1][0][1]), "=&v"(r[1][1][0]), "=&v"(r[1][1][1])
            : "v"(addr[0]), "v"(addr[1]), "i"(4 * HD * 2), "i"(16 * HD * 2), "i"(20 * HD * 2)
            : "memory");
    }
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
        v0[u] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0][u][0], r[0][u][1], 0, 1, 2, 3, 4, 5, 6, 7));
        v1[u] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[1][u][0], r[1][u][1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// ---------------------------------------------------------------------------
// On the matrix cores. The M = n G rows (node, head of the group) of a KV head
// are cut into waves of 32 and blocks of WR row waves; the WK key waves of a
// row wave take 32 positions each of the block's tiles and are joined at the end.
// Per tile, as attn_prefill_kernel's:
//   S^T = K Q^T     K rows from LDS, Q^T in registers
//   O^T += V^T P^T  V read transposed, P^T as the scores' registers lie
// Q (scaled by log2(e) / sqrt(HD)) and P are three BF16 parts each, all 24 bits
// of them. Over a BF16 cache K and V are exact: three products for one, as
// exact as f32 ones; with two parts the output would be 3.5e-6 off where f32
// products give 1e-6. An f32 cache's K and V are three parts too, and six of
// the nine part products are taken (attn_prefill_f32_kernel's).
//
// BF16 tiles of 128 positions go global to LDS, the next one while the current
// one computes; two waves a SIMD, one's softmax beside the other's products, in one
// block: two blocks of four waves a CU ran at the pace of their ages, and the younger
// alone at the end. f32 tiles of 64 come in registers, two ahead: while the scores
// are multiplied the next one is cut into its parts, which take the keys' place in
// LDS when those are read (200 nodes on 2,000, 32 / 8 heads of 128: 90 us when a tile
// was cut between two others, so 79; its products alone would take 34).
// The queries then sit in accumulation registers, which products read as well.
//
// Splits are runs of positions, joined by tree_merge_kernel. Blocks with
// the same (split, KV head) and other rows are 8 apart, on one XCD: they read
// the same tiles through its L2.
//
// Bound, long contexts: the matrix cores. 64 nodes on 16k (32 / 8 heads of 128)
// take 51.0 us for 17.2 Gflop, 51.5 Gflop of them executed, 1.2 PFLOP/s in the loop,
// what a large BF16 matrix product reaches (1.21). Around the loop's 43: 2.7 before
// the first product, 1.2 for the key waves' join, 0.8 to write the partials, 2.5 a
// launch, 4 the merge. Priorities or a late start for half of the waves change
// nothing. Short contexts: those steps. 16 nodes on 2k 14.3 us, its tile 2.2 of
// them; 5 on 60 (14 / 2 heads of 64) 6.2, one launch.
// ---------------------------------------------------------------------------
template <class KT>
constexpr int tree_tile() { return sizeof(KT) == 2 ? 128 : 64; }
template <int HD, class KT>
constexpr size_t tree_tile_lds() {  // two BF16 tiles; K of three parts and V, at head_dim 128 two of it
    return (size_t)(sizeof(KT) == 2 ? 4 : HD == 128 ? 9 : 6) * tree_tile<KT>() * HD * 2;
}
template <int HD, class KT>
constexpr size_t tree_lds_bytes() { return tree_tile_lds<HD, KT>() + sizeof(TreeLds); }

template <int HD, int WR, int WK, class KT>
__global__ __launch_bounds__(64 * WR * WK) __attribute__((amdgpu_waves_per_eu(sizeof(KT) == 4 && HD == 64 ? 2 : WR * WK / 4)))
void tree_attn_kernel(TreeArgs a, int S) {
    constexpr bool F32 = sizeof(KT) == 4;
    constexpr int NW = WR * WK, T = tree_tile<KT>();
    static_assert(WK > 1 && T == 32 * WK, "32 positions of a tile for each key wave");
    constexpr int KSTEPS = HD / 16, UT = HD / 32;
    constexpr int CPR = HD / 8;       // 16-byte chunks per LDS row
    constexpr int HC = HD / 8 / NW;   // BF16: a wave's copies for 64 positions; f32: a thread's 8-dim units of a tile
    constexpr int PL = F32 ? 3 : 1;   // parts (planes) of K and V
    constexpr int TB = T * HD * 2;    // bytes of a tile's plane
    constexpr bool V2 = F32 && HD == 128;  // the next tile's V has a place of its own
    extern __shared__ __attribute__((aligned(256))) uint8_t smem[];
    uint8_t *ks = smem, *vs = smem + PL * TB;  // the second BF16 tile, 2 TB on
    TreeLds &tree = *(TreeLds *)(smem + tree_tile_lds<HD, KT>());
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
    // A run of tiles a split, the first ones one more. (Block-uniform, said to the
    // compiler: the quotients come from vector registers.)
    const int tiles = (a.offset + a.n - 1) / T + 1, each = tiles / S, extra = tiles % S;
    const int first = split * each + min(split, extra);
    const int start = __builtin_amdgcn_readfirstlane(first * T);
    const int end = __builtin_amdgcn_readfirstlane(
        (int)min((unsigned)(first + each + (split < extra)) * T, (unsigned)(a.offset + (min(M, m0 + 32 * WR) - 1) / G + 1)));
    const size_t at_part = ((size_t)node * a.q_heads + head) * S + split;
    if (start >= end) {  // no row of the block reaches the split
        if (rvalid && wk == 0 && half == 0) a.ml[at_part] = make_float2(-INFINITY, 0.f);
        return;
    }
    const bool in_tree = end > a.offset;  // block-uniform
    // Page table entries held_0 .. + 63, a lane each: the loop looks pages up
    // without a load (a scalar load in flight would make each wait for an LDS
    // read a wait for all of them).
    const int last_page = (end - 1) / a.page_size;
    int page_i = __builtin_amdgcn_readfirstlane(start / a.page_size), held_0 = page_i;
    int page_at = start - page_i * a.page_size;
    // The first ones by one wave, for all: a CU's loads return in order, and the
    // second four waves' own would come behind the first four's copies (at 2.7 us
    // where the first four's come at 0.7).
    int held = wave == 0 ? a.page_table[min(held_0 + lane, last_page)] : 0;
    int page[T / 64], row0[T / 64];  // of the next tile to fetch
    auto next_pages = [&](int t0) {
#pragma unroll
        for (int x = 0; x < T / 64; ++x) {
            if (t0 + 64 * x >= end) break;
            if (page_i - held_0 == 64) {
                held_0 = page_i;
                held = a.page_table[min(held_0 + lane, last_page)];
                asm volatile("" : "+v"(held));  // waited for here, not by every lookup
            }
            page[x] = __builtin_amdgcn_readlane(held, page_i - held_0);
            row0[x] = page_at;
            page_at += 64;
            if (page_at == a.page_size) page_at = 0, ++page_i;
        }
    };

    // BF16 copies of a tile: copy c of a wave fills 1 KB, 64 / CPR rows, of the
    // block's NW KB; K rows at krow_of, chunks swizzled (attn_prefill_kernel's).
    // Positions past the block's rows may hold stale bytes: masked, and V cleared.
    const int lr = wave * (64 / CPR) + lane / CPR;
    const int koff = krow_of(lr) * HD * 2 + 16 * ((lane % CPR) ^ (lr % CPR));
    const int voff = lr * HD * 2 + 16 * ((lane % CPR) ^ vseg<HD>(lr));
    // f32 units: 8 dims of position idx / CPR, in registers.
    f32x4 kr[F32 ? HC : 1][2], vr[F32 ? HC : 1][2];
    auto fetch = [&](int t0, int b) {
#pragma unroll
        for (int x = 0; x < T / 64; ++x) {
            if (t0 + 64 * x >= end) break;
            const size_t tile = (((size_t)page[x] * a.kv_heads + g) * a.page_size + row0[x]) * HD;
            if constexpr (F32) {
#pragma unroll
                for (int c = 0; c < HC; ++c) {
                    const int idx = (int)threadIdx.x + 64 * NW * c;
                    const float *kp = (const float *)a.k + tile + (size_t)idx * 8;
                    const float *vp = (const float *)a.v + tile + (size_t)idx * 8;
                    kr[c][0] = *(const f32x4 *)kp;
                    kr[c][1] = *(const f32x4 *)(kp + 4);
                    vr[c][0] = *(const f32x4 *)vp;
                    vr[c][1] = *(const f32x4 *)(vp + 4);
                }
            } else {
                const int at = b * 2 * TB + x * 64 * HD * 2 + wave * 1024;
                const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)((const uint16_t *)a.k + tile), (short)0, 64 * HD * 2, 0x00020000);
                const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)((const uint16_t *)a.v + tile), (short)0, 64 * HD * 2, 0x00020000);
#pragma unroll
                for (int c = 0; c < HC; ++c) buf_to_lds<16>(rk, ks + at + 1024 * NW * c, koff, 1024 * NW * c);
#pragma unroll
                for (int c = 0; c < HC; ++c) buf_to_lds<16>(rv, vs + at + 1024 * NW * c, voff, 1024 * NW * c);
            }
        }
    };
    // V rows past the block's rows become zeros (unwritten memory: a probability
    // of 0 does not clear a NaN), and so do nodes' with an infinity or NaN, which
    // are marked. (The prefix's reach every row; they show in the result.) BF16: in
    // a landed tile that reaches the tree, a row by the wave that copied it. f32:
    // when its parts are stored.
    auto mark = [&](int p) {
        const int x = p - a.offset;
        atomicOr((unsigned long long *)&tree.sick[x >> 6], 1ull << (x & 63));
    };
    auto clean_v = [&](int t0, int b) {
        for (int c = 0; c < HC * T / 64; ++c) {
            const int p = t0 + lr + 64 * NW / CPR * c;
            if (p < a.offset) continue;
            u32x4 *at = (u32x4 *)(vs + b * 2 * TB + wave * 1024 + 1024 * NW * c + 16 * lane);
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
    // f32: unit c of the next tile, cut into its parts while the matrix cores work
    // on the current one; then all of them into the tile's place.
    bf16x8 kp[F32 ? HC : 1][3], vp[F32 ? HC : 1][3];
    uint32_t vmost[F32 ? HC : 1];  // largest magnitude of a unit's V, as bits
    auto cut_unit = [&](int c) {
        const float kv[8] = {kr[c][0][0], kr[c][0][1], kr[c][0][2], kr[c][0][3],
                             kr[c][1][0], kr[c][1][1], kr[c][1][2], kr[c][1][3]};
        const float vv[8] = {vr[c][0][0], vr[c][0][1], vr[c][0][2], vr[c][0][3],
                             vr[c][1][0], vr[c][1][1], vr[c][1][2], vr[c][1][3]};
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(vv[i]) & 0x7FFFFFFFu);
        vmost[c] = most;
        cut3x8(kv, kp[c]);
        cut3x8(vv, vp[c]);
        if constexpr (HD == 128)
#pragma unroll
            for (int k = 0; k < 3; ++k) {  // here, not where they are stored
                pin_v(kp[c][k]);
                pin_v(vp[c][k]);
            }
    };
    auto store_k = [&]() {
#pragma unroll
        for (int c = 0; c < (F32 ? HC : 0); ++c) {
            const int idx = (int)threadIdx.x + 64 * NW * c, ch = idx % CPR, kr_ = krow_of(idx / CPR);
#pragma unroll
            for (int k = 0; k < 3; ++k) *(bf16x8 *)(ks + k * TB + kr_ * HD * 2 + 16 * (ch ^ (kr_ % CPR))) = kp[c][k];
        }
    };
    auto store_v = [&](int t0, int b) {
#pragma unroll
        for (int c = 0; c < (F32 ? HC : 0); ++c) {
            const int idx = (int)threadIdx.x + 64 * NW * c, r = idx / CPR, ch = idx % CPR;
            const bool past = t0 + r >= end, sick = t0 + r >= a.offset && vmost[c] >= 0x7F800000u;
            if (__any(past || sick)) {
                if (sick && !past) mark(t0 + r);
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    if (past || sick) vp[c][k] = bf16x8{};
            }
#pragma unroll
            for (int k = 0; k < 3; ++k) *(bf16x8 *)(vs + (3 * b + k) * TB + r * HD * 2 + 16 * (ch ^ vseg<HD>(r))) = vp[c][k];
        }
    };

    // What the tile's copies would hold up is asked for before them: the parents,
    // and the queries. The key waves of a row wave load and cut a part of its
    // fragments each (cutting all of them takes a wave 0.8 us) and hand them on in
    // LDS, where the first tile does not come: BF16 in the second tile's place, f32
    // in its own.
    constexpr int OWN = KSTEPS / WK, kFragments = 3 * 1024;  // a step's three parts, 16 bytes a lane
    static_assert(WR * KSTEPS * kFragments <= (F32 ? 6 : 2) * TB, "room for the fragments");
    const int parent = in_tree && (int)threadIdx.x < a.n ? a.parents[threadIdx.x] : -1;
    f32x4 raw[OWN][2];
    {
        const float *qp = a.q + ((size_t)node * a.q_heads + head) * HD + 8 * half;
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            raw[i][0] = *(const f32x4 *)(qp + 16 * (i * WK + wk));
            raw[i][1] = *(const f32x4 *)(qp + 16 * (i * WK + wk) + 4);
        }
    }
    if (wave == 0) tree.pages[lane] = held;
    if (threadIdx.x < 4) tree.odd[threadIdx.x] = 0;
    lds_barrier();
    held = tree.pages[lane];
    next_pages(start);
    fetch(start, 0);
    next_pages(start + T);

    bf16x8 q3[KSTEPS][3];
    const float sq = rvalid ? (1.0f / sqrtf((float)HD)) * 1.44269504088896340736f : 0.f;  // (no query: scores not used)
    uint8_t *at = smem + (F32 ? 0 : 2 * TB) + wr * KSTEPS * kFragments + lane * 16;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        const float v[8] = {raw[i][0][0] * sq, raw[i][0][1] * sq, raw[i][0][2] * sq, raw[i][0][3] * sq,
                            raw[i][1][0] * sq, raw[i][1][1] * sq, raw[i][1][2] * sq, raw[i][1][3] * sq};
        bf16x8 w[3];
        cut3x8(v, w);
#pragma unroll
        for (int k = 0; k < 3; ++k)
            *(bf16x8 *)(at + ((i * WK + wk) * 3 + k) * 1024) = w[k];
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i)
#pragma unroll
        for (int k = 0; k < 3; ++k) q3[i][k] = *(const bf16x8 *)(at + (i * 3 + k) * 1024);
    if constexpr (F32 && HD == 128)
#pragma unroll
        for (int i = 0; i < KSTEPS; ++i)
#pragma unroll
            for (int k = 0; k < 3; ++k) pin_a(q3[i][k]);
    if constexpr (F32) lds_barrier();  // read before the tile comes in their place
    if (in_tree) find_ancestors(parent, a.n, tree);
    // This lane's transposing V reads in a 16-position block: rows
    // 8 half + i / 4 (and + 4), dims 32 u + 16 ((lane / 16) % 2) + 4 (i % 4).
    const int vi = lane & 15, vrow = 8 * half + (vi >> 2);
    // The chunk swizzles touch address bits that u and s alone set besides them:
    // one base, and an exclusive or for each read.
    const uint32_t vbase = (uint32_t)(uintptr_t)(vs + vrow * HD * 2 + 8 * (vi & 1) +
                                                 16 * ((2 * ((lane >> 4) & 1) + ((vi & 3) >> 1)) ^ vseg<HD>(vrow)));
    const int kbase = n * HD * 2 + 16 * (half ^ (n % CPR));

    f32x16 oacc[UT];
#pragma unroll
    for (int u = 0; u < UT; ++u) oacc[u] = f32x16{};
    float m2 = -INFINITY, l = 0.f;
    if constexpr (!F32) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (start + T > a.offset) {
            __syncthreads();  // the marks start at none
            clean_v(start, 0);
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int c = 0; c < HC; ++c) cut_unit(c);
        if (start + T < end) {
            fetch(start + T, 0);
            next_pages(start + 2 * T);
        }
        lds_barrier();
        store_k();
        store_v(start, 0);
        lds_barrier();
    }
    int b = 0;
    for (int t0 = start; t0 < end; t0 += T) {
        const bool more = t0 + T < end;
        if (!F32 && more) {
            fetch(t0 + T, b ^ 1);
            next_pages(t0 + 2 * T);
        }
        const int p0 = 32 * wk;
        if (t0 + p0 < end) {  // a tile with another behind it is full
            uint32_t vad[UT];
#pragma unroll
            for (int u = 0; u < UT; ++u) vad[u] = (vbase + b * (F32 ? 3 : 2) * TB + p0 * HD * 2) ^ (64 * u);
            const int kat = kbase + (F32 ? 0 : b * 2 * TB) + p0 * HD * 2;
            // BF16: every K fragment of the step in flight at once. (f32: three parts
            // of each would take the registers of the second wave at head_dim 64.)
            bf16x8 ka[F32 ? 1 : KSTEPS][PL];
            auto read_k = [&](int s, bf16x8 (&k)[PL]) {
#pragma unroll
                for (int x = 0; x < PL; ++x) k[x] = *(const bf16x8 *)(ks + (kat ^ (32 * s)) + x * TB);
            };
            if constexpr (!F32) {
#pragma unroll
                for (int s = 0; s < KSTEPS; ++s) read_k(s, ka[s]);
                __builtin_amdgcn_sched_barrier(0);
            }
            // f32 caches add the small products up by themselves.
            f32x16 sacc = f32x16{}, small = f32x16{};
            f32x16 &slow = F32 ? small : sacc;
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) {
                auto &k = ka[F32 ? 0 : s];
                if constexpr (F32) {
                    read_k(s, k);
                    slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[2], q3[s][0], slow, 0, 0, 0);
                    slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[1], q3[s][1], slow, 0, 0, 0);
                }
                slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], q3[s][2], slow, 0, 0, 0);
                if constexpr (F32) slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[1], q3[s][0], slow, 0, 0, 0);
                slow = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], q3[s][1], slow, 0, 0, 0);
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], q3[s][0], sacc, 0, 0, 0);
                if constexpr (F32) {
                    constexpr int EVERY = KSTEPS / HC;  // k-steps a unit of the next tile
                    if (s % EVERY == EVERY - 1) cut_unit(s / EVERY);
                }
            }
            if (F32 && more) {
                lds_barrier();  // the tile's keys are read
                store_k();
                if constexpr (V2) store_v(t0 + T, b ^ 1);
                if (t0 + 2 * T < end) {
                    fetch(t0 + 2 * T, 0);
                    next_pages(t0 + 3 * T);
                }
            }
            if constexpr (F32) sacc += small;
            // The step's V^T fragments, while the score products drain.
            bf16x8 va[2][UT];
            if constexpr (!F32) read_vt2<HD>(vad, va[0], va[1]);
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
            // Exponentials against a maximum that is raised only by more than 8
            // (log2 units), so weights are at most 256 and rescaling is rare. The
            // two lanes of a row share it; each sums its own weights.
            if (__any(tmax > m2 + 8.0f)) {
                tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
                const bool raise = tmax > m2 + 8.0f;
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
            l += tsum;
            auto mix = [&](auto block) {
                constexpr int s2 = decltype(block)::value;
                float pv[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) pv[j] = sacc[8 * s2 + j];
                bf16x8 p3[3];
                cut3x8(pv, p3);
                auto product = [&](const bf16x8 (&v)[UT], const bf16x8 &p) {
#pragma unroll
                    for (int u = 0; u < UT; ++u)
                        oacc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[u], p, oacc[u], 0, 0, 0);
                };
                if constexpr (F32) {
                    bf16x8 v[3][UT];
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
                    product(va[s2], p3[2]);
                    product(va[s2], p3[1]);
                    product(va[s2], p3[0]);
                }
            };
            mix(std::integral_constant<int, 0>{});
            mix(std::integral_constant<int, 1>{});
        }
        if constexpr (!F32) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (more && t0 + 2 * T > a.offset) clean_v(t0 + T, b ^ 1);
            b ^= 1;
            __syncthreads();
        } else {
            lds_barrier();
            if (V2) {
                b ^= 1;
            } else if (more) {
                store_v(t0 + T, 0);
                lds_barrier();
            }
        }
    }

    l += __shfl_xor(l, 32, 64);
    // The key waves of a row join in LDS, in the tiles' place: each leaves the
    // blocks of 32 dims that others own (block u: wave u % WK) and adds up its own,
    // in wave order. Rows padded by 16 bytes, off each other's banks.
    {
        constexpr int LD = 32 + 4;
        static_assert((size_t)WR * UT * (WK - 1) * 32 * LD * 4 + (size_t)NW * 32 * 8 <= tree_tile_lds<HD, KT>(),
                      "joined in the tiles' LDS");
        auto block = [&](int w, int u) {  // of key wave w, without its own ones
            const int own_before = WK <= UT ? w * (UT / WK) : min(w, UT), own_below = u > w ? (u - w - 1) / WK + 1 : 0;
            return (float *)smem + (wr * UT * (WK - 1) + w * UT - own_before + u - own_below) * 32 * LD + n * LD + 4 * half;
        };
        float2 *ml = (float2 *)((float *)smem + WR * UT * (WK - 1) * 32 * LD) + wr * WK * 32 + n;
#pragma unroll
        for (int u = 0; u < UT; ++u)
            if (u % WK != wk)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4 *)(block(wk, u) + 8 * q) =
                        f32x4{oacc[u][4 * q], oacc[u][4 * q + 1], oacc[u][4 * q + 2], oacc[u][4 * q + 3]};
        if (half == 0) ml[32 * wk] = make_float2(m2, l);
        __syncthreads();
        float2 x[WK];
        m2 = -INFINITY;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            x[w] = ml[32 * w];
            m2 = fmaxf(m2, x[w].x);
        }
        l = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) {  // a wave that saw no key (-inf) adds nothing
            x[w].x = x[w].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[w].x - m2);
            l = fmaf(x[w].x, x[w].y, l);
        }
#pragma unroll
        for (int u = 0; u < UT; ++u)
            if (u % WK == wk) {
                const f32x16 own = oacc[u];
                oacc[u] = f32x16{};
#pragma unroll
                for (int w = 0; w < WK; ++w)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 v = w == wk ? f32x4{own[4 * q], own[4 * q + 1], own[4 * q + 2], own[4 * q + 3]}
                                                : *(const f32x4 *)(block(w, u) + 8 * q);
#pragma unroll
                        for (int e = 0; e < 4; ++e) oacc[u][4 * q + e] = fmaf(x[w].x, v[e], oacc[u][4 * q + e]);
                    }
            }
    }
    if (rvalid) {
        float zero = 0.f;  // NaN with a value that is not finite
#pragma unroll
        for (int u = 0; u < UT; ++u)
            if (u % WK == wk)
#pragma unroll
                for (int r = 0; r < 16; ++r) zero = fmaf(oacc[u][r], 0.f, zero);
        bool odd = l != l || zero != zero;
        if (in_tree)
#pragma unroll
            for (int k = 0; k < kAncWords; ++k) odd |= (tree.anc[node][k] & tree.sick[k]) != 0;
        const float inv = 1.0f / l;
        if (odd) {
            atomicOr(&tree.odd[wr], 1u << n);
        } else {
            const size_t ob = ((size_t)node * a.q_heads + head) * HD + 4 * half;
#pragma unroll
            for (int u = 0; u < UT; ++u)
                if (u % WK == wk)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 v = {oacc[u][4 * q], oacc[u][4 * q + 1], oacc[u][4 * q + 2], oacc[u][4 * q + 3]};
                        if (S == 1) store_out4(a, ob + 32 * u + 8 * q, v * inv);
                        else *(f32x4 *)(a.part + at_part * HD + 32 * u + 8 * q + 4 * half) = v;
                    }
            if (S > 1 && wk == 0 && half == 0) a.ml[at_part] = make_float2(m2, l);
        }
    }
    __syncthreads();
    uint32_t odd_rows = 0;
#pragma unroll
    for (int w = 0; w < WR; ++w) odd_rows |= tree.odd[w];
    if (odd_rows == 0) return;
    // Waves whose share of such a row was finite have written it: before it is
    // written again.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (int r = wave; r < 32 * WR; r += NW)
        if (tree.odd[r >> 5] >> (r & 31) & 1) {
            const int i = (m0 + r) / G;
            plain_row<HD, KT>(a, tree, i, g * G + (m0 + r) % G, g, start, min(end, a.offset + i + 1), S, split);
        }
}

// Joins the splits of one (row, head): W waves of a block each add up every
// W-th split's values in order, then their sums in order. Every load of a batch
// is in flight at once, the first batch beside the maxima. The sums are taken of
// 2^-7 of the values (at most 2^7 splits), so that they stay finite where each
// split's are; a power of two rounds nothing.
constexpr int kMergeSplits = 128;  // two a lane
template <int HD, int W>
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(TreeArgs a, int S, int items) {
    constexpr int D = HD / 64, B = 8;
    typedef float vec __attribute__((ext_vector_type(D)));
    __shared__ float so[kThreads / 64][HD];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int item = (int)blockIdx.x * (kThreads / 64 / W) + wave / W, w0 = wave % W;
    if (W == 1 && item >= items) return;
    const float2 *ml = a.ml + (size_t)item * S;
    const float *part = a.part + (size_t)item * S * HD + D * lane;
    vec v[B];
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < B; ++i) v[i] = *(const vec *)(part + (size_t)min(s0 + W * i, S - 1) * HD);
    };
    const float2 x = ml[min(lane, S - 1)], y = ml[min(lane + 64, S - 1)];
    load(w0);
    const float m0 = lane < S ? x.x : -INFINITY, m1 = lane + 64 < S ? y.x : -INFINITY;
    const float M = wave_max(fmaxf(m0, m1));
    const float f0 = m0 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m0 - M);
    const float f1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - M);
    const float L = wave_sum((f0 != 0.f ? f0 * x.y : 0.f) + (f1 != 0.f ? f1 * y.y : 0.f));
    // A split without a key of the row (and what a lane past S read) holds no values
    // and is told apart by a factor of -1: one whose factor rounds to 0 holds them,
    // and an infinity among them shows, as it does within a split.
    static_assert(kMergeSplits == 1 << 7, "the scale of the sums");
    const float g0 = m0 == -INFINITY ? -1.f : f0 * 0x1p-7f, g1 = m1 == -INFINITY ? -1.f : f1 * 0x1p-7f;
    vec o = {};
    for (int s0 = w0; s0 < S; s0 += W * B) {
        if (s0 != w0) load(s0);
#pragma unroll
        for (int i = 0; i < B; ++i) {
            // Selected, not branched around: a load would sink into the branch.
            const int s = s0 + W * i;
            const float f = s >= S ? -1.f : s < 64 ? lane_read(g0, s) : lane_read(g1, s - 64);
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] = fmaf(f, f == -1.f ? 0.f : v[i][d], o[d]);
        }
    }
    if constexpr (W > 1) {
        *(vec *)&so[wave][D * lane] = o;
        __syncthreads();
        if (w0) return;
#pragma unroll
        for (int w = 1; w < W; ++w) o += *(const vec *)&so[wave + w][D * lane];
    }
    const float inv = 1.0f / L * 0x1p7f;
    const size_t at = (size_t)item * HD + D * lane;
#pragma unroll
    for (int d = 0; d < D; ++d) {
        const float r = o[d] * inv;
        if (a.out) a.out[at + d] = r;
        if (a.out_hi) {
            const __bf16 hb = (__bf16)r;
            a.out_hi[at + d] = __builtin_bit_cast(uint16_t, hb);
            a.out_lo[at + d] = __builtin_bit_cast(uint16_t, (__bf16)(r - (float)hb));
        }
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

// A block moves one KV head's K or V rows in one view. nodes[j] >= j and rises,
// so the row a move overwrites was the source of an earlier move or of none:
// kMoves rows of 16-byte columns a thread at a time are read by the whole block
// before any of them is written, and a later batch's sources are past everything
// an earlier one wrote. Bound: three dependent round trips to memory, the page
// table's, the reads' and the writes' (a thread that walked the branch down its
// own column took one for each eight rows: 40 rows of 32 f32 caches 21.3 us, so
// 6.4; 3 rows of 24 BF16 caches 4.9, a launch).
constexpr int kMoves = 8;
__global__ __launch_bounds__(kThreads) void tree_commit_kernel(CommitArgs a) {
    __shared__ size_t row[2][kMaxTreeNodes];  // byte offsets of the sources, the destinations
    const int cols = a.row_bytes / 16, head = blockIdx.x % a.kv_heads, which = blockIdx.x / a.kv_heads;
    const CommitArgs::View &w = a.view[which >> 1];
    uint8_t *pool = which & 1 ? w.v : w.k;
    for (int j = threadIdx.x; j < a.count; j += kThreads)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = a.offset + (k ? j : a.node[j]), lp = p / a.page_size;
            row[k][j] = (((size_t)w.page_table[lp] * a.kv_heads + head) * a.page_size + (p - lp * a.page_size)) * a.row_bytes;
        }
    __syncthreads();
    const int units = a.count * cols;
    for (int u0 = 0; u0 < units; u0 += kMoves * kThreads) {
        u32x4 r[kMoves];
#pragma unroll
        for (int k = 0; k < kMoves; ++k) {
            const int u = u0 + kThreads * k + (int)threadIdx.x;
            if (u < units) r[k] = *(const u32x4 *)(pool + row[0][u / cols] + 16 * (u % cols));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kMoves; ++k) {
            const int u = u0 + kThreads * k + (int)threadIdx.x;
            if (u < units && row[0][u / cols] != row[1][u / cols]) *(u32x4 *)(pool + row[1][u / cols] + 16 * (u % cols)) = r[k];
        }
    }
}

}  // namespace

namespace {

// Splits of whole tiles that a KV head's rows could use: a tile each, but up to two
// BF16 tiles in one, which a block walks sooner than two blocks join (5 nodes on
// 250, 14 / 2 heads of 64: 7.4 and 9.0 us; 24 on 120, 32 / 8 of 128: 10.4 and 11.2).
size_t tree_wanted(const TreeJob &j) {
    const size_t tile = j.g.kv_f32 ? tree_tile<float>() : tree_tile<uint16_t>();
    const size_t tiles = (j.offset + j.n + tile - 1) / tile;
    return !j.g.kv_f32 && tiles <= 2 ? 1 : tiles;
}

// Splits that one block a CU (f32 at head_dim 64: two) lets a KV head have, with wr
// row waves a block.
size_t tree_room(const TreeJob &j, int wr) {
    const size_t rows = j.n * (size_t)(j.q_heads / j.g.kv_heads), rb = (rows + 32 * wr - 1) / (32 * wr);
    const size_t slots = (j.g.kv_f32 && j.g.head_dim == 64 ? 2 : 1) * (size_t)std::max(device_cus(), 8);
    return std::max<size_t>(std::max<size_t>(slots / 8 / rb, 1) * 8 / (size_t)j.g.kv_heads, 1);
}

// Row waves of a block: two; over a BF16 cache one for up to 32 rows, and while every
// split wanted then has a block of its own anyway: short walks, and CUs that would
// stand idle otherwise (16 nodes on 700, 28 / 4 heads of 128: two 12.8 us, one 11.6).
// Four with half the key waves halve the tiles' traffic and double the partials':
// 64 nodes on 16k, 32 / 8 heads of 128, 53.9 us, with two 51.4; 18 on 16k, 28 / 4, 27.6
// and 22.3; f32, 18 on 6k, 30.3 and 25.8 (128 on 3k, 32 / 8, 58.6 and 60.8).
int tree_row_waves(const TreeJob &j) {
    if (j.g.kv_f32) return 2;
    const size_t rows = j.n * (size_t)(j.q_heads / j.g.kv_heads);
    return rows <= 32 || tree_wanted(j) <= tree_room(j, 1) ? 1 : 2;
}

template <int HD, int WR, int WK, class KT>
int launch_tree_blocks(const TreeArgs &a, int S, hipStream_t s) {
    constexpr size_t lds = tree_lds_bytes<HD, KT>();
    static std::atomic<uint64_t> lds_set{0};
    CHIP_TRY(allow_dynamic_lds((const void *)tree_attn_kernel<HD, WR, WK, KT>, lds, lds_set));
    const int rb = (a.n * (a.q_heads / a.kv_heads) + 32 * WR - 1) / (32 * WR);
    const size_t blocks = ((size_t)S * a.kv_heads + 7) / 8 * 8 * (size_t)rb;
    if (blocks > (size_t)INT32_MAX) return fail("HIP backend: tree attention grid out of range.");
    hipLaunchKernelGGL((tree_attn_kernel<HD, WR, WK, KT>), dim3((unsigned)blocks), dim3(64 * WR * WK), lds, s, a, S);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

template <int HD>
int launch_tree_rows(const TreeJob &j, const TreeArgs &a, int S, hipStream_t s) {
    if (j.g.kv_f32) return launch_tree_blocks<HD, 2, 2, float>(a, S, s);
    if (tree_row_waves(j) == 1) return launch_tree_blocks<HD, 1, 4, uint16_t>(a, S, s);
    return launch_tree_blocks<HD, 2, 4, uint16_t>(a, S, s);
}

template <int HD>
int launch_tree_h(const TreeJob &j, const TreeArgs &a, int S, hipStream_t s) {
    CHIP_TRY(launch_tree_rows<HD>(j, a, S, s));
    if (S == 1) return 0;
    const int items = (int)j.n * j.q_heads;
    if (S > 16)
        hipLaunchKernelGGL((tree_merge_kernel<HD, 4>), dim3((unsigned)items), dim3(kThreads), 0, s, a, S, items);
    else
        hipLaunchKernelGGL((tree_merge_kernel<HD, 1>), dim3((unsigned)((items + 3) / 4)), dim3(kThreads), 0, s, a, S, items);
    CHIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace

// Splits of the keys: as many as fill the chip with one block a CU (f32 at
// head_dim 64: two), of a tile at least; at least 8 (split, KV head) pairs go to the
// XCDs in turn, so that their number is brought down to a multiple of 8.
int tree_attention_splits(const TreeJob &j) {
    return (int)std::min({tree_wanted(j), tree_room(j, tree_row_waves(j)), (size_t)attention_max_splits(), (size_t)kMergeSplits});
}

int launch_tree_attention(const TreeJob &j, hipStream_t s) {
    if (!j.q || (!j.out && !j.out_hi) || !j.out_hi != !j.out_lo || !j.k || !j.v || !j.g.page_table || !j.parents)
        return fail("HIP backend: tree attention is missing a buffer.");
    if (j.n == 0 || j.n > (size_t)kMaxTreeNodes || j.offset > kMaxTreePositions - j.n)
        return fail("HIP backend: tree attention shape out of range.");
    int S = tree_attention_splits(j);
    const size_t split_floats = attention_part_floats(j.n, j.q_heads, 1, j.g.head_dim);
    if (S > 1) S = (int)std::min<size_t>((size_t)S, std::max<size_t>(j.part ? j.part_floats / split_floats : 1, 1));
    const int items = (int)j.n * j.q_heads;
    TreeArgs a{};
    a.q = j.q;
    a.k = j.k;
    a.v = j.v;
    a.page_table = j.g.page_table;
    a.parents = j.parents;
    a.part = j.part;
    a.ml = (float2 *)(j.part + (size_t)items * S * j.g.head_dim);
    a.out = j.out;
    a.out_hi = j.out_hi;
    a.out_lo = j.out_lo;
    a.page_size = j.g.page_size;
    a.kv_heads = j.g.kv_heads;
    a.q_heads = j.q_heads;
    a.offset = (int)j.offset;
    a.n = (int)j.n;
    if (j.g.head_dim == 64) return launch_tree_h<64>(j, a, S, s);
    return launch_tree_h<128>(j, a, S, s);
}

int launch_tree_commit(const KvLayer *layers, const int32_t *const *page_tables, size_t views, const KvGeom &g,
                       size_t offset, const uint32_t *nodes, size_t count, hipStream_t s) {
    size_t first = 0;  // nodes already in place
    while (first < count && nodes[first] == first) ++first;
    if (first == count) return 0;
    CommitArgs a{};
    for (size_t j = first; j < count; ++j) a.node[j - first] = (uint8_t)(nodes[j] - first);
    a.count = (int)(count - first);
    a.offset = (int)(offset + first);
    a.page_size = g.page_size;
    a.kv_heads = g.kv_heads;
    a.row_bytes = g.head_dim * (g.kv_f32 ? 4 : 2);
    for (size_t v0 = 0; v0 < views; v0 += kCommitViews) {
        const size_t n = std::min(views - v0, (size_t)kCommitViews);
        for (size_t i = 0; i < n; ++i)
            a.view[i] = {(uint8_t *)layers[v0 + i].k, (uint8_t *)layers[v0 + i].v, page_tables[v0 + i]};
        hipLaunchKernelGGL(tree_commit_kernel, dim3((unsigned)(2 * n * (size_t)g.kv_heads)), dim3(kThreads), 0, s, a);
        CHIP_CHECK(hipGetLastError());
    }
    return 0;
}

}  // namespace chip
