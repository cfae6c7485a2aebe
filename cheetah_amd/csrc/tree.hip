// Attention for a tree of drafted tokens over the paged KV cache, and the move
// of its accepted branch's K/V rows into place.
//
// Node i of n has its parent parents[i] < i (anything else: none, a root). Its
// K/V row sits at cache position offset + i. With the cached prefix [0, offset)
// every node sees its ancestors and itself:
//   out[i, h] = sum_p w_p v[p, h / G],  w = softmax_p(q[i, h] . k[p, h / G] / sqrt(head_dim))
// over p in [0, offset) and offset + a, a = i or an ancestor of i.
#include <algorithm>

#include "kernels.hpp"

namespace chip {
namespace {

constexpr int kThreads = 256;

struct TreeArgs {
    const float *q;
    const void *k, *v;
    const int32_t *page_table;
    const int32_t *parents;
    float *out;
    int page_size, kv_heads, q_heads, offset;
};

__device__ __forceinline__ float kv_value(const uint16_t *p) { return bf16_f32(*p); }
__device__ __forceinline__ float kv_value(const float *p) { return *p; }

// One wave per (node, q head), a lane per HD / 64 dims, key by key.
template <int HD, class KT>
__global__ __launch_bounds__(64) void tree_attn_kernel(TreeArgs a) {
    constexpr int D = HD / 64;
    __shared__ uint8_t seen[kMaxTreeNodes];
    const int lane = threadIdx.x, node = blockIdx.y, head = blockIdx.x;
    const int g = head / (a.q_heads / a.kv_heads);
    for (int i = lane; i < kMaxTreeNodes; i += 64) seen[i] = 0;
    __syncthreads();
    if (lane == 0)
        for (int i = node;;) {
            seen[i] = 1;
            const int up = a.parents[i];
            if (up < 0 || up >= i) break;
            i = up;
        }
    __syncthreads();
    const float scale = 1.0f / sqrtf((float)HD);
    const size_t row = ((size_t)node * a.q_heads + head) * HD;
    float q[D], o[D], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) {
        q[d] = a.q[row + lane + 64 * d];
        o[d] = 0.f;
    }
    for (int p = 0; p <= a.offset + node; ++p) {
        if (p >= a.offset && !seen[p - a.offset]) continue;
        const size_t at = (((size_t)a.page_table[p / a.page_size] * a.kv_heads + g) * a.page_size + p % a.page_size) * HD;
        float dot = 0.f;
#pragma unroll
        for (int d = 0; d < D; ++d) dot = fmaf(q[d], kv_value((const KT *)a.k + at + lane + 64 * d), dot);
        const float s = wave_sum(dot) * scale, mn = fmaxf(m, s);
        const float alpha = m == -INFINITY ? 0.f : expf(m - mn), w = s == -INFINITY ? 0.f : expf(s - mn);
        m = mn;
        l = l * alpha + w;
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = fmaf(w, kv_value((const KT *)a.v + at + lane + 64 * d), o[d] * alpha);
    }
#pragma unroll
    for (int d = 0; d < D; ++d) a.out[row + lane + 64 * d] = o[d] / l;
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

int launch_tree_attention(const TreeJob &j, hipStream_t s) {
    TreeArgs a{};
    a.q = j.q;
    a.k = j.k;
    a.v = j.v;
    a.page_table = j.g.page_table;
    a.parents = j.parents;
    a.out = j.out;
    a.page_size = j.g.page_size;
    a.kv_heads = j.g.kv_heads;
    a.q_heads = j.q_heads;
    a.offset = (int)j.offset;
    const dim3 grid((unsigned)j.q_heads, (unsigned)j.n);
    if (j.g.head_dim == 64) {
        if (j.g.kv_f32) hipLaunchKernelGGL((tree_attn_kernel<64, float>), grid, dim3(64), 0, s, a);
        else hipLaunchKernelGGL((tree_attn_kernel<64, uint16_t>), grid, dim3(64), 0, s, a);
    } else {
        if (j.g.kv_f32) hipLaunchKernelGGL((tree_attn_kernel<128, float>), grid, dim3(64), 0, s, a);
        else hipLaunchKernelGGL((tree_attn_kernel<128, uint16_t>), grid, dim3(64), 0, s, a);
    }
    CHIP_CHECK(hipGetLastError());
    return 0;
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
