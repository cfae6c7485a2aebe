// Fragments of the matrix-core attention kernels over LDS tiles of 64 cached
// positions: the row order and swizzles of staged K and V rows, transposing V
// reads, f32 operands as BF16 parts.
#pragma once

#include "common.hpp"

namespace chip {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// LDS row of a position within a 64-position tile (an involution).
__device__ __forceinline__ int krow_of(int p) { return (p & ~12) | ((p & 4) << 1) | ((p & 8) >> 1); }

// Chunk swizzle of V row r: the rows a transposing read takes together (four
// consecutive ones, 64 bytes each) fall on distinct banks, and rows r and
// r + 4 share it.
template <int HD>
__device__ __forceinline__ int vseg(int r) {
    return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
}

// The V^T fragments of 16 positions, all HD dims, by transposing LDS reads at
// the UT lane addresses + OFF (rows 0..3) and + OFF + 4 rows. Inline assembly:
// for the builtin the compiler waits for every copy in flight (the next tile's)
// first; each block waits for its own data.
template <int HD, int OFF>
__device__ __forceinline__ void read_vt(const uint32_t (&addr)[HD / 32], bf16x8 (&va)[HD / 32]) {
    constexpr int OFF4 = OFF + 4 * HD * 2;
    s16x4_t r[HD / 32][2];
    if constexpr (HD == 128) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
            "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
            "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
            "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[2][0]), "=&v"(r[2][1]),
              "=&v"(r[3][0]), "=&v"(r[3][1])
            : "v"(addr[0]), "v"(addr[1]), "v"(addr[2]), "v"(addr[3]), "i"(OFF), "i"(OFF4)
            : "memory");
    } else {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
            "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1])
            : "v"(addr[0]), "v"(addr[1]), "i"(OFF), "i"(OFF4)
            : "memory");
    }
#pragma unroll
    for (int u = 0; u < HD / 32; ++u)
        va[u] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[u][0], r[u][1], 0, 1, 2, 3, 4, 5, 6, 7));
}

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

struct Parts2 {  // two values' parts, packed
    uint32_t h, m, l;
};
__device__ __forceinline__ Parts2 split3(float a, float b) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    const float ra = a - __uint_as_float(ua & 0xFFFF0000u), rb = b - __uint_as_float(ub & 0xFFFF0000u);
    const __bf16 ma = (__bf16)ra, mb = (__bf16)rb;
    const __bf16 la = (__bf16)(ra - (float)ma), lb = (__bf16)(rb - (float)mb);
    Parts2 p;
    p.h = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    p.m = (uint32_t)__builtin_bit_cast(uint16_t, ma) | ((uint32_t)__builtin_bit_cast(uint16_t, mb) << 16);
    p.l = (uint32_t)__builtin_bit_cast(uint16_t, la) | ((uint32_t)__builtin_bit_cast(uint16_t, lb) << 16);
    return p;
}
// Eight values' parts as three matrix operands.
__device__ __forceinline__ void split3x8(const float (&v)[8], bf16x8 (&out)[3]) {
    u32x4 w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Parts2 p = split3(v[2 * i], v[2 * i + 1]);
        w[0][i] = p.h;
        w[1][i] = p.m;
        w[2][i] = p.l;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) out[k] = __builtin_bit_cast(bf16x8, w[k]);
}

}  // namespace
}  // namespace chip
