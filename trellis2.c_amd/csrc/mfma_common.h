// mfma_common.h - device helpers shared by the MFMA kernels (conv, linear).
#pragma once
#include <type_traits>

#include "tsh_internal.h"

namespace tsh {
namespace {

// Maps a linear block id onto a logical tile so that each of the 8 XCDs
// (which receive block ids round-robin) works on one contiguous range of
// tiles and its L2 sees neighbouring gathers.
__device__ __forceinline__ int64_t xcd_remap(int64_t bid, int64_t grid) {
    constexpr int64_t kXcd = 8;
    const int64_t q = grid / kXcd, r = grid % kXcd;
    const int64_t xcd = bid % kXcd, slot = bid / kXcd;
    return xcd < r ? xcd * (q + 1) + slot : r * (q + 1) + (xcd - r) * q + slot;
}

// Workgroup barrier that orders LDS only.  __syncthreads() also drains every
// outstanding global load (vmcnt(0)), which would empty the register prefetch
// ring of the streamed kernel at each barrier; its global loads only read
// data that no block writes.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// s_waitcnt vmcnt(N) alone (gfx9 encoding: vmcnt in bits 3:0 and 15:14;
// expcnt and lgkmcnt left at their maxima, i.e. not waited for).
template <int N> __device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}

// Direct-to-LDS load of 16 bytes per lane: the bytes at voff + soff of the
// buffer land at LDS address lds + 16 * lane (exec-masked lanes load and
// write nothing).  Inline assembly, so that the compiler neither counts it
// nor waits for it before later LDS reads (it cannot tell LDS regions apart
// and would drain every such load at the next read); the caller waits with
// wait_vmcnt.  M0, which holds the LDS address, is saved and restored, with
// the wait state that a write of M0 needs before an LDS-DMA instruction.
__device__ __forceinline__ void dma_b128(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, uint32_t voff, uint32_t soff) {
    uint32_t keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
        : "memory");
}

// The same without keeping M0, which nothing else here uses.
__device__ __forceinline__ void dma_b128_m0(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, uint32_t voff, uint32_t soff) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, %3 offen lds"
        :
        : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
        : "memory", "m0");
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int DT> struct Mfma;
template <> struct Mfma<kBF16> {
    typedef bf16x8 V;
    __device__ static f32x4 mac(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<kF16> {
    typedef f16x8 V;
    __device__ static f32x4 mac(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// Lane layout of v_mfma_f32_16x16x32 (64 lanes): A fragment = row (lane%16),
// 8 consecutive K values starting at 8*(lane/16); B fragment = column
// (lane%16), the same 8 K values; D = rows 4*(lane/16)+i, column lane%16.
// Any consistent K permutation of A and B gives the same product, so only
// the row/column mapping matters for correctness.

// LDS layout of one 16-row block of A (64 granules of 16 bytes: 16 rows x 4
// chunks).  ds_read_b128 / ds_write_b128 serve 16 lanes per cycle from the 64
// banks without conflict when lanes 0-7 of each 16-lane group touch granules
// 0-7 (mod 16) and lanes 8-15 granules 8-15, each once.  Row i, chunk c sits at
//   16 * (i1 + 2 i2) + 8 i3 + 4 (c1 ^ i2) + 2 (c0 ^ i1) + i0     (bits of i, c),
// which meets that for the fragment reads (lane i + 16 c reads row i, chunk c)
// and, with quad j fetching row a_quad_row(j) (bits 1 and 3 of j exchanged),
// for the stores (lane 4 j + c stores row a_quad_row(j), chunk c).
__device__ __forceinline__ int a_granule(int i, int c) {
    const int i0 = i & 1, i1 = (i >> 1) & 1, i2 = (i >> 2) & 1, i3 = (i >> 3) & 1;
    return 16 * (i1 + 2 * i2) + 8 * i3 + 4 * (((c >> 1) & 1) ^ i2) + 2 * ((c & 1) ^ i1) + i0;
}
__device__ __forceinline__ int a_quad_row(int j) { return (j & 5) | (((j >> 1) & 1) << 3) | (((j >> 3) & 1) << 1); }

// Sum over the 16 lanes of a DPP row, left in every lane of the row:
// rotations by 8, 4, 2 and 1 within the row (row_ror), each one VALU add.
__device__ __forceinline__ float row16_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x122, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x121, 0xf, 0xf, false));
    return v;
}

// A lane's value and that of the lane 32 (16) further on, in both lanes the same
// way round: v_permlane32_swap exchanges the upper half of a with the lower half
// of b (v_permlane16_swap every odd row of 16 lanes of a with the even one before it
// of b).  In assembly because the builtin's two results come out as one; the
// waits are those that the instruction needs after a vector write.
__device__ __forceinline__ void both_halves(float v, float & a, float & b) {
    a = b = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void both_rows(float v, float & a, float & b) {
    a = b = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}

// op over aligned groups of G lanes (a power of two), left in each of them: the
// neighbour and the next pair by DPP, then mirror images (a partial result is the
// same in all lanes that it covers), then the exchanges above.
template <int G, class Op> __device__ __forceinline__ float group_reduce(float v, Op op) {
    const auto dpp = [&](auto ctrl) {
        return __builtin_bit_cast(
            float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    if constexpr (G > 1) v = op(v, dpp(std::integral_constant<int, 0xB1>()));
    if constexpr (G > 2) v = op(v, dpp(std::integral_constant<int, 0x4E>()));
    if constexpr (G > 4) v = op(v, dpp(std::integral_constant<int, 0x141>()));
    if constexpr (G > 8) v = op(v, dpp(std::integral_constant<int, 0x140>()));
    float a, b;
    if constexpr (G > 16) {
        both_rows(v, a, b);
        v = op(a, b);
    }
    if constexpr (G > 32) {
        both_halves(v, a, b);
        v = op(a, b);
    }
    return v;
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
    return group_reduce<G>(v, [](float a, float b) { return a + b; });
}
// In 64 bits: the halves of a value go the same ways.
template <int G, class Op> __device__ __forceinline__ double group_reduce(double v, Op op) {
    const auto halves = [](double d) { return __builtin_bit_cast(int2, d); };
    const auto dpp = [&](auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        const int2 h = halves(v);
        return __builtin_bit_cast(double, int2{__builtin_amdgcn_mov_dpp(h.x, C, 0xf, 0xf, false),
                                               __builtin_amdgcn_mov_dpp(h.y, C, 0xf, 0xf, false)});
    };
    if constexpr (G > 1) v = op(v, dpp(std::integral_constant<int, 0xB1>()));
    if constexpr (G > 2) v = op(v, dpp(std::integral_constant<int, 0x4E>()));
    if constexpr (G > 4) v = op(v, dpp(std::integral_constant<int, 0x141>()));
    if constexpr (G > 8) v = op(v, dpp(std::integral_constant<int, 0x140>()));
    const auto join = [&](auto both) {
        const int2 h = halves(v);
        float ax, bx, ay, by;
        both(__builtin_bit_cast(float, h.x), ax, bx);
        both(__builtin_bit_cast(float, h.y), ay, by);
        v = op(__builtin_bit_cast(double, int2{__builtin_bit_cast(int, ax), __builtin_bit_cast(int, ay)}),
               __builtin_bit_cast(double, int2{__builtin_bit_cast(int, bx), __builtin_bit_cast(int, by)}));
    };
    if constexpr (G > 16) join([](float f, float & a, float & b) { both_rows(f, a, b); });
    if constexpr (G > 32) join([](float f, float & a, float & b) { both_halves(f, a, b); });
    return v;
}
template <int G> __device__ __forceinline__ double group_sum(double v) {
    return group_reduce<G>(v, [](double a, double b) { return a + b; });
}
// The largest of non-negative values as bits (a NaN's are larger than any number's).
template <int G> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
    return __builtin_bit_cast(uint32_t, group_reduce<G>(__builtin_bit_cast(float, v), [](float a, float b) {
                                  const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
                                  return __builtin_bit_cast(float, x > y ? x : y);
                              }));
}

}  // namespace
}  // namespace tsh
