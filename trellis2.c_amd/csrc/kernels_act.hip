// kernels_act.hip - linear with activation and residual in its epilogue, from rows of the storage type or 8-bit rows.
#include <cmath>
#include <type_traits>

#include "mfma_common.h"

namespace tsh {
namespace {

// ---- activations --------------------------------------------------------------------------------

// For 16-bit outputs the hardware exponential and reciprocal (about 2^-21
// relative) stay far below the output's rounding; fp32 outputs of SiLU and of GELU
// with tanh take the accurate functions.  Both are v times a logistic function: of v,
// and of 2 sqrt(2 / pi) (v + 0.044715 v^3).
//
// GELU is v Phi(v), and below zero Phi is small beside 1: one minus an erf, or a
// polynomial that is right to some 1e-6 of 1, loses it.  16 bits: Phi(-a), a = |v|, is
// 2 to a polynomial, fitted to its logarithm for the least error of Phi, relative and
// absolute, as the output's rounding needs it, and falling beyond the fit so that the
// exponential is zero there.  bf16: degree 9, 2^-12.4 relative down to v = -13.2 (below
// that bf16 has no normal numbers for the result), 2^-20.2 absolute.  fp16: degree 7,
// 2^-16 relative down to -4.05, below that 2^-29.6 of GELU (half a step is 2^-25), 2^-21
// absolute.  14 instructions a value: 79,523 x 512 -> 2048 from 8-bit rows 181 us; with the
// form of fp32 below 184; as a logistic function of v R(v^2), which is 5.7e-6 off, 165.
// fp32: exp(-a^2 / 2) t Q(t), t = 1 / (1 + p a), as the tail falls like 1 / a beside the
// exponential; Q of degree 8, 2^-25.2 relative.  t, Q, their products and the exponential
// add some 16 roundings, the exponential's argument 1.5 a^2.
template <int DT> struct GeluTail {
    static constexpr int degree = 9;
    static constexpr float c[10] = {-0.999997854f,    -1.15119767f,    -0.458608121f,   -0.0538811572f,  0.00854993984f,
                                    -0.000976997311f, 7.58256283e-05f, -3.73059152e-06f, 1.03579488e-07f, -1.21999999e-09f};
};
template <> struct GeluTail<kF16> {
    static constexpr int degree = 7;
    static constexpr float c[8] = {-0.999998927f,  -1.15115595f,     -0.458844155f,   -0.0534294285f,
                                   0.00817629881f, -0.000829449506f, 4.70212144e-05f, -1.05048525e-06f};
};
template <> struct GeluTail<kF32> {
    static constexpr int degree = 8;
    static constexpr float p = 0.34f;
    static constexpr float c[9] = {0.135618851f, 0.136142388f,  0.11496748f,  0.116314463f, -0.0470853858f,
                                   0.205778807f, -0.276415288f, 0.141150713f, -0.0264720283f};
};
template <int DT> __device__ __forceinline__ float gelu(float v) {
    using G = GeluTail<DT>;
    float x = fabsf(v);
    if constexpr (DT == kF32) x = __builtin_amdgcn_rcpf(fmaf(G::p, x, 1.0f));
    float q = G::c[G::degree];
#pragma unroll
    for (int i = G::degree - 1; i >= 0; --i) q = fmaf(q, x, G::c[i]);
    float tail;
    if constexpr (DT == kF32) {
        tail = q * x * __builtin_amdgcn_exp2f(v * (v * -0.72134752f));
    } else {
        tail = __builtin_amdgcn_exp2f(q);
    }
    return v * (v > 0.0f ? 1.0f - tail : tail);
}
template <int DT, int ACT> __device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_SILU) {
        if constexpr (DT == kF32) return v / (1.0f + expf(-v));
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
    } else if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_GELU) {
        return gelu<DT>(v);
    } else if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_GELU_TANH) {
        // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u))
        const float r = 1.5957691216057308f + 0.0713548162726f * v * v;
        if constexpr (DT == kF32) return v / (1.0f + expf(-v * r));
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v * r));
    } else {
        return v;
    }
}

// f(the activation as a constant).
template <class F> __device__ __forceinline__ void by_act(int act, F && f) {
    switch (act) {
        case TRELLIS_SPARSE_HIP_ACT_SILU: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_SILU>()); break;
        case TRELLIS_SPARSE_HIP_ACT_GELU: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_GELU>()); break;
        case TRELLIS_SPARSE_HIP_ACT_GELU_TANH: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_GELU_TANH>()); break;
        default: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_NONE>()); break;
    }
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// N (1, 2 or 4) adjacent values at byte voff + soff of a buffer, whole and
// aligned; beyond the buffer loads give zeros and stores nothing.
template <int DT, int N> union Adjacent {
    typename Store<DT>::T h[N];
    uint16_t b2;
    uint32_t b4;
    u32x2 b8;
    u32x4 b16;
};
template <int DT, int N>
__device__ __forceinline__ Adjacent<DT, N> load_adjacent(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff) {
    constexpr int B = N * sizeof(typename Store<DT>::T);
    Adjacent<DT, N> w;
    if constexpr (B == 2) w.b2 = __builtin_amdgcn_raw_buffer_load_b16(rsrc, (int) voff, (int) soff, 0);
    if constexpr (B == 4) w.b4 = __builtin_amdgcn_raw_buffer_load_b32(rsrc, (int) voff, (int) soff, 0);
    if constexpr (B == 8) w.b8 = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int) voff, (int) soff, 0);
    if constexpr (B == 16) w.b16 = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int) voff, (int) soff, 0);
    return w;
}
template <int DT, int N>
__device__ __forceinline__ void store_adjacent(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff, const float * v) {
    constexpr int B = N * sizeof(typename Store<DT>::T);
    Adjacent<DT, N> w;
#pragma unroll
    for (int u = 0; u < N; ++u) w.h[u] = round_to_store<DT>(v[u]);
    if constexpr (B == 2) __builtin_amdgcn_raw_buffer_store_b16(w.b2, rsrc, (int) voff, (int) soff, 0);
    if constexpr (B == 4) __builtin_amdgcn_raw_buffer_store_b32(w.b4, rsrc, (int) voff, (int) soff, 0);
    if constexpr (B == 8) __builtin_amdgcn_raw_buffer_store_b64(w.b8, rsrc, (int) voff, (int) soff, 0);
    // 16 bytes: no scalar offset.  With one, the compiler leaves out the wait
    // before the data's registers are written again, and lanes 12-15 and 28-31 of
    // a half have stored values that were written after the store (measured).
    if constexpr (B == 16) __builtin_amdgcn_raw_buffer_store_b128(w.b16, rsrc, (int) (voff + soff), 0, 0);
}

// ---- MFMA GEMM ----------------------------------------------------------------------------------

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// A fragment is two 16-byte chunks, h and h + 2 for lane half h = lane / 32, of
// row lane % 32 (of x or of W) in a step of 64 bytes: 16, 32 or 64 K values in
// fp32, 16 or 8 bits.  The scaled MFMA takes the chunks as K values 16 h .. and
// 32 + 16 h .., and from lane half h the scale of K values 32 h .. 32 h + 31.  It
// adds eight neighbouring products at a time on the scale of the largest, cutting
// each at 2^-13 of it (measured: 2^-13 stays, 2^-14 goes), before the fp32 sums: an
// error near 2e-5 of a sum's size, a hundredth of a bf16 rounding, for twice the
// rate of bf16.
struct Frag {
    int4 c[2];
};

// SEL: which of a scale register's bytes counts (0 or 2).
template <int MT, int SEL> __device__ __forceinline__ f32x16 mac(const Frag & a, const Frag & b, f32x16 c, int sa, int sb) {
    if constexpr (MT == kF32) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const f32x4 x = __builtin_bit_cast(f32x4, a.c[e]), w = __builtin_bit_cast(f32x4, b.c[e]);
#pragma unroll
            for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], w[j], c, 0, 0, 0);
        }
        return c;
    } else if constexpr (MT == kRows8) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_bit_cast(i32x8, a), __builtin_bit_cast(i32x8, b),
                                                               c, 0, 0, SEL, sa, SEL, sb);
    } else {
        using V = typename Mfma<MT>::V;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const V x = __builtin_bit_cast(V, a.c[e]), w = __builtin_bit_cast(V, b.c[e]);
            if constexpr (MT == kBF16) {
                c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, w, c, 0, 0, 0);
            } else {
                c = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w, c, 0, 0, 0);
            }
        }
        return c;
    }
}

// Direct-to-LDS load of 4 bytes per lane (see dma_b128).
__device__ __forceinline__ void dma_b32(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, uint32_t voff, uint32_t soff) {
    uint32_t keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "buffer_load_dword %2, %3, %4 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
        : "memory");
}

// The same value in every lane, in a scalar register.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

constexpr uint32_t kOutside = 0x80000000u;  // beyond every buffer here: loads fetch zeros

// A block of RW x CW wavefronts multiplies BM rows of x by BN rows of W (output
// channels), a wavefront RB blocks of 32 rows by NT tiles of 32 channels, in
// steps of 128 bytes of K (whole cache lines: with 64 bytes a step each line
// comes twice from the L2 and the loads bound the kernel, 16,384 x 4096 -> 4096
// bf16 474 us).  Two steps are in LDS or on their way there.  A step is two
// halves of 64 bytes: while the first half's products run, the second half's fragments
// are read; then comes the one barrier, after which the step's slot is free for
// the loads of the step after next, and the next step, whose loads were issued
// a step ago, has landed for the reads under the second half's products.
//
// LDS: a slot holds the rows of x and of W, 128 bytes each, chunk c of row r at c ^ f(r),
// f(r) the bits 1, 2, 3 of r in reverse: the 16 lanes that ds_read_b128 serves at
// once (0-3, 12-15, 20-23 and 24-27 of each 32, and the others) touch each of
// the 64 banks once, and eight lanes of a load fetch one row's 128 bytes.
// Of 32 NT channels, tile t's lane i has channel NT i + t: a lane ends with NT
// adjacent ones, and a row leaves in pieces of 32 NT adjacent channels.
// 8-bit rows: a step's scales are 4 bytes a row.
//
// More tiles than fit at once are walked by blocks that stay: the loads of a tile's
// last two steps are those of the next one's first two, so that they arrive while
// outputs are activated and stored (79,523 rows 512 -> 2048 with GELU of 8-bit rows
// 201 -> 181 us, in bf16 259 -> 239).
//
// Bound by the matrix unit and what feeds it where K is long: 16,384 x 4096 ->
// 4096 bf16 430 us, 1,280 TFLOP/s (the library's largest product 1,590); of 8-bit rows
// 268 us, 2,050 TFLOP/s (2,790), where a step's reads of LDS take as long as its
// products.  With short K by the outputs: their activation (GELU some 60 clocks for 64
// values) and their way to memory run while nothing is multiplied, as there are
// registers for one block of 256 x 256 per CU only.
template <int MT, int DT, int RW, int CW, int RB, int NT, int PER_CU>
__global__ void __launch_bounds__(64 * RW * CW, RW * CW * PER_CU / 4) k_linear_act(LinearAct p) {
    using T = typename Store<DT>::T;
    constexpr int NW = RW * CW, BM = RW * RB * 32, BN = CW * NT * 32;
    constexpr bool kScaled = MT == kRows8;
    constexpr bool kMaySplit = BM * BN < 256 * 256;  // the largest blocks have no registers for it
    constexpr int kRows = BM + BN, kBytes = kRows * 128, kSlot = kBytes + (kScaled ? kRows * 4 : 0);
    // Loads of 1 KB (8 rows) per step and wavefront, of x and of W.
    constexpr int NA = BM / 8 / NW, NB = BN / 8 / NW, kPer = NA + NB;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "as many loads for every wavefront");
    static_assert(!kScaled || (BM % 64 == 0 && kRows / 64 <= NW), "one load of scales per wavefront, all of x or of W");
    __shared__ __attribute__((aligned(1024))) unsigned char s_slot[2 * kSlot];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RW, cw = wave / RW;
    const int l32 = lane & 31, half = lane >> 5;

    // An XCD (blocks b, b + 8, ...) takes a contiguous range of the tiles, row
    // block by row block with every channel block in turn: the rows stay in its
    // L2, and few tiles spread over all XCDs.  More tiles than blocks: its blocks
    // take every so many of them.
    const int split = kMaySplit ? (int) (blockIdx.x / p.split_blocks) : 0;
    int unit, end, stride = 1;
    if (p.blocks == p.split_blocks) {
        unit = scalar((int) xcd_remap(blockIdx.x - (int64_t) split * p.split_blocks, p.split_blocks));
        end = unit + 1;
    } else {
        const int xcd = (int) (blockIdx.x % 8);
        stride = p.blocks / 8;
        unit = (int) ((int64_t) p.split_blocks * xcd / 8 + blockIdx.x / 8);
        end = (int) ((int64_t) p.split_blocks * (xcd + 1) / 8);
        if (unit >= end) return;
    }
    // This tile's first row and channel, and those of the one to load.
    int64_t row0, next_row0;
    int col0, next_col0;
    const auto place = [&](int u) {
        const int r = scalar(u / p.col_tiles);
        next_row0 = (int64_t) r * BM;
        next_col0 = (u - r * p.col_tiles) * BN;
    };
    place(unit);
    row0 = next_row0;
    col0 = next_col0;

    const uint32_t slots = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) unsigned char *) s_slot;

    // The channel of a row of W in LDS.
    const auto channel_of = [](int r) { return r / (32 * NT) * (32 * NT) + r % 32 * NT + r % (32 * NT) / 32; };
    const auto swizzle = [](int r) { return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1); };
    // This lane's piece of load g, of 8 rows of 128 bytes: row lane / 8, whose
    // chunk's lowest bit is g's.  The rest of the place is the same in all lanes
    // and added at each load (registers are what the largest blocks lack).
    const int chunk = (lane & 7) ^ swizzle(lane >> 3);
    uint32_t x_at[2], w_at[2];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        x_at[o] = (uint32_t) ((lane >> 3) * p.row_bytes + (chunk ^ o) * 16);
        w_at[o] = (uint32_t) ((lane >> 3) * NT * p.w_bytes + (chunk ^ o) * 16);
    }
    // Scales: 64 rows a wavefront (the last ones again for wavefronts beyond them).
    const int scale_load = min(wave, kRows / 64 - 1);
    const bool scales_of_x = scale_load * 64 < BM;
    const int scale_pitch = (scales_of_x ? p.row_bytes : p.w_bytes) / 32;
    const int scale_row = scale_load * 64 + lane;
    const uint32_t scale_at = (uint32_t) ((scales_of_x ? scale_row : channel_of(scale_row - BM)) * scale_pitch);

    // This split's steps; and the tile to load, as buffers.  Rows past the last,
    // and all after the last tile, are beyond them: zeros.
    const int all = p.w_bytes / 128;
    const int first_step = kMaySplit ? scalar(all * split / p.splits) : 0;
    const int steps = kMaySplit ? scalar(all * (split + 1) / p.splits) : all;
    __amdgpu_buffer_rsrc_t xres, wres, sres;
    const auto aim = [&](bool some) {
        const int rows = (int) min((int64_t) BM, p.n - next_row0);
        xres = __builtin_amdgcn_make_buffer_rsrc((void *) ((const char *) p.x + next_row0 * p.row_bytes), 0,
                                                 some ? rows * p.row_bytes : 0, 0x00020000);
        wres = __builtin_amdgcn_make_buffer_rsrc((void *) ((const char *) p.w + (int64_t) next_col0 * p.w_bytes), 0,
                                                 some ? BN * p.w_bytes : 0, 0x00020000);
        if constexpr (kScaled) {
            const uint8_t * base =
                scales_of_x ? p.x_scales + next_row0 * scale_pitch : p.w_scales + (int64_t) next_col0 * scale_pitch;
            sres = __builtin_amdgcn_make_buffer_rsrc((void *) base, 0, some ? (scales_of_x ? rows : BN) * scale_pitch : 0,
                                                     0x00020000);
        }
    };
    aim(true);
    // (What follows a row of x in memory is the next one.)
    const auto load = [&](int step, uint32_t slot, int j) {
        if (j < NA) {
            const int g = wave * NA + j, o = NA % 2 == 0 ? j % 2 : g % 2;
            uint32_t row = (uint32_t) (g * 8 * p.row_bytes);
            asm volatile("" : "+s"(row));
            dma_b128_m0(xres, slot + g * 1024u,
                        step * 128 + (chunk ^ o) * 16 < p.row_bytes ? x_at[o] + row : kOutside, step * 128u);
        } else {
            const int g = wave * NB + j - NA, o = NB % 2 == 0 ? (j - NA) % 2 : g % 2;
            uint32_t row = (uint32_t) (channel_of(g * 8) * p.w_bytes);
            asm volatile("" : "+s"(row));
            dma_b128_m0(wres, slot + BM * 128 + g * 1024u, w_at[o] + row, step * 128u);
        }
    };
    const auto load_scales = [&](int step, uint32_t slot) {
        if constexpr (kScaled) dma_b32(sres, slot + kBytes + scale_load * 256u, scale_at, step * 4u);
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (first_step + s >= steps) aim(false);
        const int step = first_step + s < steps ? first_step + s : 0;
        load_scales(step, slots + s * kSlot);
#pragma unroll
        for (int j = 0; j < kPer; ++j) load(step, slots + s * kSlot, j);
    }

    // The channels of this lane in a tile begin at its col0 + ch0.
    const int ch0 = (cw * 32 + l32) * NT;
    const __amdgpu_buffer_rsrc_t bres = __builtin_amdgcn_make_buffer_rsrc(
        (void *) p.bias, 0, p.bias != nullptr && (!kMaySplit || p.splits == 1) ? p.co * 4 : 0, 0x00020000);
    Adjacent<kF32, NT> bias;
    const auto load_bias = [&]() { bias = load_adjacent<kF32, NT>(bres, (uint32_t) ((col0 + ch0) * 4), 0); };
    load_bias();
    f32x16 acc[RB][NT];
    const auto begin = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int q = 0; q < RB; ++q) {
                float b = bias.h[t];
                asm volatile("" : "+v"(b));  // else 16 copies of it are made with the load, and wait in memory
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[q][t][i] = b;
            }
    };
    begin();

    Frag fa[2][RB], fb[2][NT];
    int sa[RB], sb[NT];
    const uint32_t c0 = (uint32_t) (l32 * 128 + ((half ^ swizzle(l32)) * 16));  // chunk c: c0 ^ 16 c for even c
    const auto read_a = [&](int h, uint32_t slot, int q) {
        const unsigned char * r = s_slot + slot + (rw * RB + q) * 4096;
        fa[h][q].c[0] = *(const int4 *) (r + (c0 ^ (h * 64)));
        fa[h][q].c[1] = *(const int4 *) (r + (c0 ^ (h * 64 + 32)));
    };
    const auto read_b = [&](int h, uint32_t slot, int t) {
        const unsigned char * r = s_slot + slot + BM * 128 + (cw * NT + t) * 4096;
        fb[h][t].c[0] = *(const int4 *) (r + (c0 ^ (h * 64)));
        fb[h][t].c[1] = *(const int4 *) (r + (c0 ^ (h * 64 + 32)));
    };
    // Byte 2 h + half of a row's four scales, moved down by the half.
    const auto read_scales = [&](uint32_t slot) {
        if constexpr (kScaled) {
            const unsigned char * r = s_slot + slot + kBytes;
#pragma unroll
            for (int q = 0; q < RB; ++q)
                sa[q] = (int) (*(const uint32_t *) (r + ((rw * RB + q) * 32 + l32) * 4) >> (8 * half));
#pragma unroll
            for (int t = 0; t < NT; ++t)
                sb[t] = (int) (*(const uint32_t *) (r + (BM + (cw * NT + t) * 32 + l32) * 4) >> (8 * half));
        }
    };
    // The products of half h; between one tile and the next a fragment of the
    // other half is read from `from`, and in the second half a load is issued.
    const auto products = [&](auto h_c, uint32_t from, int step, uint32_t to) {
        constexpr int H = decltype(h_c)::value, READS = RB + NT, TILES = RB * NT;
#pragma unroll
        for (int k = 0; k < TILES; ++k) {
#pragma unroll
            for (int i = READS * k / TILES; i < READS * (k + 1) / TILES; ++i) {
                if (i < RB) {
                    read_a(H ^ 1, from, i);
                } else {
                    read_b(H ^ 1, from, i - RB);
                }
            }
            if constexpr (H == 1) {
                if (k == 0) load_scales(step, slots + to);
#pragma unroll
                for (int j = kPer * k / TILES; j < kPer * (k + 1) / TILES; ++j) load(step, slots + to, j);
            }
            const int q = k / NT, t = k % NT;
            acc[q][t] = mac<MT, 2 * H>(fa[H][q], fb[H][t], acc[q][t], kScaled ? sa[q] : 0, kScaled ? sb[t] : 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Lane (l32, half) holds rows 8 (i / 4) + 4 half + i % 4 of each row block.
    // Buffer offsets: the lane's place, and the row's in a scalar; rows past
    // the last and channels past co (a multiple of NT) fall outside.
    const auto leave = [&](int64_t row0, int col0) {
        const int rows = (int) min((int64_t) BM, p.n - row0), ch = col0 + ch0;
        if constexpr (kMaySplit) if (p.splits > 1) {
            // The sums of this split, as they are.
            const __amdgpu_buffer_rsrc_t pres = __builtin_amdgcn_make_buffer_rsrc(
                p.partial + ((int64_t) split * p.n + row0) * p.co, 0, rows * p.co * 4, 0x00020000);
            const uint32_t to = ch < p.co ? (uint32_t) (((rw * RB * 32 + 4 * half) * p.co + ch) * 4) : kOutside;
#pragma unroll
            for (int q = 0; q < RB; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float v[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) v[t] = acc[q][t][i];
                    store_adjacent<kF32, NT>(pres, to, (uint32_t) ((q * 32 + i / 4 * 8 + i % 4) * p.co * 4), v);
                }
            return;
        }
        const int pitch = p.co * (int) sizeof(T);
        const __amdgpu_buffer_rsrc_t yres =
            __builtin_amdgcn_make_buffer_rsrc((char *) p.y + row0 * pitch, 0, rows * pitch, 0x00020000);
        const __amdgpu_buffer_rsrc_t rres = __builtin_amdgcn_make_buffer_rsrc(
            (char *) (p.residual != nullptr ? p.residual : p.y) + row0 * pitch, 0, rows * pitch, 0x00020000);
        const uint32_t at =
            ch < p.co ? (uint32_t) ((rw * RB * 32 + 4 * half) * pitch + ch * (int) sizeof(T)) : kOutside;
        const auto finish = [&](auto act_c, auto res_c) {
            // Four rows at a time, the next four's residuals on their way.
            constexpr bool kRes = decltype(res_c)::value;
            Adjacent<DT, NT> r[2][4];
            const auto fetch = [&](int k) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if constexpr (kRes)
                        r[k % 2][i] = load_adjacent<DT, NT>(rres, at, (uint32_t) ((k / 4 * 32 + k % 4 * 8 + i) * pitch));
            };
            fetch(0);
#pragma unroll
            for (int k = 0; k < 4 * RB; ++k) {
                if (k + 1 < 4 * RB) fetch(k + 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        v[t] = activate<DT, decltype(act_c)::value>(acc[k / 4][t][4 * (k % 4) + i]);
                        if constexpr (kRes) v[t] += Store<DT>::ld(r[k % 2][i].h, t);
                    }
                    store_adjacent<DT, NT>(yres, at, (uint32_t) ((k / 4 * 32 + k % 4 * 8 + i) * pitch), v);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        by_act(p.act, [&](auto act_c) {
            if (p.residual != nullptr) {
                finish(act_c, std::true_type());
            } else {
                finish(act_c, std::false_type());
            }
        });
    };

    const auto first_half = [&](uint32_t slot) {
        read_scales(slot);
#pragma unroll
        for (int q = 0; q < RB; ++q) read_a(0, slot, q);
#pragma unroll
        for (int t = 0; t < NT; ++t) read_b(0, slot, t);
    };
    wait_vmcnt<0>();
    lds_barrier();
    first_half(0);
    uint32_t here = 0, there = kSlot;
    using std::integral_constant;
    // Up to the step before the last two of a tile the loads are of its own
    // steps; those of the last two are of the next tile's first two (a block with
    // several tiles has at least two steps), which then arrive while it leaves.
    int s = first_step, stop = max(first_step, steps - 2), load_step = first_step + 2, more = 1;
    for (;;) {
        for (; s < stop; ++s) {
            products(integral_constant<int, 0>(), here, 0, 0);
            // Step s + 1 (or the next tile's first) has landed, and every wavefront has read all of step s.
            wait_vmcnt<0>();
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
            products(integral_constant<int, 1>(), there, scalar(load_step), here);
            read_scales(there);
            load_step += more;
            const uint32_t swap = here;
            here = there;
            there = swap;
        }
        if (stop < steps) {
            stop = steps;
            more = unit + stride < end ? 1 : 0;
            if (more) place(unit + stride);
            aim(more);
            load_step = more ? first_step : 0;
            continue;
        }
        const int64_t row = row0;
        const int col = col0;
        row0 = next_row0;
        col0 = next_col0;
        unit += stride;
        if (unit < end) load_bias();
        leave(row, col);
        if (unit >= end) break;
        s = first_step;
        stop = steps - 2;
        load_step = first_step + 2;
        begin();
        first_half(here);  // again, as the registers were of use for the outputs
    }
    wait_vmcnt<0>();
}

// Joins the splits' sums in their order, then bias, activation and residual: N
// adjacent outputs a thread (N divides co).  One row 1024 -> 4096 fp16: 4.8 us of products
// and 2.6 here.
template <int DT, int N> __global__ void __launch_bounds__(256) k_linear_join(LinearAct p) {
    using T = typename Store<DT>::T;
    const int64_t e = ((int64_t) blockIdx.x * 256 + threadIdx.x) * N, count = p.n * p.co;
    if (e >= count) return;
    const int ch = (int) (e % p.co);
    float v[N];
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = p.bias != nullptr ? p.bias[ch + u] : 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float * q = p.partial + s * count + e;
        if constexpr (N == 4) {
            const float4 c = *(const float4 *) q;
            v[0] += c.x;
            v[1] += c.y;
            v[2] += c.z;
            v[3] += c.w;
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) v[u] += q[u];
        }
    }
    const T * residual = (const T *) p.residual;
    by_act(p.act, [&](auto act_c) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            v[u] = activate<DT, decltype(act_c)::value>(v[u]);
            if (residual != nullptr) v[u] += Store<DT>::ld(residual, e + u);
        }
    });
    if constexpr (N == 4 && DT != kF32) {
        union {
            T h[4];
            uint2 c;
        } w;
#pragma unroll
        for (int u = 0; u < 4; ++u) w.h[u] = round_to_store<DT>(v[u]);
        *(uint2 *) ((T *) p.y + e) = w.c;
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u) Store<DT>::st((T *) p.y, e + u, v[u]);
    }
}

// Rows that are no whole number of 16-byte chunks (odd widths, which the 16-byte
// loads cannot take): 64 x 64 outputs a block from fp32 copies in LDS, four by four
// a thread on the vector unit, which bounds it.
template <int DT> __global__ void __launch_bounds__(256) k_linear_act_any(LinearAct p) {
    using T = typename Store<DT>::T;
    constexpr int K = 16;
    __shared__ float s_x[K][68], s_w[K][68];
    const int t = threadIdx.x, tr = t / 16, tc = t % 16;
    const int64_t row0 = (int64_t) (blockIdx.x / p.col_tiles) * 64;
    const int col0 = (int) (blockIdx.x % p.col_tiles) * 64;
    const T * x = (const T *) p.x;
    const T * w = (const T *) p.w;
    const int wp = p.w_bytes / (int) sizeof(T);
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.ci; k0 += K) {
        __syncthreads();
#pragma unroll
        for (int i = t; i < 64 * K; i += 256) {
            const int r = i / K, k = i % K;
            s_x[k][r] = row0 + r < p.n && k0 + k < p.ci ? Store<DT>::ld(x, (row0 + r) * p.ci + k0 + k) : 0.0f;
            s_w[k][r] = col0 + r < p.co && k0 + k < p.ci ? Store<DT>::ld(w, (int64_t) (col0 + r) * wp + k0 + k) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float a[4], b[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                a[u] = s_x[k][tr * 4 + u];
                b[u] = s_w[k][tc * 4 + u];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
    }
    const T * residual = (const T *) p.residual;
    by_act(p.act, [&](auto act_c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = row0 + tr * 4 + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int ch = col0 + tc * 4 + j;
                if (row >= p.n || ch >= p.co) continue;
                const int64_t e = row * p.co + ch;
                float v = activate<DT, decltype(act_c)::value>(acc[i][j] + (p.bias != nullptr ? p.bias[ch] : 0.0f));
                if (residual != nullptr) v += Store<DT>::ld(residual, e);
                Store<DT>::st((T *) p.y, e, v);
            }
        }
    });
}

// ---- which blocks, and how many splits --------------------------------------------------------------

// Block shapes: rows, channels, adjacent channels per lane (which divide co),
// blocks per CU, and what a step of 128 bytes and the rest of a block take with
// all CUs busy, in us (measured on whole rounds of blocks, 1,024 channels, K of 4
// and of 32 steps, four rounds of 16 or 8 bits and two of fp32; the first loads and
// the last outputs of all, kOnce, are not in it).
struct Blocks {
    int rows, channels, adjacent, per_cu;
    float step16, step8, step32, rest, rest32;
};
constexpr Blocks kBlocks[] = {
    {256, 256, 4, 1, 1.78f, 2.10f, 7.1f, 4.2f, 13.7f},
    {192, 256, 2, 1, 1.52f, 1.75f, 5.4f, 2.7f, 12.0f},
    {128, 128, 2, 2, 1.27f, 1.58f, 3.85f, 1.1f, 7.3f},
    {64, 128, 2, 3, 1.20f, 1.57f, 3.1f, 0.9f, 5.5f},
    {128, 128, 1, 2, 1.31f, 1.70f, 3.9f, 1.8f, 7.5f},
    {64, 64, 1, 4, 0.88f, 1.24f, 2.3f, 1.6f, 4.7f},
};
constexpr double kOnce = 1.5;
constexpr int kShapes = sizeof(kBlocks) / sizeof(kBlocks[0]);

inline float step_us(const Blocks & b, int mt) { return mt == kF32 ? b.step32 : (mt == kRows8 ? b.step8 : b.step16); }

struct Choice {
    int shape = -1, splits = 1;
    float us = 0.0f;
};

// The shape and splits with the least estimated time for n rows.  Of a round that
// is not full each CU has its share of blocks, which take their part of a full
// round's time, but not less than kAlone (one block of three or four a CU: 0.33 to
// 0.45 measured), nor a step less than its loads' way, kWay (warm 0.5 us, from
// memory 1).  Splits pay for their sums' way out and back, which the caches
// hold, and for the join's launch: 5,003 x 300 -> 77 fp32 unsplit 10.7 us, in four 14.1;
// 1,832 x 4096 -> 1024 bf16 in four 28.
constexpr double kAlone = 0.4, kWay = 0.85, kJoin = 3.0, kJoinBytesPerUs = 8e6;
Choice choose(int mt, int64_t n, int co, int w_bytes, int cus, bool may_split) {
    const int steps = w_bytes / 128;
    Choice best;
    for (int i = 0; i < kShapes; ++i) {
        const Blocks & b = kBlocks[i];
        if (co % b.adjacent != 0) continue;
        const double blocks = (double) ((n + b.rows - 1) / b.rows) * ((co + b.channels - 1) / b.channels);
        const double step = step_us(b, mt), rest = mt == kF32 ? b.rest32 : b.rest;
        for (int s = 1; s <= (may_split ? 16 : 1); s *= 2) {
            if (s > 1 && (s > steps / 2 || i == 0)) break;  // (the largest blocks do not split)
            const double rounds = blocks * s / ((double) cus * b.per_cu), whole = std::floor(rounds);
            const double last = rounds - whole;
            const double tail = std::max(kAlone, std::ceil(last * b.per_cu) / b.per_cu);
            const int each = (steps + s - 1) / s;
            double us = kOnce + whole * (each * step + rest);
            if (last > 0.0) us += each * std::max(tail * step, kWay) + tail * rest;
            if (s > 1) us += kJoin + (double) s * n * co * 8.0 / kJoinBytesPerUs;
            if (best.shape < 0 || us < best.us) {
                best.shape = i;
                best.splits = s;
                best.us = (float) us;
            }
        }
    }
    return best;
}

template <int MT, int DT, int RW, int CW, int RB, int NT, int PER_CU>
hipError_t launch_shape(LinearAct p, const Blocks & b, hipStream_t s) {
    constexpr int BM = RW * RB * 32, BN = CW * NT * 32;
    if (b.rows != BM || b.channels != BN || b.adjacent != NT || b.per_cu != PER_CU) return hipErrorInvalidValue;
    p.row_tiles = (p.n + BM - 1) / BM;
    p.col_tiles = (p.co + BN - 1) / BN;
    const int64_t grid = p.row_tiles * p.col_tiles;
    if (grid * p.splits > 0x7fffffffLL) return hipErrorInvalidValue;
    p.split_blocks = (int) grid;
    p.blocks = (int) grid;
    // More tiles than fit at once: blocks that stay, each with several of them.
    const int64_t fit = (int64_t) p.cus / 8 * 8 * PER_CU;
    if (p.splits == 1 && p.w_bytes >= 256 && fit > 0 && grid > fit) p.blocks = (int) fit;
    k_linear_act<MT, DT, RW, CW, RB, NT, PER_CU><<<(unsigned) (p.blocks * (int64_t) p.splits), 64 * RW * CW, 0, s>>>(p);
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && p.splits > 1) {
        const bool four = p.co % 4 == 0;
        const int64_t joins = (p.n * p.co + (four ? 1023 : 255)) / (four ? 1024 : 256);
        if (joins > 0x7fffffffLL) return hipErrorInvalidValue;
        if (four) {
            k_linear_join<DT, 4><<<(unsigned) joins, 256, 0, s>>>(p);
        } else {
            k_linear_join<DT, 1><<<(unsigned) joins, 256, 0, s>>>(p);
        }
        err = hipGetLastError();
    }
    return err;
}

template <int MT, int DT> hipError_t launch_gemm(LinearAct p, int shape, int splits, hipStream_t s) {
    p.splits = splits;
    const Blocks & b = kBlocks[shape];
    switch (shape) {
        case 0: return launch_shape<MT, DT, 4, 2, 2, 4, 1>(p, b, s);
        case 1: return launch_shape<MT, DT, 2, 4, 3, 2, 1>(p, b, s);
        case 2: return launch_shape<MT, DT, 2, 2, 2, 2, 2>(p, b, s);
        case 3: return launch_shape<MT, DT, 2, 2, 1, 2, 3>(p, b, s);
        case 4: return launch_shape<MT, DT, 2, 4, 2, 1, 2>(p, b, s);
        case 5: return launch_shape<MT, DT, 2, 2, 1, 1, 4>(p, b, s);
        default: return hipErrorInvalidValue;
    }
}

template <int DT> hipError_t launch_any(LinearAct p, hipStream_t s) {
    p.col_tiles = (p.co + 63) / 64;
    const int64_t grid = (p.n + 63) / 64 * p.col_tiles;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    k_linear_act_any<DT><<<(unsigned) grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

template <int DT> hipError_t launch_dt(const LinearAct & p, int x_type, const LinearActPlan & plan, hipStream_t s) {
    if (plan.parts == 0) return launch_any<DT>(p, s);
    int64_t row = 0;
    for (int i = 0; i < plan.parts; ++i) {
        const auto & part = plan.part[i];
        LinearAct q = p;
        const int64_t e = (int64_t) sizeof(typename Store<DT>::T);
        q.x = (const char *) p.x + row * p.row_bytes;
        if (p.x_scales != nullptr) q.x_scales = p.x_scales + row * (p.row_bytes / 32);
        if (p.residual != nullptr) q.residual = (const char *) p.residual + row * p.co * e;
        q.y = (char *) p.y + row * p.co * e;
        q.n = part.rows;
        const int splits = p.partial != nullptr ? part.splits : 1;
        const hipError_t err = x_type == kRows8 ? launch_gemm<kRows8, DT>(q, part.shape, splits, s)
                                                : launch_gemm<DT, DT>(q, part.shape, splits, s);
        if (err != hipSuccess) return err;
        row += part.rows;
    }
    return hipSuccess;
}

}  // namespace

// All rows in one launch, or whole rounds of large blocks in one and the rows that
// are left in another, with blocks and splits of their own (18,216 x 4096 ->
// 1024 bf16: 288 blocks of 256 x 256 are one round of 256 and one of 32).
LinearActPlan linear_act_plan(int dtype, int x_type, int64_t n, int co, int row_bytes, int w_bytes, int cus,
                              bool may_split) {
    LinearActPlan plan{};
    if (x_type != kRows8 && row_bytes % 16 != 0) return plan;
    const int mt = x_type == kRows8 ? kRows8 : dtype;
    const auto scratch = [&](const LinearActPart & part) {
        return part.splits > 1 ? (size_t) part.splits * part.rows * co * sizeof(float) : 0;
    };
    const Choice one = choose(mt, n, co, w_bytes, cus, may_split);
    plan.parts = 1;
    plan.part[0] = {n, one.shape, one.splits};
    plan.scratch = scratch(plan.part[0]);
    float least = one.us;
    for (int i = 0; i < 2; ++i) {
        const Blocks & b = kBlocks[i];
        if (co % b.adjacent != 0) continue;
        const int64_t col_tiles = (co + b.channels - 1) / b.channels, row_tiles = n / b.rows;
        const int64_t rounds = row_tiles * col_tiles / cus;
        const int64_t rows = rounds * cus / col_tiles * b.rows;
        if (rounds < 1 || rows <= 0 || rows >= n) continue;
        const Choice rest = choose(mt, n - rows, co, w_bytes, cus, may_split);
        const double block = w_bytes / 128 * step_us(b, mt) + (mt == kF32 ? b.rest32 : b.rest);
        const float us = (float) (kOnce + rounds * block) + rest.us + 3.0f;
        if (us >= least) continue;
        least = us;
        plan.parts = 2;
        plan.part[0] = {rows, i, 1};
        plan.part[1] = {n - rows, rest.shape, rest.splits};
        plan.scratch = scratch(plan.part[1]);
    }
    return plan;
}

hipError_t launch_linear_act(int dtype, int x_type, const LinearAct & p, const LinearActPlan & plan, hipStream_t s) {
    switch (dtype) {
        case kF32: return launch_dt<kF32>(p, x_type, plan, s);
        case kF16: return launch_dt<kF16>(p, x_type, plan, s);
        default: return launch_dt<kBF16>(p, x_type, plan, s);
    }
}

}  // namespace tsh
