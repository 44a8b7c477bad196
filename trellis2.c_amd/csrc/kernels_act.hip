// kernels_act.hip - linear with activation and residual in its epilogue, from rows of the storage type or 8-bit rows.
#include "mfma_common.h"

namespace tsh {
namespace {

// ---- activations --------------------------------------------------------------------------------

// For 16-bit outputs the hardware exponential and reciprocal (about 2^-21
// relative) and an erf of 1.5e-7 (Abramowitz and Stegun 7.1.26) stay far below the
// output's rounding; fp32 outputs take the accurate functions.
template <int DT, int ACT> __device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_SILU) {
        if constexpr (DT == kF32) return v / (1.0f + expf(-v));
        return v * __builtin_amdgcn_rcpf(1.0f + __expf(-v));
    } else if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_GELU) {
        if constexpr (DT == kF32) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        // erf(|z|) = 1 - t (a1 + t (a2 + ...)) exp(-z^2), t = 1 / (1 + 0.3275911 |z|).
        const float z = fabsf(v) * 0.70710678118654752f;
        const float t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * z);
        const float poly =
            t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
        const float tail = 0.5f * poly * __expf(-z * z);  // (1 - erf(z)) / 2
        return v * (v < 0.0f ? tail : 1.0f - tail);
    } else if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_GELU_TANH) {
        // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u))
        const float u2 = 1.5957691216057308f * (v + 0.044715f * v * v * v);
        if constexpr (DT == kF32) return v / (1.0f + expf(-u2));
        return v * __builtin_amdgcn_rcpf(1.0f + __expf(-u2));
    } else {
        return v;
    }
}

// ---- MFMA GEMM ----------------------------------------------------------------------------------

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

// A fragment is two 16-byte chunks, g and g + 4 for lane group g = lane / 16, of
// row lane % 16 (of x or of W) in a step of 128 bytes: 32, 64 or 128 K values in
// fp32, 16 or 8 bits.  The scaled MFMA takes the chunks as K values 16 g .. and
// 64 + 16 g .., and from lane group g the scale of K values 32 g .. 32 g + 31.  It
// adds eight neighbouring products at a time on the scale of the largest, cutting
// each at 2^-13 of it (measured: 2^-13 stays, 2^-14 goes), before the fp32 sums: an
// error near 2e-5 of a sum's size, a hundredth of a bf16 rounding, for twice the
// rate of bf16.
struct Frag {
    int4 c[2];
};

template <int MT> __device__ __forceinline__ f32x4 mac(const Frag & a, const Frag & b, f32x4 c, int sa, int sb) {
    if constexpr (MT == kF32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4v x = __builtin_bit_cast(f32x4v, a.c[h]), w = __builtin_bit_cast(f32x4v, b.c[h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], w[j], c, 0, 0, 0);
        }
        return c;
    } else if constexpr (MT == kRows8) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(i32x8, a), __builtin_bit_cast(i32x8, b),
                                                                c, 0, 0, 0, sa, 0, sb);
    } else {
        using V = typename Mfma<MT>::V;
        c = Mfma<MT>::mac(__builtin_bit_cast(V, a.c[0]), __builtin_bit_cast(V, b.c[0]), c);
        return Mfma<MT>::mac(__builtin_bit_cast(V, a.c[1]), __builtin_bit_cast(V, b.c[1]), c);
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

constexpr uint32_t kOutside = 0x80000000u;  // beyond every buffer here: loads fetch zeros

// A block multiplies BM rows of x by BN rows of W (output channels), RW x CW
// wavefronts of BM / RW rows and 128 channels each, 128 bytes of both a step.
//
// LDS: a step's slot holds 16-row blocks of 2 KB, row i at (i % 8) * 256 + (i / 8)
// * 128, its chunk c at ((c ^ i) % 8) * 16: the 16 lanes that read one chunk of
// 16 rows touch each of the 64 banks once, and eight lanes of a load fetch one
// row's 128 contiguous bytes.  Tile t's lane i multiplies channel 8 i + t of a
// wavefront's 128, so that a lane ends with eight adjacent channels and a row
// leaves in 16-byte pieces.
template <int MT, int DT, int ACT, int BM, int BN, int RW, int CW>
__global__ void __launch_bounds__(64 * RW * CW, 1) k_linear_act(LinearAct p) {
    using T = typename Store<DT>::T;
    constexpr int NW = RW * CW, NT = 8, QB = BM / RW / 16;
    static_assert(BN == CW * 128 && BM % (RW * 16) == 0, "128 channels per wavefront");
    constexpr bool kScaled = MT == kRows8;
    constexpr int kBytes = (BM + BN) * 128, kSlot = kBytes + (kScaled ? (BM + BN) * 4 : 0);
    constexpr int kLoads = (BM + BN) / 8, kPer = kLoads / NW;  // 1 KB each
    static_assert(kLoads % NW == 0, "as many loads for every wavefront");
    constexpr int kScaleLoads = (BM + BN) / 64;
    __shared__ __attribute__((aligned(1024))) unsigned char s_slot[2 * kSlot];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RW, cw = wave / RW;
    const int l16 = lane & 15, lg = lane >> 4;

    // Blocks b, b + 8, ... run on one XCD, which multiplies a row block by
    // every channel block in turn: the rows stay in its L2.
    const int64_t in_xcd = blockIdx.x / 8;
    const int64_t tile = in_xcd / p.col_tiles * 8 + blockIdx.x % 8;
    if (tile >= p.row_tiles) return;
    const int64_t row0 = tile * BM;
    const int col0 = (int) (in_xcd % p.col_tiles) * BN;
    const int rows = (int) min((int64_t) BM, p.n - row0);

    const __amdgpu_buffer_rsrc_t xres = __builtin_amdgcn_make_buffer_rsrc(
        (void *) ((const char *) p.x + row0 * p.row_bytes), 0, (int) (rows * p.row_bytes), 0x00020000);
    const __amdgpu_buffer_rsrc_t wres = __builtin_amdgcn_make_buffer_rsrc(
        (void *) ((const char *) p.w + (int64_t) col0 * p.w_bytes), 0, (int) (BN * p.w_bytes), 0x00020000);
    const uint32_t slot0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) unsigned char *) s_slot;

    // This lane's piece of load j of this wavefront: 8 lines of 128 bytes.
    const auto of_x = [&](int j) { return wave * kPer + j < BM / 8; };
    uint32_t at[kPer];
    int chunk[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int q = wave * kPer + j - (of_x(j) ? 0 : BM / 8);  // KB of x's or W's part
        const int line = (q & 1) * 4 + (lane >> 4), i = line + ((lane >> 3) & 1) * 8;
        chunk[j] = (lane ^ i) & 7;
        const int row = q / 2 * 16 + i;  // of x's rows or W's LDS rows
        if (of_x(j)) {
            at[j] = row < rows ? (uint32_t) (row * p.row_bytes) + chunk[j] * 16u : kOutside;
        } else {
            const int ch = row / 128 * 128 + row % 16 * 8 + row % 128 / 16;
            at[j] = (uint32_t) (ch * p.w_bytes) + chunk[j] * 16u;
        }
    }
    // Scales: 64 rows of 4 bytes a load, one wavefront each.
    uint32_t scale_at = kOutside;
    __amdgpu_buffer_rsrc_t sres = xres;
    if constexpr (kScaled) {
        static_assert(kScaleLoads <= NW, "one load per wavefront");
        const int row = wave * 64 + lane;
        const int xs = p.row_bytes / 32, ws = p.w_bytes / 32;
        if (wave * 64 < BM) {
            sres = __builtin_amdgcn_make_buffer_rsrc((void *) (p.x_scales + row0 * xs), 0, rows * xs, 0x00020000);
            if (row < rows) scale_at = (uint32_t) (row * xs);
        } else {
            sres = __builtin_amdgcn_make_buffer_rsrc((void *) (p.w_scales + (int64_t) col0 * ws), 0, BN * ws, 0x00020000);
            const int r = row - BM;
            scale_at = (uint32_t) ((r / 128 * 128 + r % 16 * 8 + r % 128 / 16) * ws);
        }
    }
    const int steps = p.w_bytes / 128;
    const auto load = [&](int s) {
        const uint32_t to = slot0 + (s & 1) * kSlot + (uint32_t) (wave * kPer) * 1024u;
        const bool end = (s + 1) * 128 > p.row_bytes;  // what follows a row of x is the next one
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (of_x(j)) {
                dma_b128(xres, to + j * 1024u, end && s * 128 + chunk[j] * 16 >= p.row_bytes ? kOutside : at[j],
                         s * 128u);
            } else {
                dma_b128(wres, to + j * 1024u, at[j], s * 128u);
            }
        }
        if constexpr (kScaled) {
            if (wave < kScaleLoads) dma_b32(sres, slot0 + (s & 1) * kSlot + kBytes + wave * 256u, scale_at, s * 4u);
        }
    };

    f32x4 acc[QB][NT];
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int line = (l16 & 7) * 256 + (l16 >> 3) * 128;
    const int c0 = line + ((lg ^ l16) & 7) * 16;
    const int c1 = line + (((lg + 4) ^ l16) & 7) * 16;
    load(0);
    for (int s = 0; s < steps; ++s) {
        wait_vmcnt<0>();
        lds_barrier();
        if (s + 1 < steps) load(s + 1);
        const unsigned char * sx = s_slot + (s & 1) * kSlot + rw * QB * 2048;
        const unsigned char * sw = s_slot + (s & 1) * kSlot + BM * 128 + cw * NT * 2048;
        const unsigned char * ss = s_slot + (s & 1) * kSlot + kBytes;
        Frag a[QB], b[NT];
        int sa[QB], sb[NT];
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            a[q].c[0] = *(const int4 *) (sx + q * 2048 + c0);
            a[q].c[1] = *(const int4 *) (sx + q * 2048 + c1);
            sa[q] = kScaled ? ss[((rw * QB + q) * 16 + l16) * 4 + lg] : 0;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            b[t].c[0] = *(const int4 *) (sw + t * 2048 + c0);
            b[t].c[1] = *(const int4 *) (sw + t * 2048 + c1);
            sb[t] = kScaled ? ss[(BM + (cw * NT + t) * 16 + l16) * 4 + lg] : 0;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int q = 0; q < QB; ++q) acc[q][t] = mac<MT>(a[q], b[t], acc[q][t], sa[q], sb[t]);
    }

    // Lane (l16, lg) holds rows 4 lg + i of each row block, channels 8 l16 .. 8 l16 + 7 of the wavefront's 128.
    const int ch = col0 + cw * 128 + l16 * 8;
    float bias[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) bias[u] = p.bias != nullptr && ch + u < p.co ? p.bias[ch + u] : 0.0f;
    const bool whole = p.co % 8 == 0 && ch < p.co;  // all eight channels, 16-byte aligned
    const T * residual = (const T *) p.residual;
    T * y = (T *) p.y;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = row0 + rw * (BM / RW) + q * 16 + lg * 4 + i;
            if (row >= p.n) continue;
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = activate<DT, ACT>(acc[q][u][i] + bias[u]);
            const int64_t e = row * p.co + ch;
            if (whole) {
                if (residual != nullptr) {
                    float r[8];
                    if constexpr (DT == kF32) {
#pragma unroll
                        for (int u = 0; u < 8; ++u) r[u] = residual[e + u];
                    } else {
                        unpack_chunk<DT>(*(const int4 *) (residual + e), r);
                    }
#pragma unroll
                    for (int u = 0; u < 8; ++u) v[u] += r[u];
                }
                if constexpr (DT == kF32) {
                    *(float4 *) (y + e) = float4{v[0], v[1], v[2], v[3]};
                    *(float4 *) (y + e + 4) = float4{v[4], v[5], v[6], v[7]};
                } else {
                    *(int4 *) (y + e) = pack_chunk<DT>(v);
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (ch + u >= p.co) break;
                    Store<DT>::st(y, e + u, residual != nullptr ? v[u] + Store<DT>::ld(residual, e + u) : v[u]);
                }
            }
        }
    }
}

// Rows that are no whole number of 16-byte chunks: 64 x 64 outputs a block
// from fp32 copies in LDS, four by four a thread.
template <int DT, int ACT> __global__ void __launch_bounds__(256) k_linear_act_any(LinearAct p) {
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
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + tr * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int ch = col0 + tc * 4 + j;
            if (row >= p.n || ch >= p.co) continue;
            const int64_t e = row * p.co + ch;
            float v = activate<DT, ACT>(acc[i][j] + (p.bias != nullptr ? p.bias[ch] : 0.0f));
            if (residual != nullptr) v += Store<DT>::ld(residual, e);
            Store<DT>::st((T *) p.y, e, v);
        }
    }
}

template <int MT, int DT, int ACT, int BM, int BN, int RW, int CW>
hipError_t launch_gemm_t(LinearAct p, hipStream_t s) {
    p.row_tiles = (p.n + BM - 1) / BM;
    p.col_tiles = (p.co + BN - 1) / BN;
    const int64_t grid = (p.row_tiles + 7) / 8 * 8 * p.col_tiles;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    k_linear_act<MT, DT, ACT, BM, BN, RW, CW><<<(unsigned) grid, 64 * RW * CW, 0, s>>>(p);
    return hipGetLastError();
}

template <int MT, int DT, int ACT> hipError_t launch_act_t(const LinearAct & p, int cus, hipStream_t s) {
    const auto blocks = [&](int bm, int bn) { return (p.n + bm - 1) / bm * ((p.co + bn - 1) / bn); };
    if (blocks(256, 256) >= 2 * (int64_t) cus) return launch_gemm_t<MT, DT, ACT, 256, 256, 4, 2>(p, s);
    if (blocks(128, 128) >= cus) return launch_gemm_t<MT, DT, ACT, 128, 128, 4, 1>(p, s);
    return launch_gemm_t<MT, DT, ACT, 64, 128, 4, 1>(p, s);
}

template <int DT, int ACT> hipError_t launch_any_t(LinearAct p, hipStream_t s) {
    p.col_tiles = (p.co + 63) / 64;
    const int64_t grid = (p.n + 63) / 64 * p.col_tiles;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    k_linear_act_any<DT, ACT><<<(unsigned) grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

template <int DT, int ACT> hipError_t launch_dt(const LinearAct & p, int x_type, int cus, hipStream_t s) {
    if (x_type == kRows8) return launch_act_t<kRows8, DT, ACT>(p, cus, s);
    if (p.row_bytes % 16 == 0) return launch_act_t<DT, DT, ACT>(p, cus, s);
    return launch_any_t<DT, ACT>(p, s);
}

template <int DT> hipError_t launch_act(const LinearAct & p, int x_type, int act, int cus, hipStream_t s) {
    switch (act) {
        case TRELLIS_SPARSE_HIP_ACT_SILU: return launch_dt<DT, TRELLIS_SPARSE_HIP_ACT_SILU>(p, x_type, cus, s);
        case TRELLIS_SPARSE_HIP_ACT_GELU: return launch_dt<DT, TRELLIS_SPARSE_HIP_ACT_GELU>(p, x_type, cus, s);
        case TRELLIS_SPARSE_HIP_ACT_GELU_TANH:
            return launch_dt<DT, TRELLIS_SPARSE_HIP_ACT_GELU_TANH>(p, x_type, cus, s);
        default: return launch_dt<DT, TRELLIS_SPARSE_HIP_ACT_NONE>(p, x_type, cus, s);
    }
}

}  // namespace

hipError_t launch_linear_act(int dtype, int x_type, const LinearAct & p, int act, int cus, hipStream_t s) {
    switch (dtype) {
        case kF32: return launch_act<kF32>(p, x_type, act, cus, s);
        case kF16: return launch_act<kF16>(p, x_type, act, cus, s);
        default: return launch_act<kBF16>(p, x_type, act, cus, s);
    }
}

}  // namespace tsh
