// kernels_rows.hip - row operators of transformer blocks over voxel rows: RMS norm, 8-bit rows, rotary positions.
#include <type_traits>

#include "mfma_common.h"

namespace tsh {
namespace {

// ---- chunks of 16 bytes -------------------------------------------------------------------------

// Values per 16-byte chunk.
template <int DT> constexpr int kChunk = DT == kF32 ? 4 : 8;

template <int DT> __device__ __forceinline__ void unpack_chunk_of(const int4 & c, float * v) {
    if constexpr (DT == kF32) {
        v[0] = __builtin_bit_cast(float, c.x);
        v[1] = __builtin_bit_cast(float, c.y);
        v[2] = __builtin_bit_cast(float, c.z);
        v[3] = __builtin_bit_cast(float, c.w);
    } else {
        unpack_chunk<DT>(c, v);
    }
}

template <int DT> __device__ __forceinline__ void store_chunk(typename Store<DT>::T * p, const float * v) {
    if constexpr (DT == kF32) {
        *(float4 *) p = float4{v[0], v[1], v[2], v[3]};
    } else {
        *(int4 *) p = pack_chunk<DT>(v);
    }
}

// ---- 8-bit rows ---------------------------------------------------------------------------------

// A block of 32 channels has one scale 2^e, e >= -126 the least with
// max|v| <= 448 * 2^e (448 is e4m3's largest value), so that codes never
// saturate and every product with the scale is exact: a code times its scale
// has four significant bits and fits bf16.  Returned as the biased byte that
// the scaled MFMA takes (127 + e); 127 for a block of zeros; 255 (NaN) for a block
// with an infinity or a NaN, which leaves no finite scale.
// max_bits: the largest |v| as bits (larger for NaN than for any number).
__device__ __forceinline__ uint32_t block_scale(uint32_t max_bits) {
    if (max_bits >= 0x7f800000u) return 255;
    if (max_bits == 0) return 127;
    // 448 = 1.75 * 2^8: one more where the mantissa exceeds 1.75.
    const int e = (int) (max_bits >> 23) - 127 - 8 + ((max_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t) (127 + (e < -126 ? -126 : e));
}

// 1 / scale (scale bytes 1..247 appear; 255 gives codes apart).
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
    return __builtin_bit_cast(float, (254u - byte) << 23);
}

// Four values to four e4m3 codes, to nearest even (|v| <= 448: no saturation).
__device__ __forceinline__ uint32_t codes4(const float * v, float inv, uint32_t scale) {
    if (scale == 255) return 0x7f7f7f7fu;
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
    return (uint32_t) w;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// 1 / sqrt(sum / c + eps), for 8-bit outputs as two floats from 64 bits: there a
// value on the other side of a code's border is off by a whole code, so the last
// bit of the norm counts.  The squares are exact and summed in 64 bits (with squares
// in fp32, joined 8 at a time, 2 of 12 M codes were beside the exact ones), and a
// value is not rounded to nearest before it is rounded to its code, but cut and
// made odd where something was cut (twice to nearest had 10 of 12 M).
struct Inverse {
    float hi, lo;
};
template <bool FINE> using NormSum = typename std::conditional<FINE, double, float>::type;
__device__ __forceinline__ float add_square(float sum, float v) { return sum + v * v; }
__device__ __forceinline__ double add_square(double sum, float v) { return fma((double) v, (double) v, sum); }
template <bool FINE> __device__ __forceinline__ Inverse inverse_rms(NormSum<FINE> sum, int c, double per_c, float eps) {
    if constexpr (FINE) {
        // The hardware's estimate and one Newton step in 64 bits (1e-13).
        const double m = sum * per_c + (double) eps;  // (per_c: 1 / c)
        const double y = (double) __builtin_amdgcn_rsqf((float) m);
        double d = fma(0.5 * y, fma(-m * y, y, 1.0), y);
        if (!(m > 1e-30 && m < 1e38)) d = 1.0 / sqrt(m);
        const float hi = (float) d;
        return {hi, (float) (d - (double) hi)};
    }
    return {1.0f / sqrtf(sum / (float) c + eps), 0.0f};
}
// v * inv * g; where FINE to odd: what a later rounding to fewer bits sees is the exact value's side.
template <bool FINE> __device__ __forceinline__ float scaled(float v, const Inverse & inv, float g) {
    if constexpr (FINE) {
        const float p = v * g;
        const float low = fmaf(fmaf(v, g, -p), inv.hi, p * inv.lo);
        const float h = fmaf(p, inv.hi, low);
        const float rest = fmaf(p, inv.hi, -h) + low;
        const uint32_t b = __builtin_bit_cast(uint32_t, h);
        // Nearest went past the value: one step back towards zero.
        const uint32_t past = (__builtin_bit_cast(uint32_t, rest) ^ b) >> 31;
        constexpr int kNonzeroFinite = 0x198;
        return __builtin_amdgcn_classf(rest, kNonzeroFinite) ? __builtin_bit_cast(float, (b - past) | 1u) : h;
    }
    return v * inv.hi * g;
}

// Where the norm's rows go.
struct NormOut {
    void * y;          // storage type [n][c], or null
    uint8_t * codes;   // 8-bit rows: [n][cp] codes, [n][cp / 32] scales
    uint8_t * scales;
    int cp;
};

// y = s / sqrt(mean(s^2) + eps) * gamma, s = x + residual in fp32 (total: s in
// the storage type; y comes from the unrounded s, so each output is rounded
// once).  NORM = false packs x itself into 8-bit rows.  LPR lanes hold a row in
// registers, CPL chunks of 16 bytes each, and keep gamma from row to row: one
// pass over memory, which bounds it.  The next row's loads are issued before this
// row's sum is reduced, and the sum is reduced by DPP (18,216 rows of 1024 to 8-bit
// rows 38 -> 31 us for both).  79,523 rows of 512 in bf16 with residual and total 62 us, 5.2
// TB/s (a copy of the size 5.3); 18,216 of 1024 to 8-bit rows with total 31 us,
// 4.2 TB/s; one row 4 us.
template <int DT, int LPR, int CPL, bool Q8, bool NORM>
__global__ void __launch_bounds__(256) k_norm_vec(const typename Store<DT>::T * x,
                                                  const typename Store<DT>::T * residual,
                                                  const float * __restrict__ gamma, typename Store<DT>::T * total,
                                                  NormOut out, int64_t n, int c, float eps) {
    using T = typename Store<DT>::T;
    constexpr int V = kChunk<DT>, RPB = 256 / LPR;
    const int l = threadIdx.x % LPR;
    float g[CPL][V];
#pragma unroll
    for (int i = 0; i < CPL; ++i)
#pragma unroll
        for (int u = 0; u < V; ++u) {
            const int at = (i * LPR + l) * V + u;
            g[i][u] = NORM && gamma != nullptr && at < c ? gamma[at] : 1.0f;
        }
    const double per_c = 1.0 / c;
    // The next row's loads run under this one's sums and stores.
    int4 xc[CPL], rc[CPL];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int at = (i * LPR + l) * V;
            xc[i] = rc[i] = int4{0, 0, 0, 0};
            if (at < c) {
                xc[i] = *(const int4 *) (x + row * c + at);
                if (residual != nullptr) rc[i] = *(const int4 *) (residual + row * c + at);
            }
        }
    };
    int64_t row = (int64_t) blockIdx.x * RPB + threadIdx.x / LPR;
    const int64_t stride = (int64_t) gridDim.x * RPB;
    if (row < n) fetch(row);
    for (; row < n; row += stride) {
        float v[CPL][V];
        NormSum<Q8> sum = 0;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            unpack_chunk_of<DT>(xc[i], v[i]);
            if (residual != nullptr) {
                float r[V];
                unpack_chunk_of<DT>(rc[i], r);
#pragma unroll
                for (int u = 0; u < V; ++u) v[i][u] += r[u];
            }
        }
        if (row + stride < n) fetch(row + stride);
        if (total != nullptr) {
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int at = (i * LPR + l) * V;
                if (at < c) store_chunk<DT>(total + row * c + at, v[i]);
            }
        }
        if constexpr (NORM) {
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                NormSum<Q8> part = 0;
#pragma unroll
                for (int u = 0; u < V; ++u) part = add_square(part, v[i][u]);
                sum += part;
            }
            const Inverse inv = inverse_rms<Q8>(group_sum<LPR>(sum), c, per_c, eps);
#pragma unroll
            for (int i = 0; i < CPL; ++i)
#pragma unroll
                for (int u = 0; u < V; ++u) v[i][u] = scaled<Q8>(v[i][u], inv, g[i][u]);
        }
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int at = (i * LPR + l) * V;
            if constexpr (Q8) {
                // The 32 / V lanes of a block are neighbours; values beyond c are zeros (or NaN, as all of the row).
                uint32_t m = 0;
#pragma unroll
                for (int u = 0; u < V; ++u) m = max(m, abs_bits(v[i][u]));
                const uint32_t scale = block_scale(group_max<32 / V>(m));
                const float inv = inverse_scale(scale);
                if (at < out.cp) {
                    const float * z = v[i];
                    uint8_t * p = out.codes + row * out.cp + at;
                    if constexpr (V == 8) {
                        *(uint2 *) p = uint2{codes4(z, inv, scale), codes4(z + 4, inv, scale)};
                    } else {
                        *(uint32_t *) p = codes4(z, inv, scale);
                    }
                    if (at % 32 == 0) out.scales[row * (out.cp / 32) + at / 32] = (uint8_t) scale;
                }
            } else {
                if (at < c) store_chunk<DT>((T *) out.y + row * c + at, v[i]);
            }
        }
    }
}

// Any width: one wavefront per row, which it reads twice (widths that are no
// whole number of chunks, or beyond what a wavefront holds in registers), the
// second time from the caches.
template <int DT, bool Q8, bool NORM>
__global__ void __launch_bounds__(256) k_norm_any(const typename Store<DT>::T * x,
                                                  const typename Store<DT>::T * residual,
                                                  const float * __restrict__ gamma, typename Store<DT>::T * total,
                                                  NormOut out, int64_t n, int c, float eps) {
    using T = typename Store<DT>::T;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= n) return;
    const auto at = [&](int i) {
        const float v = Store<DT>::ld(x, row * c + i);
        return residual != nullptr ? v + Store<DT>::ld(residual, row * c + i) : v;
    };
    Inverse inv{1.0f, 0.0f};
    if constexpr (NORM) {
        NormSum<Q8> sum = 0;
        for (int i = lane; i < c; i += 64) {
            sum = add_square(sum, at(i));
        }
        inv = inverse_rms<Q8>(group_sum<64>(sum), c, 1.0 / c, eps);
    }
    const int end = Q8 ? out.cp : c;
    for (int i = lane; i < end; i += 64) {
        float v = 0.0f;
        if (i < c) {
            const float s = at(i);
            // An element of total may be the same memory as that of x or residual: read first.
            if (total != nullptr) Store<DT>::st(total, row * c + i, s);
            v = s;
            if constexpr (NORM) v = scaled<Q8>(v, inv, gamma != nullptr ? gamma[i] : 1.0f);
        }
        if constexpr (Q8) {
            const uint32_t scale = block_scale(group_max<32>(abs_bits(v)));
            const float z[4] = {v, 0.0f, 0.0f, 0.0f};
            out.codes[row * out.cp + i] = (uint8_t) codes4(z, inverse_scale(scale), scale);
            if (lane % 32 == 0) out.scales[row * (out.cp / 32) + i / 32] = (uint8_t) scale;
        } else {
            Store<DT>::st((T *) out.y, row * c + i, v);
        }
    }
}

// The values that 8-bit rows stand for: 16 codes a thread, rows found once (whole
// 16-byte chunks of y where a row is a whole number of them).  Bound by memory:
// 18,216 rows of 1024 to bf16 12 us, 4.8 TB/s.
template <int DT, bool WHOLE>
__global__ void __launch_bounds__(256) k_expand8(const uint8_t * __restrict__ codes, const uint8_t * __restrict__ scales,
                                                 typename Store<DT>::T * __restrict__ y, int64_t n, int c, int cp) {
    constexpr int V = kChunk<DT>;
    const int pieces = (c + 15) / 16;
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= n * pieces) return;
    const int64_t row = n * pieces <= INT32_MAX ? (int64_t) ((uint32_t) i / (uint32_t) pieces) : i / pieces;
    const int at = (int) (i - row * pieces) * 16;
    const int4 w = *(const int4 *) (codes + row * cp + at);
    const uint32_t byte = scales[row * (cp / 32) + at / 32];
    const float scale = byte == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, byte << 23);
    const int quad[4] = {w.x, w.y, w.z, w.w};
    float v[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(quad[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(quad[k], true);
        v[4 * k] = lo[0] * scale;
        v[4 * k + 1] = lo[1] * scale;
        v[4 * k + 2] = hi[0] * scale;
        v[4 * k + 3] = hi[1] * scale;
    }
    typename Store<DT>::T * yr = y + row * c + at;
    if constexpr (WHOLE) {
#pragma unroll
        for (int u = 0; u < 16; u += V)
            if (at + u < c) store_chunk<DT>(yr + u, v + u);
    } else {
#pragma unroll
        for (int u = 0; u < 16; ++u)
            if (at + u < c) Store<DT>::st(yr, u, v[u]);
    }
}

template <int DT, bool Q8, bool NORM>
hipError_t norm_dt(const void * x, const void * residual, const float * gamma, void * total, const NormOut & out,
                   int64_t n, int c, float eps, int cus, hipStream_t s) {
    using T = typename Store<DT>::T;
    constexpr int V = kChunk<DT>;
    const int width = Q8 ? out.cp : c;
    const int chunks = (width + V - 1) / V;
    if (c % V != 0 || chunks > 64 * 8) {
        const int64_t g = (n + 3) / 4;
        if (g > 0x7fffffffLL) return hipErrorInvalidValue;
        k_norm_any<DT, Q8, NORM><<<(unsigned) g, 256, 0, s>>>((const T *) x, (const T *) residual, gamma, (T *) total,
                                                              out, n, c, eps);
        return hipGetLastError();
    }
    const auto launch = [&](auto lpr, auto cpl) {
        constexpr int LPR = decltype(lpr)::value, CPL = decltype(cpl)::value;
        constexpr int RPB = 256 / LPR;
        const int64_t g = std::min<int64_t>((n + RPB - 1) / RPB, (int64_t) cus * 4);
        k_norm_vec<DT, LPR, CPL, Q8, NORM><<<(unsigned) g, 256, 0, s>>>((const T *) x, (const T *) residual, gamma,
                                                                        (T *) total, out, n, c, eps);
        return hipGetLastError();
    };
    using std::integral_constant;
    if (chunks <= 8) return launch(integral_constant<int, 8>(), integral_constant<int, 1>());
    if constexpr (Q8) {
        // The inverse's 64-bit arithmetic counts: two rows a wavefront share it (79,523 rows of 512 in bf16 43 -> 38 us).
        if (chunks <= 16) return launch(integral_constant<int, 8>(), integral_constant<int, 2>());
        if (chunks <= 32) return launch(integral_constant<int, 16>(), integral_constant<int, 2>());
        if (chunks <= 64) return launch(integral_constant<int, 32>(), integral_constant<int, 2>());
    } else {
        if (chunks <= 16) return launch(integral_constant<int, 16>(), integral_constant<int, 1>());
        if (chunks <= 32) return launch(integral_constant<int, 32>(), integral_constant<int, 1>());
        if (chunks <= 64) return launch(integral_constant<int, 64>(), integral_constant<int, 1>());
    }
    if (chunks <= 128) return launch(integral_constant<int, 64>(), integral_constant<int, 2>());
    if (chunks <= 256) return launch(integral_constant<int, 64>(), integral_constant<int, 4>());
    return launch(integral_constant<int, 64>(), integral_constant<int, 8>());
}

// ---- rotary positions ---------------------------------------------------------------------------

// Each head's D channels are D / 2 pairs: (2p, 2p + 1), or (p, p + D / 2) with
// `split`.  Pair p of axis a turns by pos_a * base^(-j / P_a), j its place
// among the axis' P_a pairs; pairs beyond the three axes' pass unturned.  With
// `norm` each head is divided by its root mean square (and multiplied by
// gamma) first.
//
// Angles are kept in turns: pos * (freq / 2 pi) in 64 bits, less its nearest
// whole number, so that far positions lose nothing (pos = 32,767 at frequency 1
// is 5,215 turns, of which 32 bits keep 2^-12).  A block turns RB rows: sine and
// cosine of a row's pairs are computed once, into LDS, and used by all of its
// heads; then lanes of 4 pairs (two 8-byte or one 16-byte load) take one head
// each over all rows, gamma in registers, two items ahead of the one in hand (one:
// 79 us).  Bound by memory: 79,523 rows, q and k of 8 heads of 64 in a buffer of q, k
// and v, bf16 with norm 67.5 us, 4.8 TB/s (a copy of the size 5.4); packed fp32 rows of 8
// heads 66 us, 4.9 TB/s; 997 rows of 6 x 48 in fp32 4 us.
struct RotaryShape {
    int64_t n, x_stride, y_stride;
    int heads, dim, total;  // total: turned pairs
    int axis1, axis2;              // first pair of the y and z axes
    float eps;
    int rows;                      // rows per block
};
struct RotaryFreq {
    double turns[kRotaryMaxDim / 2];  // freq / 2 pi per pair
};

template <int DT, int GP, bool NORM, bool SPLIT>
__global__ void __launch_bounds__(256) k_rotary(const typename Store<DT>::T * x, const int32_t * __restrict__ coords,
                                                const float * __restrict__ gamma, typename Store<DT>::T * y,
                                                RotaryShape p, RotaryFreq f) {
    using T = typename Store<DT>::T;
    extern __shared__ float2 s_turn[];  // [rows][dim / 2]: cosine, sine
    const int64_t row0 = (int64_t) blockIdx.x * p.rows;
    const int rows = (int) min((int64_t) p.rows, p.n - row0);
    const int half = p.dim / 2;

    constexpr int GROUPS = 256 / GP;  // (row, head) items at a time
    const int lanes = p.dim / 8;      // lanes with channels in a group of GP
    const int l = threadIdx.x % GP, item = threadIdx.x / GP;
    const int heads = min(p.heads, GROUPS);
    const int step = GROUPS / heads;  // rows at a time
    const int hi = item % heads, ri = item / heads;
    const bool on = l < lanes && ri < step;
    // A lane's two runs of four channels, and its first pair.
    const int a_at = SPLIT ? 4 * l : 8 * l, b_at = SPLIT ? half + 4 * l : 8 * l + 4, pair = 4 * l;
    // Two runs as they are in memory; the next two items' are on their way while one is turned.
    using Run = typename std::conditional<DT == kF32, int4, int2>::type;
    struct Item {
        Run a, b;
    } next[2];
    const auto fetch = [&](Item & to, int h, int r) {
        to = Item{};
        if (!on || h >= p.heads || r >= rows) return;
        const T * xr = x + (row0 + r) * p.x_stride + (int64_t) h * p.dim;
        if constexpr (DT != kF32 && !SPLIT) {
            const int4 c = *(const int4 *) (xr + a_at);
            to = Item{int2{c.x, c.y}, int2{c.z, c.w}};
        } else {
            to = Item{*(const Run *) (xr + a_at), *(const Run *) (xr + b_at)};
        }
    };
    fetch(next[0], hi, ri);
    fetch(next[1], hi, ri + step);
    for (int i = threadIdx.x; i < rows * half; i += 256) {
        const int r = i / half, j = i % half;
        float sn = 0.0f, cs = 1.0f;
        if (j < p.total) {
            const int axis = j < p.axis1 ? 1 : (j < p.axis2 ? 2 : 3);
            const double t = (double) coords[(row0 + r) * 4 + axis] * f.turns[j];
            sincospif(2.0f * (float) (t - rint(t)), &sn, &cs);
        }
        s_turn[i] = float2{cs, sn};
    }
    __syncthreads();
    if (ri >= step) return;
    for (int h = hi; h < p.heads; h += heads) {
        float g[8];
        if constexpr (NORM) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                g[u] = on && gamma != nullptr ? gamma[(int64_t) h * p.dim + (u < 4 ? a_at + u : b_at + u - 4)] : 1.0f;
        }
        const auto turn = [&](Item & item, int r) {
            if (r >= rows) return;
            float v[8];
            if constexpr (DT == kF32) {
                unpack_chunk_of<DT>(item.a, v);
                unpack_chunk_of<DT>(item.b, v + 4);
            } else {
                unpack_chunk<DT>(int4{item.a.x, item.a.y, item.b.x, item.b.y}, v);
            }
            fetch(item, h, r + 2 * step);
            if constexpr (NORM) {
                float sum = 0.0f;
#pragma unroll
                for (int u = 0; u < 8; ++u) sum += v[u] * v[u];
                const float inv = 1.0f / sqrtf(group_sum<GP>(sum) / (float) p.dim + p.eps);
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = v[u] * inv * g[u];
            }
            if (on) {
                float o[8];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float2 t = s_turn[r * half + pair + u];
                    const float a = v[SPLIT ? u : 2 * u], b = v[SPLIT ? u + 4 : 2 * u + 1];
                    const float oa = a * t.x - b * t.y, ob = a * t.y + b * t.x;
                    o[SPLIT ? u : 2 * u] = oa;
                    o[SPLIT ? u + 4 : 2 * u + 1] = ob;
                }
                T * yr = y + (row0 + r) * p.y_stride + (int64_t) h * p.dim;
                if constexpr (DT == kF32) {
                    store_chunk<DT>(yr + a_at, o);
                    store_chunk<DT>(yr + b_at, o + 4);
                } else {
                    const int4 c = pack_chunk<DT>(o);
                    if constexpr (SPLIT) {
                        *(int2 *) (yr + a_at) = int2{c.x, c.y};
                        *(int2 *) (yr + b_at) = int2{c.z, c.w};
                    } else {
                        *(int4 *) (yr + a_at) = c;
                    }
                }
            }
        };
        for (int r = ri; r < rows; r += 2 * step) {
            turn(next[0], r);
            turn(next[1], r + step);
        }
        fetch(next[0], h + heads, ri);
        fetch(next[1], h + heads, ri + step);
    }
}

template <int DT>
hipError_t rotary_dt(const void * x, const int32_t * coords, const float * gamma, void * y, RotaryShape p,
                     const RotaryFreq & f, bool norm, bool split, int cus, hipStream_t s) {
    using T = typename Store<DT>::T;
    // Blocks of 16 rows share the sines' latency; with few rows smaller ones fill the CUs.
    p.rows = p.n >= (int64_t) cus * 64 ? 16 : 4;
    const int64_t g = (p.n + p.rows - 1) / p.rows;
    if (g > 0x7fffffffLL) return hipErrorInvalidValue;
    const size_t lds = (size_t) p.rows * (p.dim / 2) * sizeof(float2);
    const auto launch_as = [&](auto gp, auto norm_c, auto split_c) {
        k_rotary<DT, decltype(gp)::value, decltype(norm_c)::value, decltype(split_c)::value>
            <<<(unsigned) g, 256, lds, s>>>((const T *) x, coords, gamma, (T *) y, p, f);
        return hipGetLastError();
    };
    const auto launch = [&](auto gp) {
        using std::bool_constant;
        if (norm) return split ? launch_as(gp, bool_constant<true>(), bool_constant<true>()) : launch_as(gp, bool_constant<true>(), bool_constant<false>());
        return split ? launch_as(gp, bool_constant<false>(), bool_constant<true>()) : launch_as(gp, bool_constant<false>(), bool_constant<false>());
    };
    if (p.dim <= 32) return launch(std::integral_constant<int, 4>());
    if (p.dim <= 64) return launch(std::integral_constant<int, 8>());
    if (p.dim <= 128) return launch(std::integral_constant<int, 16>());
    return launch(std::integral_constant<int, 32>());
}

}  // namespace

hipError_t launch_rms_norm(int dtype, const void * x, const void * residual, const float * gamma, void * total,
                           void * y, int64_t n, int c, float eps, int cus, hipStream_t s) {
    const NormOut out{y, nullptr, nullptr, 0};
    switch (dtype) {
        case kF32: return norm_dt<kF32, false, true>(x, residual, gamma, total, out, n, c, eps, cus, s);
        case kF16: return norm_dt<kF16, false, true>(x, residual, gamma, total, out, n, c, eps, cus, s);
        default: return norm_dt<kBF16, false, true>(x, residual, gamma, total, out, n, c, eps, cus, s);
    }
}

hipError_t launch_rms_norm8(int dtype, const void * x, const void * residual, const float * gamma, void * total,
                            uint8_t * codes, uint8_t * scales, int64_t n, int c, float eps, int cus, hipStream_t s) {
    const NormOut out{nullptr, codes, scales, rows8_width(c)};
    switch (dtype) {
        case kF32: return norm_dt<kF32, true, true>(x, residual, gamma, total, out, n, c, eps, cus, s);
        case kF16: return norm_dt<kF16, true, true>(x, residual, gamma, total, out, n, c, eps, cus, s);
        default: return norm_dt<kBF16, true, true>(x, residual, gamma, total, out, n, c, eps, cus, s);
    }
}

hipError_t launch_pack8(int dtype, const void * x, uint8_t * codes, uint8_t * scales, int64_t n, int c, int cus,
                        hipStream_t s) {
    const NormOut out{nullptr, codes, scales, rows8_width(c)};
    switch (dtype) {
        case kF32: return norm_dt<kF32, true, false>(x, nullptr, nullptr, nullptr, out, n, c, 0.0f, cus, s);
        case kF16: return norm_dt<kF16, true, false>(x, nullptr, nullptr, nullptr, out, n, c, 0.0f, cus, s);
        default: return norm_dt<kBF16, true, false>(x, nullptr, nullptr, nullptr, out, n, c, 0.0f, cus, s);
    }
}

hipError_t launch_expand8(int dtype, const uint8_t * codes, const uint8_t * scales, void * y, int64_t n, int c,
                          hipStream_t s) {
    const int64_t g = (n * ((c + 15) / 16) + 255) / 256;
    if (g > 0x7fffffffLL) return hipErrorInvalidValue;
    const int cp = rows8_width(c);
    const auto launch = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        using T = typename Store<DT>::T;
        if (c % kChunk<DT> == 0) {
            k_expand8<DT, true><<<(unsigned) g, 256, 0, s>>>(codes, scales, (T *) y, n, c, cp);
        } else {
            k_expand8<DT, false><<<(unsigned) g, 256, 0, s>>>(codes, scales, (T *) y, n, c, cp);
        }
        return hipGetLastError();
    };
    switch (dtype) {
        case kF32: return launch(std::integral_constant<int, kF32>());
        case kF16: return launch(std::integral_constant<int, kF16>());
        default: return launch(std::integral_constant<int, kBF16>());
    }
}

hipError_t launch_rotary(int dtype, const void * x, const int32_t * coords, const float * gamma, void * y,
                         const RotaryPlan & plan, int cus, hipStream_t s) {
    RotaryShape p{};
    p.n = plan.n;
    p.x_stride = plan.x_stride;
    p.y_stride = plan.y_stride;
    p.heads = plan.heads;
    p.dim = plan.dim;
    p.axis1 = plan.pairs[0];
    p.axis2 = plan.pairs[0] + plan.pairs[1];
    p.total = p.axis2 + plan.pairs[2];
    p.eps = plan.eps;
    RotaryFreq f;
    int at = 0;
    for (int a = 0; a < 3; ++a)
        for (int j = 0; j < plan.pairs[a]; ++j)
            f.turns[at++] = pow(plan.base, -(double) j / plan.pairs[a]) / (2.0 * M_PI);
    for (; at < kRotaryMaxDim / 2; ++at) f.turns[at] = 0.0;
    switch (dtype) {
        case kF32: return rotary_dt<kF32>(x, coords, gamma, y, p, f, plan.norm, plan.split != 0, cus, s);
        case kF16: return rotary_dt<kF16>(x, coords, gamma, y, p, f, plan.norm, plan.split != 0, cus, s);
        default: return rotary_dt<kBF16>(x, coords, gamma, y, p, f, plan.norm, plan.split != 0, cus, s);
    }
}

}  // namespace tsh
