// kernels_rows.hip - row operators of transformer blocks over voxel rows: RMS norm, 8-bit rows, rotary positions.
#include "tsh_internal.h"

namespace tsh {
namespace {

// ---- chunks of 16 bytes -------------------------------------------------------------------------

// Values per 16-byte chunk.
template <int DT> constexpr int kChunk = DT == kF32 ? 4 : 8;

template <int DT> __device__ __forceinline__ void load_chunk(const typename Store<DT>::T * p, float * v) {
    if constexpr (DT == kF32) {
        const float4 c = *(const float4 *) p;
        v[0] = c.x;
        v[1] = c.y;
        v[2] = c.z;
        v[3] = c.w;
    } else {
        unpack_chunk<DT>(*(const int4 *) p, v);
    }
}

template <int DT> __device__ __forceinline__ void store_chunk(typename Store<DT>::T * p, const float * v) {
    if constexpr (DT == kF32) {
        *(float4 *) p = float4{v[0], v[1], v[2], v[3]};
    } else {
        *(int4 *) p = pack_chunk<DT>(v);
    }
}

// Sum over groups of G lanes (G a power of two, groups aligned), left in each of them.
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ float wave_sum(float v) { return group_sum<64>(v); }

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

template <int G> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
        const uint32_t o = (uint32_t) __shfl_xor((int) v, d);
        v = o > v ? o : v;
    }
    return v;
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
// registers, CPL chunks of 16 bytes each, and keep gamma from row to row.
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
    for (int64_t row = (int64_t) blockIdx.x * RPB + threadIdx.x / LPR; row < n; row += (int64_t) gridDim.x * RPB) {
        float v[CPL][V];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int at = (i * LPR + l) * V;
            if (at < c) {
                load_chunk<DT>(x + row * c + at, v[i]);
            } else {
#pragma unroll
                for (int u = 0; u < V; ++u) v[i][u] = 0.0f;
            }
        }
        if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int at = (i * LPR + l) * V;
                if (at < c) {
                    float r[V];
                    load_chunk<DT>(residual + row * c + at, r);
#pragma unroll
                    for (int u = 0; u < V; ++u) v[i][u] += r[u];
                }
            }
        }
        if (total != nullptr) {
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int at = (i * LPR + l) * V;
                if (at < c) store_chunk<DT>(total + row * c + at, v[i]);
            }
        }
        if constexpr (NORM) {
#pragma unroll
            for (int i = 0; i < CPL; ++i)
#pragma unroll
                for (int u = 0; u < V; ++u) sum += v[i][u] * v[i][u];
            const float inv = 1.0f / sqrtf(group_sum<LPR>(sum) / (float) c + eps);
#pragma unroll
            for (int i = 0; i < CPL; ++i)
#pragma unroll
                for (int u = 0; u < V; ++u) v[i][u] = v[i][u] * inv * g[i][u];
        }
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int at = (i * LPR + l) * V;
            if constexpr (Q8) {
                // The 32 / V lanes of a block are neighbours.
                uint32_t m = 0;
#pragma unroll
                for (int u = 0; u < V; ++u) m = max(m, at < c ? abs_bits(v[i][u]) : 0u);
                const uint32_t scale = block_scale(group_max<32 / V>(m));
                const float inv = inverse_scale(scale);
                if (at < out.cp) {
                    float z[V];
#pragma unroll
                    for (int u = 0; u < V; ++u) z[u] = at < c ? v[i][u] : 0.0f;
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
// whole number of chunks, or beyond what a wavefront holds in registers).
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
    float inv = 1.0f;
    if constexpr (NORM) {
        float sum = 0.0f;
        for (int i = lane; i < c; i += 64) {
            const float v = at(i);
            sum += v * v;
        }
        inv = 1.0f / sqrtf(wave_sum(sum) / (float) c + eps);
    }
    const int end = Q8 ? out.cp : c;
    for (int i = lane; i < end; i += 64) {
        float v = 0.0f;
        if (i < c) {
            const float s = at(i);
            // An element of total may be the same memory as that of x or residual: read first.
            if (total != nullptr) Store<DT>::st(total, row * c + i, s);
            v = s;
            if constexpr (NORM) v = v * inv * (gamma != nullptr ? gamma[i] : 1.0f);
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

// The values that 8-bit rows stand for, 4 per thread (cp is a multiple of 128).
template <int DT>
__global__ void __launch_bounds__(256) k_expand8(const uint8_t * __restrict__ codes, const uint8_t * __restrict__ scales,
                                                 typename Store<DT>::T * __restrict__ y, int64_t n, int c, int cp) {
    const int quads = (c + 3) / 4;
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= n * quads) return;
    const int64_t row = i / quads;
    const int at = (int) (i % quads) * 4;
    const int w = *(const int *) (codes + row * cp + at);
    const uint32_t byte = scales[row * (cp / 32) + at / 32];
    const float scale = byte == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, byte << 23);
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    const float v[4] = {lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (at + u < c) Store<DT>::st(y, row * c + at + u, v[u]);
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
        const int64_t g = std::min<int64_t>((n + RPB - 1) / RPB, (int64_t) cus * 8);
        k_norm_vec<DT, LPR, CPL, Q8, NORM><<<(unsigned) g, 256, 0, s>>>((const T *) x, (const T *) residual, gamma,
                                                                        (T *) total, out, n, c, eps);
        return hipGetLastError();
    };
    using std::integral_constant;
    if (chunks <= 8) return launch(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (chunks <= 16) return launch(integral_constant<int, 16>(), integral_constant<int, 1>());
    if (chunks <= 32) return launch(integral_constant<int, 32>(), integral_constant<int, 1>());
    if (chunks <= 64) return launch(integral_constant<int, 64>(), integral_constant<int, 1>());
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
// each over all rows, gamma in registers.
struct RotaryShape {
    int64_t n, x_stride, y_stride;
    int heads, dim, split, total;  // total: turned pairs
    int axis1, axis2;              // first pair of the y and z axes
    float eps;
    int rows;                      // rows per block
};
struct RotaryFreq {
    double turns[kRotaryMaxDim / 2];  // freq / 2 pi per pair
};

template <int DT, int GP, bool NORM>
__global__ void __launch_bounds__(256) k_rotary(const typename Store<DT>::T * x, const int32_t * __restrict__ coords,
                                                const float * __restrict__ gamma, typename Store<DT>::T * y,
                                                RotaryShape p, RotaryFreq f) {
    using T = typename Store<DT>::T;
    extern __shared__ float2 s_turn[];  // [rows][dim / 2]: cosine, sine
    const int64_t row0 = (int64_t) blockIdx.x * p.rows;
    const int rows = (int) min((int64_t) p.rows, p.n - row0);
    const int half = p.dim / 2;
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

    constexpr int GROUPS = 256 / GP;  // (row, head) items at a time
    const int lanes = p.dim / 8;      // lanes with channels in a group of GP
    const int l = threadIdx.x % GP, item = threadIdx.x / GP;
    const int heads = min(p.heads, GROUPS);
    const int step = GROUPS / heads;  // rows at a time
    const int hi = item % heads, ri = item / heads;
    if (ri >= step) return;
    const bool on = l < lanes;
    // A lane's two runs of four channels, and its first pair.
    const int a_at = p.split ? 4 * l : 8 * l, b_at = p.split ? half + 4 * l : 8 * l + 4, pair = 4 * l;
    for (int h = hi; h < p.heads; h += heads) {
        float g[8];
        if constexpr (NORM) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                g[u] = on && gamma != nullptr ? gamma[(int64_t) h * p.dim + (u < 4 ? a_at + u : b_at + u - 4)] : 1.0f;
        }
        for (int r = ri; r < rows; r += step) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            const T * xr = x + (row0 + r) * p.x_stride + (int64_t) h * p.dim;
            if (on) {
                if constexpr (DT == kF32) {
                    load_chunk<DT>(xr + a_at, v);
                    load_chunk<DT>(xr + b_at, v + 4);
                } else if (p.split) {
                    const int2 a = *(const int2 *) (xr + a_at), b = *(const int2 *) (xr + b_at);
                    unpack_chunk<DT>(int4{a.x, a.y, b.x, b.y}, v);
                } else {
                    load_chunk<DT>(xr + a_at, v);
                }
            }
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
                    const float a = p.split ? v[u] : v[2 * u], b = p.split ? v[u + 4] : v[2 * u + 1];
                    const float oa = a * t.x - b * t.y, ob = a * t.y + b * t.x;
                    if (p.split) {
                        o[u] = oa;
                        o[u + 4] = ob;
                    } else {
                        o[2 * u] = oa;
                        o[2 * u + 1] = ob;
                    }
                }
                T * yr = y + (row0 + r) * p.y_stride + (int64_t) h * p.dim;
                if constexpr (DT == kF32) {
                    store_chunk<DT>(yr + a_at, o);
                    store_chunk<DT>(yr + b_at, o + 4);
                } else {
                    const int4 c = pack_chunk<DT>(o);
                    if (p.split) {
                        *(int2 *) (yr + a_at) = int2{c.x, c.y};
                        *(int2 *) (yr + b_at) = int2{c.z, c.w};
                    } else {
                        *(int4 *) (yr + a_at) = c;
                    }
                }
            }
        }
    }
}

template <int DT>
hipError_t rotary_dt(const void * x, const int32_t * coords, const float * gamma, void * y, RotaryShape p,
                     const RotaryFreq & f, bool norm, int cus, hipStream_t s) {
    using T = typename Store<DT>::T;
    // Blocks of 16 rows share the sines' latency; with few rows smaller ones fill the CUs.
    p.rows = p.n >= (int64_t) cus * 64 ? 16 : 4;
    const int64_t g = (p.n + p.rows - 1) / p.rows;
    if (g > 0x7fffffffLL) return hipErrorInvalidValue;
    const size_t lds = (size_t) p.rows * (p.dim / 2) * sizeof(float2);
    const auto launch = [&](auto gp) {
        constexpr int GP = decltype(gp)::value;
        if (norm) {
            k_rotary<DT, GP, true><<<(unsigned) g, 256, lds, s>>>((const T *) x, coords, gamma, (T *) y, p, f);
        } else {
            k_rotary<DT, GP, false><<<(unsigned) g, 256, lds, s>>>((const T *) x, coords, gamma, (T *) y, p, f);
        }
        return hipGetLastError();
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
    const int64_t g = (n * ((c + 3) / 4) + 255) / 256;
    if (g > 0x7fffffffLL) return hipErrorInvalidValue;
    const int cp = rows8_width(c);
    switch (dtype) {
        case kF32: k_expand8<kF32><<<(unsigned) g, 256, 0, s>>>(codes, scales, (float *) y, n, c, cp); break;
        case kF16: k_expand8<kF16><<<(unsigned) g, 256, 0, s>>>(codes, scales, (_Float16 *) y, n, c, cp); break;
        default: k_expand8<kBF16><<<(unsigned) g, 256, 0, s>>>(codes, scales, (uint16_t *) y, n, c, cp); break;
    }
    return hipGetLastError();
}

hipError_t launch_rotary(int dtype, const void * x, const int32_t * coords, const float * gamma, void * y,
                         const RotaryPlan & plan, int cus, hipStream_t s) {
    RotaryShape p{};
    p.n = plan.n;
    p.x_stride = plan.x_stride;
    p.y_stride = plan.y_stride;
    p.heads = plan.heads;
    p.dim = plan.dim;
    p.split = plan.split;
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
        case kF32: return rotary_dt<kF32>(x, coords, gamma, y, p, f, plan.norm, cus, s);
        case kF16: return rotary_dt<kF16>(x, coords, gamma, y, p, f, plan.norm, cus, s);
        default: return rotary_dt<kBF16>(x, coords, gamma, y, p, f, plan.norm, cus, s);
    }
}

}  // namespace tsh
