// kernels_gnorm.hip - group norm over the rows of each sequence, channels last, with the activation that follows.
#include <type_traits>

#include "rows_common.h"

namespace tsh {
namespace {

// A group's mean m and the inverse of its root variance; the mean in two parts, so that
// x - m keeps its digits where the mean is far larger than the deviations.
struct GroupStat {
    float mean, mean_low, inverse, pad;
};

// Sums over a group are of d = x - k and d^2 in 64 bits, k the group's first value in its
// sequence: as k is one of them, (k - m)^2 is at most as many variances as there are
// values, and var = mean d^2 - (mean d)^2 loses no more than that many of 2^53.
struct GroupSum {
    double d, d2;
};
__device__ __forceinline__ void add_value(GroupSum & s, float x, float k) {
    const double d = (double) x - (double) k;
    s.d += d;
    s.d2 = fma(d, d, s.d2);
}
__device__ __forceinline__ GroupStat stat_of(const GroupSum & s, double count, float k, float eps) {
    const double off = s.d / count, var = s.d2 / count - off * off;
    const double mean = (double) k + off;
    const float hi = (float) mean;
    const double low = mean - (double) hi;
    // (A NaN stays one; a negative variance is a rounding of zero.)
    return {hi, hi - hi == 0.0f ? (float) low : 0.0f, (float) (1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double) eps)), 0.0f};
}

__device__ __forceinline__ float gn_act(float v, int act) {
    if (act == TRELLIS_SPARSE_HIP_ACT_SILU) return v / (1.0f + expf(-v));
    if (act == TRELLIS_SPARSE_HIP_ACT_GELU) return 0.5f * v * erfcf(-0.70710678f * v);
    if (act == TRELLIS_SPARSE_HIP_ACT_GELU_TANH)
        return v / (1.0f + expf(-v * (1.5957691216057308f + 0.0713548162726f * v * v)));
    return v;
}

__device__ __forceinline__ int64_t row_of(const int32_t * at, int i, int64_t n) {
    const int64_t v = at[i];
    return v < 0 ? 0 : (v > n ? n : v);
}

// Any sizes: a block per sequence and group, which reads its values twice.
template <int DT> __global__ void __launch_bounds__(256) k_group_norm(GroupNorm p) {
    using T = typename Store<DT>::T;
    __shared__ GroupSum s_sum[4];
    const int seq = blockIdx.x / p.groups, g = blockIdx.x % p.groups, size = p.c / p.groups;
    const int64_t first = p.at != nullptr ? row_of(p.at, seq, p.n) : 0;
    const int64_t end = p.at != nullptr ? row_of(p.at, seq + 1, p.n) : p.n;
    if (end <= first) return;
    const T * x = (const T *) p.x + first * p.c + g * size;
    T * y = (T *) p.y + first * p.c + g * size;
    // Lanes on neighbouring channels, then rows.
    int wide = 1;
    while (wide < size && wide < 256) wide *= 2;
    const int ch0 = threadIdx.x % wide, r0 = threadIdx.x / wide, step = 256 / wide;
    const float k = Store<DT>::ld(x, 0);
    GroupSum s{0.0, 0.0};
    for (int64_t r = r0; r < end - first; r += step)
        for (int ch = ch0; ch < size; ch += wide) add_value(s, Store<DT>::ld(x, r * p.c + ch), k);
    s.d = group_sum<64>(s.d);
    s.d2 = group_sum<64>(s.d2);
    if (threadIdx.x % 64 == 0) s_sum[threadIdx.x / 64] = s;
    __syncthreads();
    s = s_sum[0];
    for (int i = 1; i < 4; ++i) {
        s.d += s_sum[i].d;
        s.d2 += s_sum[i].d2;
    }
    const GroupStat st = stat_of(s, (double) (end - first) * size, k, p.eps);
    for (int ch = ch0; ch < size; ch += wide) {
        const float scale = st.inverse * (p.gamma != nullptr ? p.gamma[g * size + ch] : 1.0f);
        const float shift = p.beta != nullptr ? p.beta[g * size + ch] : 0.0f;
        for (int64_t r = r0; r < end - first; r += step) {
            const float v = (Store<DT>::ld(x, r * p.c + ch) - st.mean - st.mean_low) * scale + shift;
            Store<DT>::st(y, r * p.c + ch, gn_act(v, p.act));
        }
    }
}

}  // namespace

hipError_t launch_group_norm(int dtype, const GroupNorm & p, hipStream_t s) {
    const int64_t grid = (int64_t) p.seqs * p.groups;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    switch (dtype) {
        case kF32: k_group_norm<kF32><<<(unsigned) grid, 256, 0, s>>>(p); break;
        case kF16: k_group_norm<kF16><<<(unsigned) grid, 256, 0, s>>>(p); break;
        default: k_group_norm<kBF16><<<(unsigned) grid, 256, 0, s>>>(p); break;
    }
    return hipGetLastError();
}

}  // namespace tsh
