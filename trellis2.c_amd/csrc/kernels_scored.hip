// kernels_scored.hip - attention whose scores are capped by a tanh, lowered by a distance, or masked:
// out_i = sum_j softmax_j(cap tanh(scale q_i . k_j / cap) - slope d(i, j)) v_j over the keys that i sees.
#include "attn_common.h"

namespace tsh {
namespace {

// Any head width and alignment, fp32 arithmetic, as k_attention_any: 16 queries of one
// head a block, keys in tiles of 32 as fp32 in LDS.
template <int DT> __global__ void __launch_bounds__(256) k_scored_any(Attention p, Scores sc) {
    using T = typename Store<DT>::T;
    constexpr int TQ = 16, TK = 32;
    extern __shared__ float s_mem[];
    const int pitch = p.dim + 1;
    float * s_q = s_mem;                 // [TQ][pitch]
    float * s_k = s_q + TQ * pitch;      // [TK][pitch]
    float * s_v = s_k + TK * pitch;      // [TK][pitch]
    float * s_p = s_v + TK * pitch;      // [TQ][TK + 1], -1 where the query does not see the key
    const int head = blockIdx.x % p.heads;
    const Place at = find_place<TQ>(p, blockIdx.x / p.heads, 1);
    if (at.nq <= 0) return;
    const int kv = head / (p.heads / p.kv_heads);
    const T * q = (const T *) p.q + (int64_t) head * p.dim;
    const T * k = (const T *) p.k + (int64_t) kv * p.dim;
    const T * v = (const T *) p.v + (int64_t) kv * p.dim;
    const int t = threadIdx.x, row = t / 16, l = t % 16;
    for (int i = t; i < TQ * p.dim; i += 256) {
        const int r = i / p.dim, c = i % p.dim;
        s_q[r * pitch + c] = r < at.nq ? Store<DT>::ld(q, (at.q0 + at.first + r) * p.q_stride + c) : 0.0f;
    }
    // The query's place among the keys, and the keys that it sees.
    const int64_t place = at.first + row + at.nk - at.rows;
    const int64_t prefix = sc.prefix != nullptr ? sc.prefix[at.seq] : 0;
    const auto sees = [&](int64_t j) { return sc.causal == 0 || j <= place || j < prefix; };
    const int seen = (int) keys_seen(at, sc, at.first + at.nq - 1);
    const float slope = sc.slopes != nullptr ? sc.slopes[head] * 1.44269504f : 0.0f;
    int3 here{0, 0, 0};
    if (sc.q_xyz != nullptr && row < at.nq) here = voxel_of(sc.q_xyz, at.q0 + at.first + row);
    const auto score = [&](float dot, int j) {
        float s = dot * p.scale;
        if (sc.cap > 0.0f) s = sc.cap * tanhf(dot * sc.cap_scale);
        if (sc.slopes != nullptr && j < at.nk) {
            const float d = sc.q_xyz != nullptr ? distance_of(here, voxel_of(sc.k_xyz, at.k0 + j)) : fabsf((float) (place - j));
            s -= slope * d;
        }
        return s;
    };
    float most = -__builtin_inff(), sum = 0.0f;
    float acc[kAttentionMaxDim / 16];
#pragma unroll
    for (int u = 0; u < kAttentionMaxDim / 16; ++u) acc[u] = 0.0f;
    for (int j0 = 0; j0 < seen; j0 += TK) {
        const int keys = min(TK, at.nk - j0);
        __syncthreads();
        for (int i = t; i < TK * p.dim; i += 256) {
            const int r = i / p.dim, c = i % p.dim;
            const int64_t key = at.k0 + j0 + r;
            s_k[r * pitch + c] = r < keys ? Store<DT>::ld(k, key * p.k_stride + c) : 0.0f;
            s_v[r * pitch + c] = r < keys ? Store<DT>::ld(v, key * p.v_stride + c) : 0.0f;
        }
        __syncthreads();
        // Lane l of a row's 16 has keys l and l + 16.
        float s0 = 0.0f, s1 = 0.0f;
        for (int c = 0; c < p.dim; ++c) {
            const float a = s_q[row * pitch + c];
            s0 = fmaf(a, s_k[l * pitch + c], s0);
            s1 = fmaf(a, s_k[(l + 16) * pitch + c], s1);
        }
        const bool see0 = l < keys && sees(j0 + l), see1 = l + 16 < keys && sees(j0 + l + 16);
        s0 = see0 ? score(s0, j0 + l) : -__builtin_inff();
        s1 = see1 ? score(s1, j0 + l + 16) : -__builtin_inff();
        float m = fmaxf(s0, s1);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        m = fmaxf(m, most);
        const float base = m == -__builtin_inff() ? 0.0f : m;
        const float keep = exp2f(most - base);
        const float p0 = exp2f(s0 - base), p1 = exp2f(s1 - base);
        most = m;
        sum = sum * keep + row16_sum(p0 + p1);
        s_p[row * (TK + 1) + l] = see0 ? p0 : -1.0f;
        s_p[row * (TK + 1) + l + 16] = see1 ? p1 : -1.0f;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kAttentionMaxDim / 16; ++u) {
            const int c = u * 16 + l;
            if (c >= p.dim) break;
            float a = acc[u] * keep;
            for (int j = 0; j < keys; ++j) {
                const float w = s_p[row * (TK + 1) + j];
                if (!(w < 0.0f)) a = fmaf(w, s_v[j * pitch + c], a);
            }
            acc[u] = a;
        }
    }
    if (row < at.nq) {
        // No keys (or none above -inf): zeros.
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T * y = (T *) p.y + (at.q0 + at.first + row) * p.y_stride + (int64_t) head * p.dim;
#pragma unroll
        for (int u = 0; u < kAttentionMaxDim / 16; ++u) {
            const int c = u * 16 + l;
            if (c < p.dim) Store<DT>::st(y, c, acc[u] * inv);
        }
    }
}

template <int DT> hipError_t launch_any(const Attention & p, const Scores & sc, hipStream_t s) {
    const int64_t tiles = p.nq / 16 + (p.q_at != nullptr ? p.seqs : 1);
    const int64_t grid = tiles * p.heads;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    const size_t lds = ((size_t) (16 + 32 + 32) * (p.dim + 1) + 16 * 33) * sizeof(float);
    k_scored_any<DT><<<(unsigned) grid, 256, lds, s>>>(p, sc);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_scored(int dtype, const Attention & p, const Scores & sc, hipStream_t s) {
    switch (dtype) {
        case kF32: return launch_any<kF32>(p, sc, s);
        case kF16: return launch_any<kF16>(p, sc, s);
        default: return launch_any<kBF16>(p, sc, s);
    }
}

}  // namespace tsh
