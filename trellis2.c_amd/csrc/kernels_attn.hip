// kernels_attn.hip - attention within sequences of rows: out_i = sum_j softmax_j(scale q_i . k_j) v_j.
#include "mfma_common.h"

namespace tsh {
namespace {

// A block's place: rows [q0, q0 + nq) of one sequence's queries, keys [k0, k0 + nk).
struct Place {
    int64_t q0, k0;
    int nq, nk;
};

__device__ __forceinline__ int64_t offset_of(const int32_t * at, int i, int64_t n) {
    const int64_t v = at[i];
    return v < 0 ? 0 : (v > n ? n : v);
}

// Tile `tile` of TQ queries among all sequences' tiles, in order; nq = 0 past
// the last.  Offsets are read on the device, so a grid has an upper bound of
// tiles; they are clamped to the rows that there are, and a sequence whose
// offsets fall is empty.
template <int TQ> __device__ Place find_place(const Attention & p, int64_t tile) {
    Place r{0, 0, 0, 0};
    if (p.q_at == nullptr) {
        r.q0 = tile * TQ;
        r.nq = (int) max((int64_t) 0, min((int64_t) TQ, p.nq - r.q0));
        r.nk = (int) p.nk;
        return r;
    }
    // 64 sequences at a time: an inclusive scan of their tile counts, then the first that reaches past `tile`.
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < p.seqs; s0 += 64) {
        const int i = s0 + lane;
        int64_t lo = 0, len = 0;
        if (i < p.seqs) {
            lo = offset_of(p.q_at, i, p.nq);
            len = max((int64_t) 0, offset_of(p.q_at, i + 1, p.nq) - lo);
        }
        int64_t sum = (len + TQ - 1) / TQ;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const unsigned long long past = __ballot(sum > tile);
        if (past != 0) {
            const int at = __ffsll(past) - 1;
            const int64_t tiles = (len + TQ - 1) / TQ;
            const int64_t in = tile - __shfl(sum - tiles, at);
            const int seq = s0 + at;
            r.q0 = __shfl(lo, at) + in * TQ;
            r.nq = (int) min((int64_t) TQ, __shfl(len, at) - in * TQ);
            r.k0 = offset_of(p.k_at, seq, p.nk);
            r.nk = (int) max((int64_t) 0, offset_of(p.k_at, seq + 1, p.nk) - r.k0);
            return r;
        }
        tile -= __shfl(sum, 63);
    }
    return r;
}

// Any head width and alignment, fp32 arithmetic: 16 queries of one head a
// block, keys in tiles of 32 as fp32 in LDS; the running maximum and sum of
// each query's softmax rescale its output as the maximum grows.
template <int DT> __global__ void __launch_bounds__(256) k_attention_any(Attention p) {
    using T = typename Store<DT>::T;
    constexpr int TQ = 16, TK = 32;
    extern __shared__ float s_mem[];
    const int pitch = p.dim + 1;
    float * s_q = s_mem;                 // [TQ][pitch]
    float * s_k = s_q + TQ * pitch;      // [TK][pitch]
    float * s_v = s_k + TK * pitch;      // [TK][pitch]
    float * s_p = s_v + TK * pitch;      // [TQ][TK + 1]
    const int head = blockIdx.x % p.heads;
    const Place at = find_place<TQ>(p, blockIdx.x / p.heads);
    if (at.nq <= 0) return;
    const int kv = head / (p.heads / p.kv_heads);
    const T * q = (const T *) p.q + (int64_t) head * p.dim;
    const T * k = (const T *) p.k + (int64_t) kv * p.dim;
    const T * v = (const T *) p.v + (int64_t) kv * p.dim;
    const int t = threadIdx.x, row = t / 16, l = t % 16;
    for (int i = t; i < TQ * p.dim; i += 256) {
        const int r = i / p.dim, c = i % p.dim;
        s_q[r * pitch + c] = r < at.nq ? Store<DT>::ld(q, (at.q0 + r) * p.q_stride + c) : 0.0f;
    }
    float most = -__builtin_inff(), sum = 0.0f;
    float acc[kAttentionMaxDim / 16];
#pragma unroll
    for (int u = 0; u < kAttentionMaxDim / 16; ++u) acc[u] = 0.0f;
    for (int j0 = 0; j0 < at.nk; j0 += TK) {
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
        s0 = l < keys ? s0 * p.scale : -__builtin_inff();
        s1 = l + 16 < keys ? s1 * p.scale : -__builtin_inff();
        float m = fmaxf(s0, s1);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        m = fmaxf(m, most);
        const float base = m == -__builtin_inff() ? 0.0f : m;
        const float keep = exp2f(most - base);
        const float p0 = exp2f(s0 - base), p1 = exp2f(s1 - base);
        most = m;
        sum = sum * keep + row16_sum(p0 + p1);
        s_p[row * (TK + 1) + l] = p0;
        s_p[row * (TK + 1) + l + 16] = p1;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kAttentionMaxDim / 16; ++u) {
            const int c = u * 16 + l;
            if (c >= p.dim) break;
            float a = acc[u] * keep;
            for (int j = 0; j < keys; ++j) a = fmaf(s_p[row * (TK + 1) + j], s_v[j * pitch + c], a);
            acc[u] = a;
        }
    }
    if (row < at.nq) {
        // No keys (or none above -inf): zeros.
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T * y = (T *) p.y + (at.q0 + row) * p.y_stride + (int64_t) head * p.dim;
#pragma unroll
        for (int u = 0; u < kAttentionMaxDim / 16; ++u) {
            const int c = u * 16 + l;
            if (c < p.dim) Store<DT>::st(y, c, acc[u] * inv);
        }
    }
}

template <int DT> hipError_t launch_any(const Attention & p, hipStream_t s) {
    // Every sequence may add one partly filled tile.
    const int64_t tiles = p.nq / 16 + (p.q_at != nullptr ? p.seqs : 1);
    const int64_t grid = tiles * p.heads;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    const size_t lds = ((size_t) (16 + 32 + 32) * (p.dim + 1) + 16 * 33) * sizeof(float);
    k_attention_any<DT><<<(unsigned) grid, 256, lds, s>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(int dtype, const Attention & p, hipStream_t s) {
    switch (dtype) {
        case kF32: return launch_any<kF32>(p, s);
        case kF16: return launch_any<kF16>(p, s);
        default: return launch_any<kBF16>(p, s);
    }
}

}  // namespace tsh
