// attn_common.h - what the attention kernels share: their queries' places, products on the matrix unit, outputs and the
// join of split keys.
#pragma once
#include "mfma_common.h"

namespace tsh {
namespace {

// A block's place: nq queries from `first` of sequence `seq`, whose `rows` rows begin at q0, its keys [k0, k0 + nk).
struct Place {
    int64_t q0, first, k0;
    int nq, nk;
    int64_t rows;
    int seq;
};

// The same value in every lane, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t) (((uint64_t) (uint32_t) uniform((int) (v >> 32)) << 32) | (uint32_t) uniform((int) v));
}

__device__ __forceinline__ int64_t offset_of(const int32_t * at, int i, int64_t n) {
    const int64_t v = at[i];
    return v < 0 ? 0 : (v > n ? n : v);
}

// Tile `tile` of TQ queries among all sequences' tiles, in order; nq = 0 where
// there is none.  A query is a row and one of the `group` heads that share a kv
// head: query i of a sequence is its row i / group, head i % group of them.
// Offsets are read on the device, so tiles are numbered by what holds for any
// lengths: sequence s, whose queries begin at a, has its tiles from a / TQ + s
// on, and never reaches past the next one's first.  They are clamped to the rows
// that there are, and a sequence whose offsets fall is empty.  The sequence is
// found 64 offsets at a time: 18,216 rows in 2,024 sequences of 9, 8 heads of 64,
// took 284 us with all sequences counted up to the tile, 89 so.
template <int TQ> __device__ Place find_place(const Attention & p, int64_t tile, int group) {
    Place r{0, 0, 0, 0, 0, 0, 0};
    if (p.q_at == nullptr) {
        r.first = tile * TQ;
        r.nq = (int) max((int64_t) 0, min((int64_t) TQ, p.nq * group - r.first));
        r.nk = (int) p.nk;
        r.rows = p.nq;
        return r;
    }
    const int lane = threadIdx.x & 63;
    const auto first_tile = [&](int s) { return offset_of(p.q_at, s, p.nq) * group / TQ + s; };
    // The last sequence of [seq, seq + many) whose tiles begin at or before `tile`.
    int seq = 0, many = p.seqs;
    while (many > 1) {
        const int step = (many + 63) / 64, i = lane * step;
        const unsigned long long before = __ballot(i < many && first_tile(seq + i) <= tile);
        if (before == 0) return r;
        const int at = 63 - __clzll(before);
        seq += at * step;
        many = min(step, many - at * step);
    }
    r.q0 = uniform(offset_of(p.q_at, seq, p.nq));
    r.first = (tile - (r.q0 * group / TQ + seq)) * TQ;
    r.seq = seq;
    r.rows = uniform(offset_of(p.q_at, seq + 1, p.nq)) - r.q0;
    const int64_t left = r.rows * group - r.first;
    if (r.first < 0 || left <= 0) return r;
    r.nq = (int) min((int64_t) TQ, left);
    r.k0 = uniform(offset_of(p.k_at, seq, p.nk));
    r.nk = (int) max((int64_t) 0, uniform(offset_of(p.k_at, seq + 1, p.nk)) - r.k0);
    return r;
}

// How many of its sequence's keys row `row` of a place sees: all, or those up to its own
// place (the last row's is the last key's) and the prefix.
__device__ __forceinline__ int64_t keys_seen(const Place & at, const Scores & sc, int64_t row) {
    if (sc.causal == 0) return at.nk;
    const int64_t prefix = sc.prefix != nullptr ? sc.prefix[at.seq] : 0;
    return max((int64_t) 0, min((int64_t) at.nk, max(row + 1 + at.nk - at.rows, prefix)));
}

__device__ __forceinline__ int3 voxel_of(const int32_t * xyz, int64_t row) {
    const int4 c = *(const int4 *) (xyz + row * 4);
    return {c.y, c.z, c.w};
}
__device__ __forceinline__ float distance_of(const int3 & a, const int3 & b) {
    const float x = (float) (a.x - b.x), y = (float) (a.y - b.y), z = (float) (a.z - b.z);
    return sqrtf(fmaf(x, x, fmaf(y, y, z * z)));
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT> __device__ __forceinline__ f32x16 mac32(s16x8 a, s16x8 b, f32x16 c) {
    using V = typename Mfma<DT>::V;
    if constexpr (DT == kBF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
}

// Weights e >= 0 as two each of the storage type: e cut, and what is left, rounded.  The
// second is above zero wherever the first is, so that an infinite value's products agree.
template <int DT> __device__ __forceinline__ void two_parts(const float * e, s16x8 & w, s16x8 & rest) {
    if constexpr (DT == kBF16) {
        union {
            uint32_t c[4];
            s16x8 v;
        } cut;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint32_t b0 = __builtin_bit_cast(uint32_t, e[i]), b1 = __builtin_bit_cast(uint32_t, e[i + 1]);
            cut.c[i / 2] = __builtin_amdgcn_perm(b1, b0, 0x07060302);  // the upper halves
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // A step of fp32 more than what is left.
                const float h = __builtin_bit_cast(float, (j == 0 ? b0 : b1) & 0xffff0000u);
                rest[i + j] = __builtin_bit_cast(short, round_to_store<DT>(fmaf(e[i + j], 1.00000012f, -h)));
            }
        }
        w = cut.v;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const auto cut = __builtin_amdgcn_cvt_pkrtz(e[i], e[i + 1]);
            const f16x2 left{(_Float16) (e[i] - (float) cut[0]), (_Float16) (e[i + 1] - (float) cut[1])};
            const u16x2 h = __builtin_bit_cast(u16x2, cut);
            const u16x2 l = __builtin_elementwise_max(__builtin_bit_cast(u16x2, left),
                                                      __builtin_elementwise_min(h, u16x2{1, 1}));  // 2^-24 at least
            w[i] = (short) h[0];
            w[i + 1] = (short) h[1];
            rest[i] = (short) l[0];
            rest[i + 1] = (short) l[1];
        }
    }
}

__device__ __forceinline__ float max_halves(float v) {
    float a, b;
    both_halves(v, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_halves(float v) {
    float a, b;
    both_halves(v, a, b);
    return a + b;
}

// Where the keys are split over blocks: each split's reference, sum and
// unnormalised output of every query (row * heads + head), joined by k_join.
// (Sums and outputs of all splits are lifted alike.)
struct Partial {
    float * out;   // [splits][nq * heads][dim]
    float2 * stat; // [splits][nq * heads]: maximum (log2 units), sum
    int splits;
};

// Lane (query, half) leaves channels d * 32 + 8 i + 4 half + 0 .. 3: of its split, at place
// at_q() of part, or of y.
template <int DT, int N, class At>
__device__ __forceinline__ void leave_at(const Attention & p, const Partial & part, const f32x16 (&out)[N], float ref,
                                         float sum, bool live, bool some, At && place, int64_t row, int head, int half) {
    using T = typename Store<DT>::T;
    if (!live) return;
    if (part.splits > 1) {
        const int64_t at_q = place();
        if (half == 0) part.stat[at_q] = float2{ref, sum};
        if (!some) return;
        float * o = part.out + at_q * p.dim;
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = d * 32 + i * 8 + half * 4;
                if (c < p.dim)
                    *(float4 *) (o + c) = float4{out[d][4 * i], out[d][4 * i + 1], out[d][4 * i + 2], out[d][4 * i + 3]};
            }
        return;
    }
    // No keys (or none above -inf): zeros.
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T * y = (T *) p.y + row * p.y_stride + (int64_t) head * p.dim;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = d * 32 + i * 8 + half * 4;
            struct alignas(4 * sizeof(T)) {
                T h[4];
            } w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w.h[j] = round_to_store<DT>(out[d][4 * i + j] * inv);
            if (c < p.dim) *(decltype(w) *) (y + c) = w;
        }
}

template <int DT, int N>
__device__ __forceinline__ void leave(const Attention & p, const Partial & part, const f32x16 (&out)[N], float ref,
                                      float sum, bool live, bool some, int split, int64_t row, int head, int half) {
    const auto place = [&] { return ((int64_t) split * p.nq + row) * p.heads + head; };
    leave_at<DT>(p, part, out, ref, sum, live, some, place, row, head, half);
}

// The splits of a query, at places q + split * step of part, joined by WAVES wavefronts (see k_join).
template <int DT, int WAVES>
__device__ __forceinline__ void join_query(const Attention & p, const Partial & part, int qp, int64_t q, int64_t step,
                                           int64_t row, int head, float (&s_sum)[WAVES > 4 ? WAVES : 4][64][5]) {
    using T = typename Store<DT>::T;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float most = -__builtin_inff();
    for (int s = lane; s < part.splits; s += 64) most = fmaxf(most, part.stat[s * step + q].x);
    most = group_reduce<64>(most, [](float a, float b) { return fmaxf(a, b); });
    const float base = most == -__builtin_inff() ? 0.0f : most;
    const int c = lane % qp * 4;
    float sum = 0.0f, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.dim) {
#pragma unroll 4
        for (int s = (wave % WAVES * 64 + lane) / qp; s < part.splits; s += WAVES * 64 / qp) {
            const float2 st = part.stat[s * step + q];
            // No keys: nothing was written.
            const bool some = st.x != -__builtin_inff() || st.y != 0.0f;
            const float w = some ? exp2f(st.x - base) : 0.0f;
            const float4 o = some ? *(const float4 *) (part.out + (s * step + q) * p.dim + c) : float4{0.f, 0.f, 0.f, 0.f};
            sum += w * st.y;
            v[0] += w * o.x;
            v[1] += w * o.y;
            v[2] += w * o.z;
            v[3] += w * o.w;
        }
    }
    for (int d = qp; d < 64; d <<= 1) {
        sum += __shfl_xor(sum, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += __shfl_xor(v[j], d);
    }
    if constexpr (WAVES > 1) {
        s_sum[wave][lane][4] = sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) s_sum[wave][lane][j] = v[j];
        __syncthreads();
        if (wave > 0) return;
        for (int w = 1; w < WAVES; ++w) {
            sum += s_sum[w][lane][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += s_sum[w][lane][j];
        }
    }
    if (lane < qp && c < p.dim) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T * y = (T *) p.y + row * p.y_stride + (int64_t) head * p.dim + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) Store<DT>::st(y, j, v[j] * inv);
    }
}

// Joins the splits, a query to WAVES wavefronts (one with few splits, four with
// many): QP lanes (a power of two) have four channels each, and the 64 WAVES / QP
// groups of them every so many splits.  Queries are found as k_attention<.., NW>
// does, TQ blocks' worth for each of its tiles.
template <int DT, int TQ, int WAVES>
__global__ void __launch_bounds__(256) k_join(Attention p, Partial part, int tiles, int qp) {
    constexpr int QUERIES = 4 / WAVES, PER = TQ / QUERIES;
    __shared__ float s_sum[4][64][5];
    const int group = p.heads / p.kv_heads, kv = blockIdx.x / PER / tiles;
    const Place at = find_place<TQ>(p, blockIdx.x / PER % tiles, group);
    const int i = blockIdx.x % PER * QUERIES + (threadIdx.x >> 6) / WAVES;
    // With one wavefront a query no barrier follows.
    if (WAVES == 1 ? i >= at.nq : (int) (blockIdx.x % PER) * QUERIES >= at.nq) return;
    const int64_t vq = at.first + i;
    const int64_t row = at.q0 + vq / group;
    const int head = kv * group + (int) (vq % group);
    join_query<DT, WAVES>(p, part, qp, row * p.heads + head, p.nq * p.heads, row, head, s_sum);
}

}  // namespace
}  // namespace tsh
