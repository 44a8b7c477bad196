// kernels_scored.hip - attention whose scores are capped by a tanh, lowered by a distance, or masked:
// out_i = sum_j softmax_j(cap tanh(scale q_i . k_j / cap) - slope d(i, j)) v_j over the keys that i sees.
#include <type_traits>

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
        // (Below that tanh(u) is u, which may have lost digits where the cap is very large.)
        const float u = dot * sc.cap_scale;
        if (sc.cap > 0.0f && !(fabsf(u) < 0x1p-13f)) s = sc.cap * tanhf(u);
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

// ---- MFMA ---------------------------------------------------------------------------------------

// Units of work, a tile of queries with a kv head each, neighbouring units of the same kv
// head, in causal calls within a head from the last queries, which see most, to the first.  The first
// `whole` take all of their keys; the rest, which the CUs would not share evenly, are split
// over blocks of their own, started last.
struct Split {
    Partial part;      // of the rest: its splits
    int whole, rest;
    __host__ __device__ int64_t blocks() const { return whole + (int64_t) rest * part.splits; }
    // Where query i of a unit of the rest leaves its split's part.
    struct Unit {
        int64_t unit;
        int split, splits;
    };
    __device__ __forceinline__ int64_t place(const Unit & u, int tq, int i) const {
        return ((int64_t) u.split * rest + (u.unit - whole)) * tq + i;
    }
};
using Unit = Split::Unit;
// Each XCD takes contiguous ranges of both.
__device__ __forceinline__ Unit unit_of(const Split & s) {
    const int64_t b = blockIdx.x;
    if (b < s.whole) return {xcd_remap(b, s.whole), 0, 1};
    const int64_t r = xcd_remap(b - s.whole, gridDim.x - s.whole);
    return {s.whole + r / s.part.splits, (int) (r % s.part.splits), s.part.splits};
}

// Joins the rest's splits as k_join does, many by 16 wavefronts a query: 77 splits of 64
// channels 7.4 us, where four take 6.1, 310 8.2 (the call 39 -> 35).
template <int DT, int TQ, int WAVES>
__global__ void __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) k_scored_join(Attention p, Split shape, int tiles, int qp,
                                                                              int causal) {
    constexpr int BLOCK = WAVES > 4 ? WAVES : 4, QUERIES = BLOCK / WAVES, PER = TQ / QUERIES;
    __shared__ float s_sum[BLOCK][64][5];
    const int64_t unit = shape.whole + blockIdx.x / PER;
    const int group = p.heads / p.kv_heads, kv = (int) (unit / tiles);
    const Place at = find_place<TQ>(p, causal != 0 ? tiles - 1 - unit % tiles : unit % tiles, group);
    const int i = blockIdx.x % PER * QUERIES + (threadIdx.x >> 6) / WAVES;
    if (WAVES == 1 ? i >= at.nq : (int) (blockIdx.x % PER) * QUERIES >= at.nq) return;
    const int64_t vq = at.first + i;
    join_query<DT, WAVES>(p, shape.part, qp, shape.place({unit, 0, 0}, TQ, i), (int64_t) shape.rest * TQ, at.q0 + vq / group,
                          kv * group + (int) (vq % group), s_sum);
}

// The coordinates of a tile's 64 keys: as they are, and, counted from an origin, as the A
// operand of the squared distances, |p - k|^2 = |p|^2 - 2 p . k + |k|^2 as one product of
// seven terms in fp16: coordinates, and squares in two parts, all whole numbers of 11 bits.
// The sums are exact as long as no voxel is more than 1,023 from the origin on an axis
// (|p|^2 + |k|^2 + 2 |p . k| then stays below 2^24).
struct VoxelTile {
    int4 terms[64];
    int3 at[64];
    int far;  // some key is farther

    __device__ __forceinline__ void set(int key, const int3 & xyz, const int3 & origin);
};

__device__ __forceinline__ short f16_whole(int v) { return __builtin_bit_cast(short, (_Float16) (float) v); }
// Whether d (a difference that may have wrapped) is beyond what the products hold.
__device__ __forceinline__ bool beyond(int d) { return (uint32_t) (d + 1023) > 2046u; }

__device__ __forceinline__ void VoxelTile::set(int key, const int3 & xyz, const int3 & origin) {
    int x = xyz.x - origin.x, y = xyz.y - origin.y, z = xyz.z - origin.z;
    const bool out = beyond(x) || beyond(y) || beyond(z);
    at[key] = xyz;
    if (out) x = y = z = 0;
    const int sq = x * x + y * y + z * z;
    const s16x8 a{f16_whole(x), f16_whole(y), f16_whole(z), f16_whole(sq >> 11), f16_whole(sq & 2047), f16_whole(2048),
                  f16_whole(1), 0};
    terms[key] = __builtin_bit_cast(int4, a);
    const unsigned long long any = __ballot(out);
    if (key == 0) far = any != 0 ? 1 : 0;
}

// A query's terms (those of the lanes' first half; the other's are zeros); whether a lane's are beyond the products.
__device__ __forceinline__ bool voxel_terms(const int3 & xyz, const int3 & origin, int half, s16x8 & terms) {
    int x = xyz.x - origin.x, y = xyz.y - origin.y, z = xyz.z - origin.z;
    const bool out = beyond(x) || beyond(y) || beyond(z);
    if (out) x = y = z = 0;
    const int sq = x * x + y * y + z * z;
    const s16x8 b{f16_whole(-2 * x), f16_whole(-2 * y), f16_whole(-2 * z), f16_whole(2048), f16_whole(1),
                  f16_whole(sq >> 11), f16_whole(sq & 2047), 0};
    terms = half == 0 ? b : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
    return (bool) __any(out);
}

// top tanh(u) for a product z, u = |z by| and top = 1 / by, to 16 roundings of its own value: z times the series of
// tanh(u) / u below 0.35 (the next term is 2^-26 of it), where u's own digits matter little, else 1 - t over 1 + t,
// t = exp(-2 u).
__device__ __forceinline__ float capped(float z, float by, float top) {
    const float u = fabsf(z * by), q = u * u;
    const float t = __builtin_amdgcn_exp2f(-2.88539008f * u);
    const float far = copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t) * top, z);
    float s = fmaf(q, -8.86323553e-3f, 2.18694885e-2f);
    s = fmaf(q, s, -5.39682540e-2f);
    s = fmaf(q, s, 1.33333333e-1f);
    s = fmaf(q, s, -3.33333333e-1f);
    return u < 0.35f ? fmaf(z * q, s, z) : far;
}

// 16-bit values: whether one of eight is an infinity or a NaN, and zeros in place of those.
template <int DT> __device__ __forceinline__ bool any_not_finite(const int4 & c) {
    constexpr uint32_t E = DT == kBF16 ? 0x7f80u : 0x7c00u;
    bool some = false;
#pragma unroll
    for (uint32_t w : {(uint32_t) c.x, (uint32_t) c.y, (uint32_t) c.z, (uint32_t) c.w})
        some |= (w & E) == E || ((w >> 16) & E) == E;
    return some;
}
template <int DT> __device__ __forceinline__ s16x8 finite_part(s16x8 v) {
    constexpr short E = DT == kBF16 ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (v[i] & E) == E ? (short) 0 : v[i];
    return v;
}

// As k_attention, its scores changed between the products and the softmax.  What that adds
// runs on the vector unit, which bounds attention already; squared distances of voxels are the
// matrix unit's, counted from the block's first query, but where some are too far for that.
// The cap's constant part and the scale are the softmax's own: a cap adds a product, two
// transcendental instructions and a sum a score, a distance one product and, of voxels, a
// root.  A tile's scores are not computed under the softmax of the one before: without their
// registers one more wavefront per SIMD fits, which hides as much and spills nothing (18,216
// rows of 8 x 64 bf16 by voxel distance 1.62 -> 1.30 ms).
// Bound by the vector unit, 76 % busy there (matrix unit 31 %): now 1.07 ms, 637 TFLOP/s of its
// products; 16,384 rows of 8 x 128 fp16 capped 1.36 ms, 808 TFLOP/s.
//
// Weights meet the values in the storage type, rounded to nearest (their sum is of fp32 ones): an error
// of the size of the output's own rounding (fp16 2.9e-4 of the output's root mean square where that
// rounding alone leaves 2.1e-4).  FINE: in two parts, which few blocks hide in their
// latencies; for many they cost 23 % (18,216 rows of 8 x 64 bf16 by voxel distance) to 41 %
// (9,001 causal rows of 8 x 128 fp16).
template <int DT, int DC, int NW, bool FINE, bool VOXELS, bool TANH>
__global__ void __launch_bounds__(64 * NW, DC <= 64 ? (VOXELS ? 3 : 4) : 2) k_scored(Attention p, Scores sc, Split shape, int tiles) {
    using T = typename Store<DT>::T;
    constexpr int TQ = 32 * NW, TK = 64;
    constexpr int LP = DC <= 64 ? 64 : 128;      // values per LDS row
    constexpr int ROW = LP * 2, CH = LP / 8;     // its bytes and chunks
    constexpr int KS = DC / 16, DT32 = DC / 32;  // K steps of the scores, 32-row tiles of the output
    constexpr int TILE = TK * ROW;
    constexpr int RPL = 64 / CH;                 // rows per load of 1 KB
    constexpr int LOADS = TILE / 1024;
    constexpr int PER = LOADS / NW;              // of K, and of V, per wavefront
    static_assert(LOADS % NW == 0, "whole loads");
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[4 * TILE];  // K, V of two tiles
    __shared__ typename std::conditional<VOXELS, VoxelTile, char>::type s_voxel[2];
    __shared__ int s_odd[NW];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int group = p.heads / p.kv_heads;

    const Unit u = unit_of(shape);
    const Partial part = u.splits > 1 ? shape.part : Partial{nullptr, nullptr, 1};
    const int split = u.split, kv = (int) (u.unit / tiles);
    const int64_t tile_at = u.unit % tiles;
    const Place at = find_place<TQ>(p, sc.causal != 0 ? tiles - 1 - tile_at : tile_at, group);
    if (at.nq <= 0) return;
    const int seen = (int) keys_seen(at, sc, (at.first + at.nq - 1) / group);
    const int all = (seen + TK - 1) / TK;
    const int t0 = (int) ((int64_t) all * split / part.splits), t1 = (int) ((int64_t) all * (split + 1) / part.splits);

    // This lane's query.
    const int qi = wave * 32 + l32;
    const int64_t vq = at.first + qi;
    const int64_t row = at.q0 + vq / group;
    const int head = kv * group + (int) (vq % group);
    const bool live = qi < at.nq;
    s16x8 q[KS];
    {
        const T * qr = (const T *) p.q + row * p.q_stride + (int64_t) head * p.dim;
        const int flip = p.scale < 0.0f ? (int) 0x80008000u : 0;  // the reference follows the largest score
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int c = (2 * k + half) * 8;
            int4 v{0, 0, 0, 0};
            if (live && c < p.dim) v = *(const int4 *) (qr + c);
            q[k] = __builtin_bit_cast(s16x8, int4{v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip});
        }
    }
    const float scale = sc.by;
    // The query's place among the keys, and the last key that it sees.
    const int64_t query = vq / group;
    const int place = (int) (query + at.nk - at.rows);
    const int limit = (live ? (int) keys_seen(at, sc, query) : seen) - 1;  // (lanes without one mask nothing)
    const float slope = sc.slopes != nullptr && live ? -sc.slopes[head] * sc.over : 0.0f;
    s16x8 voxel;
    bool far = false;
    int3 origin{0, 0, 0};
    if constexpr (VOXELS) {
        origin = voxel_of(sc.q_xyz, at.q0 + at.first / group);
        far = voxel_terms(live ? voxel_of(sc.q_xyz, row) : origin, origin, half, voxel);
    }
    // The coordinates of tile t's keys, a key a lane of the first wavefront: fetched, and left in LDS.
    int3 key_xyz{0, 0, 0};
    const auto fetch_xyz = [&](int t) {
        if (!VOXELS || wave != 0) return;
        key_xyz = t * TK + lane < at.nk ? voxel_of(sc.k_xyz, at.k0 + t * TK + lane) : origin;
    };
    const auto leave_xyz = [&](int j) {
        if (!VOXELS || wave != 0) return;
        if constexpr (VOXELS) s_voxel[j & 1].set(lane, key_xyz, origin);
    };

    const auto swizzle = [](int r) {
        if constexpr (LP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
        return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);
    };
    // Loads: row lane / CH of RPL, the chunk that lands at place lane % CH.
    // Rows of one load and the next differ in bits that swizzle sees, so each
    // load has its own chunk.
    const char * kb = (const char *) ((const T *) p.k + at.k0 * p.k_stride + (int64_t) kv * p.dim);
    const char * vb = (const char *) ((const T *) p.v + at.k0 * p.v_stride + (int64_t) kv * p.dim);
    const int ks = (int) p.k_stride * 2, vs = (int) p.v_stride * 2;
    constexpr uint32_t kOutside = 0x80000000u;
    uint32_t k_off[PER], v_off[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int r = (wave * PER + j) * RPL + lane / CH;
        const int c = (lane % CH) ^ swizzle(r);
        const bool in = c * 8 < p.dim;
        k_off[j] = in ? (uint32_t) (r * ks + c * 16) : kOutside;
        v_off[j] = in ? (uint32_t) (r * vs + c * 16) : kOutside;
    }
    const uint32_t lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) unsigned char *) s_tile;
    const auto load = [&](const char * base, int pitch, const uint32_t (&off)[PER], int rows, uint32_t to) {
        if (rows >= TK) {
            const __amdgpu_buffer_rsrc_t res =
                __builtin_amdgcn_make_buffer_rsrc((void *) base, 0, (TK - 1) * pitch + p.dim * 2, 0x00020000);
#pragma unroll
            for (int j = 0; j < PER; ++j) dma_b128_m0(res, lds0 + to + (wave * PER + j) * 1024u, off[j], 0);
        } else {
            // Rows past the end are zeros.
            const __amdgpu_buffer_rsrc_t res =
                __builtin_amdgcn_make_buffer_rsrc((void *) base, 0, (rows - 1) * pitch + p.dim * 2, 0x00020000);
#pragma unroll
            for (int j = 0; j < PER; ++j)
                dma_b128_m0(res, lds0 + to + (wave * PER + j) * 1024u,
                            (wave * PER + j) * RPL + lane / CH < rows ? off[j] : kOutside, 0);
        }
    };
    // Tile t's keys go to buffer (t - t0) % 2, its values to the same of two more;
    // the next tile to load of each, and where it is.
    int tk = t0, tv = t0;
    const char * k_at = kb + (int64_t) t0 * TK * ks;
    const char * v_at = vb + (int64_t) t0 * TK * vs;
    const auto load_k = [&]() {
        load(k_at, ks, k_off, at.nk - tk * TK, (uint32_t) (((tk - t0) & 1) * TILE));
        ++tk;
        k_at += (int64_t) TK * ks;
    };
    const auto load_v = [&]() {
        load(v_at, vs, v_off, at.nk - tv * TK, (uint32_t) (((tv - t0) & 1) * TILE + 2 * TILE));
        ++tv;
        v_at += (int64_t) TK * vs;
    };

    // Reads: K row l32 (+ 32), chunk 2 k + half; V rows 4 half + (lane % 16) / 4
    // (+ 8, + 16 g), 16-value column block (lane / 16) % 2 of each 32.
    uint32_t k_read[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) k_read[k] = (uint32_t) (l32 * ROW + (((2 * k + half) ^ swizzle(l32)) * 16));
    uint32_t v_read[DT32][2];
#pragma unroll
    for (int d = 0; d < DT32; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * e + 4 * half + ((lane & 15) >> 2);
            const int c = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            v_read[d][e] = (uint32_t) (r * ROW + ((c ^ swizzle(r)) * 16) + (lane & 1) * 8);
        }

    f32x16 out[DT32];
#pragma unroll
    for (int d = 0; d < DT32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[d][i] = 0.0f;
    float ref = -__builtin_inff(), sum0 = 0.0f, sum1 = 0.0f;

    // The scores' product k (of KS) of keys n (of 2).
    const auto read_k = [&](const unsigned char * sk, int n, int k) {
        return *(const s16x8 *) (sk + n * 32 * ROW + k_read[k]);
    };
    const auto zero = [](f32x16 & v) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    };
    // Products with keys n * 32 .. of tile t to what times `scale` is a score in log2 units: the
    // cap, then the distance.
    const auto change_scores = [&](int t, int n, f32x16 & cur, bool near, const int4 & terms) {
        if constexpr (TANH) {
#pragma unroll
            for (int i = 0; i < 16; ++i) cur[i] = capped(cur[i], sc.cap_scale, sc.top);
        } else if (sc.cap > 0.0f) {
            // cap tanh(z) is cap less 2 cap / (1 + exp(2 z)), the cap the same for all keys: off by
            // some 2^-22.5 of the cap, whatever the score.
#pragma unroll
            for (int i = 0; i < 16; ++i) cur[i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(cur[i] * sc.twice));
        }
        if (sc.slopes == nullptr) return;
        if constexpr (VOXELS) {
            if (near) {
                f32x16 d2;
                zero(d2);
                d2 = mac32<kF16>(__builtin_bit_cast(s16x8, terms), voxel, d2);
#pragma unroll
                for (int i = 0; i < 16; ++i) cur[i] = fmaf(slope, __builtin_amdgcn_sqrtf(d2[i]), cur[i]);
            } else {
                const VoxelTile & keys = (const VoxelTile &) s_voxel[(t - t0) & 1];
                const int3 here = voxel_of(sc.q_xyz, live ? row : at.q0);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    cur[i] = fmaf(slope, distance_of(here, keys.at[n * 32 + 8 * (i / 4) + 4 * half + i % 4]), cur[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
            const float from = (float) (place - t * TK - 4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                cur[i] = fmaf(slope, fabsf(from - (float) (n * 32 + 8 * (i / 4) + i % 4)), cur[i]);
        }
    };

    // What a query does not see has weight zero, but zero times an infinity or a NaN is a
    // NaN: of tiles with keys that some query of the block does not see, such values are
    // added to the queries that see them here, and are zeros for the products.
    const int least_seen = (int) keys_seen(at, sc, at.first / group);
    const auto set_aside = [&](unsigned char * sv, int last) {
        constexpr int PART = TILE / NW;
        unsigned char * mine = sv + wave * PART + lane * 16;
        bool some = false;
#pragma unroll
        for (int i = 0; i < PART; i += 1024) some |= any_not_finite<DT>(*(const int4 *) (mine + i));
        const bool any = __any(some);
        if (lane == 0) s_odd[wave] = any;
        lds_barrier();
        int odd = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) odd |= s_odd[w];
        if (uniform(odd) == 0) return;
#pragma unroll 1
        for (int r = 0; r < TK; ++r) {
            if (r - 4 * half > last) break;
#pragma unroll
            for (int d = 0; d < DT32; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = d * 32 + i * 8 + half * 4;
                    const T * v = (const T *) (sv + r * ROW + (((c / 8) ^ swizzle(r)) * 16) + half * 8);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float x = Store<DT>::ld(v, u);
                        if (!(fabsf(x) < __builtin_inff())) out[d][4 * i + u] += x;
                    }
                }
        }
        lds_barrier();
#pragma unroll 1
        for (int i = 0; i < PART; i += 1024) {
            int4 * c = (int4 *) (mine + i);
            *c = __builtin_bit_cast(int4, finite_part<DT>(__builtin_bit_cast(s16x8, *c)));
        }
        lds_barrier();
    };

    // One tile: its scores, their softmax, and the products of weights and values a group of
    // 16 keys behind the exponentials.
    const auto tile = [&](int t) {
        const int j = (t - t0) & 1;
        // Keys and values of t have landed; every wavefront is done with those of t - 1.
        wait_vmcnt<0>();
        leave_xyz(j);
        lds_barrier();
        if (t + 1 < t1) {
            load_k();
            load_v();
            fetch_xyz(t + 1);
        }
        const unsigned char * sk = s_tile + j * TILE;
        unsigned char * sv = s_tile + (j + 2) * TILE;
        bool near = false;
        int4 terms[2];
        if constexpr (VOXELS) {
            const VoxelTile & keys = (const VoxelTile &) s_voxel[j];
            near = uniform(keys.far) == 0 && !far;
#pragma unroll
            for (int n = 0; n < 2; ++n) terms[n] = keys.terms[n * 32 + l32];
        }
        f32x16 cur[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            zero(cur[n]);
#pragma unroll
            for (int k = 0; k < KS; ++k) cur[n] = mac32<DT>(read_k(sk, n, k), q[k], cur[n]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) change_scores(t, n, cur[n], near, terms[n]);
        const int last = limit - t * TK - 4 * half;  // of this tile's keys, less what the lane's half adds
        const bool masked = __any(last < TK - 5);
        if (masked) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (n * 32 + 8 * (i / 4) + i % 4 > last) cur[n][i] = -__builtin_inff();
        }
        float m = cur[0][0];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, cur[n][i]);
        m = max_halves(m) * scale;
        if (__any(m > ref + 8.0f)) {
            const float next = m > ref + 8.0f ? m : ref;  // each query by itself: what it does not see moves nothing
            const float keep = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(ref - next);
            ref = next;
            sum0 *= keep;
            sum1 *= keep;
#pragma unroll
            for (int d = 0; d < DT32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) out[d][i] *= keep;
        }
        constexpr float kLift = DT == kF16 ? 7.0f : 0.0f;
        const float base = ref == -__builtin_inff() ? 0.0f : ref - kLift;
        if (t * TK + TK > least_seen) set_aside(sv, last);
        s16x8 vf[DT32], w, rest;
        const auto values = [&](int d) {
            out[d] = mac32<DT>(vf[d], w, out[d]);
            if constexpr (FINE) out[d] = mac32<DT>(vf[d], rest, out[d]);
        };
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float e[8];
            const auto weight = [&](int i) {
                e[i] = __builtin_amdgcn_exp2f(fmaf(cur[g / 2][8 * (g % 2) + i], scale, -base));
            };
            if (g > 0) {
#pragma unroll
                for (int d = 0; d < DT32; ++d) {
                    values(d);
#pragma unroll
                    for (int i = 8 * d / DT32; i < 8 * (d + 1) / DT32; ++i) weight(i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) weight(i);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int d = 0; d < DT32; ++d) {
                union {
                    s16x4 h[2];
                    s16x8 v;
                } a;
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    a.h[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4 *) (sv + g * 16 * ROW + v_read[d][x]));
                vf[d] = a.v;
            }
            union {
                T h[8];
                s16x8 v;
            } r;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (!FINE) r.h[i] = round_to_store<DT>(e[i]);
                if (i % 2 == 0) {
                    sum0 += e[i];
                } else {
                    sum1 += e[i];
                }
            }
            if constexpr (FINE) {
                two_parts<DT>(e, w, rest);
            } else {
                w = r.v;
            }
        }
#pragma unroll
        for (int d = 0; d < DT32; ++d) values(d);
    };

    if (t0 < t1) {
        fetch_xyz(t0);
        load_k();
        load_v();
        for (int t = t0; t < t1; ++t) tile(t);
    }

    const auto left = [&] { return shape.place(u, TQ, qi); };
    leave_at<DT>(p, part, out, ref, sum_halves(sum0 + sum1), live, t0 < t1, left, row, head, half);
}

// fp32, as k_attention32: its products leave the vector unit time for exact changes.
template <int DC, int NW>
__global__ void __launch_bounds__(64 * NW, 2) k_scored32(Attention p, Scores sc, Split shape, int tiles) {
    constexpr int TQ = 32 * NW, TK = 32;
    constexpr int LP = DC <= 32 ? 32 : (DC <= 64 ? 64 : 128);  // values per LDS row
    constexpr int ROW = LP * 4, CH = LP / 4;
    constexpr int KS = DC / 8, DT32 = DC / 32;
    constexpr int TILE = TK * ROW;
    constexpr int RPL = 64 / CH;
    constexpr int PER = TILE / 1024 / NW;
    static_assert(TILE / 1024 % NW == 0, "whole loads");
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[4 * TILE];  // K, V of two tiles
    __shared__ int4 s_xyz[2][TK];  // the coordinates of their keys
    __shared__ int s_odd[NW];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int group = p.heads / p.kv_heads;
    const Unit u = unit_of(shape);
    const Partial part = u.splits > 1 ? shape.part : Partial{nullptr, nullptr, 1};
    const int split = u.split, kv = (int) (u.unit / tiles);
    const int64_t tile_at = u.unit % tiles;
    const Place at = find_place<TQ>(p, sc.causal != 0 ? tiles - 1 - tile_at : tile_at, group);
    if (at.nq <= 0) return;
    const int seen = (int) keys_seen(at, sc, (at.first + at.nq - 1) / group);
    const int all = (seen + TK - 1) / TK;
    const int t0 = (int) ((int64_t) all * split / part.splits), t1 = (int) ((int64_t) all * (split + 1) / part.splits);

    const int qi = wave * 32 + l32;
    const int64_t vq = at.first + qi;
    const int64_t row = at.q0 + vq / group;
    const int head = kv * group + (int) (vq % group);
    const bool live = qi < at.nq;
    const float sign = p.scale < 0.0f ? -1.0f : 1.0f, scale = sc.by;
    const int64_t query = vq / group;
    const int place = (int) (query + at.nk - at.rows);
    const int limit = (live ? (int) keys_seen(at, sc, query) : seen) - 1;  // (lanes without one mask nothing)
    const float slope = sc.slopes != nullptr && live ? -sc.slopes[head] * sc.over : 0.0f;
    const int3 here = sc.q_xyz != nullptr && live ? voxel_of(sc.q_xyz, row) : int3{0, 0, 0};
    float q[KS][4];
    {
        const float * qr = (const float *) p.q + row * p.q_stride + (int64_t) head * p.dim;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int c = 8 * k + 4 * half;
            float4 v{0.f, 0.f, 0.f, 0.f};
            if (live && c < p.dim) v = *(const float4 *) (qr + c);
            q[k][0] = v.x * sign;
            q[k][1] = v.y * sign;
            q[k][2] = v.z * sign;
            q[k][3] = v.w * sign;
        }
    }

    const auto swizzle = [](int r) {
        if constexpr (CH == 8) return (r >> 1) & 7;
        return ((r & 4) << 1) | ((r & 8) >> 1) | (r & 3);
    };
    const char * kb = (const char *) ((const float *) p.k + at.k0 * p.k_stride + (int64_t) kv * p.dim);
    const char * vb = (const char *) ((const float *) p.v + at.k0 * p.v_stride + (int64_t) kv * p.dim);
    const int ks = (int) p.k_stride * 4, vs = (int) p.v_stride * 4;
    constexpr uint32_t kOutside = 0x80000000u;
    const uint32_t lds0 = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) unsigned char *) s_tile;
    // Rows past the last and channels past dim are zeros.
    const auto load = [&](int t) {
        const int rows = min(TK, at.nk - t * TK);
        const uint32_t to = lds0 + (uint32_t) (((t - t0) & 1) * TILE);
        const __amdgpu_buffer_rsrc_t kres = __builtin_amdgcn_make_buffer_rsrc(
            (void *) (kb + (int64_t) t * TK * ks), 0, (rows - 1) * ks + p.dim * 4, 0x00020000);
        const __amdgpu_buffer_rsrc_t vres = __builtin_amdgcn_make_buffer_rsrc(
            (void *) (vb + (int64_t) t * TK * vs), 0, (rows - 1) * vs + p.dim * 4, 0x00020000);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = (wave * PER + j) * RPL + lane / CH;
            const int c = (lane % CH) ^ swizzle(r);
            const bool in = r < rows && c * 4 < p.dim;
            dma_b128_m0(kres, to + (wave * PER + j) * 1024u, in ? (uint32_t) (r * ks + c * 16) : kOutside, 0);
            dma_b128_m0(vres, to + 2 * TILE + (wave * PER + j) * 1024u, in ? (uint32_t) (r * vs + c * 16) : kOutside, 0);
        }
    };

    int4 key_xyz{0, 0, 0, 0};
    const auto fetch_xyz = [&](int t) {
        if (sc.k_xyz != nullptr && wave == 0 && lane < TK && t * TK + lane < at.nk)
            key_xyz = *(const int4 *) (sc.k_xyz + (at.k0 + t * TK + lane) * 4);
    };

    f32x16 out[DT32];
#pragma unroll
    for (int d = 0; d < DT32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[d][i] = 0.0f;
    // As k_scored's.
    const int least_seen = (int) keys_seen(at, sc, at.first / group);
    const auto set_aside = [&](unsigned char * sv, int last) {
        constexpr int PART = TILE / NW;
        unsigned char * mine = sv + wave * PART + lane * 16;
        const auto odd_value = [](float v) { return !(fabsf(v) < __builtin_inff()); };
        bool some = false;
#pragma unroll 1
        for (int i = 0; i < PART; i += 1024) {
            const float4 v = *(const float4 *) (mine + i);
            some |= odd_value(v.x) || odd_value(v.y) || odd_value(v.z) || odd_value(v.w);
        }
        const bool any = __any(some);
        if (lane == 0) s_odd[wave] = any;
        lds_barrier();
        int odd = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) odd |= s_odd[w];
        if (uniform(odd) == 0) return;
#pragma unroll 1
        for (int r = 0; r < TK; ++r) {
            if (r - 4 * half > last) break;
#pragma unroll
            for (int d = 0; d < DT32; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float * v = (const float *) (sv + r * ROW + (((d * 8 + i * 2 + half) ^ swizzle(r)) * 16));
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (odd_value(v[u])) out[d][4 * i + u] += v[u];
                }
        }
        lds_barrier();
#pragma unroll 1
        for (int i = 0; i < PART; i += 1024) {
            float4 * c = (float4 *) (mine + i);
            const float4 v = *c;
            *c = float4{odd_value(v.x) ? 0.0f : v.x, odd_value(v.y) ? 0.0f : v.y, odd_value(v.z) ? 0.0f : v.z,
                        odd_value(v.w) ? 0.0f : v.w};
        }
        lds_barrier();
    };
    float ref = -__builtin_inff(), sum0 = 0.0f, sum1 = 0.0f;
    if (t0 < t1) {
        load(t0);
        fetch_xyz(t0);
    }
    for (int t = t0; t < t1; ++t) {
        // Tile t has landed; every wavefront is done with tile t - 1.
        wait_vmcnt<0>();
        if (sc.k_xyz != nullptr && wave == 0 && lane < TK) s_xyz[(t - t0) & 1][lane] = key_xyz;
        lds_barrier();
        if (t + 1 < t1) {
            load(t + 1);
            fetch_xyz(t + 1);
        }
        const unsigned char * sk = s_tile + ((t - t0) & 1) * TILE;
        unsigned char * sv = s_tile + ((t - t0) & 1) * TILE + 2 * TILE;
        f32x16 cur;
#pragma unroll
        for (int i = 0; i < 16; ++i) cur[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const float4 a = *(const float4 *) (sk + l32 * ROW + (((2 * k + half) ^ swizzle(l32)) * 16));
            cur = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, q[k][0], cur, 0, 0, 0);
            cur = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, q[k][1], cur, 0, 0, 0);
            cur = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, q[k][2], cur, 0, 0, 0);
            cur = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, q[k][3], cur, 0, 0, 0);
        }
        if (sc.top > 0.0f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) cur[i] = capped(cur[i], sc.cap_scale, sc.top);
        }
        if (sc.slopes != nullptr && sc.q_xyz == nullptr) {
            const float from = (float) (place - t * TK - 4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) cur[i] = fmaf(slope, fabsf(from - (float) (8 * (i / 4) + i % 4)), cur[i]);
        }
        if (sc.q_xyz != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int4 key = s_xyz[(t - t0) & 1][8 * (i / 4) + 4 * half + i % 4];
                const float x = (float) (here.x - key.y), y = (float) (here.y - key.z), z = (float) (here.z - key.w);
                cur[i] = fmaf(slope, __builtin_amdgcn_sqrtf(fmaf(x, x, fmaf(y, y, z * z))), cur[i]);
            }
        }
        const int last = limit - t * TK - 4 * half;
        if (__any(last < TK - 5)) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i / 4) + i % 4 > last) cur[i] = -__builtin_inff();
        }
        float m = cur[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) m = fmaxf(m, cur[i]);
        m = max_halves(m) * scale;
        if (__any(m > ref + 8.0f)) {
            const float next = m > ref + 8.0f ? m : ref;  // each query by itself: what it does not see moves nothing
            const float keep = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(ref - next);
            ref = next;
            sum0 *= keep;
            sum1 *= keep;
#pragma unroll
            for (int d = 0; d < DT32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) out[d][i] *= keep;
        }
        const float base = ref == -__builtin_inff() ? 0.0f : ref;
        if (t * TK + TK > least_seen) set_aside(sv, last);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(cur[i], scale, -base));
            (i % 2 == 0 ? sum0 : sum1) += e;
            const int r = 8 * (i / 4) + 4 * half + i % 4;
#pragma unroll
            for (int d = 0; d < DT32; ++d) {
                const float a = *(const float *) (sv + r * ROW + (((8 * d + l32 / 4) ^ swizzle(r)) * 16) + l32 % 4 * 4);
                out[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, e, out[d], 0, 0, 0);
            }
        }
    }
    const auto left = [&] { return shape.place(u, TQ, qi); };
    leave_at<kF32>(p, part, out, ref, sum_halves(sum0 + sum1), live, t0 < t1, left, row, head, half);
}

template <int DT, int DC, int NW>
hipError_t launch_nw(const Attention & p, const Scores & sc, const Split & split, const ScoredShape & sh, hipStream_t s) {
    const int64_t grid = split.blocks();
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    const int tiles = (int) sh.tiles;
    if constexpr (DT == kF32) {
        k_scored32<DC, NW><<<(unsigned) grid, 64 * NW, 0, s>>>(p, sc, split, tiles);
    } else {
        const auto launch = [&](auto fine_c, auto voxels_c, auto tanh_c) {
            k_scored<DT, DC, NW, decltype(fine_c)::value, decltype(voxels_c)::value, decltype(tanh_c)::value>
                <<<(unsigned) grid, 64 * NW, 0, s>>>(p, sc, split, tiles);
        };
        using std::false_type, std::true_type;
        // (Large caps are rare: one instance, for any number of queries.)
        const auto kind = [&](auto voxels_c) {
            if (sc.top > 0.0f) return launch(true_type(), voxels_c, true_type());
            sh.fine ? launch(true_type(), voxels_c, false_type()) : launch(false_type(), voxels_c, false_type());
        };
        sc.q_xyz != nullptr ? kind(true_type()) : kind(false_type());
    }
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && split.part.splits > 1) {
        int qp = 1;
        while (qp * 4 < p.dim) qp *= 2;
        const int splits = split.part.splits;
        const int64_t joins = (int64_t) split.rest * (splits >= 32 ? 32 * NW : 8 * NW);
        if (joins > 0x7fffffffLL) return hipErrorInvalidValue;
        if (splits >= 128) {
            k_scored_join<DT, 32 * NW, 16><<<(unsigned) joins, 1024, 0, s>>>(p, split, tiles, qp, sc.causal);
        } else if (splits >= 32) {
            k_scored_join<DT, 32 * NW, 4><<<(unsigned) joins, 256, 0, s>>>(p, split, tiles, qp, sc.causal);
        } else {
            k_scored_join<DT, 32 * NW, 1><<<(unsigned) joins, 256, 0, s>>>(p, split, tiles, qp, sc.causal);
        }
        err = hipGetLastError();
    }
    return err;
}

template <int DT, int DC>
hipError_t launch_dc(const Attention & p, const Scores & sc, const Split & split, const ScoredShape & sh, hipStream_t s) {
    return sh.waves == 1 ? launch_nw<DT, DC, 1>(p, sc, split, sh, s) : launch_nw<DT, DC, 4>(p, sc, split, sh, s);
}

template <int DT>
hipError_t launch_mfma(const Attention & p, const Scores & sc, const Split & split, const ScoredShape & sh, hipStream_t s) {
    if (p.dim <= 32) return launch_dc<DT, 32>(p, sc, split, sh, s);
    if (p.dim <= 64) return launch_dc<DT, 64>(p, sc, split, sh, s);
    if (p.dim <= 96) return launch_dc<DT, 96>(p, sc, split, sh, s);
    return launch_dc<DT, 128>(p, sc, split, sh, s);
}

}  // namespace

// Few queries: all units split as attention's are.  Many: CUs get equal numbers of whole
// units, and what is left over is split.  (Causal units are of unequal lengths; they are not
// split, and go from the longest to the shortest of each kv head.)
ScoredShape scored_shape(int dtype, const Attention & p, const Scores & sc, int cus) {
    const AttentionShape a = attention_shape(dtype, p, cus);
    ScoredShape sh{a.waves, a.tiles, a.fine, 0, 0, 1, 0};
    // (Slopes over a scale that small could leave fp32: the general kernel.)
    if (sc.slopes != nullptr && sc.by < 0x1p-30f) sh.waves = 0;
    if (sh.waves == 0) return sh;
    const int64_t units = sh.tiles * p.kv_heads;
    if (units > 0x7fffffffLL) return sh;
    sh.whole = (int) units;
    const int64_t key_tiles = (p.nk / (p.q_at != nullptr ? p.seqs : 1) + 63) / 64;
    if (a.splits > 1) {
        sh.whole = 0;
        sh.splits = a.splits;
    } else if (sc.causal == 0 && sh.waves == 4 && units > 2 * cus) {
        const int splits = (int) std::min<int64_t>(8, key_tiles / 16);
        if (splits > 1) {
            sh.whole = (int) (units / cus * cus);
            sh.splits = splits;
        }
    }
    sh.rest = (int) (units - sh.whole);
    if (sh.rest == 0) sh.splits = 1;
    if (sh.splits > 1) sh.scratch = (size_t) sh.splits * sh.rest * 32 * sh.waves * (p.dim + 2) * sizeof(float);
    return sh;
}

hipError_t launch_attention_scored(int dtype, const Attention & p, const Scores & sc, const ScoredShape & sh, void * scratch,
                                   hipStream_t s) {
    if (sh.waves == 0) {
        switch (dtype) {
            case kF32: return launch_any<kF32>(p, sc, s);
            case kF16: return launch_any<kF16>(p, sc, s);
            default: return launch_any<kBF16>(p, sc, s);
        }
    }
    if (sh.tiles * p.kv_heads > 0x7fffffffLL) return hipErrorInvalidValue;
    Split split{Partial{nullptr, nullptr, 1}, sh.whole + sh.rest, 0};
    if (scratch != nullptr && sh.splits > 1) {
        split = Split{Partial{(float *) scratch, nullptr, sh.splits}, sh.whole, sh.rest};
        split.part.stat = (float2 *) (split.part.out + (size_t) sh.splits * sh.rest * 32 * sh.waves * p.dim);
    }
    switch (dtype) {
        case kF32: return launch_mfma<kF32>(p, sc, split, sh, s);
        case kF16: return launch_mfma<kF16>(p, sc, split, sh, s);
        default: return launch_mfma<kBF16>(p, sc, split, sh, s);
    }
}

}  // namespace tsh
