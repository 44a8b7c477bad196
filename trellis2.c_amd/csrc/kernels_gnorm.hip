// kernels_gnorm.hip - group norm over the rows of each sequence, channels last, with the activation that follows.
#include <type_traits>

#include "act_common.h"
#include "rows_common.h"

namespace tsh {
namespace {

// A group's mean m and the inverse of its root variance; the mean in two parts, so that
// x - m keeps its digits where the mean is far larger than the deviations.  Of groups beyond 2^64
// values and mean are taken 2^32 (`unit`) smaller and the inverse larger, exactly: x - m
// can be twice fp32's largest, and the inverse of that is subnormal.
struct GroupStat {
    float mean, mean_low, inverse, unit;
};
// x - m in those units.  (fp16 has no such groups.)
template <int DT> __device__ __forceinline__ float centred(float x, const GroupStat & st) {
    return (DT == kF16 ? x - st.mean : fmaf(x, st.unit, -st.mean)) - st.mean_low;
}

// Sums over a group, in 64 bits: of d = x - k and of d^2, k the group's first value in its
// sequence in fp32 (as k is one of the values, (k - m)^2 is at most as many variances as
// there are values, and var = mean d^2 - (mean d)^2 loses no more than that many of
// 2^-53), zero in 16 bits (whose values are at most 2^11 of their own steps).
struct GroupSum {
    double d, d2;
};
__device__ __forceinline__ GroupStat * stats_of(const GroupNorm & p) {
    return (GroupStat *) ((GroupSum *) p.scratch + p.tiles * p.slabs * p.groups);
}
template <int DT> __device__ __forceinline__ void add_value(GroupSum & s, float x, float k) {
    const double d = DT == kF32 ? (double) x - (double) k : (double) x;
    s.d += d;
    s.d2 = fma(d, d, s.d2);
}
__device__ __forceinline__ GroupStat stat_of(const GroupSum & s, double count, float k, float eps) {
    const double off = s.d / count, var = s.d2 / count - off * off;
    // (A NaN stays one; a negative variance is a rounding of zero.)
    const double root = sqrt((var < 0.0 ? 0.0 : var) + (double) eps), most = 0x1p64;
    const double unit = root > most || fabs((double) k + off) > most ? 0x1p-32 : 1.0, mean = ((double) k + off) * unit;
    const float hi = (float) mean;
    const double low = mean - (double) hi;
    return {hi, hi - hi == 0.0f ? (float) low : 0.0f, (float) (1.0 / (root * unit)), (float) unit};
}
template <int DT> __device__ __forceinline__ float first_value(const typename Store<DT>::T * p, int64_t i) {
    return DT == kF32 ? Store<DT>::ld(p, i) : 0.0f;
}

__device__ __forceinline__ int64_t row_of(const int32_t * at, int i, int64_t n) {
    const int64_t v = at[i];
    return v < 0 ? 0 : (v > n ? n : v);
}

// ---- a block per sequence and group -----------------------------------------------------------------

// Any sizes, values read twice: where groups are small, and where there is no scratch.
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
    const float k = first_value<DT>(x, 0);
    GroupSum s{0.0, 0.0};
    for (int64_t r = r0; r < end - first; r += step)
        for (int ch = ch0; ch < size; ch += wide) add_value<DT>(s, Store<DT>::ld(x, r * p.c + ch), k);
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
    by_act(p.act, [&](auto act_c) {
        for (int ch = ch0; ch < size; ch += wide) {
            const float scale = st.inverse * (p.gamma != nullptr ? p.gamma[g * size + ch] : 1.0f);
            const float shift = p.beta != nullptr ? p.beta[g * size + ch] : 0.0f;
            for (int64_t r = r0; r < end - first; r += step) {
                const float v = centred<DT>(Store<DT>::ld(x, r * p.c + ch), st) * scale + shift;
                Store<DT>::st(y, r * p.c + ch, activate<DT, decltype(act_c)::value>(v));
            }
        }
    });
}

// ---- tiles of rows ----------------------------------------------------------------------------------

// A tile's rows [first, first + rows) of sequence seq; rows = 0 where there is none.  Tiles are
// numbered by what holds for any lengths: sequence s, whose rows begin at a, has its tiles
// from a / tile_rows + s on, and never reaches past the next one's first.
struct Tile {
    int64_t first;
    int rows, seq;
};
__device__ __forceinline__ int64_t first_tile(const GroupNorm & p, int s) {
    return p.at != nullptr ? row_of(p.at, s, p.n) / p.tile_rows + s : 0;
}
__device__ Tile find_tile(const GroupNorm & p, int64_t tile) {
    int seq = 0;
    int64_t begin = 0, end = p.n;
    if (p.at != nullptr) {
        // The last sequence whose tiles begin at or before this one, 64 of them at a time.
        const int lane = threadIdx.x & 63;
        int many = p.seqs;
        while (many > 1) {
            const int step = (many + 63) / 64, i = lane * step;
            const unsigned long long before = __ballot(i < many && first_tile(p, seq + i) <= tile);
            if (before == 0) return {0, 0, 0};
            const int at = 63 - __clzll(before);
            seq += at * step;
            many = min(step, many - at * step);
        }
        begin = row_of(p.at, seq, p.n);
        end = row_of(p.at, seq + 1, p.n);
    }
    const int64_t from = begin + (tile - first_tile(p, seq)) * p.tile_rows;
    if (from < begin || from >= end) return {0, 0, seq};
    return {from, (int) min((int64_t) p.tile_rows, end - from), seq};
}

// V adjacent channels of a row: a chunk of 16 bytes, or (rows that are no whole number of
// them) a single one.
template <int DT, int V>
using Channels = typename std::conditional<V == 1, typename Store<DT>::T, int4>::type;
template <int DT, int V> __device__ __forceinline__ void unpack_channels(const Channels<DT, V> & c, float * v) {
    if constexpr (V == 1) {
        v[0] = Store<DT>::ld(&c, 0);
    } else {
        unpack_chunk_of<DT>(c, v);
    }
}

// Sums of a tile's rows and 256 chunks of V of their channels (`slab`), per group.  A thread
// has a chunk of every so many rows, and NG sums of neighbouring channels of it: one where a
// chunk is of one group, one a channel where groups do not divide chunks.  Each block
// writes its part of every group's sums (zeros for those that it has nothing of).
template <int DT, int V, int NG> __global__ void __launch_bounds__(256) k_gn_sums(GroupNorm p) {
    using T = typename Store<DT>::T;
    constexpr int W = V / NG;
    __shared__ GroupSum s_sum[256 * NG];
    const int64_t tile = blockIdx.x / p.slabs;
    const int slab = blockIdx.x % p.slabs;
    const Tile at = find_tile(p, tile);
    if (at.rows <= 0) return;
    const int size = p.c / p.groups, chunk0 = slab * 256;
    const int chunks = min(256, p.c / V - chunk0), step = 256 / chunks;
    const int col = threadIdx.x % chunks, r0 = threadIdx.x / chunks, ch0 = (chunk0 + col) * V;
    const T * x = (const T *) p.x + at.first * p.c + ch0;
    GroupSum s[NG];
    float k[NG];
    const int64_t begin = p.at != nullptr ? row_of(p.at, at.seq, p.n) : 0;
#pragma unroll
    for (int a = 0; a < NG; ++a) {
        s[a] = {0.0, 0.0};
        k[a] = first_value<DT>((const T *) p.x, begin * p.c + (ch0 + a * W) / size * size);
    }
    if (r0 < step) {
#pragma unroll 4
        for (int r = r0; r < at.rows; r += step) {
            float v[V];
            unpack_channels<DT, V>(*(const Channels<DT, V> *) (x + (int64_t) r * p.c), v);
#pragma unroll
            for (int u = 0; u < V; ++u) add_value<DT>(s[u / W], v[u], k[u / W]);
        }
    }
#pragma unroll
    for (int a = 0; a < NG; ++a) s_sum[threadIdx.x * NG + a] = s[a];
    __syncthreads();
    // `each` (a power of two, up to a wavefront) threads a group.
    const int here = (min(p.c, (chunk0 + chunks) * V) - 1) / size + 1 - chunk0 * V / size;  // groups of the slab
    int each = 1;
    while (each < 64 && each * 2 * here <= 256) each *= 2;
    const int unit = V / NG;  // channels of a sum
    GroupSum * out = (GroupSum *) p.scratch;
    for (int g0 = 0; g0 < here; g0 += 256 / each) {
        const int g = chunk0 * V / size + g0 + threadIdx.x / each;
        // The slab's sums of group g: [from, to) of every row.
        const int from = max(0, (g * size - chunk0 * V + unit - 1) / unit);
        const int to = min(chunks * NG, ((g + 1) * size - chunk0 * V) / unit);
        GroupSum t{0.0, 0.0};
        if (g0 + (int) threadIdx.x / each < here) {
            const int wide = to - from;
            for (int i = threadIdx.x % each; i < wide * step; i += each) {
                const GroupSum & q = s_sum[i / wide * chunks * NG + from + i % wide];
                t.d += q.d;
                t.d2 += q.d2;
            }
        }
        for (int d = 1; d < each; d <<= 1) {
            t.d += __shfl_xor(t.d, d);
            t.d2 += __shfl_xor(t.d2, d);
        }
        if (g0 + (int) threadIdx.x / each < here && threadIdx.x % each == 0) out[(g * p.tiles + tile) * p.slabs + slab] = t;
    }
    if (p.slabs > 1) {
        const int g1 = chunk0 * V / size;
        for (int g = threadIdx.x; g < p.groups; g += 256)
            if (g < g1 || g >= g1 + here) out[(g * p.tiles + tile) * p.slabs + slab] = {0.0, 0.0};
    }
}

// The sums of a sequence's tiles to its groups' statistics: a block each, or, where there
// are many sequences of few tiles, a wavefront.
template <int DT, int LANES> __global__ void __launch_bounds__(256) k_gn_stats(GroupNorm p) {
    using T = typename Store<DT>::T;
    __shared__ GroupSum s_sum[4];
    const int64_t i = (int64_t) blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES, seq = (int) (i / p.groups), g = (int) (i % p.groups), size = p.c / p.groups;
    if (seq >= p.seqs) return;
    const int64_t begin = p.at != nullptr ? row_of(p.at, seq, p.n) : 0;
    const int64_t end = p.at != nullptr ? row_of(p.at, seq + 1, p.n) : p.n;
    if (end <= begin) return;
    const float k = first_value<DT>((const T *) p.x, begin * p.c + g * size);
    const GroupSum * in = (const GroupSum *) p.scratch + (g * p.tiles + first_tile(p, seq)) * p.slabs;
    const int64_t many = (end - begin + p.tile_rows - 1) / p.tile_rows * p.slabs;
    GroupSum s{0.0, 0.0};
#pragma unroll 4
    for (int64_t j = lane; j < many; j += LANES) {
        s.d += in[j].d;
        s.d2 += in[j].d2;
    }
    s.d = group_sum<64>(s.d);
    s.d2 = group_sum<64>(s.d2);
    if constexpr (LANES == 256) {
        if (threadIdx.x % 64 == 0) s_sum[threadIdx.x / 64] = s;
        __syncthreads();
        for (int w = 1; w < 4; ++w) {
            s.d += s_sum[w].d;
            s.d2 += s_sum[w].d2;
        }
    }
    if (lane == 0) stats_of(p)[i] = stat_of(s, (double) (end - begin) * size, k, p.eps);
}

// A chunk that leaves the caches to x: 419,340 x 128 fp16 73 -> 63 us for all three kernels.
template <int DT> __device__ __forceinline__ void store_past_caches(typename Store<DT>::T * p, const float * v) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    i32x4 w;
    if constexpr (DT == kF32) {
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = __builtin_bit_cast(int, v[u]);
    } else {
        w = __builtin_bit_cast(i32x4, pack_chunk<DT>(v));
    }
    __builtin_nontemporal_store(w, (i32x4 *) p);
}

// The tiles, last ones first: they are what the caches still hold of the sums' pass.
// Bound by memory: 79,523 x 512 bf16 16 us of sums (5.0 TB/s), 5 of statistics, 30 here on average (15, 4
// and 29 at best); the call 49, of which reading and writing once would take 31 at a large copy's 5.3 TB/s.
template <int DT, int V, int ACT> __global__ void __launch_bounds__(256) k_gn_apply(GroupNorm p) {
    using T = typename Store<DT>::T;
    const unsigned block = gridDim.x - 1 - blockIdx.x;
    const int slab = block % p.slabs;
    const Tile at = find_tile(p, block / p.slabs);
    if (at.rows <= 0) return;
    const int size = p.c / p.groups, chunk0 = slab * 256;
    const int chunks = min(256, p.c / V - chunk0), step = 256 / chunks;
    const int col = threadIdx.x % chunks, r0 = threadIdx.x / chunks, ch0 = (chunk0 + col) * V;
    if (r0 >= step) return;
    const T * x = (const T *) p.x + at.first * p.c + ch0;
    T * y = (T *) p.y + at.first * p.c + ch0;
    GroupStat st[V];
    float scale[V], shift[V];
#pragma unroll
    for (int u = 0; u < V; ++u) {
        st[u] = stats_of(p)[(int64_t) at.seq * p.groups + (ch0 + u) / size];
        scale[u] = st[u].inverse * (p.gamma != nullptr ? p.gamma[ch0 + u] : 1.0f);
        shift[u] = p.beta != nullptr ? p.beta[ch0 + u] : 0.0f;
    }
    // Four rows at a time, the next four on their way.
    constexpr int D = 4;
    Channels<DT, V> next[D];
    const auto fetch = [&](int r) {
#pragma unroll
        for (int i = 0; i < D; ++i)
            if (r + i * step < at.rows) next[i] = *(const Channels<DT, V> *) (x + (int64_t) (r + i * step) * p.c);
    };
    fetch(r0);
    for (int r = r0; r < at.rows; r += D * step) {
        Channels<DT, V> here[D];
#pragma unroll
        for (int i = 0; i < D; ++i) here[i] = next[i];
        fetch(r + D * step);
#pragma unroll
        for (int i = 0; i < D; ++i) {
            if (r + i * step >= at.rows) break;
            float v[V];
            unpack_channels<DT, V>(here[i], v);
#pragma unroll
            for (int u = 0; u < V; ++u) v[u] = activate<DT, ACT>(centred<DT>(v[u], st[u]) * scale[u] + shift[u]);
            if constexpr (V == 1) {
                Store<DT>::st(y + (int64_t) (r + i * step) * p.c, 0, v[0]);
            } else {
                store_past_caches<DT>(y + (int64_t) (r + i * step) * p.c, v);
            }
        }
    }
}

template <int DT, int V> hipError_t launch_tiles(const GroupNorm & p, hipStream_t s) {
    const int64_t grid = p.tiles * p.slabs, stats = (int64_t) p.seqs * p.groups;
    const bool blocks = p.tiles >= (int64_t) p.seqs * 64;
    if (grid > 0x7fffffffLL || stats > 0x7fffffffLL) return hipErrorInvalidValue;
    const int size = p.c / p.groups;
    if (size % V == 0) {
        k_gn_sums<DT, V, 1><<<(unsigned) grid, 256, 0, s>>>(p);
    } else if (size * 2 == V) {
        k_gn_sums<DT, V, V == 1 ? 1 : 2><<<(unsigned) grid, 256, 0, s>>>(p);
    } else {
        k_gn_sums<DT, V, V><<<(unsigned) grid, 256, 0, s>>>(p);
    }
    if (blocks) {
        k_gn_stats<DT, 256><<<(unsigned) stats, 256, 0, s>>>(p);
    } else {
        k_gn_stats<DT, 64><<<(unsigned) ((stats + 3) / 4), 256, 0, s>>>(p);
    }
    switch (p.act) {
        case TRELLIS_SPARSE_HIP_ACT_SILU:
            k_gn_apply<DT, V, TRELLIS_SPARSE_HIP_ACT_SILU><<<(unsigned) grid, 256, 0, s>>>(p);
            break;
        case TRELLIS_SPARSE_HIP_ACT_GELU:
            k_gn_apply<DT, V, TRELLIS_SPARSE_HIP_ACT_GELU><<<(unsigned) grid, 256, 0, s>>>(p);
            break;
        case TRELLIS_SPARSE_HIP_ACT_GELU_TANH:
            k_gn_apply<DT, V, TRELLIS_SPARSE_HIP_ACT_GELU_TANH><<<(unsigned) grid, 256, 0, s>>>(p);
            break;
        default: k_gn_apply<DT, V, TRELLIS_SPARSE_HIP_ACT_NONE><<<(unsigned) grid, 256, 0, s>>>(p); break;
    }
    return hipGetLastError();
}

template <int DT> hipError_t launch_dt(const GroupNorm & p, hipStream_t s) {
    if (p.scratch != nullptr)
        return p.c % kChunk<DT> == 0 ? launch_tiles<DT, kChunk<DT>>(p, s) : launch_tiles<DT, 1>(p, s);
    const int64_t grid = (int64_t) p.seqs * p.groups;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    k_group_norm<DT><<<(unsigned) grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace

// Tiles of rows where a group has many values: as many as give each CU four blocks, of at least four rows a
// thread.
size_t group_norm_scratch(int dtype, GroupNorm & p, int cus) {
    const int whole = dtype == kF32 ? 4 : 8, chunk = p.c % whole == 0 ? whole : 1;
    const int chunks = p.c / chunk, wide = chunks < 256 ? chunks : 256;
    const int64_t size = p.c / p.groups;
    if (p.n * size < kGroupNormTiled) return 0;
    p.slabs = (chunks + 255) / 256;
    const int64_t step = 256 / wide, want = std::max<int64_t>(1, (int64_t) cus * 4 / p.slabs);
    const int64_t rows = std::max<int64_t>((p.n + want - 1) / want, 4 * step);
    p.tile_rows = (int) std::min<int64_t>((rows + step - 1) / step * step, 1 << 20);
    p.tiles = (p.n + p.tile_rows - 1) / p.tile_rows + (p.at != nullptr ? p.seqs : 0);
    return (size_t) p.tiles * p.slabs * p.groups * sizeof(GroupSum) + (size_t) p.seqs * p.groups * sizeof(GroupStat);
}

hipError_t launch_group_norm(int dtype, const GroupNorm & p, hipStream_t s) {
    switch (dtype) {
        case kF32: return launch_dt<kF32>(p, s);
        case kF16: return launch_dt<kF16>(p, s);
        default: return launch_dt<kBF16>(p, s);
    }
}

}  // namespace tsh
