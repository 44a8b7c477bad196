// kernels_attn.hip - attention within sequences of rows: out_i = sum_j softmax_j(scale q_i . k_j) v_j.
#include "attn_common.h"

namespace tsh {
namespace {

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
        T * y = (T *) p.y + (at.q0 + at.first + row) * p.y_stride + (int64_t) head * p.dim;
#pragma unroll
        for (int u = 0; u < kAttentionMaxDim / 16; ++u) {
            const int c = u * 16 + l;
            if (c < p.dim) Store<DT>::st(y, c, acc[u] * inv);
        }
    }
}

template <int DT> hipError_t launch_any(const Attention & p, hipStream_t s) {
    const int64_t tiles = p.nq / 16 + (p.q_at != nullptr ? p.seqs : 1);
    const int64_t grid = tiles * p.heads;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    const size_t lds = ((size_t) (16 + 32 + 32) * (p.dim + 1) + 16 * 33) * sizeof(float);
    k_attention_any<DT><<<(unsigned) grid, 256, lds, s>>>(p);
    return hipGetLastError();
}

// ---- MFMA ---------------------------------------------------------------------------------------

// NW wavefronts of 32 queries each, keys in tiles of 64 straight into LDS, two
// tiles deep.  Scores are computed transposed (keys x queries, K as the A
// operand): a lane then holds 32 of one query's 64 scores, its softmax needs
// one exchange with the lane 32 further on, and the weights are, rounded to the
// storage type, the B operand of V^T x weights as they stand: rows 8 i + 4 h + j
// of a 32 x 32 result (h the lane's half) are K values 8 h + .. of the next
// product if V^T's columns are read in the same order, which the transposing
// LDS read gives (16 lanes read four rows of 16 values and get a column each).
//
// Weights are 2^(score - reference), in [0, 2^8]: the reference is a running
// maximum that moves only when some query's scores exceed it by 8, so most
// tiles leave the output unscaled.  They meet the values in the storage type, as the
// matrix unit takes no other; their sum is that of the fp32 weights.  Rounded once, by
// half a step, they have as much error as the output's own rounding (with random values
// 0.0023 of the output's root mean square against 0.0017 in bf16, 0.00029 against
// 0.00021 in fp16); FINE takes what is left of each as a second weight, and the output's
// rounding is all (0.0017), for products twice and a third more vector instructions.
// fp16's steps end at 2^-24, which many keys far below the maximum would feel (80,000 of
// them 25.05 below it: 0.0023 of the result, five half steps): its weights are 2^7 times
// as large, up to 2^15, and what is lost is 2^-32 a key.
//
// Bound by issue: a tile of 32 queries x 64 keys x 64 channels is 16 products, 512
// clocks of the matrix unit, and its softmax about 580 of the vector unit (per
// value an exponential 8.3, scale and sum 2.7 each, maximum and rounding 2.2), which
// stands still for half of each product's 32.  Counted: 1,060 clocks a tile, and CUs without
// a block for 15 % of the time.  18,216 rows, 8 heads of 64, bf16 768 us (885 TFLOP/s);
// 16,384 rows of 128 channels 986 us, 1,115 TFLOP/s, with twice the products to the same
// softmax.  Products and exponentials written down in turns, and the next tile's scores
// under this one's softmax: 812 -> 791 us.
//
// LDS: rows of 64 or 128 values, chunk c of row r at c ^ f(r): the 16 lanes of
// a K read (16 rows, one chunk) and the 32 of a V read (4 rows x 4 chunks, two of
// them) touch different banks.
template <int DT, int DC, int NW, bool FINE>
__global__ void __launch_bounds__(64 * NW, DC <= 64 ? 3 : 2) k_attention(Attention p, Partial part, int tiles) {
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

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int group = p.heads / p.kv_heads;

    // Neighbouring blocks share a kv head; each XCD takes a contiguous range.
    const int64_t unit = xcd_remap(blockIdx.x, gridDim.x);
    const int split = (int) (unit % part.splits);
    const int kv = (int) (unit / part.splits / tiles);
    const Place at = find_place<TQ>(p, unit / part.splits % tiles, group);
    if (at.nq <= 0) return;
    const int all = (at.nk + TK - 1) / TK;
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
    const float scale = fabsf(p.scale);

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
    // One tile: softmax of `cur`, the scores of tile t, and their products with
    // its values, and the scores of tile t + 1 into `nxt`.  Products and
    // exponentials are written down in turns, in four steps of 16 keys:
    //   step g: weights of group g; the values' products of group g - 1 beside the
    //   first half of them, a quarter of the next scores beside the second.
    // Fragments are read half a step before their products.
    const auto tile = [&](int t, int j, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
        const int left = at.nk - t * TK;
        if (left < TK) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (n * 32 + 8 * (i / 4) + 4 * half + i % 4 >= left) cur[n][i] = -__builtin_inff();
        }
        float m = cur[0][0];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, cur[n][i]);
        m = max_halves(m) * scale;
        if (__any(m > ref + 8.0f)) {
            const float next = fmaxf(ref, m);
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
        // Keys of t + 1 and values of t have landed; every wavefront is done with
        // the keys of t and the values of t - 1.
        wait_vmcnt<0>();
        lds_barrier();
        if (t + 2 < t1) load_k();
        if (t + 1 < t1) load_v();
        // (Past the last tile these are old keys, and the scores are not used.)
        const unsigned char * sk = s_tile + ((j & 1) ^ 1) * TILE;
        const unsigned char * sv = s_tile + (j & 1) * TILE + 2 * TILE;
        zero(nxt[0]);
        zero(nxt[1]);
        constexpr int QPS = KS / 2;  // products of the next scores per step
        s16x8 kf[QPS], vf[DT32], w, rest;
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
#pragma unroll
            for (int i = 0; i < QPS; ++i) kf[i] = read_k(sk, g / 2, g % 2 * QPS + i);
            __builtin_amdgcn_sched_barrier(0);
            if (g > 0) {
#pragma unroll
                for (int d = 0; d < DT32; ++d) {
                    values(d);
#pragma unroll
                    for (int i = 4 * d / DT32; i < 4 * (d + 1) / DT32; ++i) weight(i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) weight(i);
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
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < QPS; ++i) {
                nxt[g / 2] = mac32<DT>(kf[i], q[g % 2 * QPS + i], nxt[g / 2]);
#pragma unroll
                for (int x = 4 + 4 * i / QPS; x < 4 + 4 * (i + 1) / QPS; ++x) weight(x);
                __builtin_amdgcn_sched_barrier(0);
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
        load_k();
        load_v();
        if (t0 + 1 < t1) load_k();
        wait_vmcnt<0>();
        lds_barrier();
        f32x16 sa[2], sb[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            zero(sa[n]);
#pragma unroll
            for (int k = 0; k < KS; ++k) sa[n] = mac32<DT>(read_k(s_tile, n, k), q[k], sa[n]);
        }
        for (int t = t0; t < t1; t += 2) {
            tile(t, 0, sa, sb);
            if (t + 1 >= t1) break;
            tile(t + 1, 1, sb, sa);
        }
    }

    leave<DT>(p, part, out, ref, sum_halves(sum0 + sum1), live, t0 < t1, split, row, head, half);
}

// fp32: as k_attention, with products of two channels, or two keys, at a time.
// The two halves of a wavefront have 4 channels each of every 8 of K's and q's
// rows (the order of a sum's terms is free, so a chunk of 16 bytes serves four
// products as it is read), and score i of a lane, key 8 (i / 4) + 4 half + i % 4, is
// the B operand of the values' product with the rows of V that the halves read.
// These products take 64 clocks each, 4,096 of a tile of 32 queries x 32 keys x
// 64 channels against some 300 of its softmax, which is why nothing is
// interleaved by hand: 18,216 rows, 8 heads of 64 in 5.7 ms, 118 TFLOP/s (129 at
// 128 channels; a large fp32 matrix product of the library reaches 136 to 153),
// where k_attention_any takes 44 ms.  Keys in tiles of 32 straight into LDS, two tiles deep;
// chunk c of row r at c ^ f(r), so that the 16 lanes of a K read (16 rows, one
// chunk) touch different banks.
template <int DC, int NW>
__global__ void __launch_bounds__(64 * NW, 2) k_attention32(Attention p, Partial part, int tiles) {
    constexpr int TQ = 32 * NW, TK = 32;
    constexpr int LP = DC <= 32 ? 32 : (DC <= 64 ? 64 : 128);  // values per LDS row
    constexpr int ROW = LP * 4, CH = LP / 4;
    constexpr int KS = DC / 8, DT32 = DC / 32;
    constexpr int TILE = TK * ROW;
    constexpr int RPL = 64 / CH;
    constexpr int PER = TILE / 1024 / NW;
    static_assert(TILE / 1024 % NW == 0, "whole loads");
    __shared__ __attribute__((aligned(1024))) unsigned char s_tile[4 * TILE];  // K, V of two tiles

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int group = p.heads / p.kv_heads;
    const int64_t unit = xcd_remap(blockIdx.x, gridDim.x);
    const int split = (int) (unit % part.splits);
    const int kv = (int) (unit / part.splits / tiles);
    const Place at = find_place<TQ>(p, unit / part.splits % tiles, group);
    if (at.nq <= 0) return;
    const int all = (at.nk + TK - 1) / TK;
    const int t0 = (int) ((int64_t) all * split / part.splits), t1 = (int) ((int64_t) all * (split + 1) / part.splits);

    const int qi = wave * 32 + l32;
    const int64_t vq = at.first + qi;
    const int64_t row = at.q0 + vq / group;
    const int head = kv * group + (int) (vq % group);
    const bool live = qi < at.nq;
    const float sign = p.scale < 0.0f ? -1.0f : 1.0f, scale = fabsf(p.scale);
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

    f32x16 out[DT32];
#pragma unroll
    for (int d = 0; d < DT32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[d][i] = 0.0f;
    float ref = -__builtin_inff(), sum0 = 0.0f, sum1 = 0.0f;
    if (t0 < t1) load(t0);
    for (int t = t0; t < t1; ++t) {
        // Tile t has landed; every wavefront is done with tile t - 1.
        wait_vmcnt<0>();
        lds_barrier();
        if (t + 1 < t1) load(t + 1);
        const unsigned char * sk = s_tile + ((t - t0) & 1) * TILE;
        const unsigned char * sv = sk + 2 * TILE;
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
        const int left = at.nk - t * TK;
        if (left < TK) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i / 4) + 4 * half + i % 4 >= left) cur[i] = -__builtin_inff();
        }
        float m = cur[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) m = fmaxf(m, cur[i]);
        m = max_halves(m) * scale;
        if (__any(m > ref + 8.0f)) {
            const float next = fmaxf(ref, m);
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
    leave<kF32>(p, part, out, ref, sum_halves(sum0 + sum1), live, t0 < t1, split, row, head, half);
}

template <int DT, int DC, int NW>
hipError_t launch_nw(const Attention & p, const Partial & part, int64_t tiles, bool fine, hipStream_t s) {
    const int64_t grid = tiles * p.kv_heads * part.splits;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    if constexpr (DT == kF32) {
        k_attention32<DC, NW><<<(unsigned) grid, 64 * NW, 0, s>>>(p, part, (int) tiles);
    } else {
        if (fine) {
            k_attention<DT, DC, NW, true><<<(unsigned) grid, 64 * NW, 0, s>>>(p, part, (int) tiles);
        } else {
            k_attention<DT, DC, NW, false><<<(unsigned) grid, 64 * NW, 0, s>>>(p, part, (int) tiles);
        }
    }
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && part.splits > 1) {
        int qp = 1;
        while (qp * 4 < p.dim) qp *= 2;
        // 77 splits of 64 channels: 12 us with a wavefront a query, 6.5 with four.
        const bool wide = part.splits >= 32;
        const int64_t joins = tiles * p.kv_heads * (wide ? 32 * NW : 8 * NW);
        if (joins > 0x7fffffffLL) return hipErrorInvalidValue;
        if (wide) {
            k_join<DT, 32 * NW, 4><<<(unsigned) joins, 256, 0, s>>>(p, part, (int) tiles, qp);
        } else {
            k_join<DT, 32 * NW, 1><<<(unsigned) joins, 256, 0, s>>>(p, part, (int) tiles, qp);
        }
        err = hipGetLastError();
    }
    return err;
}

template <int DT, int DC>
hipError_t launch_dc(const Attention & p, const Partial & part, const AttentionShape & sh, hipStream_t s) {
    return sh.waves == 1 ? launch_nw<DT, DC, 1>(p, part, sh.tiles, sh.fine, s)
                         : launch_nw<DT, DC, 4>(p, part, sh.tiles, sh.fine, s);
}

template <int DT>
hipError_t launch_mfma(const Attention & p, const Partial & part, const AttentionShape & sh, hipStream_t s) {
    if (p.dim <= 32) return launch_dc<DT, 32>(p, part, sh, s);
    if (p.dim <= 64) return launch_dc<DT, 64>(p, part, sh, s);
    if (p.dim <= 96) return launch_dc<DT, 96>(p, part, sh, s);
    return launch_dc<DT, 128>(p, part, sh, s);
}

}  // namespace

AttentionShape attention_shape(int dtype, const Attention & p, int cus) {
    AttentionShape sh{0, 0, 1, 0, false};
    const int chunk = dtype == kF32 ? 4 : 8;  // of 16 bytes
    const auto aligned = [&](const void * ptr, int64_t stride) { return (uintptr_t) ptr % 16 == 0 && stride % chunk == 0; };
    // A tile's rows (64, of fp32 32) stay within a buffer's 2 GiB of offsets.
    constexpr int64_t kMaxStride = 1 << 23;
    if (p.dim % chunk != 0 || p.dim > 128 || !aligned(p.q, p.q_stride) || !aligned(p.k, p.k_stride) ||
        !aligned(p.v, p.v_stride) || !aligned(p.y, p.y_stride) || p.k_stride > kMaxStride || p.v_stride > kMaxStride) {
        return sh;
    }
    const int group = p.heads / p.kv_heads;
    const int64_t queries = p.nq * group, seqs = p.q_at != nullptr ? p.seqs : 1;
    // Sequences of up to 32 queries: one wavefront a block, as the others would only help to load.
    sh.waves = queries <= 32 * seqs ? 1 : 4;
    const int tq = 32 * sh.waves;
    sh.tiles = queries / tq + seqs;
    const int64_t blocks = (queries + tq - 1) / tq * p.kv_heads;
    const int64_t want = (int64_t) cus * 8 / sh.waves;  // two wavefronts per SIMD
    // Few queries: the keys split over more blocks, at least four tiles of 64 each.
    const int64_t key_tiles = (p.nk / seqs + 63) / 64;
    if (blocks < want) sh.splits = (int) std::max<int64_t>(1, std::min(want / std::max<int64_t>(blocks, 1), key_tiles / 4));
    // Few blocks: weights in two parts, for the output's own rounding alone.  Their time is
    // that of loads and latencies: 4 queries on 79,523 keys 33.5 -> 34.9 us, in four sequences
    // 26 -> 29, 1,000 rows of 8 x 64 17.8 -> 18.9, 2,000 30.3 -> 33.6, but 5,003 85 -> 120 and
    // 18,216 792 -> 1,097.
    sh.fine = blocks <= cus / 2;
    if (sh.splits > 1) sh.scratch = (size_t) sh.splits * p.nq * p.heads * (p.dim + 2) * sizeof(float);
    return sh;
}

hipError_t launch_attention(int dtype, const Attention & p, const AttentionShape & sh, void * scratch, hipStream_t s) {
    if (sh.waves == 0) {
        switch (dtype) {
            case kF32: return launch_any<kF32>(p, s);
            case kF16: return launch_any<kF16>(p, s);
            default: return launch_any<kBF16>(p, s);
        }
    }
    Partial part{nullptr, nullptr, 1};
    if (scratch != nullptr && sh.splits > 1) {
        part.splits = sh.splits;
        part.out = (float *) scratch;
        part.stat = (float2 *) (part.out + (size_t) sh.splits * p.nq * p.heads * p.dim);
    }
    if (sh.tiles > 0x7fffffffLL) return hipErrorInvalidValue;
    switch (dtype) {
        case kF32: return launch_mfma<kF32>(p, part, sh, s);
        case kF16: return launch_mfma<kF16>(p, part, sh, s);
        default: return launch_mfma<kBF16>(p, part, sh, s);
    }
}

}  // namespace tsh
