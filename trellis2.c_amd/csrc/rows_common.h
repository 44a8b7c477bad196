// rows_common.h - device helpers of the row operators: rows as chunks of 16 bytes.
#pragma once
#include "mfma_common.h"

namespace tsh {
namespace {

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

}  // namespace
}  // namespace tsh
