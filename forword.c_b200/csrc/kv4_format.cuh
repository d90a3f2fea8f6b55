// kv4_format.cuh — the paged cache of 4-bit keys and values.
//
// cache [n_page][n_head_kv] lines of page_size / 16 tiles; a tile holds 16
// positions: the codes of their keys (16 rows), the keys' scales, the codes of
// the values, the values' scales.  A row has NB = ceil(head_dim / 32) blocks of
// 32 values: 16 NB bytes of codes and NB fp16 scales; dimensions past head_dim
// stand for zeros.  A code q (0..15) stands for (q - 8) * d.
//
// The codes lie as the m16n8k16 products take them, so that a lane's part of
// a tile is one aligned read and unpacking needs no shuffles:
// * keys: lane (g, c) of a warp (g = lane / 4, c = lane % 4) reads dimensions
//   8c..8c+7 of every block of one row: word (c, b) of the row at byte
//   4 NB c + 4 b; nibble j holds dimension 8c + 2j and nibble j + 4 dimension
//   8c + 2j + 1, so that one mask leaves a pair of neighbours as two halves.
// * values: the products take dimensions as rows and positions as columns.
//   Lane (g, c) reads dimensions 4g..4g+3 of every block of the positions c,
//   c + 4, c + 8, c + 12: the unit of 2 NB bytes at 2 NB (g ^ 4 (p / 2 % 2)) of
//   row p, block b's 16 bits at byte 2 b of it.  The exclusive or spreads the
//   units that a warp reads over all banks.
// Every byte belongs to one position, so positions are written independently.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace fwb {

constexpr uint32_t kKvTile = 16;      // positions of a tile
constexpr uint32_t kKvMaxBlocks = 4;  // of a row: head_dim at most 128

__host__ __device__ constexpr uint32_t kv4_blocks(uint32_t hd) { return (hd + 31) / 32; }
__host__ __device__ constexpr uint32_t kv4_codes(uint32_t nb) { return kKvTile * 16 * nb; }
__host__ __device__ constexpr uint32_t kv4_scales(uint32_t nb) { return kKvTile * 2 * nb; }
__host__ __device__ constexpr uint32_t kv4_tile(uint32_t nb) { return 2 * (kv4_codes(nb) + kv4_scales(nb)); }

__device__ __forceinline__ uint32_t kv4_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 kv4_unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }

// Four elements at element `at`, by type and by GGML's id of it (0, 1, 30).
template <typename T> __device__ __forceinline__ float4 kv4_load4(const void *p, uint64_t at);
template <> __device__ __forceinline__ float4 kv4_load4<float>(const void *p, uint64_t at) {
    return *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
}
template <> __device__ __forceinline__ float4 kv4_load4<__half>(const void *p, uint64_t at) {
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
    const float2 a = kv4_unpack(w.x), b = kv4_unpack(w.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
template <> __device__ __forceinline__ float4 kv4_load4<__nv_bfloat16>(const void *p, uint64_t at) {
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ void kv4_store4(void *p, uint64_t at, float4 v);
template <> __device__ __forceinline__ void kv4_store4<float>(void *p, uint64_t at, float4 v) {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = v;
}
template <> __device__ __forceinline__ void kv4_store4<__half>(void *p, uint64_t at, float4 v) {
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) = make_uint2(kv4_pack(v.x, v.y), kv4_pack(v.z, v.w));
}
template <> __device__ __forceinline__ void kv4_store4<__nv_bfloat16>(void *p, uint64_t at, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
// Eight 16-bit elements.
template <typename T>
__device__ __forceinline__ void kv4_floats8(uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = std::is_same<T, __half>::value ? kv4_unpack(w[i])
                                                        : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
// Eight elements, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void kv4_load8(const void *p, uint64_t at, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = kv4_load4<float>(p, at), b = kv4_load4<float>(p, at + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        kv4_floats8<T>(*reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at), x);
    }
}
template <typename T>
__device__ __forceinline__ void kv4_store8(void *p, uint64_t at, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        kv4_store4<float>(p, at, make_float4(x[0], x[1], x[2], x[3]));
        kv4_store4<float>(p, at + 4, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                w[i] = kv4_pack(x[2 * i], x[2 * i + 1]);
            } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&b);
            }
        }
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ float4 kv4_load4(const void *p, uint64_t at, uint32_t type) {
    return type == 0 ? kv4_load4<float>(p, at) : type == 1 ? kv4_load4<__half>(p, at) : kv4_load4<__nv_bfloat16>(p, at);
}
__device__ __forceinline__ void kv4_store4(void *p, uint64_t at, uint32_t type, float4 v) {
    if (type == 0) kv4_store4<float>(p, at, v);
    else if (type == 1) kv4_store4<__half>(p, at, v);
    else kv4_store4<__nv_bfloat16>(p, at, v);
}

// What a kernel met in its tables, until fwb_kv4_status takes it.
constexpr uint32_t kKvBadPage = 1;      // a page outside the cache
constexpr uint32_t kKvBadPosition = 2;  // a position past the page table or the rotation's tables

}  // namespace fwb
