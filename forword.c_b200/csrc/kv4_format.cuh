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

// Four elements of type F32 (0), F16 (1) or BF16 (30) at element `at`.
__device__ __forceinline__ float4 kv4_load4(const void *p, uint64_t at, uint32_t type) {
    if (type == 0) return *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
    if (type == 1) {
        const float2 a = kv4_unpack(w.x), b = kv4_unpack(w.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ void kv4_store4(void *p, uint64_t at, uint32_t type, float4 v) {
    if (type == 0) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = v;
        return;
    }
    uint2 w;
    if (type == 1) {
        w = make_uint2(kv4_pack(v.x, v.y), kv4_pack(v.z, v.w));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) = w;
}

// What a kernel met in its tables, until fwb_kv4_status takes it.
constexpr uint32_t kKvBadPage = 1;      // a page outside the cache
constexpr uint32_t kKvBadPosition = 2;  // a position past the page table or the rotation's tables

}  // namespace fwb
