// What the 4-bit operators share: the storage format's sizes, element types, and the arithmetic of codes and scales.
//
// A quantised matrix of `rows` x K (K the summed dimension of a product) is two arrays:
//   codes   rows x ceil(K / 32) * 16 bytes; byte b of a row holds k = 2b in its lower half and 2b + 1 in its upper one.
//   scales  one byte per block of k, in tiles of 128 rows x 4 blocks: 512 bytes, row r and block c at
//           (r % 32) * 16 + (r % 128) / 32 * 4 + c % 4.  Tiles of one band of 128 rows follow each other along k.  This
//           is the order in which tensor memory wants them, so a product copies tiles without touching them.
#pragma once
#include "../../include/b200_sgemm.h"

#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace sgemm_b200
{
constexpr int MX4_BAND       = 128; // rows of one scale tile
constexpr int MX4_TILE_BYTES = 512;

__host__ __device__ constexpr int mx4_block(int format) { return format == B200_SGEMM_NVFP4 ? 16 : 32; }
__host__ __device__ constexpr size_t mx4_pitch(size_t K) { return (K + 31) / 32 * 16; }
// scale tiles along k: four blocks each
__host__ __device__ constexpr size_t mx4_tiles(int format, size_t K)
{
    return (K + 4 * mx4_block(format) - 1) / (4 * mx4_block(format));
}
inline bool   mx4_format_ok(int format) { return format == B200_SGEMM_NVFP4 || format == B200_SGEMM_MXFP4; }
inline bool   type_ok(int type) { return type == B200_SGEMM_F32 || type == B200_SGEMM_F16 || type == B200_SGEMM_BF16; }
inline size_t type_bytes(int type) { return type == B200_SGEMM_F32 ? 4 : 2; }
inline bool   misaligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
constexpr size_t MAX_EXTENT = size_t(1) << 30; // of a dimension, as in the other entries

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template<class T> __device__ __forceinline__ T from_float(float v);
template<> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template<> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template<> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of T
template<class T>
struct Vec16
{
    static constexpr int N = 16 / sizeof(T);
    union
    {
        uint4 raw;
        T     v[N];
    };
    __device__ __forceinline__ Vec16() {}
};

// e4m3 byte (0..0x7E) to its value
__device__ __forceinline__ float e4m3_value(unsigned byte)
{
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(__half(h));
}
// value of an e8m0 byte below 0xFF: 2^(byte - 127)
__device__ __forceinline__ float e8m0_value(unsigned byte) { return byte ? __uint_as_float(byte << 23) : __uint_as_float(1u << 22); }

// f(type as a C++ type) for a checked element type
template<class F>
int with_type(int type, F f)
{
    switch(type)
    {
    case B200_SGEMM_F32: return f(float());
    case B200_SGEMM_F16: return f(__half());
    default: return f(__nv_bfloat16());
    }
}
} // namespace sgemm_b200
