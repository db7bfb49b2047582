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

// 32 bytes of T, in one access
template<class T>
struct Vec32
{
    static constexpr int N = 32 / sizeof(T);
    union
    {
        uint32_t raw[8];
        T        v[N];
    };
    __device__ __forceinline__ Vec32() {}
    __device__ __forceinline__ void load(const T* p) // of read-only data
    {
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]), "=r"(raw[7])
                     : "l"(p));
    }
    __device__ __forceinline__ void store(T* p) const
    {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(p), "r"(raw[0]), "r"(raw[1]), "r"(raw[2]), "r"(raw[3]), "r"(raw[4]), "r"(raw[5]), "r"(raw[6]), "r"(raw[7])
                     : "memory");
    }
};

// e4m3 byte (0..0x7E) to its value: its bits are those of an FP32 number 2^120 times smaller, subnormals included
__device__ __forceinline__ float e4m3_value(unsigned byte) { return __uint_as_float(byte << 20) * 0x1p120f; }
// value of an e8m0 byte below 0xFF: 2^(byte - 127)
__device__ __forceinline__ float e8m0_value(unsigned byte) { return byte ? __uint_as_float(byte << 23) : __uint_as_float(1u << 22); }

constexpr unsigned NAN_E4M3 = 0x7Fu;
constexpr unsigned NAN_E8M0 = 0xFFu;
// the value of a scale byte
template<int FMT>
__device__ __forceinline__ float scale_value(unsigned byte)
{
    const float nan = __uint_as_float(0x7FC00000u);
    if(FMT == B200_SGEMM_NVFP4)
        return (byte & 0x7Fu) == NAN_E4M3 ? nan : e4m3_value(byte);
    return byte == NAN_E8M0 ? nan : e8m0_value(byte);
}

// Launches a kernel and returns this launch's own status; cudaPeekAtLastError would also give what an earlier call that failed
// (an allocation that another entry did not get) left behind.
template<class Args>
int launch_kernel(void (*kernel)(Args), unsigned grid, int threads, cudaStream_t stream, const Args& a)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(grid);
    cfg.blockDim           = dim3((unsigned)threads);
    cfg.stream             = stream;
    return (int)cudaLaunchKernelEx(&cfg, kernel, a);
}

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
