// b200_sgemm_mx4_quantize / b200_sgemm_mx4_dequantize: FP32, FP16 or BF16 matrices to microscaled 4-bit floating point
// and back.  Both are bound by HBM: each value is read once and each code written once, in one kernel.
//
// Definition, in exact arithmetic (RN = round to nearest, ties to the even code; a block is 16 or 32 neighbours along k):
//   nvfp4   s = RN_e4m3(amax / (6 g)), at most 448;      code = RN_e2m1(x / (s g)), at most 6
//   mxfp4   s = 2^(floor(log2 amax) - 2), in 2^+-127;    code = RN_e2m1(x / s),     at most 6
// amax is the block's largest magnitude, g the matrix's FP32 scale.  s = 0 (nvfp4, a block far below g) gives codes 0.
// A block that holds an infinity or a NaN has the NaN scale and codes 0, so whatever is computed from it is NaN.
//
// How the kernel stays exact without dividing in 64 bits.  mxfp4: x / s is a multiplication by a power of two.  nvfp4:
//   * the scale: the quotient in FP32 is off by a few units, so its rounding is off by one step at most; the sign of
//     amax - 6 m g for the midpoints m on both sides of it, which one fused multiply-add gives exactly (6 m has seven
//     bits), says whether to move.
//   * the codes, g with at most 17 significant bits (1.0, powers of two): s g is exact in 21 bits, so every midpoint
//     t s g is an FP32 number; the correctly rounded quotient (one product and two fused multiply-adds) is then on the
//     same side of t as x / (s g), or on t when that is.
//   * any other g: the quotient is a product with the reciprocal, off by three units at most.  Midpoints have two bits
//     after the leading one; where a quotient comes within eight units of such a number (one in 10^5) the block is done
//     again by the signs of |x| - (t s) g, exact as above.
#include "mx4_common.cuh"

namespace
{
using namespace sgemm_b200;

constexpr int Q_THREADS = 256;
constexpr int Q_LANE_K  = 16;            // k of one lane: a block of nvfp4, half of one of mxfp4
constexpr int Q_TILE_K  = 32 * Q_LANE_K; // k of one warp's step, and of one CTA
constexpr int Q_COL_K   = 128;           // k of one CTA when the rows are the contiguous dimension

constexpr unsigned INF_BITS  = 0x7F800000u;
constexpr unsigned NAN_E4M3  = 0x7Fu;
constexpr unsigned NAN_E8M0  = 0xFFu;

// the matrix's scale, as every thread needs it
struct Global
{
    float g, r6;   // 1 / (6 g)
    bool  ok, few; // ok: finite and in 2^+-90, where none of the products below can leave FP32's range; few: <= 17 bits
};
__device__ __forceinline__ Global load_global(const float* p)
{
    Global G;
    G.g   = p ? *p : 1.f;
    G.r6  = __frcp_rn(6.f * G.g);
    G.ok  = G.g >= 0x1p-90f && G.g <= 0x1p90f;
    G.few = (__float_as_uint(G.g) & 0x7Fu) == 0;
    return G;
}

struct Scale
{
    unsigned byte;
    float    s, sg, inv; // value, s * g, 1 / (s g); inv = 0 for a block whose codes are all 0
};

__device__ __forceinline__ Scale scale_nvfp4(unsigned amax_bits, const Global& G)
{
    Scale       r;
    const float amax = __uint_as_float(amax_bits);
    unsigned    c    = __nv_cvt_float_to_fp8(amax * G.r6, __NV_SATFINITE, __NV_E4M3);
    float       v    = e4m3_value(c);
    if(c < 0x7Eu)
    {
        const float up = e4m3_value(c + 1);
        const float d  = fmaf(-3.f * (v + up), G.g, amax); // amax - 6 * (v + up) / 2 * g
        if(d > 0.f || (d == 0.f && (c & 1u)))
        {
            ++c;
            v = up;
        }
    }
    if(c > 0u)
    {
        const float dn = e4m3_value(c - 1);
        const float d  = fmaf(-3.f * (v + dn), G.g, amax);
        if(d < 0.f || (d == 0.f && (c & 1u)))
        {
            --c;
            v = dn;
        }
    }
    const bool bad = amax_bits >= INF_BITS || !G.ok;
    r.byte = bad ? NAN_E4M3 : c;
    r.s    = v;
    r.sg   = v * G.g;
    r.inv  = bad || c == 0u ? 0.f : __frcp_rn(r.sg);
    return r;
}
__device__ __forceinline__ Scale scale_mxfp4(unsigned amax_bits)
{
    Scale     r;
    const int e = max((int)(amax_bits >> 23) - 129, -127); // floor(log2 amax) - 2; subnormal amax: -127
    const bool bad = amax_bits >= INF_BITS;
    r.byte = bad ? NAN_E8M0 : (unsigned)(e + 127);
    r.s = r.sg = 0.f;
    r.inv = bad ? 0.f : __uint_as_float((unsigned)(127 - e) << 23);
    return r;
}

// code of one value by exact comparison with the midpoints
__device__ __noinline__ unsigned code_exact(float x, float s, float g)
{
    const float a    = fabsf(x);
    unsigned    code = 0;
    const float mid[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.f};
#pragma unroll
    for(int i = 0; i < 7; ++i)
    {
        const float d = fmaf(-(mid[i] * s), g, a);
        code += d > 0.f || (d == 0.f && (i & 1)) ? 1u : 0u;
    }
    return code | (__float_as_uint(x) >> 31 << 3);
}

// sixteen codes, eight bytes
template<int FMT>
__device__ __forceinline__ uint2 encode(const float (&x)[Q_LANE_K], const Scale& sc, const Global& G)
{
    uint2 out = make_uint2(0u, 0u);
    if(sc.inv == 0.f)
        return out;
    float y[Q_LANE_K];
    bool  near = false;
    if(FMT == B200_SGEMM_MXFP4)
    {
#pragma unroll
        for(int i = 0; i < Q_LANE_K; ++i)
            y[i] = x[i] * sc.inv;
    }
    else if(G.few)
    {
#pragma unroll
        for(int i = 0; i < Q_LANE_K; ++i)
        {
            const float q = x[i] * sc.inv;
            y[i]          = copysignf(fmaf(fmaf(-q, sc.sg, x[i]), sc.inv, q), x[i]); // -0 keeps its sign
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < Q_LANE_K; ++i)
        {
            y[i] = x[i] * sc.inv;
            near = near || ((__float_as_uint(y[i]) + 8u) & 0x1FFFFFu) <= 16u;
        }
    }
    if(near)
    {
#pragma unroll
        for(int i = 0; i < Q_LANE_K; ++i)
        {
            const unsigned c = code_exact(x[i], sc.s, G.g);
            if(i < 8)
                out.x |= c << (4 * i);
            else
                out.y |= c << (4 * (i - 8));
        }
        return out;
    }
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        out.x |= (unsigned)__nv_cvt_float2_to_fp4x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_E2M1, cudaRoundNearest) << (8 * i);
        out.y |= (unsigned)__nv_cvt_float2_to_fp4x2(make_float2(y[8 + 2 * i], y[9 + 2 * i]), __NV_E2M1, cudaRoundNearest) << (8 * i);
    }
    return out;
}

__device__ __forceinline__ unsigned amax16(const float (&x)[Q_LANE_K])
{
    unsigned m = 0;
#pragma unroll
    for(int i = 0; i < Q_LANE_K; ++i)
        m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu); // NaN orders above infinity
    return m;
}

struct QArgs
{
    const void*  x;
    const float* global;
    const int*   row_index; // gather: matrix row r is X row row_index[r] / index_div; a negative index leaves row r out
    uint8_t*     codes;
    uint8_t*     scales;
    long long    ld, pitch;
    int          rows, source_rows, K, tiles, index_div;
    int          vector; // base and pitch of X allow 16-byte loads
};

// position of (row in band, block in CTA) in the staged scale tiles; the pad keeps tiles in different banks
constexpr int Q_TILE_PAD = MX4_TILE_BYTES + 16;
__device__ __forceinline__ int scale_at(int row, int block)
{
    return (block >> 2) * Q_TILE_PAD + (row & 31) * 16 + (row >> 5) * 4 + (block & 3);
}
// staged tiles to their place; the band's tiles from `first` on
__device__ __forceinline__ void store_scales(const uint8_t* staged, const QArgs& a, int band, int first, int count)
{
    count = min(count, a.tiles - first);
    uint4* dst = reinterpret_cast<uint4*>(a.scales + ((size_t)band * a.tiles + first) * MX4_TILE_BYTES);
    for(int i = threadIdx.x; i < count * (MX4_TILE_BYTES / 16); i += Q_THREADS)
        dst[i] = *reinterpret_cast<const uint4*>(staged + (i >> 5) * Q_TILE_PAD + (i & 31) * 16);
}

// K-contiguous source.  One CTA: a band of 128 rows x 512 k; a warp takes a row at a time, a lane 16 neighbours of it,
// so a row is read and written in contiguous pieces of a warp's width.  The scales of the band meet in shared memory
// and leave as whole tiles.
template<int FMT, class T>
__global__ void __launch_bounds__(Q_THREADS) quantize_rows_kernel(const __grid_constant__ QArgs a)
{
    constexpr int BLOCKS = Q_TILE_K / (FMT == B200_SGEMM_NVFP4 ? 16 : 32), TILES = BLOCKS / 4;
    __shared__ __align__(16) uint8_t staged[TILES * Q_TILE_PAD];
    __shared__ int any;
    const int  k_ctas = (a.K + Q_TILE_K - 1) / Q_TILE_K;
    const int  band = blockIdx.x / k_ctas, kc = blockIdx.x % k_ctas;
    const int  warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int  k0 = kc * Q_TILE_K + lane * Q_LANE_K;
    const T*   X  = static_cast<const T*>(a.x);
    if(a.row_index) // a band of the sorted rows that holds none is left alone
    {
        if(threadIdx.x == 0)
            any = 0;
        __syncthreads();
        const int r = band * MX4_BAND + threadIdx.x;
        if(threadIdx.x < MX4_BAND && r < a.rows && a.row_index[r] >= 0)
            any = 1;
        __syncthreads();
        if(!any)
            return;
    }
    const Global G = load_global(a.global);
    for(int i = threadIdx.x; i < TILES * Q_TILE_PAD / 16; i += Q_THREADS)
        reinterpret_cast<uint4*>(staged)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int in_band = min(MX4_BAND, a.rows - band * MX4_BAND);
#pragma unroll 2
    for(int r = warp; r < in_band; r += Q_THREADS / 32)
    {
        const long long row = (long long)band * MX4_BAND + r;
        long long       src = row;
        if(a.row_index)
        {
            const int index = a.row_index[row];
            src             = index < 0 ? -1 : index / a.index_div;
            if(src < 0 || src >= a.source_rows)
                continue; // uniform over the warp
        }
        const T* from = X + src * a.ld + k0;
        float    x[Q_LANE_K];
        if(a.vector && k0 + Q_LANE_K <= a.K)
        {
            constexpr int N = Vec16<T>::N;
            Vec16<T>      v[Q_LANE_K / N];
#pragma unroll
            for(int i = 0; i < Q_LANE_K / N; ++i)
                v[i].raw = __ldg(reinterpret_cast<const uint4*>(from) + i);
#pragma unroll
            for(int i = 0; i < Q_LANE_K; ++i)
                x[i] = to_float(v[i / N].v[i % N]);
        }
        else
        {
#pragma unroll
            for(int i = 0; i < Q_LANE_K; ++i)
                x[i] = k0 + i < a.K ? to_float(from[i]) : 0.f;
        }
        unsigned amax = amax16(x);
        if(FMT == B200_SGEMM_MXFP4)
            amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        const Scale sc = FMT == B200_SGEMM_NVFP4 ? scale_nvfp4(amax, G) : scale_mxfp4(amax);
        const uint2 c  = encode<FMT>(x, sc, G);
        if(k0 < 2 * a.pitch)
            *reinterpret_cast<uint2*>(a.codes + row * a.pitch + k0 / 2) = c;
        if(FMT == B200_SGEMM_NVFP4)
            staged[scale_at(r, lane)] = (uint8_t)sc.byte;
        else if((lane & 1) == 0)
            staged[scale_at(r, lane >> 1)] = (uint8_t)sc.byte;
    }
    __syncthreads();
    store_scales(staged, a, band, kc * TILES, TILES);
}

// Row-contiguous source (a col-major A, a row-major B).  One CTA: a band of 128 rows x 128 k; a thread takes one row and
// 64 k, lanes take neighbouring rows, so every load is contiguous over the warp and a thread has whole blocks in
// registers; its 32 code bytes are one sector.
template<int FMT, class T>
__global__ void __launch_bounds__(Q_THREADS) quantize_cols_kernel(const __grid_constant__ QArgs a)
{
    constexpr int BLOCKS = Q_COL_K / (FMT == B200_SGEMM_NVFP4 ? 16 : 32), TILES = BLOCKS / 4;
    __shared__ __align__(16) uint8_t staged[TILES * Q_TILE_PAD];
    const int       k_ctas = (a.K + Q_COL_K - 1) / Q_COL_K;
    const int       band = blockIdx.x / k_ctas, kc = blockIdx.x % k_ctas;
    const int       r = threadIdx.x & (MX4_BAND - 1), half = threadIdx.x / MX4_BAND;
    const long long row = (long long)band * MX4_BAND + r;
    const T*        X   = static_cast<const T*>(a.x);
    const Global    G   = load_global(a.global);
    const bool      in  = row < a.rows;
#pragma unroll
    for(int j = 0; j < 2; ++j) // 32 k at a time
    {
        const int k0 = kc * Q_COL_K + half * 64 + j * 32;
        float     x[2][Q_LANE_K];
#pragma unroll
        for(int i = 0; i < 32; ++i)
            x[i / 16][i % 16] = in && k0 + i < a.K ? to_float(X[(long long)(k0 + i) * a.ld + row]) : 0.f;
        unsigned amax[2] = {amax16(x[0]), amax16(x[1])};
        Scale    sc[2];
        if(FMT == B200_SGEMM_MXFP4)
            sc[0] = sc[1] = scale_mxfp4(max(amax[0], amax[1]));
        else
        {
            sc[0] = scale_nvfp4(amax[0], G);
            sc[1] = scale_nvfp4(amax[1], G);
        }
        const uint2 lo = encode<FMT>(x[0], sc[0], G), hi = encode<FMT>(x[1], sc[1], G);
        if(in && k0 < 2 * a.pitch)
            *reinterpret_cast<uint4*>(a.codes + row * a.pitch + k0 / 2) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        const int block = (half * 64 + j * 32) / (FMT == B200_SGEMM_NVFP4 ? 16 : 32);
        staged[scale_at(r, block)] = in ? (uint8_t)sc[0].byte : 0;
        if(FMT == B200_SGEMM_NVFP4)
            staged[scale_at(r, block + 1)] = in ? (uint8_t)sc[1].byte : 0;
    }
    __syncthreads();
    store_scales(staged, a, band, kc * TILES, TILES);
}

struct DArgs
{
    const uint8_t* codes;
    const uint8_t* scales;
    const float*   global;
    void*          x;
    long long      ld, pitch;
    int            rows, K, tiles;
    int            vector;
};

// One CTA: a band of 128 rows x 512 k.  The scale tiles come in whole; a lane turns 16 bytes of output at a time, so that
// a warp's stores are contiguous.
template<int FMT, class T>
__global__ void __launch_bounds__(Q_THREADS) dequantize_kernel(const __grid_constant__ DArgs a)
{
    constexpr int BLOCK = FMT == B200_SGEMM_NVFP4 ? 16 : 32, TILES = Q_TILE_K / BLOCK / 4;
    constexpr int N = Vec16<T>::N;
    __shared__ __align__(16) uint8_t staged[TILES * Q_TILE_PAD];
    const int k_ctas = (a.K + Q_TILE_K - 1) / Q_TILE_K;
    const int band = blockIdx.x / k_ctas, kc = blockIdx.x % k_ctas;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    {
        const int    count = min(TILES, a.tiles - kc * TILES);
        const uint4* src = reinterpret_cast<const uint4*>(a.scales + ((size_t)band * a.tiles + kc * TILES) * MX4_TILE_BYTES);
        for(int i = threadIdx.x; i < count * (MX4_TILE_BYTES / 16); i += Q_THREADS)
            *reinterpret_cast<uint4*>(staged + (i >> 5) * Q_TILE_PAD + (i & 31) * 16) = __ldg(src + i);
    }
    const float g = a.global ? *a.global : 1.f;
    __syncthreads();
    const int in_band = min(MX4_BAND, a.rows - band * MX4_BAND);
    for(int r = warp; r < in_band; r += Q_THREADS / 32)
    {
        const long long row = (long long)band * MX4_BAND + r;
#pragma unroll
        for(int step = 0; step < Q_TILE_K / (32 * N); ++step)
        {
            const int kl = step * 32 * N + lane * N, k0 = kc * Q_TILE_K + kl;
            if(k0 >= a.K)
                break;
            const uint8_t* from = a.codes + row * a.pitch + k0 / 2;
            unsigned       c;
            if(N == 8)
                c = __ldg(reinterpret_cast<const unsigned*>(from));
            else
                c = __ldg(reinterpret_cast<const unsigned short*>(from));
            const unsigned byte = staged[scale_at(r, kl / BLOCK)];
            const float    s    = FMT == B200_SGEMM_NVFP4
                                      ? ((byte & 0x7Fu) == NAN_E4M3 ? __uint_as_float(0x7FC00000u) : e4m3_value(byte))
                                      : (byte == NAN_E8M0 ? __uint_as_float(0x7FC00000u) : e8m0_value(byte));
            Vec16<T> out;
#pragma unroll
            for(int i = 0; i < N / 2; ++i)
            {
                const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(c >> (8 * i) & 0xFFu), __NV_E2M1);
                const float2      f = __half22float2(__half2(h));
                out.v[2 * i]     = from_float<T>(f.x * s * g); // f * s is exact
                out.v[2 * i + 1] = from_float<T>(f.y * s * g);
            }
            T* to = static_cast<T*>(a.x) + row * a.ld + k0;
            if(a.vector && k0 + N <= a.K)
                *reinterpret_cast<uint4*>(to) = out.raw;
            else
            {
#pragma unroll
                for(int i = 0; i < N; ++i)
                    if(k0 + i < a.K)
                        to[i] = out.v[i];
            }
        }
    }
}

// CTAs of bands x pieces of k, or 0 when that is more than a grid holds
unsigned grid_of(size_t rows, size_t K, size_t tile_k)
{
    const unsigned long long n = (unsigned long long)((rows + MX4_BAND - 1) / MX4_BAND) * ((K + tile_k - 1) / tile_k);
    return n > 0x7fffffffull ? 0u : (unsigned)n;
}
} // namespace

extern "C" size_t b200_sgemm_mx4_code_bytes(int format, size_t rows, size_t K)
{
    return !mx4_format_ok(format) || rows > MAX_EXTENT || K > MAX_EXTENT ? 0 : rows * mx4_pitch(K);
}

extern "C" size_t b200_sgemm_mx4_scale_bytes(int format, size_t rows, size_t K)
{
    return !mx4_format_ok(format) || rows > MAX_EXTENT || K > MAX_EXTENT
               ? 0
               : (rows + MX4_BAND - 1) / MX4_BAND * mx4_tiles(format, K) * MX4_TILE_BYTES;
}

extern "C" int b200_sgemm_mx4_quantize(int format, int layout, int type, const void* X, size_t rows, size_t K, size_t ldx,
                                       const int* row_index, size_t source_rows, int index_div, const float* global_scale,
                                       void* codes, void* scales, void* cuda_stream)
{
    if(!X || !codes || !scales || rows == 0 || K == 0 || !mx4_format_ok(format) || !type_ok(type) || layout & ~1)
        return B200_SGEMM_INVALID_ARGUMENT;
    if(rows > MAX_EXTENT || K > MAX_EXTENT || source_rows > MAX_EXTENT)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    const bool row_major = layout == B200_SGEMM_ROW_MAJOR;
    if(row_index ? (!row_major || source_rows == 0 || index_div < 1) : source_rows != 0)
        return B200_SGEMM_INVALID_ARGUMENT;
    const size_t extent = row_major ? K : rows;
    if(ldx == 0)
        ldx = extent;
    if(ldx < extent || misaligned(X, type_bytes(type)) || misaligned(codes, 16) || misaligned(scales, 16)
       || misaligned(row_index, 4) || misaligned(global_scale, 4) || (format == B200_SGEMM_MXFP4 && global_scale))
        return B200_SGEMM_INVALID_ARGUMENT;
    const unsigned grid = grid_of(rows, K, row_major ? Q_TILE_K : Q_COL_K);
    if(!grid || ldx > (size_t(1) << 40))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    QArgs a;
    a.x           = X;
    a.global      = global_scale;
    a.row_index   = row_index;
    a.codes       = static_cast<uint8_t*>(codes);
    a.scales      = static_cast<uint8_t*>(scales);
    a.ld          = (long long)ldx;
    a.pitch       = (long long)mx4_pitch(K);
    a.rows        = (int)rows;
    a.source_rows = (int)source_rows;
    a.K           = (int)K;
    a.tiles       = (int)mx4_tiles(format, K);
    a.index_div   = index_div;
    a.vector      = !misaligned(X, 16) && ldx * type_bytes(type) % 16 == 0;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if(row_major)
        {
            if(format == B200_SGEMM_NVFP4)
                quantize_rows_kernel<B200_SGEMM_NVFP4, T><<<grid, Q_THREADS, 0, stream>>>(a);
            else
                quantize_rows_kernel<B200_SGEMM_MXFP4, T><<<grid, Q_THREADS, 0, stream>>>(a);
        }
        else
        {
            if(format == B200_SGEMM_NVFP4)
                quantize_cols_kernel<B200_SGEMM_NVFP4, T><<<grid, Q_THREADS, 0, stream>>>(a);
            else
                quantize_cols_kernel<B200_SGEMM_MXFP4, T><<<grid, Q_THREADS, 0, stream>>>(a);
        }
        return (int)cudaPeekAtLastError();
    });
}

extern "C" int b200_sgemm_mx4_dequantize(int format, int type, const void* codes, const void* scales, size_t rows, size_t K,
                                         const float* global_scale, void* X, size_t ldx, void* cuda_stream)
{
    if(!X || !codes || !scales || rows == 0 || K == 0 || !mx4_format_ok(format) || !type_ok(type))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(rows > MAX_EXTENT || K > MAX_EXTENT)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    if(ldx == 0)
        ldx = K;
    if(ldx < K || misaligned(X, type_bytes(type)) || misaligned(codes, 16) || misaligned(scales, 16)
       || misaligned(global_scale, 4) || (format == B200_SGEMM_MXFP4 && global_scale))
        return B200_SGEMM_INVALID_ARGUMENT;
    const unsigned grid = grid_of(rows, K, Q_TILE_K);
    if(!grid || ldx > (size_t(1) << 40))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    DArgs a;
    a.codes  = static_cast<const uint8_t*>(codes);
    a.scales = static_cast<const uint8_t*>(scales);
    a.global = global_scale;
    a.x      = X;
    a.ld     = (long long)ldx;
    a.pitch  = (long long)mx4_pitch(K);
    a.rows   = (int)rows;
    a.K      = (int)K;
    a.tiles  = (int)mx4_tiles(format, K);
    a.vector = !misaligned(X, 16) && ldx * type_bytes(type) % 16 == 0;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if(format == B200_SGEMM_NVFP4)
            dequantize_kernel<B200_SGEMM_NVFP4, T><<<grid, Q_THREADS, 0, stream>>>(a);
        else
            dequantize_kernel<B200_SGEMM_MXFP4, T><<<grid, Q_THREADS, 0, stream>>>(a);
        return (int)cudaPeekAtLastError();
    });
}
