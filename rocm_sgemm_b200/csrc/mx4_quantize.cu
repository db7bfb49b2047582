// b200_sgemm_mx4_quantize / b200_sgemm_mx4_dequantize: FP32, FP16 or BF16 matrices to microscaled 4-bit floating point
// and back.  Both are bound by HBM: each value is read once and each code written once, in one kernel.
//
// Definition, in exact arithmetic (RN = round to nearest, ties to the even code; a block is 16 or 32 neighbours along k):
//   nvfp4   s = RN_e4m3(amax / (6 g)), at most 448;      code = RN_e2m1(x / (s g)), at most 6
//   mxfp4   s = 2^(floor(log2 amax) - 2), in 2^+-127;    code = RN_e2m1(x / s),     at most 6
// amax is the block's largest magnitude, g the matrix's FP32 scale.  s = 0 (nvfp4, a block far below g) gives codes 0; a block
// of zeros has s = 0 for every finite g >= 0, so that g = amax / 2688 of a matrix of zeros does.
// A block that holds an infinity or a NaN has the NaN scale and codes 0, so whatever is computed from it is NaN.
//
// How the kernel stays exact without dividing in 64 bits.  mxfp4: x / s is a multiplication by a power of two.  nvfp4:
//   * the scale: the quotient in FP32 is off by a few units, so its rounding is off by one step at most; the sign of
//     amax - 6 m g for the midpoints m on both sides of it, which one fused multiply-add gives exactly (6 m has seven
//     bits), says whether to move.
//   * the codes, g with at most 12 significant bits (1.0, powers of two): s g is exact in 16 bits and every midpoint t s g an
//     FP32 number, which the next FP32 number x is so far from that the quotient in FP32 (one product and two fused
//     multiply-adds, off by 2^-45 before its rounding) is t only if x / (s g) is: the closest case, t = 1/4 and s g just below a
//     power of two, leaves 2^-40.  A block with the largest scale, the only one whose x / (s g) can leave FP32's range, goes the
//     other way, where a product may become infinite: here the fused multiply-adds would take infinities from each other.
//   * any other g: products with the reciprocal, made a little too small and a little too large (2^-21, five roundings of
//     2^-24 lie in between), bracket the quotient.  Where their codes differ the value is read again and the sign of
//     |x| - (t s) g decides, exact as above.  That is rare for random g, but g = amax / 2688 of BF16 data makes every
//     hundredth block hold such a value, so a warp meets one in most rows: the repair has to be cheap (doing all sixteen
//     values again by comparisons took 271 us for 16384 x 8192 BF16 where g was of that kind, 151 us where not).
#include "mx4_common.cuh"

#include <type_traits>

namespace
{
using namespace sgemm_b200;

constexpr int Q_THREADS = 256;
constexpr int Q_LANE_K  = 16;            // k of one lane: a block of nvfp4, half of one of mxfp4
constexpr int Q_TILE_K  = 32 * Q_LANE_K; // k of one warp's step, and of one CTA
constexpr int Q_WARP_ROWS = 4;           // rows of one warp
constexpr int Q_ROWS      = Q_THREADS / 32 * Q_WARP_ROWS;
static_assert(Q_ROWS == 32, "the rows of a CTA lie 16 bytes apart in a scale tile");
constexpr int Q_COL_K   = 128;           // k of one CTA when the rows are the contiguous dimension

constexpr unsigned INF_BITS  = 0x7F800000u;
constexpr unsigned MAX_E4M3  = 0x7Eu; // 448

// the matrix's scale, as every thread needs it
struct Global
{
    float    g, r6; // 1 / (6 g), or 0 where g is not in 2^+-90, in which none of the products below can leave FP32's range
    unsigned limit; // largest magnitudes from these bits on give NaN: infinity; 1 where g is not in 2^+-90, 0 where it is no scale
    bool     few;   // g has <= 12 bits
};
__device__ __forceinline__ Global load_global(const float* p)
{
    Global G;
    G.g = p ? *p : 1.f;
    const bool ok = G.g >= 0x1p-90f && G.g <= 0x1p90f;
    G.r6    = ok ? __frcp_rn(6.f * G.g) : 0.f;
    G.limit = ok ? INF_BITS : (G.g >= 0.f && G.g < __uint_as_float(INF_BITS) ? 1u : 0u);
    G.few   = (__float_as_uint(G.g) & 0xFFFu) == 0;
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
    // amax - 6 m g for the midpoints m above and below c (half a step on in the bits)
    const float above = fmaf(-(__uint_as_float((2 * c + 1) << 19) * (6.f * 0x1p120f)), G.g, amax);
    const float below = fmaf(-(__uint_as_float((2 * c - 1) << 19) * (6.f * 0x1p120f)), G.g, amax);
    if(c < MAX_E4M3 && (above > 0.f || (above == 0.f && (c & 1u))))
        ++c;
    else if(c > 0u && (below < 0.f || (below == 0.f && (c & 1u))))
        --c;
    const bool bad = amax_bits >= G.limit;
    r.byte = bad ? NAN_E4M3 : c;
    r.s    = e4m3_value(c);
    r.sg   = r.s * G.g;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inv) : "f"(r.sg)); // within 2^-23; s g is in 2^+-100
    r.inv = bad || c == 0u ? 0.f : r.inv;
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

// what a code 0..7 stands for
__device__ __forceinline__ float e2m1_value(unsigned code) { return __uint_as_float(code << 22) * 0x1p126f; }

// the codes nearest to y[0..7], four bytes, without moving bytes by hand
__device__ __forceinline__ unsigned codes8(const float2* y)
{
    unsigned r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(y[0].x), "f"(y[0].y), "f"(y[1].x), "f"(y[1].y), "f"(y[2].x), "f"(y[2].y), "f"(y[3].x), "f"(y[3].y));
    return r;
}
__device__ __forceinline__ uint2 codes16(const float2 (&y)[Q_LANE_K / 2]) { return make_uint2(codes8(y), codes8(y + 4)); }
// y = x * f, two values an instruction
__device__ __forceinline__ void scaled16(float2 (&y)[Q_LANE_K / 2], const float (&x)[Q_LANE_K], float f)
{
#pragma unroll
    for(int i = 0; i < Q_LANE_K / 2; ++i)
        y[i] = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(f, f));
}

// Sign of |x| minus the midpoint above code `code`: exact.
__device__ __forceinline__ float beyond_midpoint(float x, unsigned code, const Scale& sc, const Global& G)
{
    const float mid = 0.5f * (e2m1_value(code) + e2m1_value(code + 1));
    return fmaf(-(mid * sc.s), G.g, fabsf(x));
}

// Settles the nibbles in which `low` and `high` (one more) differ.  again(i) is x[i].
//   FP32    one by one.
//   FP16 and BF16, all at once: such an x lies within 2^-20 of t s g, so the quotient x / (t s), eleven bits over seven, is
//           that close to g.  Two such quotients of one binade are at least 2^-18 apart, so all values of the matrix that need
//           settling have the same quotient and lie on the same side, or all on their midpoints.
template<class T, class Again>
__device__ __forceinline__ uint2 settle(uint2 low, uint2 high, const Scale& sc, const Global& G, Again again)
{
    if constexpr(sizeof(T) == 2)
    {
        const bool     second = low.x == high.x;
        const unsigned word = second ? low.y : low.x, left = second ? low.y ^ high.y : low.x ^ high.x;
        const int      i = (__ffs(left) - 1) >> 2;
        const float    d = beyond_midpoint(again(second ? 8 + i : i), word >> (4 * i) & 7u, sc, G);
        if(d > 0.f)
            return high;
        if(d == 0.f) // each to the even one: up by one where the nibbles differ and the lower is odd
        {
            const unsigned x = low.x ^ high.x, y = low.y ^ high.y;
            low.x += (x | x >> 1 | x >> 2) & low.x & 0x11111111u;
            low.y += (y | y >> 1 | y >> 2) & low.y & 0x11111111u;
        }
    }
    else
    {
#pragma unroll
        for(int half = 0; half < 2; ++half)
        {
            unsigned& word = half ? low.y : low.x;
            for(unsigned left = word ^ (half ? high.y : high.x); left;)
            {
                const int      i    = (__ffs(left) - 1) >> 2;
                const unsigned code = word >> (4 * i) & 7u;
                const float    d    = beyond_midpoint(again(8 * half + i), code, sc, G);
                if(d > 0.f || (d == 0.f && (code & 1u)))
                    word += 1u << (4 * i);
                left &= ~(0xFu << (4 * i));
            }
        }
    }
    return low;
}

// sixteen codes, eight bytes
template<int FMT, class T, class Again>
__device__ __forceinline__ uint2 encode(const float (&x)[Q_LANE_K], const Scale& sc, const Global& G, Again again)
{
    if(sc.inv == 0.f)
        return make_uint2(0u, 0u);
    float2 y[Q_LANE_K / 2];
    if(FMT == B200_SGEMM_MXFP4)
    {
        scaled16(y, x, sc.inv);
        return codes16(y);
    }
    if(G.few && sc.byte != MAX_E4M3)
    {
#pragma unroll
        for(int i = 0; i < Q_LANE_K; ++i)
        {
            const float q = x[i] * sc.inv;
            const float v = copysignf(fmaf(fmaf(-q, sc.sg, x[i]), sc.inv, q), x[i]); // -0 keeps its sign
            if(i & 1)
                y[i / 2].y = v;
            else
                y[i / 2].x = v;
        }
        return codes16(y);
    }
    scaled16(y, x, sc.inv * (1.f - 0x1p-21f));
    uint2 low = codes16(y);
    scaled16(y, x, sc.inv * (1.f + 0x1p-21f));
    const uint2 high = codes16(y);
    if(low.x != high.x || low.y != high.y)
        low = settle<T>(low, high, sc, G, again);
    return low;
}

// largest magnitude as bits; NaN where there is one
__device__ __forceinline__ unsigned amax16(const float (&x)[Q_LANE_K])
{
    float m = 0.f;
#pragma unroll
    for(int i = 0; i < Q_LANE_K; i += 2)
        asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(x[i])), "f"(fabsf(x[i + 1])));
    return __float_as_uint(m);
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
    int          vector; // base and pitch of X allow loads of 32 (rows) or 4 bytes (columns)
};

// address of (row, block) in the scales
__device__ __forceinline__ size_t scale_at(long long row, int block, int tiles)
{
    return ((size_t)(row / MX4_BAND) * tiles + (block >> 2)) * MX4_TILE_BYTES + (row & 31) * 16 + ((row & (MX4_BAND - 1)) >> 5) * 4
           + (block & 3);
}

// K-contiguous source.  One CTA: 32 rows (a quarter of a band) x 512 k.  A warp takes four rows, the next fetched while one is
// worked on, a lane 16 neighbours of each in one or two 32-byte loads; codes leave in contiguous pieces of a warp's width.  Scales meet in shared
// memory and leave as words of four blocks.  Rows off 32 bytes are read element by element: 16384 x 8192 BF16 70 us for nvfp4, 16384 x
// 8200 140.  (With a whole band per CTA, 16 rows per warp one after the other, 16384 x 8192
// BF16 took 163 us and 4097 x 2050 had only 165 CTAs.)
template<int FMT, class T>
__global__ void __launch_bounds__(Q_THREADS) quantize_rows_kernel(const __grid_constant__ QArgs a)
{
    constexpr int BLOCKS = Q_TILE_K / (FMT == B200_SGEMM_NVFP4 ? 16 : 32), TILES = BLOCKS / 4;
    __shared__ __align__(16) uint8_t staged[Q_ROWS][BLOCKS];
    const int       k_ctas = (a.K + Q_TILE_K - 1) / Q_TILE_K;
    const int       slice = blockIdx.x / k_ctas, kc = blockIdx.x - slice * k_ctas;
    const long long row0 = (long long)slice * Q_ROWS;
    const int       warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int       k0 = kc * Q_TILE_K + lane * Q_LANE_K;
    const T*        X  = static_cast<const T*>(a.x);
    if(a.row_index) // a band of the gathered rows that holds none is left alone
    {
        const long long r = row0 / MX4_BAND * MX4_BAND + threadIdx.x;
        const int       index = threadIdx.x < MX4_BAND && r < a.rows ? __ldg(a.row_index + r) : -1;
        if(!__syncthreads_or(index >= 0 && index / a.index_div < a.source_rows))
            return;
    }
    const bool vector = a.vector && k0 + Q_LANE_K <= a.K;
    // the row of X behind row r of the slice, uniform over the warp; -1: none
    auto source = [&](int r) -> long long {
        const long long row = row0 + r;
        if(row >= a.rows)
            return -1;
        if(!a.row_index)
            return row;
        const int index = __ldg(a.row_index + row), src = index < 0 ? -1 : index / a.index_div;
        return src < a.source_rows ? src : -1;
    };
    constexpr int V = Q_LANE_K / Vec32<T>::N;
    Vec32<T>      ahead[V]; // a row is fetched while the one before is worked on
    auto fetch = [&](long long src) {
        if(vector && src >= 0)
        {
#pragma unroll
            for(int j = 0; j < V; ++j)
                ahead[j].load(X + src * a.ld + k0 + j * Vec32<T>::N);
        }
    };
    long long next = source(warp);
    fetch(next);
    const Global G = load_global(a.global);
#pragma unroll 1
    for(int r = warp; r < Q_ROWS; r += Q_THREADS / 32)
    {
        const long long src = next;
        float           x[Q_LANE_K];
        if(vector)
        {
#pragma unroll
            for(int j = 0; j < Q_LANE_K; ++j)
                x[j] = to_float(ahead[j / Vec32<T>::N].v[j % Vec32<T>::N]);
        }
        else
        {
#pragma unroll
            for(int j = 0; j < Q_LANE_K; ++j)
                x[j] = src >= 0 && k0 + j < a.K ? to_float(X[src * a.ld + k0 + j]) : 0.f;
        }
        next = r + Q_THREADS / 32 < Q_ROWS ? source(r + Q_THREADS / 32) : -1;
        fetch(next);
        Scale sc;
        sc.byte = 0;
        if(src >= 0)
        {
            unsigned amax = amax16(x);
            if(FMT == B200_SGEMM_MXFP4)
                amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1)); // NaN orders above infinity
            sc            = FMT == B200_SGEMM_NVFP4 ? scale_nvfp4(amax, G) : scale_mxfp4(amax);
            const uint2 c = encode<FMT, T>(x, sc, G, [&](int i) { return to_float(X[src * a.ld + k0 + i]); });
            if(k0 < 2 * a.pitch)
                *reinterpret_cast<uint2*>(a.codes + (row0 + r) * a.pitch + k0 / 2) = c;
        }
        if(FMT == B200_SGEMM_NVFP4)
            staged[r][lane] = (uint8_t)sc.byte;
        else if((lane & 1) == 0)
            staged[r][lane >> 1] = (uint8_t)sc.byte;
    }
    __syncthreads();
    for(int i = threadIdx.x; i < Q_ROWS * TILES; i += Q_THREADS)
    {
        const int tile = i / Q_ROWS, r = i % Q_ROWS;
        if(kc * TILES + tile < a.tiles)
            *reinterpret_cast<uint32_t*>(a.scales + scale_at(row0 + r, (kc * TILES + tile) * 4, a.tiles)) =
                *reinterpret_cast<const uint32_t*>(&staged[r][tile * 4]);
    }
}

// Row-contiguous source (a col-major A, a row-major B).  One CTA: a band of 128 rows x 128 k.  A thread takes one row (FP32) or
// two neighbours (16 bits, one load of both), 32 k at a time; lanes take neighbouring rows, so a warp loads 128 contiguous
// bytes of a k, and a thread has whole blocks in registers; three CTAs an SM.  (16384 x 8192 BF16: 93 us for nvfp4, with the matrix scale
// amax / 2688 98, 68 us for mxfp4; with two CTAs an SM 123 us for nvfp4; with one row per thread of 16-bit types, 64 bytes a load, 270 us for
// 16384 x 8192 BF16.)
template<int FMT, class T>
__global__ void __launch_bounds__(Q_THREADS, 3) quantize_cols_kernel(const __grid_constant__ QArgs a)
{
    constexpr int   BLOCK = FMT == B200_SGEMM_NVFP4 ? 16 : 32;
    constexpr int   R = 4 / sizeof(T), SPAN = 64 / R; // rows and k of a thread
    const int       k_ctas = (a.K + Q_COL_K - 1) / Q_COL_K;
    const int       band = blockIdx.x / k_ctas, kc = blockIdx.x - band * k_ctas;
    const int       pair = threadIdx.x % (MX4_BAND / R), part = threadIdx.x / (MX4_BAND / R);
    const long long row0 = (long long)band * MX4_BAND + pair * R;
    const T*        X    = static_cast<const T*>(a.x);
    const Global    G    = load_global(a.global);
#pragma unroll
    for(int j = 0; j < SPAN / 32; ++j)
    {
        const int k0 = kc * Q_COL_K + part * SPAN + j * 32;
        if(k0 >= a.tiles * 4 * BLOCK)
            break;
        uint32_t raw[32];
        if(a.vector && row0 + R <= a.rows) // both rows (the only one) and aligned
        {
#pragma unroll
            for(int i = 0; i < 32; ++i)
                raw[i] = k0 + i < a.K ? __ldg(reinterpret_cast<const uint32_t*>(X + (long long)(k0 + i) * a.ld + row0)) : 0u;
        }
        else
        {
#pragma unroll
            for(int i = 0; i < 32; ++i)
            {
                T v[R];
#pragma unroll
                for(int m = 0; m < R; ++m)
                    v[m] = row0 + m < a.rows && k0 + i < a.K ? X[(long long)(k0 + i) * a.ld + row0 + m] : from_float<T>(0.f);
                if constexpr(R == 1)
                    raw[i] = __float_as_uint(to_float(v[0]));
                else
                    raw[i] = *reinterpret_cast<const uint16_t*>(&v[0]) | (uint32_t)*reinterpret_cast<const uint16_t*>(&v[R - 1]) << 16;
            }
        }
#pragma unroll
        for(int m = 0; m < R; ++m)
        {
            const long long row = row0 + m;
            float           x[2][Q_LANE_K];
#pragma unroll
            for(int i = 0; i < 32; ++i)
            {
                if constexpr(R == 1)
                    x[i / 16][i % 16] = __uint_as_float(raw[i]);
                else
                {
                    const uint16_t bits = (uint16_t)(raw[i] >> (16 * m));
                    x[i / 16][i % 16]   = to_float(*reinterpret_cast<const T*>(&bits));
                }
            }
            const unsigned amax[2] = {amax16(x[0]), amax16(x[1])};
            Scale          sc[2];
            if(FMT == B200_SGEMM_MXFP4)
                sc[0] = sc[1] = scale_mxfp4(max(amax[0], amax[1]));
            else
            {
                sc[0] = scale_nvfp4(amax[0], G);
                sc[1] = scale_nvfp4(amax[1], G);
            }
            auto        again = [&](int i) { return to_float(X[(long long)(k0 + i) * a.ld + row]); };
            const uint2 lo = encode<FMT, T>(x[0], sc[0], G, again);
            const uint2 hi = encode<FMT, T>(x[1], sc[1], G, [&](int i) { return again(16 + i); });
            const bool  in = row < a.rows;
            if(in && k0 < 2 * a.pitch)
                *reinterpret_cast<uint4*>(a.codes + row * a.pitch + k0 / 2) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            uint8_t* to = a.scales + scale_at(row, k0 / BLOCK, a.tiles);
            if(FMT == B200_SGEMM_NVFP4)
                *reinterpret_cast<uint16_t*>(to) = in ? (uint16_t)(sc[0].byte | sc[1].byte << 8) : (uint16_t)0;
            else
                *to = in ? (uint8_t)sc[0].byte : (uint8_t)0;
        }
    }
}

struct DArgs
{
    const uint8_t* codes;
    const uint8_t* scales;
    const float*   global;
    void*          x;
    long long      ld, pitch;
    int            rows, K, tiles;
};

// the two values of a byte of codes
__device__ __forceinline__ float2 levels2(unsigned byte)
{
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)byte, __NV_E2M1);
    return __half22float2(__half2(h));
}
// One CTA: 32 rows x 512 k, a warp four rows.  A lane turns 32 bytes of output at a time, with the codes and scales of all four
// rows in flight at once.
template<int FMT, class T>
__global__ void __launch_bounds__(Q_THREADS) dequantize_kernel(const __grid_constant__ DArgs a)
{
    constexpr int   BLOCK = FMT == B200_SGEMM_NVFP4 ? 16 : 32, N = Vec32<T>::N, STEPS = Q_TILE_K / (32 * N);
    const int       k_ctas = (a.K + Q_TILE_K - 1) / Q_TILE_K;
    const int       slice = blockIdx.x / k_ctas, kc = blockIdx.x - slice * k_ctas;
    const int       warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row0 = (long long)slice * Q_ROWS + warp;
    const float     g = a.global ? *a.global : 1.f;
    uint2           c[Q_WARP_ROWS][STEPS];
    uint8_t         byte[Q_WARP_ROWS][STEPS];
#pragma unroll
    for(int i = 0; i < Q_WARP_ROWS; ++i)
    {
        const long long row = row0 + i * (Q_THREADS / 32);
#pragma unroll
        for(int step = 0; step < STEPS; ++step)
        {
            const int k = kc * Q_TILE_K + (step * 32 + lane) * N;
            if(row < a.rows && k < a.K)
            {
                const uint8_t* from = a.codes + row * a.pitch + k / 2;
                if(N == 16)
                    c[i][step] = __ldg(reinterpret_cast<const uint2*>(from));
                else
                    c[i][step].x = __ldg(reinterpret_cast<const unsigned*>(from));
                byte[i][step] = __ldg(a.scales + scale_at(row, k / BLOCK, a.tiles));
            }
        }
    }
#pragma unroll
    for(int i = 0; i < Q_WARP_ROWS; ++i)
    {
        const long long row = row0 + i * (Q_THREADS / 32);
#pragma unroll
        for(int step = 0; step < STEPS; ++step)
        {
            const int k = kc * Q_TILE_K + (step * 32 + lane) * N;
            if(row >= a.rows || k >= a.K)
                break;
            const float s  = scale_value<FMT>(byte[i][step]);
            T*          to = static_cast<T*>(a.x) + row * a.ld + k;
            Vec32<T>    out;
#pragma unroll
            for(int j = 0; j < N / 2; ++j)
            {
                const float2 f = levels2((j < 4 ? c[i][step].x >> (8 * j) : c[i][step].y >> (8 * (j - 4))) & 0xFFu);
                out.v[2 * j]     = from_float<T>(f.x * s * g); // f * s is exact
                out.v[2 * j + 1] = from_float<T>(f.y * s * g);
            }
            if(k + N <= a.K)
                out.store(to);
            else
            {
#pragma unroll
                for(int j = 0; j < N; ++j)
                    if(k + j < a.K)
                        to[j] = out.v[j];
            }
        }
    }
}

// The same for rows that do not start on 32 bytes: lanes take neighbours, so that a warp's stores are contiguous all the same, in
// pairs (the two codes of a byte) where rows start on a pair.  Each lane turns one scale of the row into its value and the
// others fetch it from there.  (4097 x 2050 FP32, whose rows start on 8 bytes: 31.5 us with 16 neighbours per lane, 14.7 us
// with one, 10.7 us with two.)
template<int FMT, class T, int N>
__global__ void __launch_bounds__(Q_THREADS) dequantize_unaligned_kernel(const __grid_constant__ DArgs a)
{
    constexpr int   BLOCK = FMT == B200_SGEMM_NVFP4 ? 16 : 32, STEPS = Q_TILE_K / (32 * N);
    const int       k_ctas = (a.K + Q_TILE_K - 1) / Q_TILE_K;
    const int       slice = blockIdx.x / k_ctas, kc = blockIdx.x - slice * k_ctas;
    const int       warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float     g = a.global ? *a.global : 1.f;
    const int       k0 = kc * Q_TILE_K + lane * N, block = kc * (Q_TILE_K / BLOCK) + lane % (Q_TILE_K / BLOCK);
#pragma unroll
    for(int i = 0; i < Q_WARP_ROWS; ++i)
    {
        const long long row = (long long)slice * Q_ROWS + warp + i * (Q_THREADS / 32);
        if(row >= a.rows)
            break;
        const uint8_t* from = a.codes + row * a.pitch + k0 / 2;
        uint8_t        c[STEPS];
#pragma unroll
        for(int step = 0; step < STEPS; ++step)
            if(k0 + step * 32 * N < a.K)
                c[step] = __ldg(from + step * 16 * N);
        const float value = scale_value<FMT>(block >> 2 < a.tiles ? __ldg(a.scales + scale_at(row, block, a.tiles)) : 0);
        T*          to    = static_cast<T*>(a.x) + row * a.ld + k0;
#pragma unroll
        for(int step = 0; step < STEPS; ++step)
        {
            const int   k = k0 + step * 32 * N;
            const float s = __shfl_sync(0xFFFFFFFFu, value, (step * 32 + lane) * N / BLOCK);
            if(k >= a.K)
                continue;
            const float2 f = levels2(c[step]);
            if constexpr(N == 2)
            {
                struct alignas(2 * sizeof(T)) Two
                {
                    T x, y;
                };
                const Two v = {from_float<T>(f.x * s * g), from_float<T>(f.y * s * g)};
                if(k + 1 < a.K)
                    *reinterpret_cast<Two*>(to + step * 64) = v;
                else
                    to[step * 64] = v.x;
            }
            else
                to[step * 32] = from_float<T>((lane & 1 ? f.y : f.x) * s * g);
        }
    }
}

// CTAs of `parts` x pieces of k, or 0 when that is more than a grid holds
unsigned grid_of(size_t parts, size_t K, size_t tile_k)
{
    const unsigned long long n = (unsigned long long)parts * ((K + tile_k - 1) / tile_k);
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
    const size_t   bands = (rows + MX4_BAND - 1) / MX4_BAND;
    const unsigned grid  = row_major ? grid_of(bands * (MX4_BAND / Q_ROWS), K, Q_TILE_K) : grid_of(bands, K, Q_COL_K);
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
    const size_t access = row_major ? 32 : 4; // bytes of a load
    a.vector            = !misaligned(X, access) && ldx * type_bytes(type) % access == 0;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const bool nv = format == B200_SGEMM_NVFP4;
        auto kernel = row_major ? (nv ? quantize_rows_kernel<B200_SGEMM_NVFP4, T> : quantize_rows_kernel<B200_SGEMM_MXFP4, T>)
                                : (nv ? quantize_cols_kernel<B200_SGEMM_NVFP4, T> : quantize_cols_kernel<B200_SGEMM_MXFP4, T>);
        return launch_kernel(kernel, grid, Q_THREADS, stream, a);
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
    const unsigned grid = grid_of((rows + Q_ROWS - 1) / Q_ROWS, K, Q_TILE_K);
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
    auto aligned = [&](size_t bytes) { return !misaligned(X, bytes) && ldx * type_bytes(type) % bytes == 0; };
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto pick = [&](auto f) {
            constexpr int FMT = decltype(f)::value;
            return aligned(32) ? dequantize_kernel<FMT, T>
                               : (aligned(2 * sizeof(T)) ? dequantize_unaligned_kernel<FMT, T, 2> : dequantize_unaligned_kernel<FMT, T, 1>);
        };
        auto kernel = format == B200_SGEMM_NVFP4 ? pick(std::integral_constant<int, B200_SGEMM_NVFP4>())
                                                 : pick(std::integral_constant<int, B200_SGEMM_MXFP4>());
        return launch_kernel(kernel, grid, Q_THREADS, stream, a);
    });
}
