// The 4-bit product for one or two rows on one side: a token or two against a weight matrix.
//
//   c[r, m] = alpha * g * g_x * sum over blocks of s[r, b] s_x[m, b] (sum over the block of v[r, k] v_x[m, k])
//
// Bound by HBM: the long matrix is read once, 4.5 bits a value, and there are only 2 x `few` operations for each.  The tensor
// core's way (mx4_gemm.cu) brings little here: it copies scale tiles into tensor memory at 50 cycles each, as many for one
// token as for 128, and its set-up and split of K cost as much as the work: 7.0 us for 1 x 4096 x 4096.
//
// Products of two e2m1 values are multiples of 1/4 up to 36, so the sum of eight is exact in FP16 (1152 quarters): a block of 16
// is eight fused multiply-adds on pairs, whose two halves are added in FP32.  That sum has at most 12 bits, with both scales at
// most 20: blocks are added in FP32 with one rounding each.  (Integer dot products of looked-up bytes are exact too, but byte
// selection, shifts and integer products run at half the rate: 16.1 us for 1 x 16384 x 4096.)
//
// A warp takes two groups of four rows r, r + 32, r + 64, r + 96 of a band, whose scales for four blocks are 16 contiguous bytes,
// and 1024 k a step, 32 neighbours a lane, for which the short side's values are turned once; one group's codes are fetched while
// the other's are used.  Long matrices of few rows: the warps of a CTA share rows and split K; sums are then added in the
// warps' order.  What is left is the arithmetic on the way (some 70 instructions for 32 values of a lane, a quarter of them
// conversions) and the registers it takes, which leave two CTAs an SM: one row x 4096 x 4096 takes 4.0 us, where the tensor core
// takes 7.0; 1 x 16384 x 4096 11.1 us, where it takes 10.1.  One group a warp and three CTAs: 5.1 and 14.4 us.
#include "mx4_few.hpp"

#include "mx4_common.cuh"

namespace
{
using namespace sgemm_b200;

constexpr int F_THREADS = 256;
constexpr int F_WARPS   = F_THREADS / 32;
constexpr int F_LANE_K  = 32;
constexpr int F_GROUPS  = 2; // of four rows, that a warp takes

struct Args
{
    FewArgs   f;
    long long pitch;
    int       tiles, k_split, units; // scale tiles along k; warps that share rows; warps' worth of rows
};

// the four pairs of values of eight codes
__device__ __forceinline__ void pairs8(__half2* v, unsigned codes)
{
    uint32_t r[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(codes));
#pragma unroll
    for(int i = 0; i < 4; ++i)
        v[i] = *reinterpret_cast<__half2*>(&r[i]);
}
__device__ __forceinline__ void pairs16(__half2 (&v)[8], unsigned low, unsigned high)
{
    pairs8(v, low);
    pairs8(v + 4, high);
}
// whether one of sixteen scales is NaN
template<int FMT>
__device__ __forceinline__ bool any_nan(const unsigned (&scales)[4])
{
    unsigned found = 0;
#pragma unroll
    for(int i = 0; i < 4; ++i)
        found |= FMT == B200_SGEMM_NVFP4 ? (scales[i] & 0x7F7F7F7Fu) + 0x01010101u : __vcmpeq4(scales[i], 0xFFFFFFFFu);
    return (found & 0x80808080u) != 0u;
}
// a scale's bits as those of an FP32 number: e4m3 2^-120 times its value, e8m0 its value (which has to be above 2^-127: see
// scale_value)
template<int FMT>
__device__ __forceinline__ float raw_scale(unsigned byte_and_more)
{
    if(FMT == B200_SGEMM_NVFP4)
        return __uint_as_float(byte_and_more << 20 & 0x07F00000u);
    return e8m0_value(byte_and_more & 0xFFu);
}

template<int FMT, int FEW>
__global__ void __launch_bounds__(F_THREADS, 2) mx4_few_kernel(const __grid_constant__ Args a)
{
    constexpr int BLOCK = FMT == B200_SGEMM_NVFP4 ? 16 : 32, BLOCKS = F_LANE_K / BLOCK; // blocks of a lane's k
    constexpr int SUMS  = F_GROUPS * 4 * FEW;
    __shared__ float part[F_WARPS][SUMS];
    const int       warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int       share = warp % a.k_split;
    const long long unit  = (long long)blockIdx.x * (F_WARPS / a.k_split) + warp / a.k_split;
    const long long row0  = unit / (32 / F_GROUPS) * MX4_BAND + unit % (32 / F_GROUPS) * F_GROUPS; // group g: row0 + g + 0, 32, 64, 96
    const uint8_t*  codes_x  = static_cast<const uint8_t*>(a.f.codes_x);
    const uint8_t*  scales_x = static_cast<const uint8_t*>(a.f.scales_x);
    const int       step     = a.k_split * 32 * F_LANE_K;
    int             k        = unit < a.units ? (share * 32 + lane) * F_LANE_K : a.f.K;
    // where the lane's codes of each row start; rows that are not there are the last one again, and not stored
    const uint8_t* at[F_GROUPS][4];
#pragma unroll
    for(int g = 0; g < F_GROUPS; ++g)
#pragma unroll
        for(int q = 0; q < 4; ++q)
            at[g][q] = static_cast<const uint8_t*>(a.f.codes) + min(row0 + g + q * 32, (long long)a.f.rows - 1) * a.pitch + k / 2;
    const uint8_t* scales = static_cast<const uint8_t*>(a.f.scales)
                            + (row0 / MX4_BAND * a.tiles + k / BLOCK / 4) * MX4_TILE_BYTES + row0 % MX4_BAND * 16;
    float sum[F_GROUPS][4][FEW] = {};
    uint4 ahead[4], ahead_s; // one group's codes and scales (four blocks of each of its four rows), fetched while another's are used
    auto  fetch = [&](int g) {
#pragma unroll
        for(int q = 0; q < 4; ++q)
        {
            ahead[q] = __ldg(reinterpret_cast<const uint4*>(at[g][q]));
            at[g][q] += step / 2;
        }
        ahead_s = __ldg(reinterpret_cast<const uint4*>(scales + g * 16));
    };
    if(k < a.f.K)
        fetch(0);
    for(; k < a.f.K; k += step)
    {
        const size_t tile = (size_t)(k / BLOCK / 4) * MX4_TILE_BYTES;
        const int    in   = k / BLOCK % 4 * 8;
        // scales of the short side.  nvfp4: times 2^100 of the 2^120 that raw_scale lacks (448 x 2^120 is no FP32 number).  mxfp4: a
        // quarter, the smallest |v| but zero, so that the product of two scales only exceeds FP32 where the block's sum does
        float   sx[FEW][BLOCKS];
        __half2 v[FEW][2][8];
#pragma unroll
        for(int m = 0; m < FEW; ++m)
        {
            const uint4    x = __ldg(reinterpret_cast<const uint4*>(codes_x + m * a.pitch + k / 2));
            const unsigned s = __ldg(reinterpret_cast<const unsigned*>(scales_x + tile + m * 16)) >> in;
#pragma unroll
            for(int b = 0; b < BLOCKS; ++b)
                sx[m][b] = scale_value<FMT>(s >> (8 * b) & 0xFFu) * (FMT == B200_SGEMM_NVFP4 ? 0x1p100f : 0.25f);
            pairs16(v[m][0], x.x, x.y);
            pairs16(v[m][1], x.z, x.w);
        }
#pragma unroll
        for(int g = 0; g < F_GROUPS; ++g)
        {
            const uint4    w[4]  = {ahead[0], ahead[1], ahead[2], ahead[3]};
            const unsigned sw[4] = {ahead_s.x, ahead_s.y, ahead_s.z, ahead_s.w};
            if(g + 1 < F_GROUPS)
                fetch(g + 1);
            else
            {
                scales += (size_t)step / BLOCK / 4 * MX4_TILE_BYTES;
                if(k + step < a.f.K)
                    fetch(0);
            }
#pragma unroll
            for(int q = 0; q < 4; ++q)
            {
                const unsigned scale = sw[q] >> in;
#pragma unroll
                for(int h = 0; h < 2; ++h) // 16 k
                {
                    __half2 p[8];
                    pairs16(p, h ? w[q].z : w[q].x, h ? w[q].w : w[q].y);
                    const float s = raw_scale<FMT>(scale >> (8 * (h * BLOCKS / 2)));
#pragma unroll
                    for(int m = 0; m < FEW; ++m)
                    {
                        __half2 dot = __hmul2(p[0], v[m][h][0]);
#pragma unroll
                        for(int i = 1; i < 8; ++i)
                            dot = __hfma2(p[i], v[m][h][i], dot);
                        const float2 f = __half22float2(dot);
                        const float  v = f.x + f.y;
                        const float  other = sx[m][h * BLOCKS / 2];
                        // where two mxfp4 scales exceed FP32 all the same, a block that adds nothing is zero, and NaN where the
                        // short side's scale is
                        sum[g][q][m] = fmaf(v, FMT == B200_SGEMM_NVFP4 || v != 0.f ? s * other : other, sum[g][q][m]);
                    }
                }
            }
            if(any_nan<FMT>(sw)) // rare: which rows
            {
#pragma unroll
                for(int q = 0; q < 4; ++q)
                {
                    const unsigned one[4] = {sw[q], 0u, 0u, 0u};
                    if(any_nan<FMT>(one))
                    {
#pragma unroll
                        for(int m = 0; m < FEW; ++m)
                            sum[g][q][m] = __uint_as_float(0x7FC00000u);
                    }
                }
            }
        }
    }
#pragma unroll
    for(int i = 0; i < SUMS; ++i)
    {
        float v = sum[i / (4 * FEW)][i / FEW % 4][i % FEW];
#pragma unroll
        for(int d = 16; d; d >>= 1)
            v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
        if(lane == i)
            part[warp][i] = v;
    }
    __syncthreads();
    if(share != 0 || lane >= SUMS || unit >= a.units)
        return;
    const int       g = lane / (4 * FEW), q = lane / FEW % 4, m = lane % FEW;
    const long long row   = row0 + g + q * 32;
    float           total = 0.f;
    for(int i = 0; i < a.k_split; ++i)
        total += part[warp + i][lane];
    if(row >= a.f.rows)
        return;
    total *= FMT == B200_SGEMM_NVFP4 ? 0x1p20f : 4.f;
    float factor = a.f.alpha;
    if(a.f.global_x)
        factor *= *a.f.global_x;
    if(a.f.global)
        factor *= *a.f.global;
    const long long to = row * a.f.ld_long + m * a.f.ld_few;
    total *= factor;
    if(a.f.type == B200_SGEMM_F32)
        static_cast<float*>(a.f.c)[to] = total;
    else if(a.f.type == B200_SGEMM_F16)
        static_cast<__half*>(a.f.c)[to] = from_float<__half>(total);
    else
        static_cast<__nv_bfloat16*>(a.f.c)[to] = from_float<__nv_bfloat16>(total);
}

template<int FMT>
int launch(const Args& a, unsigned grid, cudaStream_t stream)
{
    return launch_kernel(a.f.few == 1 ? mx4_few_kernel<FMT, 1> : mx4_few_kernel<FMT, 2>, grid, F_THREADS, stream, a);
}
} // namespace

int sgemm_b200::mx4_few(int format, const FewArgs& f, int sms, cudaStream_t stream)
{
    Args a;
    a.f     = f;
    a.pitch = (long long)mx4_pitch((size_t)f.K);
    a.tiles = (int)mx4_tiles(format, (size_t)f.K);
    a.units   = (f.rows + MX4_BAND - 1) / MX4_BAND * (32 / F_GROUPS);
    // 24 warps an SM hide the memory's latency; each keeps two steps of K where there are that many
    a.k_split = 1;
    while(a.k_split < F_WARPS && (long long)a.units * a.k_split < 24ll * sms && f.K >= a.k_split * 2 * 1024)
        a.k_split *= 2;
    const unsigned grid = (unsigned)((a.units + F_WARPS / a.k_split - 1) / (F_WARPS / a.k_split));
    return format == B200_SGEMM_NVFP4 ? launch<B200_SGEMM_NVFP4>(a, grid, stream) : launch<B200_SGEMM_MXFP4>(a, grid, stream);
}
