// b200_sgemm_mx4 and b200_sgemm_mx4_grouped: products of matrices in microscaled 4-bit floating point on the tensor
// cores (tcgen05, block-scaled e2m1 operands, FP32 accumulators in tensor memory).
//
//   C[m, n] = alpha * global_a * global_b[e] * sum_k A[m, k] B[n, k]
//
// Both operands are K-contiguous, so either can take either side of a tile.  The kernel knows a LANE operand P (128 rows
// of it on the 128 lanes of tensor memory) and a COLUMN operand Q (BN rows of it as columns):
//   lanes    the dimension along which C is contiguous, so that a warp stores 32 neighbours of C at once; for few tokens
//            that is the weights, and the tokens cost 32 or 64 columns instead of a tile of 128 rows
//   columns  the other one; the rows of the groups in the grouped product
//
// Tiles.  128 lanes x 64 or 128 columns by one CTA, or 256 lanes x 256 columns by a pair of CTAs on neighbouring SMs: each holds
// 128 of the lanes, half of Q's rows and all of Q's scales, and the first one issues for both.  A pair reads half of Q from the
// L2 and from shared memory and issues half the scale copies per product.
//
// One persistent CTA per SM, 10 warps (12 where 128 sums a thread stay in registers: 10 and 11 only give theirs up):
//   warps 0-7  accumulate and store.  The tensor core adds into its FP32 accumulator with truncation, so for an FP32
//              result the accumulator is emptied into registers every 1024 or 2048 k and the parts are added there,
//              rounded to nearest (relative error of the whole result with scales over 2^+-8, K = 4096 and 16384 alike: 1.6e-7 in
//              parts of 512 k, 2.8e-7 of 1024, 5.3e-7 of 2048; an FP32 product on the FMA pipe 5.0e-7 and 1.0e-6).  A bias of at most 2^-23 a
//              product of 64 k: it stays below a quarter of the smallest rounding of an FP16 result (2^-12) up to 2^15 k and of
//              a BF16 one (2^-9) up to 2^18, so those keep one accumulator that long and empty it as FP32 results do beyond.
//   warp 8     fetches the stages by TMA: the two operands' codes (256 k = rows of 128 bytes, 128-byte swizzle) and the scale
//              tiles as they lie; zero beyond the matrix
//   warp 9     copies the stage's scale tiles into tensor memory (tcgen05.cp, replicated to the four lane quarters) and issues
//              the products, 64 k each.  Scales go to a tensor-memory slot of the stage's own, which is free as soon as the
//              stage is.
// Few tiles: a cluster of 2, 4 or 8 CTAs shares a tile, each with a range of K of its own; every CTA sends its part of a column
// to the one that will store it, from shared memory to shared memory, which adds the parts in ascending order of K, so the
// result does not depend on timing and no workspace is needed (a captured graph can be replayed on any stream).
// Every wait is bounded, as in the other kernels.
#include "mx4_common.cuh"
#include "mx4_few.hpp"
#include "sgemm_ws_kernel.cuh"
#include "tcgen05.cuh"

#include <cuda.h>

#include <atomic>

namespace
{
using namespace sgemm_b200;

constexpr int G_LANES      = 128; // lanes of a CTA
constexpr int G_KBLOCK     = 256; // k of one stage: a 128-byte row of codes
constexpr int G_ROW_BYTES  = G_KBLOCK / 2;
constexpr int G_KSTEP      = 64; // k of one instruction
constexpr int G_EPILOGUE   = 256;
constexpr int G_TMA_WARP   = 8;
constexpr int G_MMA_WARP   = 9;
constexpr int G_TMEM_COLS  = 512;
constexpr int G_SCALE_COL  = 256; // tensor-memory columns 0..255: accumulators; behind them a slot of scales per stage
constexpr int G_MAX_GROUPS = 1024;
constexpr int MAX_SPLIT    = 8; // CTAs that share a tile's K
constexpr int CHUNK_F32    = 4; // K blocks (1024 k, 16 products) added inside the tensor core for an FP32 result
// the same for 256 columns, whose one accumulator stands still while it is emptied: 4096 cube 38.7 us, 8192 cube 236, 8192 tokens'
// experts 162; with 1024 k 44.9, 262 and 190
constexpr int CHUNK_F32_WIDE = 8;
constexpr int CHUNK_F16    = 1 << 7, CHUNK_BF16 = 1 << 10; // 2^15 and 2^18 k
// Registers of the kernel that keeps 128 sums a thread: 12 warps are launched with 168 each; warps 8 to 11 give theirs up
// and warps 0 to 7 take them: 256 x 224 + 128 x 56 = 384 x 168, exactly the launch's allocation, so the increase is always granted.
constexpr int G_LAUNCH_REGS = 168, G_SUM_REGS = 224, G_ISSUE_REGS = 56;
static_assert(G_EPILOGUE * G_SUM_REGS + 128 * G_ISSUE_REGS == (G_EPILOGUE + 128) * G_LAUNCH_REGS, "register budgets");

constexpr int G_ERR_WAIT  = 1; // status bits: a wait gave up (bits 8.. say which)
constexpr int G_ERR_GROUP = 2; // a group's offset or count does not fit the matrix, and the group was left out

__device__ int g_mx4_status;

// PAIR: CTAs that share a tile's instructions
// SUMS: 256 columns of results whose parts are added in registers
template<int FMT, int BN, int PAIR, bool SUMS = false>
struct GLayout
{
    static constexpr int    THREADS     = SUMS ? G_EPILOGUE + 128 : G_EPILOGUE + 64;
    static constexpr int    TILE_P      = PAIR * G_LANES;
    static constexpr int    Q_ROWS      = BN / PAIR;                     // of this CTA
    static constexpr int    Q_BOX       = BN == 64 ? 32 : Q_ROWS;        // rows of one copy; a tile of up to 32 rows takes one of two
    static constexpr int    Q_BANDS     = (BN + MX4_BAND - 1) / MX4_BAND; // bands of scales that a column tile touches
    static constexpr int    TILES       = G_KBLOCK / (4 * mx4_block(FMT)); // scale tiles of a band in a stage
    static constexpr int    P_BYTES     = G_LANES * G_ROW_BYTES;
    static constexpr int    Q_BYTES     = Q_ROWS * G_ROW_BYTES;
    static constexpr int    P_SCALES    = TILES * MX4_TILE_BYTES;
    static constexpr int    Q_SCALES    = Q_BANDS * P_SCALES;
    static constexpr int    BOX_BYTES   = Q_BOX * G_ROW_BYTES;
    static constexpr int    STAGE_BYTES = (P_BYTES + Q_BYTES + P_SCALES + Q_SCALES + 1023) / 1024 * 1024;
    static constexpr int    SLOT_COLS   = 4 * TILES * (1 + Q_BANDS); // tensor-memory columns of a stage's scales
    static constexpr int    BY_SMEM     = (216 * 1024) / STAGE_BYTES;
    static constexpr int    BY_TMEM     = (G_TMEM_COLS - G_SCALE_COL) / SLOT_COLS;
    static constexpr int    STAGES      = BY_SMEM < BY_TMEM ? (BY_SMEM < 8 ? BY_SMEM : 8) : (BY_TMEM < 8 ? BY_TMEM : 8);
    // accumulators.  One of 256 columns beats two of 192 for pairs, whose tiles read a fifth more bytes a product: 8192 cube 195 us
    // against 243, experts of about 1024 rows x 4096 x 2048 130 against 152
    static constexpr int    ACCS        = BN > 128 ? 1 : 2;
    static constexpr int    BARRIERS    = 2 * STAGES + 6;
    static constexpr size_t SMEM_BYTES  = size_t(STAGES) * STAGE_BYTES + 1024 /*alignment slack*/ + 256 /*barriers, misc*/;
    static_assert(8 * BARRIERS + 16 <= 256 && BARRIERS <= 32, "barrier area, a lane each");
    static_assert(ACCS * BN <= G_SCALE_COL, "tensor memory");
    static_assert(BN % 64 == 0 && SLOT_COLS % 4 == 0 && TILES % 2 == 0, "scales start on an even column");
    static_assert(SMEM_BYTES + (G_MAX_GROUPS + 1) * 4 <= 227 * 1024, "shared memory");
    static_assert(PAIR > 1 || (BN + MAX_SPLIT) * G_LANES * 4 <= STAGES * STAGE_BYTES / 2, "a split tile's parts lie in the ring twice");
    static_assert(PAIR > 1 || STAGES * STAGE_BYTES / 2 % 16 == 0, "bulk copies start on 16 bytes");
};

struct GArgs
{
    void*          c;
    long long      sp, sq;   // element strides of C along lanes and columns; one of them is 1
    const uint8_t* scales_p; // for a single CTA, which takes the tiles by plain bulk copies (two descriptors less to build: 0.6 us)
    const uint8_t* scales_q;
    int            k_tiles; // scale tiles along k
    const int*     offsets; // grouped: first row (of Q and C) of each group, and rows
    const int*     counts;
    const float*   global_p;
    const float*   global_q;
    float          alpha;
    int            np;      // lane extent (of one group's operand)
    int            nq;      // column extent: rows of Q
    int            K, kblocks, chunk;
    int            tiles_p, bands_p; // lane tiles; bands of scales of one group's P
    int            groups;  // 0: one product
    int            most_q;  // column tiles that groups can have in all
    int            split_bits; // 2^split_bits CTAs of a cluster share a tile
    int            type;
};

// ---- instructions ----------------------------------------------------------------------------------------
// tile copies that signal a barrier of the pair's first CTA; `bar` as a cluster address
template<int PAIR>
__device__ __forceinline__ void load_codes(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar)
{
    if constexpr(PAIR == 1)
        tma_load_2d(dst, map, c0, c1, bar);
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
                     : "memory");
}
__device__ __forceinline__ void load_scales_pair(uint32_t dst, const CUtensorMap* map, int tile, int band, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(tile), "r"(band), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// a scale tile (32 rows of 16 bytes) to four columns of all four lane quarters; a pair: each CTA its own tile
template<int PAIR>
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc)
{
    if constexpr(PAIR == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
#define MX4_MMA(GROUP, VEC)                                                                                                      \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                              \
                 "tcgen05.mma.cta_group::" GROUP ".kind::mxf4nvf4.block_scale.scale_vec::" VEC " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" \
                 ::"r"(d), "l"(p_desc), "l"(q_desc), "r"(idesc), "r"(sf_p), "r"(sf_q), "r"(accumulate)                            \
                 : "memory")
template<int FMT, int PAIR>
__device__ __forceinline__ void tc_mma_mx4(uint32_t d, uint64_t p_desc, uint64_t q_desc, uint32_t idesc, uint32_t sf_p, uint32_t sf_q,
                                           uint32_t accumulate)
{
    if constexpr(FMT == B200_SGEMM_NVFP4 && PAIR == 1)
        MX4_MMA("1", "4X");
    else if constexpr(FMT == B200_SGEMM_NVFP4)
        MX4_MMA("2", "4X");
    else if constexpr(PAIR == 1)
        MX4_MMA("1", "2X");
    else
        MX4_MMA("2", "2X");
}
#undef MX4_MMA
// codes: rows of 128 bytes with the 128-byte swizzle, 1024 bytes between groups of eight rows
__device__ __forceinline__ uint64_t codes_desc(uint32_t addr)
{
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46)
           | (uint64_t(2) << 61);
}
// scale tile: rows of 16 bytes, no swizzle, 128 bytes between groups of eight rows
__device__ __forceinline__ uint64_t scales_desc(uint32_t addr)
{
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(128 >> 4) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}
// block-scaled product: e2m1 operands (1), both K-major, N >> 3, scale type (0 e4m3, 1 e8m0), M >> 4; which bytes of the
// 32-bit scale words an instruction takes is added by the issuer (bits 4-5 for Q, 29-30 for P)
template<int FMT, int PAIR>
__device__ __forceinline__ constexpr uint32_t mx4_idesc(uint32_t n)
{
    return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (FMT == B200_SGEMM_MXFP4 ? 1u << 23 : 0u)
           | (uint32_t(PAIR * G_LANES >> 4) << 24);
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the address in CTA `rank` of the cluster that corresponds to `addr` here
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank)
{
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    return at;
}
// this CTA's shared memory to another's, whose barrier counts the bytes
__device__ __forceinline__ void bulk_send(uint32_t cluster_dst, uint32_t src, uint32_t bytes, uint32_t cluster_bar)
{
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(cluster_dst), "r"(src), "r"(bytes), "r"(cluster_bar)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// what is in flight when a CTA gives up has to land before it leaves; bounded, without looking at the abort flag
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity)
{
    const uint64_t t0 = global_timer_ns();
    while(!mbar_try_wait(bar, parity) && global_timer_ns() - t0 < 100ull * 1000 * 1000) {}
}

// one thread of a converged warp
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// a bounded wait of a whole warp: all lanes see the same outcome
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag)
{
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag));
}

// ---- tiles -------------------------------------------------------------------------------------------------
struct Tile
{
    int group, p0, q0, q_end; // columns q0 .. min(q0 + BN, q_end)
};
// one product: bands of 16 lane tiles, columns advancing inside a band, so that CTAs running together share operands in
// the L2; groups: all lane tiles of a group's column tile, then the next column tile, so a group's weights stay in the L2
template<int BN, int TILE_P>
__device__ __forceinline__ Tile tile_at(const GArgs& a, const int* first_tile, int tile)
{
    Tile t;
    if(a.groups == 0)
    {
        constexpr int BAND = 16 * G_LANES / TILE_P;
        const int tiles_q = (a.nq + BN - 1) / BN;
        const int band = tile / (BAND * tiles_q), in = tile - band * BAND * tiles_q;
        const int wide = min(BAND, a.tiles_p - band * BAND);
        t.group = 0;
        t.p0    = (band * BAND + in % wide) * TILE_P;
        t.q0    = in / wide * BN;
        t.q_end = a.nq;
        return t;
    }
    const int qt = tile / a.tiles_p;
    int       lo = 0, hi = a.groups; // the group with first_tile[lo] <= qt < first_tile[lo + 1]
    while(hi - lo > 1)
    {
        const int mid = (lo + hi) >> 1;
        if(first_tile[mid] <= qt)
            lo = mid;
        else
            hi = mid;
    }
    const int off = a.offsets[lo];
    t.group = lo;
    t.p0    = (tile - qt * a.tiles_p) * TILE_P;
    t.q0    = off + (qt - first_tile[lo]) * BN;
    t.q_end = off + a.counts[lo];
    return t;
}

template<class T, int COLS>
__device__ __forceinline__ void store_columns(const GArgs& a, const float (&acc)[COLS], float factor, int p, int q0, int q_end)
{
    if(p >= a.np)
        return;
    T* c = static_cast<T*>(a.c) + (long long)p * a.sp + (long long)q0 * a.sq;
    if(a.sq == 1)
    {
        constexpr int N = Vec16<T>::N;
        const bool vector = ((reinterpret_cast<uintptr_t>(c)) & 15) == 0;
#pragma unroll
        for(int j = 0; j < COLS; j += N)
        {
            Vec16<T> v;
#pragma unroll
            for(int i = 0; i < N; ++i)
                v.v[i] = from_float<T>(acc[j + i] * factor);
            if(vector && q0 + j + N <= q_end)
                *reinterpret_cast<uint4*>(c + j) = v.raw;
            else
            {
#pragma unroll
                for(int i = 0; i < N; ++i)
                    if(q0 + j + i < q_end)
                        c[j + i] = v.v[i];
            }
        }
    }
    else
    {
        // eight columns at a time, without a test each where all are there (a test, a 64-bit product and a branch for each of 32
        // columns took 0.8 us)
        constexpr int STEP = 8;
        const int     n    = q_end - q0;
#pragma unroll
        for(int j0 = 0; j0 < COLS; j0 += STEP)
        {
            if(j0 >= n)
                break;
            if(j0 + STEP <= n)
            {
#pragma unroll
                for(int j = 0; j < STEP; ++j, c += a.sq)
                    *c = from_float<T>(acc[j0 + j] * factor);
            }
            else
            {
#pragma unroll
                for(int j = 0; j < STEP; ++j, c += a.sq)
                    if(j0 + j < n)
                        *c = from_float<T>(acc[j0 + j] * factor);
            }
        }
    }
}
template<int COLS>
__device__ __forceinline__ void store_typed(const GArgs& a, const float (&acc)[COLS], float factor, int p, int q0, int q_end)
{
    if(a.type == B200_SGEMM_F32)
        store_columns<float>(a, acc, factor, p, q0, q_end);
    else if(a.type == B200_SGEMM_F16)
        store_columns<__half>(a, acc, factor, p, q0, q_end);
    else
        store_columns<__nv_bfloat16>(a, acc, factor, p, q0, q_end);
}

template<int PAIR>
struct Maps
{
    CUtensorMap p, q, scales_p, scales_q;
};
template<>
struct Maps<1>
{
    CUtensorMap p, q;
};

// Columns that the instructions of a tile compute: the last tile of a group seldom needs all (32 experts of about 1024 rows x 4096
// x 2048: 129.7 us, 131.7 with all).  The CTAs of a pair hold the rows of the first and the second half of them.
template<int BN, int PAIR>
__device__ __forceinline__ int columns_of(const Tile& t)
{
    const int left = t.q_end - t.q0;
    if(PAIR > 1)
        return min(BN, (left + 63) / 64 * 64);
    return BN == 64 && left <= 32 ? 32 : BN;
}

// the first n of N results, `stride` elements apart
template<class T, int N>
__device__ __forceinline__ void store_strided(T* c, const float (&v)[N], float factor, long long stride, int n)
{
#pragma unroll
    for(int j = 0; j < N; ++j)
        if(j < n)
            c[j * stride] = from_float<T>(v[j] * factor);
}
// results of 16 bits, two in a word, the first in the lower half
template<int COLS>
__device__ __forceinline__ void store_packed(const GArgs& a, const uint32_t (&v)[COLS / 2], int p, int q0, int q_end)
{
    if(p >= a.np)
        return;
    uint16_t* c = static_cast<uint16_t*>(a.c) + (long long)p * a.sp + (long long)q0 * a.sq;
    if(a.sq == 1)
    {
        const bool vector = (reinterpret_cast<uintptr_t>(c) & 15) == 0;
#pragma unroll
        for(int j = 0; j < COLS; j += 8)
        {
            if(vector && q0 + j + 8 <= q_end)
                *reinterpret_cast<uint4*>(c + j) = make_uint4(v[j / 2], v[j / 2 + 1], v[j / 2 + 2], v[j / 2 + 3]);
            else
            {
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    if(q0 + j + i < q_end)
                        c[j + i] = (uint16_t)(v[(j + i) / 2] >> (16 * (i & 1)));
            }
        }
    }
    else
    {
        constexpr int STEP = 16;
        const int     n    = q_end - q0;
#pragma unroll
        for(int j0 = 0; j0 < COLS; j0 += STEP)
        {
            if(j0 >= n)
                break;
            if(j0 + STEP <= n)
            {
#pragma unroll
                for(int j = 0; j < STEP; ++j, c += a.sq)
                    *c = (uint16_t)(v[(j0 + j) / 2] >> (16 * (j & 1)));
            }
            else
            {
#pragma unroll
                for(int j = 0; j < STEP; ++j, c += a.sq)
                    if(j0 + j < n)
                        *c = (uint16_t)(v[(j0 + j) / 2] >> (16 * (j & 1)));
            }
        }
    }
}

template<int FMT, int BN, int PAIR, bool SUMS>
__global__ void __launch_bounds__(GLayout<FMT, BN, PAIR, SUMS>::THREADS, 1)
    mx4_gemm_kernel(const __grid_constant__ GArgs a, const __grid_constant__ Maps<PAIR> maps)
{
    using L = GLayout<FMT, BN, PAIR, SUMS>;
    constexpr int STAGES = L::STAGES;
    constexpr int COLS   = BN / 2; // columns of one epilogue thread
    extern __shared__ uint8_t smem_raw[];
    __shared__ int first_tile[G_MAX_GROUPS + 1];
    const uint32_t raw_addr = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t base     = (raw_addr + 1023u) & ~1023u;
    uint8_t*       ring     = smem_raw + (base - raw_addr);
    const uint32_t bar_base = base + STAGES * L::STAGE_BYTES;
    auto full      = [&](int s) { return bar_base + 8u * s; };
    auto empty     = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto acc_full  = [&](int b) { return bar_base + 8u * (2 * STAGES + b); };
    auto acc_empty = [&](int b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    const uint32_t drained = bar_base + 8u * (2 * STAGES + 4), parts = drained + 8u;
    uint8_t*       misc       = ring + STAGES * L::STAGE_BYTES + 8 * L::BARRIERS;
    uint32_t*      tmem_slot  = reinterpret_cast<uint32_t*>(misc);
    volatile int*  abort_flag = reinterpret_cast<volatile int*>(misc + 8);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int split = 1 << a.split_bits, shared_by = PAIR * split; // CTAs of the cluster, a power of two
    const int rank  = (int)(blockIdx.x & (shared_by - 1));
    const int lane0 = PAIR > 1 ? rank * G_LANES : 0; // this CTA's first lane in the tile
    const int first = blockIdx.x >> (a.split_bits + PAIR - 1), stride = gridDim.x >> (a.split_bits + PAIR - 1);
    const int part  = PAIR > 1 ? 0 : rank; // this CTA's range of K
    const int kb0 = (a.kblocks * part) >> a.split_bits, kb1 = (a.kblocks * (part + 1)) >> a.split_bits; // kblocks < 2^23
    // one stage of a tile: codes and scales of K block kb
    auto fill = [&](const Tile& t, int kb, int s) {
        const uint32_t st  = base + s * L::STAGE_BYTES;
        const uint32_t bar = PAIR > 1 ? cluster_addr(full(s), 0) : full(s);
        const bool     whole = L::Q_BOX == L::Q_ROWS || columns_of<BN, PAIR>(t) > L::Q_BOX; // or the first box alone
        // a pair's copies bring whole stages (zero beyond the matrix), a single CTA's the tiles that there are
        const int      tiles = PAIR > 1 ? L::TILES : min(L::TILES, a.k_tiles - kb * L::TILES);
        const int      band_p = t.group * a.bands_p + (t.p0 + lane0) / MX4_BAND, band_q = t.q0 / MX4_BAND;
        const uint32_t sp = st + L::P_BYTES + L::Q_BYTES, sq = sp + L::P_SCALES, bytes = tiles * MX4_TILE_BYTES;
        if(rank == 0 || PAIR == 1)
            mbar_arrive_expect_tx(full(s), PAIR * (L::P_BYTES + (whole ? L::Q_BYTES : L::BOX_BYTES) + bytes * (1 + L::Q_BANDS)));
        load_codes<PAIR>(st, &maps.p, kb * G_ROW_BYTES, t.group * a.np + t.p0 + lane0, bar);
        load_codes<PAIR>(st + L::P_BYTES, &maps.q, kb * G_ROW_BYTES, t.q0 + (PAIR > 1 ? rank * (columns_of<BN, PAIR>(t) / 2) : 0), bar);
        if(L::Q_BOX < L::Q_ROWS && whole)
            load_codes<PAIR>(st + L::P_BYTES + L::BOX_BYTES, &maps.q, kb * G_ROW_BYTES, t.q0 + L::Q_BOX, bar);
        if constexpr(PAIR > 1)
        {
            load_scales_pair(sp, &maps.scales_p, kb * L::TILES, band_p, bar);
            load_scales_pair(sq, &maps.scales_q, kb * L::TILES, band_q, bar);
        }
        else
        {
            bulk_load(sp, a.scales_p + ((size_t)band_p * a.k_tiles + kb * L::TILES) * MX4_TILE_BYTES, bytes, bar);
            bulk_load(sq, a.scales_q + ((size_t)band_q * a.k_tiles + kb * L::TILES) * MX4_TILE_BYTES, bytes, bar);
        }
    };
    int filled = 0; // stages that are on their way before the rest of the CTA is ready
    if(warp == G_TMA_WARP)
    {
        if(lane < (int)(sizeof(maps) / sizeof(CUtensorMap))) // the descriptors at once: each costs a trip to memory
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.p + lane)) : "memory");
        if(lane < L::BARRIERS) // one each: full, empty, acc_full, acc_empty, drained, parts
        {
            const bool of_epilogue = lane >= 2 * STAGES + 2 && lane < 2 * STAGES + 4;
            mbar_init(bar_base + 8u * lane, of_epilogue ? PAIR * G_EPILOGUE / 32 : 1);
            if(lane == 0)
                *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        if(PAIR == 1 && a.groups == 0) // nothing to wait for: this CTA's first tile and its barriers are known
        {
            const Tile t      = tile_at<BN, L::TILE_P>(a, nullptr, first);
            const bool issuer = elect_one();
            filled            = min(STAGES, kb1 - kb0);
            for(int i = 0; i < filled; ++i)
                if(issuer)
                    fill(t, kb0 + i, i);
            __syncwarp();
        }
    }
    if(warp == G_MMA_WARP)
    {
        tmem_alloc<PAIR>((uint32_t)__cvta_generic_to_shared(tmem_slot), G_TMEM_COLS);
        tmem_relinquish<PAIR>();
    }
    if(a.groups) // column tiles before each group
    {
        for(int e = threadIdx.x; e < a.groups; e += L::THREADS)
        {
            const int off = a.offsets[e], count = a.counts[e];
            int       n = 0;
            if(count > 0 && off >= 0 && off % MX4_BAND == 0 && count <= a.nq && off <= a.nq - count)
                n = (count + BN - 1) / BN;
            else if(count != 0 && blockIdx.x == 0)
                atomicOr(&g_mx4_status, G_ERR_GROUP);
            first_tile[e] = n;
        }
        __syncthreads();
        if(warp == G_TMA_WARP)
        {
            int  sum = 0;
            bool fits = true; // groups that do not overlap have no more tiles than that
            for(int e0 = 0; e0 < a.groups; e0 += 32)
            {
                const int e = e0 + lane, n = e < a.groups ? first_tile[e] : 0;
                int       up = n;
#pragma unroll
                for(int d = 1; d < 32; d <<= 1)
                {
                    const int v = __shfl_up_sync(0xFFFFFFFFu, up, d);
                    if(lane >= d)
                        up += v;
                }
                if(e < a.groups)
                    first_tile[e] = sum + up - n;
                sum += __shfl_sync(0xFFFFFFFFu, up, 31);
                fits = fits && sum <= a.most_q;
            }
            if(lane == 0)
            {
                first_tile[a.groups] = fits ? sum : 0;
                if(!fits && blockIdx.x == 0)
                    atomicOr(&g_mx4_status, G_ERR_GROUP);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if(PAIR > 1) // the other CTA's barriers and tensor memory are there
    {
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int      total     = (a.groups ? first_tile[a.groups] : (a.nq + BN - 1) / BN) * a.tiles_p;
    // the first wait of the CTA that gives up records where (bits 8..) and raises the abort flag for the others
    auto fail = [&](int where) {
        if(atomicExch(const_cast<int*>(abort_flag), 1) == 0)
            atomicOr(&g_mx4_status, G_ERR_WAIT | (256 << where));
    };

    if(SUMS && warp >= G_EPILOGUE / 32) // the whole warpgroup 8 to 11
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G_ISSUE_REGS));
    if(warp == G_TMA_WARP)
    {
        // here and below the whole warp walks the loop, so that addresses and descriptors are uniform, and one thread
        // issues: with the loop inside `if(lane == 0)` the compiler moved every operand of every instruction to the uniform
        // registers as if lanes could differ, and the 8192 cube took 680 us instead of 285
        const bool issuer = elect_one();
        uint32_t   s = filled % STAGES, ph = filled / STAGES;
        bool       ok = true;
        for(int tile = first; tile < total && ok; tile += stride)
        {
            const Tile t = tile_at<BN, L::TILE_P>(a, first_tile, tile);
            for(int kb = kb0 + (tile == first ? filled : 0); kb < kb1; ++kb)
            {
                if(!warp_wait(empty(s), ph ^ 1, abort_flag)) { fail(0); ok = false; break; }
                if(issuer)
                    fill(t, kb, s);
                __syncwarp();
                if(++s == STAGES)
                {
                    s = 0;
                    ph ^= 1;
                }
            }
        }
        // the copies in flight write to shared memory of this CTA (and of its pair, which stays until the end of both): wait
        // for each stage's last fill, if it had one
        if(!ok && (PAIR == 1 || rank == 0))
            for(int j = 0; j < STAGES; ++j)
            {
                const uint32_t fill = j < (int)s ? ph : ph ^ 1; // parity of the fill before the one that would come next
                drain_wait(full(j), fill);
            }
    }
    else if(warp == G_MMA_WARP)
    {
        const bool issuer = elect_one();
        uint32_t   s = 0, ph = 0, buf = 0, acc_ph = 0;
        bool       ok = true;
        for(int tile = first; tile < total && ok && (PAIR == 1 || rank == 0); tile += stride)
        {
            const Tile     t     = tile_at<BN, L::TILE_P>(a, first_tile, tile);
            // Q's rows start at column q_col of the band's scales: 0, or 2 for the second tile of 64 (an odd column is a fault)
            const uint32_t q_col = t.q0 % MX4_BAND / 32;
            const uint32_t idesc = mx4_idesc<FMT, PAIR>(columns_of<BN, PAIR>(t));
            int            in_chunk = 0;
            for(int kb = kb0; kb < kb1; ++kb)
            {
                if(in_chunk == 0 && !warp_wait(acc_empty(buf), acc_ph ^ 1, abort_flag)) { fail(1); ok = false; break; }
                if(!warp_wait(full(s), ph, abort_flag)) { fail(2); ok = false; break; }
                tc_fence_after();
                const bool last = in_chunk == a.chunk - 1 || kb == kb1 - 1;
                if(issuer)
                {
                    const uint32_t d    = tmem_base + buf * BN;
                    const uint32_t st   = base + s * L::STAGE_BYTES;
                    const uint32_t tp   = tmem_base + G_SCALE_COL + L::SLOT_COLS * s, tq = tp + 4 * L::TILES;
                    const uint64_t sp   = scales_desc(st + L::P_BYTES + L::Q_BYTES), sq = sp + (L::P_SCALES >> 4);
                    const uint64_t dp   = codes_desc(st), dq = dp + (L::P_BYTES >> 4);
                    const int      left = a.K - kb * G_KBLOCK;
#pragma unroll
                    for(int i = 0; i < L::TILES; ++i)
                        if(i * 4 * mx4_block(FMT) < left)
                        {
                            tc_copy_scales<PAIR>(tp + 4 * i, sp + i * (MX4_TILE_BYTES >> 4));
#pragma unroll
                            for(int b = 0; b < L::Q_BANDS; ++b) // an instruction takes the columns of all bands in a row
                                tc_copy_scales<PAIR>(tq + 4 * (i * L::Q_BANDS + b), sq + (b * L::TILES + i) * (MX4_TILE_BYTES >> 4));
                        }
#pragma unroll
                    for(int kk = 0; kk < G_KBLOCK / G_KSTEP; ++kk)
                        if(kk * G_KSTEP < left)
                        {
                            constexpr int  per = FMT == B200_SGEMM_NVFP4 ? 1 : 2; // instructions per scale tile
                            const uint32_t id  = kk % per * 2;                    // first byte of the scale words it takes
                            constexpr int  off = G_KSTEP / 2 >> 4;
                            tc_mma_mx4<FMT, PAIR>(d, dp + kk * off, dq + kk * off, idesc | id << 4 | id << 29,
                                                  tp + kk / per * 4, tq + kk / per * 4 * L::Q_BANDS + q_col, in_chunk > 0 || kk > 0);
                        }
                    tc_commit<PAIR>(empty(s));
                    if(last)
                        tc_commit<PAIR>(acc_full(buf));
                }
                __syncwarp();
                in_chunk = last ? 0 : in_chunk + 1;
                if(last && ++buf == L::ACCS)
                {
                    buf = 0;
                    acc_ph ^= 1;
                }
                if(++s == STAGES)
                {
                    s = 0;
                    ph ^= 1;
                }
            }
        }
        if(!ok && issuer) // the products in flight write to tensor memory that is about to be freed
        {
            tc_commit<PAIR>(drained);
            drain_wait(drained, 0);
        }
    }
    else if(warp < G_EPILOGUE / 32)
    {
        if constexpr(SUMS)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G_SUM_REGS));
        const int quarter = warp & 3, half = warp >> 2;
        uint32_t  buf = 0, acc_ph = 0;
        bool      ok     = true;
        const int n_chunks = (kb1 - kb0 + a.chunk - 1) / a.chunk;
        float     factor_q = a.alpha;
        if(a.global_q)
            factor_q *= *a.global_q;
        for(int tile = first; tile < total && ok; tile += stride)
        {
            const Tile t = tile_at<BN, L::TILE_P>(a, first_tile, tile);
            const float factor = a.global_p ? factor_q * a.global_p[t.group] : factor_q; // fetched while the tile is computed
            if constexpr(L::ACCS == 1 && !SUMS) // 16 bits, all of K: rounded into registers, so that the one accumulator is free at once
            {
                uint32_t    out[COLS / 2];
                if(!warp_wait(acc_full(0), acc_ph, abort_flag)) { fail(3); ok = false; break; }
                tc_fence_after();
                const uint32_t from = tmem_base + half * COLS + (uint32_t(quarter * 32) << 16);
                auto empty_into = [&](auto pack) { // packed while the next 32 columns are on their way
                    uint32_t v[2][32];
                    tmem_ld32(from, v[0]);
#pragma unroll
                    for(int c = 0; c < COLS; c += 32)
                    {
                        tmem_ld_wait();
                        if(c + 32 < COLS)
                            tmem_ld32(from + c + 32, v[(c / 32 + 1) % 2]);
                        else
                        {
                            tc_fence_before();
                            __syncwarp();
                            if(lane == 0)
                                mbar_arrive_cluster(cluster_addr(acc_empty(0), 0));
                        }
#pragma unroll
                        for(int j = 0; j < 32; j += 2)
                            out[(c + j) / 2] = pack(__uint_as_float(v[c / 32 % 2][j]) * factor, __uint_as_float(v[c / 32 % 2][j + 1]) * factor);
                    }
                };
                if(a.type == B200_SGEMM_F16)
                    empty_into([](float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); });
                else
                    empty_into([](float x, float y) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); });
                acc_ph ^= 1;
                store_packed<COLS>(a, out, t.p0 + lane0 + quarter * 32 + lane, t.q0 + half * COLS, t.q_end);
                continue;
            }
            else
            {
                float acc[COLS];
                for(int ch = 0; ch < n_chunks; ++ch)
                {
                    if(!warp_wait(acc_full(buf), acc_ph, abort_flag)) { fail(3); ok = false; break; }
                    tc_fence_after();
                    const uint32_t from = tmem_base + buf * BN + half * COLS + (uint32_t(quarter * 32) << 16);
                    // SUMS: 16 columns at a time, added while the next are on their way (32 at a time spill)
                    constexpr int STEP = SUMS ? 16 : COLS;
                    uint32_t      v[2][STEP];
                    auto          load = [&](int c) {
#pragma unroll
                        for(int j = 0; j < STEP; j += 16)
                            tmem_ld16(from + c + j, v[c / STEP % 2] + j);
                    };
                    load(0);
#pragma unroll
                    for(int c = 0; c < COLS; c += STEP)
                    {
                        tmem_ld_wait();
                        if(c + STEP < COLS)
                            load(c + STEP);
                        else
                        {
                            tc_fence_before();
                            __syncwarp();
                            if(lane == 0) // the accumulator is free before its last values are added
                            {
                                if(PAIR > 1)
                                    mbar_arrive_cluster(cluster_addr(acc_empty(buf), 0));
                                else
                                    mbar_arrive(acc_empty(buf));
                            }
                        }
#pragma unroll
                        for(int j = 0; j < STEP; ++j)
                        {
                            const float part = __uint_as_float(v[c / STEP % 2][j]);
                            acc[c + j]       = ch == 0 ? part : acc[c + j] + part;
                        }
                    }
                    if(++buf == L::ACCS)
                    {
                        buf = 0;
                        acc_ph ^= 1;
                    }
                }
                if(!ok)
                    break;
                const int p = lane0 + quarter * 32 + lane, q = half * COLS;
                if(PAIR > 1 || split == 1)
                    store_typed(a, acc, factor, t.p0 + p, t.q0 + q, t.q_end);
                else // park the part in the ring, which is at rest: a CTA of a split tile has no other
                {
                    float* parked = reinterpret_cast<float*>(ring);
#pragma unroll
                    for(int j = 0; j < COLS; ++j)
                        if(t.q0 + q + j < t.q_end)
                            parked[(q + j) * G_LANES + p] = acc[j];
                    fence_async_smem(); // for the copies below
                }
            }
        }
    }

    __syncwarp();
    if(PAIR == 1 && split > 1)
    {
        cluster_arrive(); // all parts are parked and all rings at rest
        cluster_wait();
        if(first < total && warp < G_EPILOGUE / 32)
        {
            // CTA r adds and stores columns r * share .. of the tile; the others' parts come by bulk copies into the upper half of
            // its ring (single words written or read across the cluster take about 60 cycles a warp: 6 us for 64 columns)
            constexpr uint32_t UPPER = STAGES * L::STAGE_BYTES / 2;
            const Tile         t       = tile_at<BN, L::TILE_P>(a, first_tile, first);
            const int          columns = min(BN, t.q_end - t.q0), share = (columns + split - 1) / split;
            const int          mine    = max(0, min(share, columns - rank * share));
            if(threadIdx.x == 0 && mine)
                mbar_arrive_expect_tx(parts, (uint32_t)(split - 1) * mine * G_LANES * 4);
            if(threadIdx.x < split && threadIdx.x != rank)
            {
                const int r = threadIdx.x, theirs = max(0, min(share, columns - r * share));
                if(theirs)
                    bulk_send(cluster_addr(base + UPPER + (uint32_t)(rank * share * G_LANES) * 4, r), base + (uint32_t)(r * share * G_LANES) * 4,
                              (uint32_t)theirs * G_LANES * 4, cluster_addr(parts, r));
            }
            __syncwarp();
            if(mine && !warp_wait(parts, 0, abort_flag))
                fail(4);
            else
            {
                float factor = a.alpha;
                if(a.global_q)
                    factor *= *a.global_q;
                if(a.global_p)
                    factor *= a.global_p[t.group];
                const float* own   = reinterpret_cast<const float*>(ring) + rank * share * G_LANES;
                const float* other = reinterpret_cast<const float*>(ring + UPPER); // [rank][column][lane]
                const int    p     = threadIdx.x & (G_LANES - 1);
                // eight columns at a time, so that their reads overlap
                constexpr int STEP = 8, STRIDE = G_EPILOGUE / G_LANES;
                for(int i0 = threadIdx.x / G_LANES; i0 < mine; i0 += STEP * STRIDE)
                {
                    float sum[STEP];
#pragma unroll
                    for(int j = 0; j < STEP; ++j)
                        sum[j] = 0.f;
                    for(int r = 0; r < split; ++r)
                    {
                        const float* from = r == rank ? own : other + r * share * G_LANES;
#pragma unroll
                        for(int j = 0; j < STEP; ++j)
                            if(i0 + j * STRIDE < mine)
                                sum[j] += from[(i0 + j * STRIDE) * G_LANES + p];
                    }
                    const long long at = (long long)(t.p0 + p) * a.sp + (long long)(t.q0 + rank * share + i0) * a.sq;
                    const int       n  = t.p0 + p < a.np ? (mine - i0 + STRIDE - 1) / STRIDE : 0;
                    if(a.type == B200_SGEMM_F32)
                        store_strided(static_cast<float*>(a.c) + at, sum, factor, STRIDE * a.sq, n);
                    else if(a.type == B200_SGEMM_F16)
                        store_strided(static_cast<__half*>(a.c) + at, sum, factor, STRIDE * a.sq, n);
                    else
                        store_strided(static_cast<__nv_bfloat16*>(a.c) + at, sum, factor, STRIDE * a.sq, n);
                }
            }
        }
        __syncwarp();
        cluster_arrive(); // nobody leaves while its part is being read
        cluster_wait();
    }
    tc_fence_before();
    if(PAIR > 1) // neither CTA leaves while the other's instructions or copies may reach it
    {
        cluster_arrive();
        cluster_wait();
    }
    else
        __syncthreads();
    if(warp == G_MMA_WARP)
    {
        tc_fence_after();
        tmem_dealloc<PAIR>(tmem_base, G_TMEM_COLS);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder()
{
    static EncodeFn fn = [] {
        void*                           p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess
           || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// rows of `pitch` code bytes; box = 128 bytes x box_rows rows, 128-byte swizzle
bool encode_codes(CUtensorMap* map, const void* codes, size_t rows, size_t pitch, int box_rows)
{
    EncodeFn fn = encoder();
    if(!fn)
        return false;
    const cuuint64_t dims[2]    = {(cuuint64_t)pitch, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2]     = {(cuuint32_t)G_ROW_BYTES, (cuuint32_t)box_rows};
    const cuuint32_t estr[2]    = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// scale tiles as (512 bytes, tile along k, band); box = the tiles of a stage x `bands`
bool encode_scales(CUtensorMap* map, const void* scales, size_t tiles, size_t bands, int box_tiles, int box_bands)
{
    EncodeFn fn = encoder();
    if(!fn)
        return false;
    const cuuint64_t dims[3]    = {MX4_TILE_BYTES / 4, (cuuint64_t)tiles, (cuuint64_t)bands};
    const cuuint64_t strides[2] = {MX4_TILE_BYTES, (cuuint64_t)tiles * MX4_TILE_BYTES};
    const cuuint32_t box[3]     = {MX4_TILE_BYTES / 4, (cuuint32_t)box_tiles, (cuuint32_t)box_bands};
    const cuuint32_t estr[3]    = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(scales), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int MAX_DEVICES = 64;

// the current device and its SMs; also binds the device's context to this thread, which the driver's encoder needs
int device_sms(int* device_out, int* sms)
{
    static std::atomic<int> known[MAX_DEVICES];
    int                     device = 0;
    cudaError_t             e      = cudaGetDevice(&device);
    if(e != cudaSuccess)
        return (int)e;
    static thread_local int bound = -1;
    if(bound != device)
    {
        if((e = cudaSetDevice(device)) != cudaSuccess)
            return (int)e;
        bound = device;
    }
    int n = device < MAX_DEVICES ? known[device].load(std::memory_order_relaxed) : 0;
    if(!n)
    {
        if((e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device)) != cudaSuccess)
            return (int)e;
        if(device < MAX_DEVICES)
            known[device].store(n, std::memory_order_relaxed);
    }
    *device_out = device;
    *sms = n;
    return B200_SGEMM_OK;
}

struct Operand
{
    const void* codes;
    const void* scales;
    size_t      rows, bands; // of the whole array: all groups
};

// How a product is cut: the columns of a tile (256: by pairs of CTAs) and the CTAs that share its K.
struct Cut
{
    int columns, split;
};
// The cut with the least estimated time, from what two dozen shapes between 100 x 1000 x 300 and 2560^3 measured (us): a K block
// takes 0.33 / 0.37 / 0.37 in tiles of 64 / 128 / 256 columns, for the SMs go through it at about the same pace whatever
// its width; storing a tile 1.1 / 1.75 / 2.3 where the next tile's blocks do not hide it, and 0.4 / 0.9 / 2 more at the end; FP32
// results (and any whose parts are added) in 256 columns 0.4 a block, 3.7 and 3.5; adding the parts of a split tile 2.2 / 3.3.
// Examples, us for (columns, split), BF16: 2048^3 (128, 1) 11.5, (256, 1) 9.1; 64 x 8192 x 8192 (64, 1) 13.9, (64, 2) 12.1,
// (128, 2) 12.9; 512 x 512 x 8192 (64, 1) 13.5, (64, 4) 9.7; 512^3 (64, 1) 4.7, (64, 2) 7.0, (128, 1) 5.4.
// lane_rows, column_rows: extents of one group; clusters of 8 and 4 CTAs do not fill every part of the chip, so they are held
// below three quarters and seven eighths of the SMs.
Cut cut_of(size_t lane_rows, size_t column_rows, size_t groups, int kblocks, bool in_parts, bool may_split, int sms)
{
    Cut   best = {64, 1};
    float least = 1e30f;
    for(int i = 0; i < 3; ++i)
    {
        const int    columns = 64 << i, lanes = i == 2 ? 256 : 128, slots = i == 2 ? sms / 2 : sms;
        const bool   sums  = in_parts && i == 2;
        const float  block = i == 0 ? 0.33f : (sums ? 0.4f : 0.37f), join = i == 0 ? 2.2f : 3.3f;
        const float  store = i == 0 ? 1.1f : (i == 1 ? 1.75f : (sums ? 3.7f : 2.3f));
        const float  end   = i == 0 ? 0.4f : (i == 1 ? 0.9f : (sums ? 3.5f : 2.f));
        const size_t tiles = (lane_rows + lanes - 1) / lanes * ((column_rows + columns - 1) / columns) * groups;
        for(int split = 1; split <= (may_split && i < 2 ? MAX_SPLIT : 1); split *= 2)
        {
            const size_t room = split == 8 ? sms * 3 / 4 : (split == 4 ? sms * 7 / 8 : slots);
            if(split > 1 && (tiles * split > room || split > kblocks))
                break;
            const float waves = (float)((tiles * split + slots - 1) / slots);
            const float one   = (float)((kblocks + split - 1) / split) * block;
            const float time  = (waves - 1.f) * (one > store ? one : store) + one + end + (split > 1 ? join : 0.f);
            if(time < least)
            {
                least = time;
                best  = {columns, split};
            }
        }
    }
    return best;
}

template<int FMT, int BN, int PAIR, bool SUMS = false>
int launch(GArgs a, const Operand& p, const Operand& q, int device, int sms, cudaStream_t stream)
{
    using L      = GLayout<FMT, BN, PAIR, SUMS>;
    auto  kernel = mx4_gemm_kernel<FMT, BN, PAIR, SUMS>;
    const size_t pitch = mx4_pitch((size_t)a.K), k_tiles = mx4_tiles(FMT, (size_t)a.K);
    Maps<PAIR> maps;
    if(!encode_codes(&maps.p, p.codes, p.rows, pitch, G_LANES) || !encode_codes(&maps.q, q.codes, q.rows, pitch, L::Q_BOX))
        return B200_SGEMM_NO_KERNEL;
    if constexpr(PAIR > 1)
    {
        if(!encode_scales(&maps.scales_p, p.scales, k_tiles, p.bands, L::TILES, 1)
           || !encode_scales(&maps.scales_q, q.scales, k_tiles, q.bands, L::TILES, L::Q_BANDS))
            return B200_SGEMM_NO_KERNEL;
    }
    a.scales_p = static_cast<const uint8_t*>(p.scales);
    a.scales_q = static_cast<const uint8_t*>(q.scales);
    a.k_tiles  = (int)k_tiles;
    a.tiles_p = (a.np + L::TILE_P - 1) / L::TILE_P;
    // no more than these hold rows: groups start on multiples of 128, for wider tiles each can add one
    const unsigned long long tiles_q = ((unsigned long long)a.nq + BN - 1) / BN + (BN > MX4_BAND ? a.groups : 0);
    const unsigned long long tiles   = tiles_q * a.tiles_p;
    if(tiles > 0x3fffffffull) // the CTAs step beyond the last one
        return B200_SGEMM_UNSUPPORTED_SIZE;
    a.most_q = (int)tiles_q;
    // one tile per cluster where K is split, otherwise as many CTAs as there are tiles or SMs
    const int      split    = 1 << a.split_bits;
    const unsigned clusters = (unsigned)(split > 1 || tiles < (unsigned long long)(sms / PAIR) ? tiles : sms / PAIR);
    static std::atomic<unsigned long long> ready{0}; // devices on which the kernel may have its shared memory
    const unsigned long long               bit = 1ull << (device % MAX_DEVICES);
    if(device >= MAX_DEVICES || !(ready.load(std::memory_order_relaxed) & bit))
    {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM_BYTES);
        if(e != cudaSuccess)
            return (int)e;
        if(SUMS)
        {
            cudaFuncAttributes f;
            if(const cudaError_t e = cudaFuncGetAttributes(&f, kernel); e != cudaSuccess)
                return (int)e;
            if(f.numRegs != G_LAUNCH_REGS) // the registers would not add up (the build refuses such a kernel)
                return B200_SGEMM_NO_KERNEL;
        }
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(clusters * PAIR * split);
    cfg.blockDim           = dim3(L::THREADS);
    cfg.dynamicSmemBytes   = L::SMEM_BYTES;
    cfg.stream             = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id               = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)(PAIR * split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs                = attr;
    cfg.numAttrs             = PAIR * split > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, kernel, a, maps);
}

template<int FMT>
int launch_tile(int columns, const GArgs& a, const Operand& p, const Operand& q, int device, int sms, cudaStream_t stream)
{
    if(columns == 256 && a.type != B200_SGEMM_F32 && a.chunk >= a.kblocks)
        return launch<FMT, 256, 2>(a, p, q, device, sms, stream);
    if(columns == 256) // a build whose registers do not add up takes narrower tiles
    {
        const int status = launch<FMT, 256, 2, true>(a, p, q, device, sms, stream);
        if(status != B200_SGEMM_NO_KERNEL)
            return status;
    }
    return columns == 64 ? launch<FMT, 64, 1>(a, p, q, device, sms, stream) : launch<FMT, 128, 1>(a, p, q, device, sms, stream);
}

// K blocks that one accumulator of a 16-bit result may hold
int most_blocks(int type) { return type == B200_SGEMM_F16 ? CHUNK_F16 : CHUNK_BF16; }
int blocks_of(size_t K) { return (int)((K + G_KBLOCK - 1) / G_KBLOCK); }
bool added_in_parts(int type, int kblocks) { return type == B200_SGEMM_F32 || kblocks > most_blocks(type); }

// The cut of a product of `lanes` rows of P and `columns` of Q, or the rows of Q to be expected in one of `groups`.
Cut cut_for(int type, size_t lanes, size_t columns, size_t groups, size_t K, int sms)
{
    const int kblocks = blocks_of(K);
    return cut_of(lanes, columns, groups ? groups : 1, kblocks, added_in_parts(type, kblocks), groups == 0, sms);
}
// whether B takes the lanes: they are C's contiguous dimension, unless that one is short and the other is not
bool lanes_from_b(bool row, size_t M, size_t N)
{
    const size_t packed = row ? N : M;
    return packed <= 64 && (row ? M : N) > packed ? !row : row;
}
size_t rows_of_group(size_t rows, size_t groups) { return (rows + groups - 1) / groups; }

// `a` holds what both entries agree on; `columns` as in cut_for
int run(int format, GArgs a, const Operand& p, const Operand& q, size_t K, size_t columns, cudaStream_t stream)
{
    int device = 0, sms = 0, status = device_sms(&device, &sms);
    if(status != B200_SGEMM_OK)
        return status;
    a.K           = (int)K;
    a.kblocks     = blocks_of(K);
    a.bands_p     = (a.np + MX4_BAND - 1) / MX4_BAND;
    const Cut cut = cut_for(a.type, (size_t)a.np, columns, (size_t)a.groups, K, sms);
    while((1 << a.split_bits) < cut.split)
        ++a.split_bits;
    if(!added_in_parts(a.type, a.kblocks))
        a.chunk = a.kblocks;
    else
        a.chunk = a.type != B200_SGEMM_F32 ? most_blocks(a.type) : (cut.columns == 256 ? CHUNK_F32_WIDE : CHUNK_F32);
    return format == B200_SGEMM_NVFP4 ? launch_tile<B200_SGEMM_NVFP4>(cut.columns, a, p, q, device, sms, stream)
                                      : launch_tile<B200_SGEMM_MXFP4>(cut.columns, a, p, q, device, sms, stream);
}
} // namespace

extern "C" int b200_sgemm_mx4(int format, int layout_c, int type_c, void* C, const void* a_codes, const void* a_scales,
                              const void* b_codes, const void* b_scales, size_t M, size_t N, size_t K, size_t ldc, float alpha,
                              const float* global_a, const float* global_b, void* cuda_stream)
{
    if(!C || !a_codes || !a_scales || !b_codes || !b_scales || M == 0 || N == 0 || K == 0 || !mx4_format_ok(format)
       || !type_ok(type_c) || layout_c & ~1)
        return B200_SGEMM_INVALID_ARGUMENT;
    if(M > MAX_EXTENT || N > MAX_EXTENT || K > MAX_EXTENT)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    const bool   row = layout_c == B200_SGEMM_ROW_MAJOR;
    const size_t packed = row ? N : M;
    if(ldc == 0)
        ldc = packed;
    if(ldc < packed || misaligned(C, type_bytes(type_c)) || misaligned(a_codes, 16) || misaligned(a_scales, 16)
       || misaligned(b_codes, 16) || misaligned(b_scales, 16) || misaligned(global_a, 4) || misaligned(global_b, 4)
       || (format == B200_SGEMM_MXFP4 && (global_a || global_b)))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(ldc > (size_t(1) << 40))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    const Operand a{a_codes, a_scales, M, (M + MX4_BAND - 1) / MX4_BAND}, b{b_codes, b_scales, N, (N + MX4_BAND - 1) / MX4_BAND};
    if(mx4_is_few(M < N ? M : N, M < N ? N : M, K))
    {
        const bool b_long = N >= M;
        int        device = 0, sms = 0, status = device_sms(&device, &sms);
        if(status != B200_SGEMM_OK)
            return status;
        FewArgs f;
        f.codes    = b_long ? b_codes : a_codes;
        f.scales   = b_long ? b_scales : a_scales;
        f.codes_x  = b_long ? a_codes : b_codes;
        f.scales_x = b_long ? a_scales : b_scales;
        f.global   = b_long ? global_b : global_a;
        f.global_x = b_long ? global_a : global_b;
        f.c        = C;
        f.ld_long  = b_long == row ? 1 : (long long)ldc;
        f.ld_few   = b_long == row ? (long long)ldc : 1;
        f.alpha    = alpha;
        f.rows     = (int)(b_long ? N : M);
        f.few      = (int)(b_long ? M : N);
        f.K        = (int)K;
        f.type     = type_c;
        return mx4_few(format, f, sms, static_cast<cudaStream_t>(cuda_stream));
    }
    const bool b_lanes = lanes_from_b(row, M, N);
    GArgs g     = {};
    g.c         = C;
    g.sp        = b_lanes == row ? 1 : (long long)ldc;
    g.sq        = b_lanes == row ? (long long)ldc : 1;
    g.global_p  = b_lanes ? global_b : global_a;
    g.global_q  = b_lanes ? global_a : global_b;
    g.alpha     = alpha;
    g.np        = (int)(b_lanes ? N : M);
    g.nq        = (int)(b_lanes ? M : N);
    g.type      = type_c;
    return run(format, g, b_lanes ? b : a, b_lanes ? a : b, K, (size_t)g.nq, static_cast<cudaStream_t>(cuda_stream));
}

extern "C" int b200_sgemm_mx4_grouped(int format, int type_c, void* C, const void* a_codes, const void* a_scales, const void* b_codes,
                                      const void* b_scales, size_t rows, size_t N, size_t K, size_t ldc, size_t groups,
                                      const int* offsets, const int* counts, size_t used_rows, float alpha,
                                      const float* global_a, const float* global_b, void* cuda_stream)
{
    if(!C || !a_codes || !a_scales || !b_codes || !b_scales || !offsets || !counts || rows == 0 || N == 0 || K == 0 || groups == 0
       || !mx4_format_ok(format) || !type_ok(type_c))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(rows > MAX_EXTENT || N > MAX_EXTENT || K > MAX_EXTENT || groups > G_MAX_GROUPS || groups * N > MAX_EXTENT)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    if(ldc == 0)
        ldc = N;
    if(ldc < N || misaligned(C, type_bytes(type_c)) || misaligned(a_codes, 16) || misaligned(a_scales, 16)
       || misaligned(b_codes, 16) || misaligned(b_scales, 16) || misaligned(offsets, 4) || misaligned(counts, 4)
       || misaligned(global_a, 4) || misaligned(global_b, 4) || (format == B200_SGEMM_MXFP4 && (global_a || global_b)))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(ldc > (size_t(1) << 40))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    GArgs g    = {};
    g.c        = C;
    g.sp       = 1;
    g.sq       = (long long)ldc;
    g.offsets  = offsets;
    g.counts   = counts;
    g.global_p = global_b;
    g.global_q = global_a;
    g.alpha    = alpha;
    g.np       = (int)N;
    g.nq       = (int)rows;
    g.groups   = (int)groups;
    g.type     = type_c;
    const size_t used = used_rows && used_rows < rows ? used_rows : rows;
    const Operand b{b_codes, b_scales, groups * N, groups * ((N + MX4_BAND - 1) / MX4_BAND)};
    const Operand a{a_codes, a_scales, rows, (rows + MX4_BAND - 1) / MX4_BAND};
    return run(format, g, b, a, K, rows_of_group(used, groups), static_cast<cudaStream_t>(cuda_stream));
}

extern "C" int b200_sgemm_mx4_plan(int layout_c, int type_c, size_t M, size_t N, size_t K, size_t groups, int sm_count, int* columns,
                                   int* split)
{
    if(!columns || !split || M == 0 || N == 0 || K == 0 || !type_ok(type_c) || layout_c & ~1 || sm_count < 2
       || (groups && layout_c != B200_SGEMM_ROW_MAJOR))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(M > MAX_EXTENT || N > MAX_EXTENT || K > MAX_EXTENT || groups > G_MAX_GROUPS || groups * N > MAX_EXTENT)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    if(groups == 0 && mx4_is_few(M < N ? M : N, M < N ? N : M, K))
    {
        *columns = 0;
        *split   = 1;
        return B200_SGEMM_OK;
    }
    const bool b_lanes = groups || lanes_from_b(layout_c == B200_SGEMM_ROW_MAJOR, M, N);
    const Cut  cut     = cut_for(type_c, b_lanes ? N : M, groups ? rows_of_group(M, groups) : (b_lanes ? M : N), groups, K, sm_count);
    *columns = cut.columns;
    *split   = cut.split;
    return B200_SGEMM_OK;
}

extern "C" int b200_sgemm_mx4_device_status(int* status)
{
    if(!status)
        return B200_SGEMM_INVALID_ARGUMENT;
    cudaError_t e = cudaDeviceSynchronize();
    if(e != cudaSuccess)
        return (int)e;
    const int zero = 0;
    if((e = cudaMemcpyFromSymbol(status, g_mx4_status, sizeof(int))) != cudaSuccess)
        return (int)e;
    if(*status)
        e = cudaMemcpyToSymbol(g_mx4_status, &zero, sizeof(int));
    return (int)e;
}
