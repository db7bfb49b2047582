// C ABI and host dispatch of the B200 SGEMM library (declarations and reference citations:
// include/b200_sgemm.h).  Host-side roles covered here:
//   * rocm_sgemm::gemm                       (rocm_sgemm/src/gemm.cpp:8-41)        -> b200_sgemm / b200_sgemm_ex
//   * kernel_launcher<...>::launch           (rocm_sgemm/include/rocm_sgemm/kernel_launcher.hpp:35-100)
//   * lookup_kernel                          (rocm_sgemm/include/rocm_sgemm/kernel_lookup.hpp:39)
//   * detail::find_best_config and the tables generated by rocm_sgemm/config/generate_config.py:97-303
#include "../../include/b200_sgemm.h"
#include "config_select.hpp"
#include "transpose.hpp"
#include "sgemm_kernel.cuh"
#include "sgemm_ws_kernel.cuh"

#include <climits>
#include <cstring>
#include <cstdint>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

namespace sgemm_b200
{
#include "generated/config_table.inc"

const void* lookup_kernel(int variant, int layout_idx, int aligned); // generated/kernel_lookup.cu

// one status word per device that loads the library; kernels write it only when a bounded wait gives up
__device__ int g_kernel_status = 0;

// ------------------------------------------------------------------------------------------------
// split-K: C = partial[0] + partial[1] + ... in ascending slice order (deterministic).
// The partial results are packed `outer` x `inner` matrices in C's own orientation (inner = the
// contiguous extent: N for row-major C, M for col-major); C itself may have a leading dimension.
// ------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) splitk_reduce_kernel(float* __restrict__ C, const float* __restrict__ partial,
                                                            long long inner, long long outer, long long ldc,
                                                            long long split_stride, int splits, int vec_ok)
{
    const long long stride = (long long)gridDim.x * blockDim.x;
    long long       i      = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if(vec_ok)
    {
        const long long inner4 = inner >> 2;
        const long long n4     = inner4 * outer;
        for(; i < n4; i += stride)
        {
            float4 s = __ldcs(reinterpret_cast<const float4*>(partial) + i);
            for(int k = 1; k < splits; ++k)
            {
                const float4 v = __ldcs(reinterpret_cast<const float4*>(partial + (long long)k * split_stride) + i);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            const long long o = i / inner4, in4 = i - o * inner4;
            *reinterpret_cast<float4*>(C + o * ldc + 4 * in4) = s;
        }
    }
    else
    {
        const long long n = inner * outer;
        for(; i < n; i += stride)
        {
            float s = partial[i];
            for(int k = 1; k < splits; ++k)
                s += partial[(long long)k * split_stride + i];
            const long long o = i / inner;
            C[o * ldc + (i - o * inner)] = s;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Pre-transposition of a K-contiguous operand: src is X rows of K contiguous floats (pitch ld_in),
// dst is K rows of X contiguous floats (pitch ld_out, a multiple of 4 so that TMA can read it).
// 64 x 64 tiles through padded shared memory; 128-bit loads along K when `vec_in`, 128-bit stores
// along X.  HBM-bound: 8 bytes moved per element.  One-dimensional grid (k-blocks fastest), so that neither extent
// is bound by the 65535 limit of gridDim.y.
// ------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) transpose_kernel(const float* __restrict__ src, float* __restrict__ dst, int X,
                                                        int K, long long ld_in, long long ld_out, int vec_in,
                                                        unsigned k_blocks)
{
    __shared__ float tile[64][65];
    const unsigned bx = blockIdx.x / k_blocks;
    const int      k0 = (int)(blockIdx.x - bx * k_blocks) * 64, x0 = (int)bx * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const int    xl = ty + 16 * i, x = x0 + xl, k = k0 + 4 * tx;
        float4       v   = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* row = src + (long long)x * ld_in + k;
        if(x < X)
        {
            if(vec_in && k + 3 < K)
                v = __ldcs(reinterpret_cast<const float4*>(row));
            else
            {
                if(k + 0 < K) v.x = row[0];
                if(k + 1 < K) v.y = row[1];
                if(k + 2 < K) v.z = row[2];
                if(k + 3 < K) v.w = row[3];
            }
        }
        tile[xl][4 * tx + 0] = v.x;
        tile[xl][4 * tx + 1] = v.y;
        tile[xl][4 * tx + 2] = v.z;
        tile[xl][4 * tx + 3] = v.w;
    }
    __syncthreads();
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const int kl = ty + 16 * i, k = k0 + kl, x = x0 + 4 * tx;
        if(k < K && x < X)
        {
            const float4 v = make_float4(tile[4 * tx + 0][kl], tile[4 * tx + 1][kl], tile[4 * tx + 2][kl],
                                         tile[4 * tx + 3][kl]);
            float* out = dst + (long long)k * ld_out + x;
            if(x + 3 < X)
                *reinterpret_cast<float4*>(out) = v;
            else
            {
                out[0] = v.x;
                if(x + 1 < X) out[1] = v.y;
                if(x + 2 < X) out[2] = v.z;
            }
        }
    }
}

cudaError_t launch_transpose(const float* src, float* dst, size_t X, size_t K, size_t ld_in, size_t ld_out,
                             cudaStream_t stream)
{
    const int                vec_in = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 && ld_in % 4 == 0;
    const unsigned long long kb = (K + 63) / 64, xb = (X + 63) / 64;
    if(X > INT_MAX || K > INT_MAX || kb * xb > 0x7fffffffull)
        return cudaErrorInvalidConfiguration;
    transpose_kernel<<<(unsigned)(kb * xb), 256, 0, stream>>>(src, dst, (int)X, (int)K, (long long)ld_in,
                                                             (long long)ld_out, vec_in, (unsigned)kb);
    return cudaPeekAtLastError();
}

// device address of the current device's status word, for the self-test's private kernel copy (sgemm_selftest.cu)
int* status_word_address();

namespace
{
    // ---- per-kernel shared-memory opt-in, once per (kernel, device) ------------------------------
    std::mutex                               g_attr_mutex;
    std::map<std::pair<const void*, int>, size_t> g_attr_done; // the size the kernel has been opted in for

    cudaError_t ensure_smem_attr(const void* fn, int device, size_t smem)
    {
        if(smem <= 48 * 1024)
            return cudaSuccess;
        std::lock_guard<std::mutex> lock(g_attr_mutex);
        auto                        key = std::make_pair(fn, device);
        auto                        it  = g_attr_done.find(key);
        if(it != g_attr_done.end() && it->second >= smem)
            return cudaSuccess;
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if(e == cudaSuccess)
            g_attr_done[key] = smem;
        return e;
    }

    // ---- internal split-K arena for the drop-in entry (which has no workspace argument) ----------
    // Layout of an arena: [flags, ARENA_FLAG_BYTES][whatever the call needs].  The flag words sit at a fixed place
    // so that they only ever hold zero or the epoch of an earlier launch (they are cleared when the block is
    // allocated and never used for anything else); `epoch` counts the launches that used them.  First the words of
    // the accumulator hand-over (one per CTA and consumer warp), then one word per block of the operands that the
    // kernel transposes itself.
    constexpr size_t ARENA_HANDOVER_FLAG_BYTES = 64 * 1024;
    constexpr size_t ARENA_FLAG_BYTES          = 1024 * 1024;
    constexpr size_t ARENA_COOP_FLAG_WORDS     = (ARENA_FLAG_BYTES - ARENA_HANDOVER_FLAG_BYTES) / sizeof(unsigned);
    struct Arena
    {
        void*    ptr   = nullptr;
        size_t   bytes = 0;
        unsigned epoch = 0;
        unsigned coop_total = 0; // what the block's "transposing warps finished" word reads after the launches so far
    };
    std::mutex                                        g_arena_mutex;
    std::map<std::pair<int, cudaStream_t>, Arena>     g_arenas;

    cudaError_t arena_get(int device, cudaStream_t stream, size_t bytes, void** out, unsigned* epoch)
    {
        bytes += ARENA_FLAG_BYTES;
        std::lock_guard<std::mutex> lock(g_arena_mutex);
        Arena&                      a = g_arenas[std::make_pair(device, stream)];
        if(a.bytes < bytes)
        {
            if(a.ptr)
            {
                // work queued on this stream may still read the old block
                cudaError_t e = cudaStreamSynchronize(stream);
                if(e != cudaSuccess)
                    return e;
                cudaFree(a.ptr);
                a.ptr   = nullptr;
                a.bytes = 0;
            }
            cudaError_t e = cudaMalloc(&a.ptr, bytes);
            if(e != cudaSuccess)
            {
                (void)cudaGetLastError(); // the caller is told: keep it out of later launches' checks
                return e;
            }
            e = cudaMemsetAsync(a.ptr, 0, ARENA_FLAG_BYTES, stream);
            if(e != cudaSuccess)
            {
                cudaFree(a.ptr);
                a.ptr = nullptr;
                return e;
            }
            a.bytes      = bytes;
            a.epoch      = 0;
            a.coop_total = 0;
        }
        *out   = a.ptr;
        *epoch = ++a.epoch;
        return cudaSuccess;
    }

    // Books `warps` more arrivals on the arena's "transposing warps finished" word for the launch that is about to be
    // enqueued on the stream, and returns the value the word will have when that launch's warps are all done.
    unsigned arena_coop_target(int device, cudaStream_t stream, unsigned warps)
    {
        std::lock_guard<std::mutex> lock(g_arena_mutex);
        Arena&                      a = g_arenas[std::make_pair(device, stream)];
        a.coop_total += warps;
        return a.coop_total;
    }

    // The arenas are released by b200_sgemm_shutdown(); at process exit they are left to the driver,
    // because CUDA calls from static destructors may run after the runtime has been torn down.

    inline size_t variant_smem(const KernelVariant& v)
    {
        const size_t tiles = size_t(v.stages) * size_t(v.block_m + v.block_n) * size_t(v.block_k) * sizeof(float);
        // the warp-specialised kernel keeps its mbarriers (stage full / empty, two staging slots full / empty) and an
        // abort flag behind the tiles
        return v.pipeline >= 1 ? tiles + size_t(2 * v.stages + 4) * 8 + 16 : tiles;
    }
    // the staging ring of K-contiguous operands: two slots of [rows][32 floats] per staged operand + alignment slack
    inline size_t staging_smem(const KernelVariant& v, bool stage_a, bool stage_b)
    {
        if(!stage_a && !stage_b)
            return 0;
        return 1024 + 2 * ((stage_a ? size_t(v.block_m) * 128 : 0) + (stage_b ? size_t(v.block_n) * 128 : 0));
    }
    constexpr size_t SMEM_PER_SM = 227 * 1024;

    // ---- per-device facts and the kernels' status word ---------------------------------------------
    struct DeviceInfo
    {
        int  sm_count = 0;
        int* status   = nullptr; // address of g_kernel_status on that device
    };
    std::mutex                g_dev_mutex;
    std::map<int, DeviceInfo> g_dev;

    // ---- TMA tensor maps (driver entry point fetched through the runtime: no link against libcuda) ---
    typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                      const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                      CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    EncodeTiledFn get_encode_fn()
    {
        static EncodeTiledFn fn = []() -> EncodeTiledFn {
            void*                           p = nullptr;
            cudaDriverEntryPointQueryResult q;
            if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess
               || q != cudaDriverEntryPointSuccess)
                return nullptr;
            return reinterpret_cast<EncodeTiledFn>(p);
        }();
        return fn;
    }

    // The encoder is a driver call and wants the device's context current in the calling thread.  A host thread that
    // has so far only made calls the runtime answers from its caches has none yet (its encodes fail): bind it once
    // per thread.
    void ensure_thread_context()
    {
        static thread_local bool bound = false;
        if(!bound)
        {
            int device = 0;
            if(cudaGetDevice(&device) == cudaSuccess)
                cudaSetDevice(device); // makes the device's primary context current in this thread
            bound = true;
        }
    }

    // Tensor map of one operand.  `inner` / `outer` are the extents along the contiguous and the pitched
    // dimension, the box is box_inner x box_outer elements; out-of-bounds elements read as zero.
    // A third dimension carries the matrices of a batch (extent `batch`, `batch_stride` elements apart, a multiple of
    // 4; extent 1 for a single or shared matrix).
    bool encode_map(CUtensorMap* map, const float* base, size_t inner, size_t outer, size_t ld, int box_inner,
                    int box_outer, bool swizzle128, size_t batch = 1, size_t batch_stride = 0)
    {
        EncodeTiledFn enc = get_encode_fn();
        if(!enc || box_inner > 256 || box_outer > 256)
            return false;
        ensure_thread_context();
        if(batch <= 1)
        {
            batch        = 1;
            batch_stride = ld * outer; // never stepped over; only has to be a legal stride
        }
        const cuuint64_t dims[3]    = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)batch};
        const cuuint64_t strides[2] = {(cuuint64_t)ld * sizeof(float), (cuuint64_t)batch_stride * sizeof(float)};
        const cuuint32_t box[3]     = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1};
        const cuuint32_t estr[3]    = {1, 1, 1};
        return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
               == CUDA_SUCCESS;
    }

    // Tensor map of a K-contiguous operand for the staging ring of the warp-specialised kernel: X rows (X % 4 == 0) of K
    // floats, pitch ld, seen as three dimensions (k, row / 4, row % 4) so that a box of 32 k x block_x rows lands in
    // shared memory with the rows ordered (row % 4, row / 4) - the order the transposing warps read without bank
    // conflicts.  128-byte swizzle; out-of-bounds k and row groups read as zero.
    bool encode_staged_map(CUtensorMap* map, const float* base, size_t X, size_t K, size_t ld, int block_x,
                           size_t batch = 1, size_t batch_stride = 0)
    {
        EncodeTiledFn enc = get_encode_fn();
        if(!enc || block_x > 1024 || X % 4 != 0)
            return false;
        ensure_thread_context();
        if(batch <= 1)
        {
            batch        = 1;
            batch_stride = ld * X;
        }
        const cuuint64_t dims[4]    = {(cuuint64_t)K, (cuuint64_t)(X / 4), 4, (cuuint64_t)batch};
        const cuuint64_t strides[3] = {(cuuint64_t)ld * 4 * sizeof(float), (cuuint64_t)ld * sizeof(float),
                                       (cuuint64_t)batch_stride * sizeof(float)};
        const cuuint32_t box[4]     = {32, (cuuint32_t)(block_x / 4), 4, 1};
        const cuuint32_t estr[4]    = {1, 1, 1, 1};
        return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<float*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
               == CUDA_SUCCESS;
    }

    // first use on a device: SM count and the device address of the status word (the symbol's name is a
    // host-side handle, not a device address)
    cudaError_t device_info(DeviceInfo* out)
    {
        int         device = 0;
        cudaError_t e      = cudaGetDevice(&device);
        if(e != cudaSuccess)
            return e;
        std::lock_guard<std::mutex> lock(g_dev_mutex);
        auto                        it = g_dev.find(device);
        if(it == g_dev.end())
        {
            DeviceInfo d;
            e = cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, device);
            if(e != cudaSuccess)
                return e;
            void* addr = nullptr;
            e          = cudaGetSymbolAddress(&addr, g_kernel_status);
            if(e != cudaSuccess)
                return e;
            d.status = static_cast<int*>(addr);
            it       = g_dev.emplace(device, d).first;
        }
        *out = it->second;
        return cudaSuccess;
    }

    void fill_params(const KernelVariant& v, int split_k, int pretranspose, b200_sgemm_params* out)
    {
        out->block_size        = v.block_size;
        out->block_m           = v.block_m;
        out->block_n           = v.block_n;
        out->block_k           = v.block_k;
        out->warp_tile_m_count = v.warp_tile_m_count;
        out->warp_tile_n_count = v.warp_tile_n_count;
        out->thread_tile_m     = v.thread_tile_m;
        out->thread_tile_n     = v.thread_tile_n;
        out->threads_n         = v.threads_n;
        out->stages            = v.stages;
        out->fma_mode          = v.fma_mode;
        out->raster            = v.raster;
        out->min_blocks        = v.min_blocks;
        out->pipeline          = v.pipeline;
        out->split_k           = split_k;
        out->pretranspose      = pretranspose;
    }

    bool bad_layout(int l)
    {
        return l != 0 && l != 1;
    }

    // table lookup (variant < 0), or the forced variant unsplit; a forced split (> 0, or -1 = equal K ranges per CTA
    // with in-kernel ordered reduction, which a table entry asks for with split_k 0) overrides either.
    // *split_k: >= 1 slices, 0 = equal ranges.
    void choose(int la, int lb, int lc, size_t M, size_t N, size_t K, int forced_variant, int forced_split,
                int* variant, int* split_k, int* pretranspose = nullptr)
    {
        int v = forced_variant, s = 1, pre = 0;
        if(v < 0)
        {
            const ConfigKey key{M, N, K, la, lb, lc};
            const int       e = find_best_config(sorted_config_map, CONFIG_ENTRIES, key);
            if(e >= 0)
            {
                v = sorted_config_map[e].variant;
                s = sorted_config_map[e].split_k;
                pre = sorted_config_map[e].pretranspose;
                // an entry reached through the any-layout fallback may name a variant that was never
                // built for this layout (the reference throws there): use the default variant instead
                if(lookup_kernel(v, layout_index(la, lb, lc), 0) == nullptr)
                {
                    v = DEFAULT_VARIANT_IDX;
                    s = 1;
                    pre = 0;
                }
            }
            else
            {
                v = DEFAULT_VARIANT_IDX;
            }
        }
        if(forced_split > 0)
            s = forced_split;
        else if(forced_split < 0)
            s = 0;
        *variant = v;
        *split_k = s < 0 ? 1 : s;
        if(pretranspose)
        {
            // only K-contiguous operands can be pre-transposed, only for the warp-specialised kernel (whose
            // TMA path it feeds), and only when the other dimension re-uses the operand often enough to pay
            // for one extra pass over it (8 bytes per element against 2 x dimension flops)
            int mask = kernel_variants[v].pipeline >= 1 ? pre : 0;
            if(la != LAYOUT_ROW || N < 1024) mask &= ~1;
            if(lb != LAYOUT_COL || M < 1024) mask &= ~2;
            *pretranspose = mask;
        }
    }

    // a warp-specialised variant that is built for this layout (the smallest tile first), or -1
    int fallback_ws_variant(int la, int lb, int lc)
    {
        for(int v = 0; v < KERNEL_VARIANTS; ++v)
            if(kernel_variants[v].pipeline >= 1 && lookup_kernel(v, layout_index(la, lb, lc), 0)
               && lookup_kernel(v, layout_index(la, lb, lc), 1))
                return v;
        return -1;
    }

    bool v_pipeline_ok(int variant)
    {
        return variant >= 0 && variant < KERNEL_VARIANTS && kernel_variants[variant].pipeline >= 1;
    }

    // K slicing: whole block_k tiles per slice, empty slices dropped
    void slice_k(size_t K, int block_k, int want, int* splits, int* k_per_split)
    {
        const long long ktiles = (long long)((K + block_k - 1) / block_k);
        long long       s      = want < 1 ? 1 : want;
        if(s > ktiles)
            s = ktiles;
        const long long per = (ktiles + s - 1) / s;
        *k_per_split        = (int)(per * block_k);
        *splits             = (int)((ktiles + per - 1) / per);
    }

    bool aligned16(const void* p)
    {
        return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
    }

    // Schedule 1 of the warp-specialised kernel (equal contiguous ranges of K tiles per CTA, accumulators handed
    // over once per CTA): used when there is no split-K, at least as many tiles as CTAs, and a last wave that the
    // round-robin schedule would leave partly empty.  Needs `slots` parking slots of one tile each plus flags.
    // Schedule 2 (`stream`): the same ranges when the tiles are fewer than the CTAs; the pieces of a tile are chains
    // of their own; the CTA that owns the tile's last piece adds the others to its chain in ascending K order.
    struct HandoverPlan
    {
        int    sched      = 0; // 0: neither
        int    ctas       = 0; // grid of schedule 2
        size_t slot_bytes = 0; // all parking slots
        size_t flag_bytes = 0;
        bool   use() const { return sched != 0; }
    };
    // A CTA's range in schedule 2 is at least this many K tiles (measured on 256^3 .. 768^3 with 1, 2, 3 and 4: 2 is
    // where the shorter chains stop paying for the longer ordered sum; 256^3 25 -> 20 us, 512^3 25.5 -> 23.4 us)
    constexpr int STREAM_MIN_KTILES = 2;
    HandoverPlan plan_handover(const KernelVariant& v, size_t M, size_t N, size_t K, int splits, bool stream, int sm_count,
                               size_t batch = 1)
    {
        HandoverPlan h;
        if(v.pipeline < 1 || splits != 1 || sm_count <= 0)
            return h;
        const long long tiles = (long long)((M + v.block_m - 1) / v.block_m) * (long long)((N + v.block_n - 1) / v.block_n)
                                * (long long)batch;
        const long long slots = (long long)sm_count * (v.min_blocks > 0 ? v.min_blocks : 1);
        long long       ctas  = slots;
        if(tiles > slots)
        {
            if(tiles % slots == 0)
                return h;
            h.sched = 1;
        }
        else
        {
            const long long kts = (long long)((K + v.block_k - 1) / v.block_k);
            ctas = tiles * kts / STREAM_MIN_KTILES;
            if(ctas > slots)
                ctas = slots;
            if(!stream || ctas <= tiles || tiles * kts > INT_MAX)
                return h;
            h.sched = 2;
        }
        h.ctas       = (int)ctas;
        h.flag_bytes = size_t(ctas) * size_t(v.block_size / 32) * sizeof(unsigned);
        h.slot_bytes = size_t(ctas) * size_t(v.block_m) * size_t(v.block_n) * sizeof(float);
        if(h.flag_bytes > ARENA_HANDOVER_FLAG_BYTES - 256) // (the last words of that part belong to the transposition)
            h.sched = 0;
        return h;
    }
    int current_sm_count()
    {
        DeviceInfo info;
        return device_info(&info) == cudaSuccess ? info.sm_count : 0;
    }

    int run(int lc, int la, int lb, float* C, const float* A, const float* B, size_t M, size_t N, size_t K,
            size_t lda, size_t ldb, size_t ldc, int forced_variant, int forced_split, void* workspace,
            size_t workspace_bytes, bool use_arena, cudaStream_t stream, float* const* extra_c = nullptr, int n_extra = 0,
            int forced_pre = -1, size_t batch = 1, size_t stride_a = 0, size_t stride_b = 0, size_t stride_c = 0,
            const float* alpha_beta = nullptr)
    {
        // alpha_beta != nullptr: C = alpha * (A B) + beta * C in the kernel's epilogue (warp-specialised kernels without
        // K slices only: B200_SGEMM_NO_KERNEL otherwise, before anything is launched, and the caller makes a second pass)
        // batch > 1: `batch` problems of the same shape at fixed strides in ONE launch (warp-specialised kernels without
        // K slices only: B200_SGEMM_NO_KERNEL otherwise, and the caller falls back to one launch per matrix)
        if(batch == 0)
            return B200_SGEMM_INVALID_ARGUMENT;
        if(n_extra < 0 || n_extra > WS_MAX_EXTRA || (n_extra > 0 && !extra_c))
            return B200_SGEMM_INVALID_ARGUMENT;
        for(int d = 0; d < n_extra; ++d)
            if(!extra_c[d])
                return B200_SGEMM_INVALID_ARGUMENT;
        if(!C || !A || !B || M == 0 || N == 0 || K == 0 || bad_layout(la) || bad_layout(lb) || bad_layout(lc))
            return B200_SGEMM_INVALID_ARGUMENT;
        if(M > INT_MAX || N > INT_MAX || K > INT_MAX)
            return B200_SGEMM_UNSUPPORTED_SIZE;
        if(forced_variant >= KERNEL_VARIANTS)
            return B200_SGEMM_INVALID_ARGUMENT;
        const size_t min_lda = la == LAYOUT_ROW ? K : M, min_ldb = lb == LAYOUT_ROW ? N : K,
                     min_ldc = lc == LAYOUT_ROW ? N : M;
        if(lda == 0) lda = min_lda;
        if(ldb == 0) ldb = min_ldb;
        if(ldc == 0) ldc = min_ldc;
        if(lda < min_lda || ldb < min_ldb || ldc < min_ldc)
            return B200_SGEMM_INVALID_ARGUMENT;

        int variant, want_split, pre = 0;
        choose(la, lb, lc, M, N, K, forced_variant, forced_split, &variant, &want_split, use_arena ? &pre : nullptr);
        if(forced_pre >= 0 && use_arena)
        {
            // a tuning trial states the entry's pre-transposition bits itself (same eligibility rules as a table entry)
            pre = v_pipeline_ok(variant) ? forced_pre & 3 : 0;
            if(la != LAYOUT_ROW || N < 1024) pre &= ~1;
            if(lb != LAYOUT_COL || M < 1024) pre &= ~2;
        }
        if((batch > 1 || n_extra > 0) && forced_variant < 0)
        {
            // A batch brings its own parallelism and the multi-destination epilogue writes whole tiles: both take a
            // warp-specialised kernel without K slices, whatever the table entry of the single problem says.
            if(kernel_variants[variant].pipeline < 1)
                variant = fallback_ws_variant(la, lb, lc);
            if(variant < 0)
                return B200_SGEMM_NO_KERNEL;
            if(want_split > 1 || batch > 1)
                want_split = batch > 1 ? 1 : 0;
        }
        if(batch > 1)
        {
            pre = 0; // the transposed copies are per matrix: a batch goes through the kernel's own staging ring
            if(kernel_variants[variant].pipeline < 1 || want_split > 1 || n_extra > 0)
                return B200_SGEMM_NO_KERNEL;
        }
        // (a batch never takes the schedule with ordered in-kernel reduction: its cut points would depend on the batch)
        const bool equal_ranges = want_split == 0 && batch == 1; // equal K ranges per CTA instead of slices (falls back to no split)
        if(equal_ranges)
            want_split = 1;
        const KernelVariant& v = kernel_variants[variant];
        int                  splits, k_per_split;
        slice_k(K, v.block_k, want_split, &splits, &k_per_split);

        if(alpha_beta && (v.pipeline < 1 || splits > 1 || n_extra > 0 || batch > 1))
            return B200_SGEMM_NO_KERNEL;

        // ---- scratch plan of the drop-in entry: [A transposed][B transposed][split-K partials | parking slots] --------
        auto         round256 = [](size_t b) { return (b + 255) / 256 * 256; };
        const size_t ldat = (M + 3) / 4 * 4, ldbt = (N + 3) / 4 * 4; // pitches of the transposed copies
        // the kernel for the transposed layouts must exist, else the operand stays as it is
        if((pre & 1) && !lookup_kernel(variant, layout_index(LAYOUT_COL, lb, lc), 0)) pre &= ~1;
        if((pre & 2) && !lookup_kernel(variant, layout_index((pre & 1) ? LAYOUT_COL : la, LAYOUT_ROW, lc), 0)) pre &= ~2;
        const size_t bytes_at = (pre & 1) ? round256(K * ldat * sizeof(float)) : 0;
        const size_t bytes_bt = (pre & 2) ? round256(K * ldbt * sizeof(float)) : 0;
        const size_t bytes_pk = splits > 1 ? size_t(splits) * M * N * sizeof(float) : 0;
        // schedule 1 (no partly filled last wave): the drop-in entry takes the parking slots from its arena, the
        // explicit entry from the caller's workspace when that is large enough, and else keeps schedule 0
        if(batch > 1 && splits > 1)
            return B200_SGEMM_NO_KERNEL;
        HandoverPlan hand = plan_handover(v, M, N, K, splits, equal_ranges, v.pipeline >= 1 && splits == 1 ? current_sm_count() : 0,
                                          batch);
        if(hand.use() && !use_arena && (!workspace || workspace_bytes < round256(hand.slot_bytes) + hand.flag_bytes))
            hand.sched = 0;
        if(hand.sched == 2 && n_extra > 0)
            hand.sched = 0; // further destinations are written by whole-tile epilogues only
        const size_t bytes_ho = hand.use() ? round256(hand.slot_bytes) : 0;
        char*        arena    = nullptr;
        unsigned     epoch    = 1;
        unsigned*    flags    = nullptr;
        if(use_arena && bytes_at + bytes_bt + bytes_pk + bytes_ho > 0)
        {
            int         device = 0;
            cudaError_t e      = cudaGetDevice(&device);
            if(e != cudaSuccess)
                return (int)e;
            void* p = nullptr;
            e       = arena_get(device, stream, bytes_at + bytes_bt + bytes_pk + bytes_ho, &p, &epoch);
            if(e != cudaSuccess)
                return (int)e;
            flags = static_cast<unsigned*>(p);
            arena = static_cast<char*>(p) + ARENA_FLAG_BYTES;
        }
        float* handover = nullptr;
        if(hand.use())
        {
            if(use_arena)
                handover = reinterpret_cast<float*>(arena + bytes_at + bytes_bt);
            else
            {
                // caller's workspace: [parking slots][flags]; its contents are unknown, so the flags are cleared
                handover = static_cast<float*>(workspace);
                flags    = reinterpret_cast<unsigned*>(static_cast<char*>(workspace) + bytes_ho);
                const cudaError_t e = cudaMemsetAsync(flags, 0, hand.flag_bytes, stream);
                if(e != cudaSuccess)
                    return (int)e;
            }
        }
        // The transposed copies are made either by the warp-specialised kernel itself (block by block, by the producer
        // warps its TMA route leaves idle: no second pass over HBM before the product starts) or, where that does not
        // apply, by a transposition kernel launched in front of the product.  Which, is decided once the tensor maps
        // are known; until then only the operands are rebound to the copies.
        const float* src_a = nullptr;
        const float* src_b = nullptr;
        const size_t src_lda = lda, src_ldb = ldb;
        if(pre & 1)
        {
            src_a = A;
            A     = reinterpret_cast<float*>(arena);
            la    = LAYOUT_COL;
            lda   = ldat;
        }
        if(pre & 2)
        {
            src_b = B;
            B     = reinterpret_cast<float*>(arena + bytes_at);
            lb    = LAYOUT_ROW;
            ldb   = ldbt;
        }
        auto transpose_in_front = [&]() -> cudaError_t {
            cudaError_t te = cudaSuccess;
            if(src_a)
                te = launch_transpose(src_a, const_cast<float*>(A), M, K, src_lda, ldat, stream);
            if(te == cudaSuccess && src_b)
                te = launch_transpose(src_b, const_cast<float*>(B), N, K, src_ldb, ldbt, stream);
            return te;
        };

        GemmArgs args;
        args.A = A;
        args.B = B;
        args.M = (int)M;
        args.N = (int)N;
        args.K = (int)K;
        args.lda = (long long)lda;
        args.ldb = (long long)ldb;
        args.grid_m      = (int)((M + v.block_m - 1) / v.block_m);
        args.grid_n      = (int)((N + v.block_n - 1) / v.block_n);
        args.splits      = splits;
        args.k_per_split = k_per_split;
        // (a batch steps its operands by the strides: they take part in the 16-byte rule)
        args.vec_a       = aligned16(A) && lda % 4 == 0 && (batch == 1 || stride_a % 4 == 0);
        args.vec_b       = aligned16(B) && ldb % 4 == 0 && (batch == 1 || stride_b % 4 == 0);

        const long long total_ctas = (long long)args.grid_m * args.grid_n * splits * (long long)batch;
        if(total_ctas > INT_MAX)
            return B200_SGEMM_UNSUPPORTED_SIZE;

        float* partial = nullptr;
        if(splits > 1)
        {
            const size_t need = bytes_pk;
            if(use_arena)
            {
                partial = reinterpret_cast<float*>(arena + bytes_at + bytes_bt);
            }
            else
            {
                if(!workspace || workspace_bytes < need)
                    return B200_SGEMM_WORKSPACE_TOO_SMALL;
                partial = static_cast<float*>(workspace);
            }
            // partial results are packed MxN in C's layout
            args.C            = partial;
            args.ldc          = (long long)min_ldc;
            args.split_stride = (long long)(M * N);
            args.vec_c        = aligned16(partial) && min_ldc % 4 == 0 && (M * N) % 4 == 0;
        }
        else
        {
            args.C            = C;
            args.ldc          = (long long)ldc;
            args.split_stride = 0;
            args.vec_c        = aligned16(C) && ldc % 4 == 0 && (batch == 1 || stride_c % 4 == 0);
            for(int d = 0; d < n_extra; ++d)
                args.vec_c = args.vec_c && aligned16(extra_c[d]);
        }
        // further destinations are written by the warp-specialised kernels' epilogue only, and only without split-K
        if(n_extra > 0 && (splits > 1 || v.pipeline < 1))
            return B200_SGEMM_NO_KERNEL;

        const bool aligned = (M % v.block_m == 0) && (N % v.block_n == 0) && (K % v.block_k == 0) && args.vec_a
                             && args.vec_b && args.vec_c;
        const void* fn = lookup_kernel(variant, layout_index(la, lb, lc), aligned ? 1 : 0);
        if(!fn)
            return B200_SGEMM_NO_KERNEL;

        // K-contiguous operands of the warp-specialised kernel come through its TMA staging ring when they meet TMA's
        // alignment rules, the K tile is 32 floats (one 128-byte swizzle row) and the ring fits beside the stages
        // (and M / N is a multiple of 4: the tensor map groups the rows by four)
        bool stage_a = v.pipeline >= 1 && v.block_k == 32 && la == LAYOUT_ROW && args.vec_a && M % 4 == 0;
        bool stage_b = v.pipeline >= 1 && v.block_k == 32 && lb == LAYOUT_COL && args.vec_b && N % 4 == 0;
        if((stage_a || stage_b)
           && ((la == LAYOUT_ROW && !stage_a) || (lb == LAYOUT_COL && !stage_b) || (la == LAYOUT_COL && !args.vec_a)
               || (lb == LAYOUT_ROW && !args.vec_b)
               || (variant_smem(v) + staging_smem(v, stage_a, stage_b)) * (v.min_blocks > 0 ? v.min_blocks : 1) > SMEM_PER_SM))
            stage_a = stage_b = false; // every operand must come by TMA on that route
        const size_t smem = variant_smem(v) + staging_smem(v, stage_a, stage_b);
        if(smem > 48 * 1024)
        {
            int         device = 0;
            cudaError_t e      = cudaGetDevice(&device);
            if(e != cudaSuccess)
                return (int)e;
            // opt the kernel in for the most it can ever ask for (the staging ring depends on the operands' alignment,
            // the kernel function does not), so that concurrent callers never lower each other's limit
            const bool   ka = v.pipeline >= 1 && v.block_k == 32 && la == LAYOUT_ROW, kb = v.pipeline >= 1 && v.block_k == 32 && lb == LAYOUT_COL;
            const size_t most = (variant_smem(v) + staging_smem(v, ka, kb)) * (v.min_blocks > 0 ? v.min_blocks : 1) <= SMEM_PER_SM
                                    ? variant_smem(v) + staging_smem(v, ka, kb)
                                    : variant_smem(v);
            e = ensure_smem_attr(fn, device, most > smem ? most : smem);
            if(e != cudaSuccess)
                return (int)e;
        }

        cudaError_t e;
        if(v.pipeline >= 1)
        {
            DeviceInfo info;
            e = device_info(&info);
            if(e != cudaSuccess)
                return (int)e;
            WsArgs w;
            w.g           = args;
            w.total_units = (int)total_ctas;
            w.status      = info.status;
            w.sched       = hand.sched;
            w.k_tiles     = (int)((K + v.block_k - 1) / v.block_k);
            w.rr_tiles    = 0;
            w.test_omit_last_fill = 0;
            w.batch    = (int)batch;
            w.bstep_a  = batch > 1 && stride_a != 0 ? 1 : 0;
            w.bstep_b  = batch > 1 && stride_b != 0 ? 1 : 0;
            w.stride_a = batch > 1 ? (long long)stride_a : 0;
            w.stride_b = batch > 1 ? (long long)stride_b : 0;
            w.stride_c = batch > 1 ? (long long)stride_c : 0;
            const size_t nb_a = w.bstep_a ? batch : 1, nb_b = w.bstep_b ? batch : 1;
            if(hand.sched == 1)
            {
                // all but the last one to two waves' worth of tiles keep the round-robin order
                const long long slots_ = (long long)info.sm_count * (v.min_blocks > 0 ? v.min_blocks : 1);
                const long long waves  = ((long long)args.grid_m * args.grid_n * (long long)batch) / slots_;
                w.rr_tiles             = waves >= 2 ? (int)((waves - 1) * slots_) : 0;
            }
            w.handover    = handover;
            w.flags       = flags;
            w.epoch       = epoch;
            w.n_extra     = n_extra;
            for(int d = 0; d < WS_MAX_EXTRA; ++d)
                w.extra_c[d] = d < n_extra ? extra_c[d] : nullptr;
            CUtensorMap map_a, map_b;
            memset(&map_a, 0, sizeof(map_a));
            memset(&map_b, 0, sizeof(map_b));
            // TMA serves the operands whose M / N extent is contiguous ([K][X] in memory: box block_x wide,
            // block_k tall); base and pitch must be 16-byte aligned (vec_a / vec_b).  K-contiguous operands
            // are transposed by the producer warps, anything unaligned is copied by them with guards.
            w.tma_a = (la == LAYOUT_COL) && args.vec_a && encode_map(&map_a, A, M, K, lda, v.block_m, v.block_k, false, nb_a, stride_a);
            w.tma_b = (lb == LAYOUT_ROW) && args.vec_b && encode_map(&map_b, B, N, K, ldb, v.block_n, v.block_k, false, nb_b, stride_b);
            // staged operands: [X rows][K] in memory, box 32 k x block_x rows, 128-byte swizzle
            w.stg_a = stage_a && encode_staged_map(&map_a, A, M, K, lda, v.block_m, nb_a, stride_a);
            w.stg_b = stage_b && encode_staged_map(&map_b, B, N, K, ldb, v.block_n, nb_b, stride_b);
            if((stage_a || stage_b) && !((w.stg_a || w.tma_a) && (w.stg_b || w.tma_b)))
            {
                return B200_SGEMM_NO_KERNEL; // tensor-map encoding failed for an operand that met every rule
            }
            w.alpha = alpha_beta ? alpha_beta[0] : 1.f;
            w.beta  = alpha_beta ? alpha_beta[1] : 0.f;
            w.coop_src_a = w.coop_src_b = nullptr;
            w.coop_ld_a = w.coop_ld_b = 0;
            w.coop_flags              = nullptr;
            w.coop_done               = nullptr;
            if(src_a || src_b)
            {
                // in-kernel transposition: both operands of the kernel come by TMA (so that producer warps are idle),
                // every 4 x 4 piece is whole and 16-byte aligned, and the blocks have a flag word each
                const int  qk       = v.block_k / 4;
                // (K tile of 32 only: with 64 the kernel in front measured 0.2 % faster, 6144x2048x8192 and 2048x6144x2048)
                const bool shape_ok = v.block_k == 32 && qk >= 1 && qk <= 32 && 32 % qk == 0
                                      && (v.block_m / 4) % (32 / qk) == 0 && (v.block_n / 4) % (32 / qk) == 0
                                      && v.block_m % 4 == 0 && v.block_n % 4 == 0;
                const bool a_ok = !src_a || (M % 4 == 0 && aligned16(src_a) && src_lda % 4 == 0);
                const bool b_ok = !src_b || (N % 4 == 0 && aligned16(src_b) && src_ldb % 4 == 0);
                const unsigned long long units = (unsigned long long)w.k_tiles
                                                 * ((src_a ? args.grid_m : 0) + (src_b ? args.grid_n : 0));
                const int  idle_warps = ws_producer_threads(v.block_size, v.warp_tile_m_count * v.thread_tile_m * v.warp_tile_n_count * v.thread_tile_n) / 32 - 1;
                // (a tuning trial may ask for the kernel in front with bit 2 of its pre-transposition argument)
                const bool in_front = forced_pre >= 0 && (forced_pre & 4);
                if(!in_front && shape_ok && a_ok && b_ok && K % 4 == 0 && batch == 1 && w.tma_a && w.tma_b && idle_warps > 0
                   && flags && units <= ARENA_COOP_FLAG_WORDS)
                {
                    w.coop_src_a = src_a;
                    w.coop_src_b = src_b;
                    w.coop_ld_a  = (long long)src_lda;
                    w.coop_ld_b  = (long long)src_ldb;
                    w.coop_flags = flags + ARENA_HANDOVER_FLAG_BYTES / sizeof(unsigned);
                    w.coop_done  = w.coop_flags - 1; // counts the warps that have finished, over all launches
                }
                else
                {
                    e = transpose_in_front();
                    if(e != cudaSuccess)
                        return (int)e;
                }
            }
            const long long slots = (long long)info.sm_count * (v.min_blocks > 0 ? v.min_blocks : 1);
            const long long grid  = hand.sched == 2 ? hand.ctas : total_ctas < slots ? total_ctas : slots;
            w.coop_done_target = 0;
            if(w.coop_flags)
            {
                int device = 0;
                e          = cudaGetDevice(&device);
                if(e != cudaSuccess)
                    return (int)e;
                const unsigned per_cta = (unsigned)(ws_producer_threads(v.block_size, v.warp_tile_m_count * v.thread_tile_m * v.warp_tile_n_count * v.thread_tile_n) / 32 - 1);
                w.coop_done_target     = arena_coop_target(device, stream, (unsigned)grid * per_cta);
            }
            w.range_q = 0;
            w.range_r = 0;
            if(hand.sched != 0)
            {
                const long long units = (total_ctas - w.rr_tiles) * (long long)w.k_tiles; // splits == 1 here
                w.range_q             = units / grid;
                w.range_r             = (unsigned)(units % grid);
            }
            void*           kargs[] = {&w, &map_a, &map_b};
            e = cudaLaunchKernel(fn, dim3((unsigned)grid), dim3((unsigned)(v.block_size + ws_producer_threads(v.block_size, v.warp_tile_m_count * v.thread_tile_m * v.warp_tile_n_count * v.thread_tile_n))), kargs,
                                 smem, stream);
        }
        else
        {
            e = transpose_in_front();
            if(e != cudaSuccess)
                return (int)e;
            void* kargs[] = {&args};
            e = cudaLaunchKernel(fn, dim3((unsigned)total_ctas), dim3((unsigned)v.block_size), kargs, smem, stream);
        }
        if(e != cudaSuccess)
            return (int)e;

        if(splits > 1)
        {
            const long long inner = (long long)min_ldc, outer = (long long)(lc == LAYOUT_ROW ? M : N);
            const int       vec   = inner % 4 == 0 && ldc % 4 == 0 && aligned16(C) && aligned16(partial);
            const long long work  = vec ? inner * outer / 4 : inner * outer;
            long long       blocks = (work + 255) / 256;
            if(blocks > 148 * 16)
                blocks = 148 * 16;
            splitk_reduce_kernel<<<(unsigned)blocks, 256, 0, stream>>>(C, partial, inner, outer, (long long)ldc,
                                                                       (long long)(M * N), splits, vec);
            e = cudaPeekAtLastError();
            if(e != cudaSuccess)
                return (int)e;
        }
        return B200_SGEMM_OK;
    }
} // namespace

int* status_word_address()
{
    DeviceInfo info;
    return device_info(&info) == cudaSuccess ? info.status : nullptr;
}

// ---- register-only FMA throughput probe ---------------------------------------------------------
// The register-tile update of the GEMM kernels with the fragments held in registers: 8 x 8 accumulators per thread,
// mode 0 as 64 scalar FMAs per step, mode 1 as 32 packed FMAs in the kernels' order (the natural pair b fixed, the
// duplicated a cycling).  Nothing but FMAs in the loop, so the rate is what the FMA pipe itself delivers.
template<int MODE>
__global__ void __launch_bounds__(256) fma_peak_kernel(float* out, int iterations, float seed)
{
    float a[8], b[8];
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        a[i] = seed * (float)(i + 1 + (threadIdx.x & 3));
        b[i] = 1.0f + seed * (float)(i + 1);
    }
    if constexpr(MODE == 0)
    {
        float acc[8][8];
#pragma unroll
        for(int i = 0; i < 8; ++i)
#pragma unroll
            for(int j = 0; j < 8; ++j)
                acc[i][j] = 0.f;
        for(int it = 0; it < iterations; ++it)
        {
#pragma unroll
            for(int r = 0; r < 4; ++r)
#pragma unroll
                for(int i = 0; i < 8; ++i)
#pragma unroll
                    for(int j = 0; j < 8; ++j)
                        acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        float s = 0.f;
#pragma unroll
        for(int i = 0; i < 8; ++i)
#pragma unroll
            for(int j = 0; j < 8; ++j)
                s += acc[i][j];
        if(s == 123.456f)
            out[0] = s;
    }
    else
    {
        uint64_t acc[8][4], a2[8], b2[4];
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            a2[i] = pack2(a[i], a[i]);
#pragma unroll
            for(int j = 0; j < 4; ++j)
                acc[i][j] = 0ull;
        }
#pragma unroll
        for(int j = 0; j < 4; ++j)
            b2[j] = pack2(b[2 * j], b[2 * j + 1]);
        for(int it = 0; it < iterations; ++it)
        {
#pragma unroll
            for(int r = 0; r < 4; ++r)
#pragma unroll
                for(int j = 0; j < 4; ++j)
#pragma unroll
                    for(int i = 0; i < 8; ++i)
                        asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i][j]) : "l"(a2[i]), "l"(b2[j]));
        }
        float s = 0.f;
#pragma unroll
        for(int i = 0; i < 8; ++i)
#pragma unroll
            for(int j = 0; j < 4; ++j)
            {
                float lo, hi;
                unpack2(acc[i][j], lo, hi);
                s += lo + hi;
            }
        if(s == 123.456f)
            out[0] = s;
    }
}

} // namespace sgemm_b200

using namespace sgemm_b200;

extern "C" {

int b200_sgemm(int layout_c, int layout_a, int layout_b, float* C, const float* A, const float* B, size_t M, size_t N,
               size_t K, void* cuda_stream)
{
    return run(layout_c, layout_a, layout_b, C, A, B, M, N, K, 0, 0, 0, -1, 0, nullptr, 0, true,
               static_cast<cudaStream_t>(cuda_stream));
}

int b200_sgemm_ex(int layout_c, int layout_a, int layout_b, float* C, const float* A, const float* B, size_t M,
                  size_t N, size_t K, size_t lda, size_t ldb, size_t ldc, int variant, int split_k, void* workspace,
                  size_t workspace_bytes, void* cuda_stream)
{
    return run(layout_c, layout_a, layout_b, C, A, B, M, N, K, lda, ldb, ldc, variant, split_k, workspace,
               workspace_bytes, false, static_cast<cudaStream_t>(cuda_stream));
}

int b200_sgemm_trial(int layout_c, int layout_a, int layout_b, float* C, const float* A, const float* B, size_t M,
                     size_t N, size_t K, int variant, int split_k, int pretranspose, void* cuda_stream)
{
    if(variant < 0 || pretranspose < 0 || pretranspose > 7)
        return B200_SGEMM_INVALID_ARGUMENT;
    return run(layout_c, layout_a, layout_b, C, A, B, M, N, K, 0, 0, 0, variant, split_k == 0 ? -1 : split_k, nullptr, 0,
               true, static_cast<cudaStream_t>(cuda_stream), nullptr, 0, pretranspose);
}

// The drop-in entry's path (table lookup, arena scratch, transposed copies, balanced schedules) with leading dimensions
// and, when alpha_beta is given, C = alpha * (A B) + beta * C formed in the kernel's epilogue (internal: b200_sgemm_blas
// in sgemm_blas.cu.  With alpha_beta it returns B200_SGEMM_NO_KERNEL before launching anything when the table's kernel
// cannot scale in its epilogue, and the caller makes a second pass over C.)
int b200_sgemm_arena_ld(int layout_c, int layout_a, int layout_b, float* C, const float* A, const float* B, size_t M,
                        size_t N, size_t K, size_t lda, size_t ldb, size_t ldc, const float* alpha_beta, void* cuda_stream)
{
    return run(layout_c, layout_a, layout_b, C, A, B, M, N, K, lda, ldb, ldc, -1, 0, nullptr, 0, true,
               static_cast<cudaStream_t>(cuda_stream), nullptr, 0, -1, 1, 0, 0, 0, alpha_beta);
}

// One launch for a whole batch (internal: b200_sgemm_strided_batched in sgemm_blas.cu falls back to a launch per
// matrix when this returns B200_SGEMM_NO_KERNEL).
int b200_sgemm_batched_launch(int layout_c, int layout_a, int layout_b, float* C, const float* A, const float* B, size_t M,
                              size_t N, size_t K, size_t stride_c, size_t stride_a, size_t stride_b, size_t batch,
                              void* cuda_stream)
{
    if(M > INT_MAX || N > INT_MAX
       || ((M + 31) / 32) * ((N + 31) / 32) * batch > (size_t)INT_MAX / 64) // the tile sequence is indexed with int
        return B200_SGEMM_NO_KERNEL;
    return run(layout_c, layout_a, layout_b, C, A, B, M, N, K, 0, 0, 0, -1, 0, nullptr, 0, true,
               static_cast<cudaStream_t>(cuda_stream), nullptr, 0, -1, batch, stride_a, stride_b, stride_c);
}

int b200_sgemm_multi(int layout_c, int layout_a, int layout_b, float* const* C_list, int n_dst, const float* A,
                     const float* B, size_t M, size_t N, size_t K, size_t lda, size_t ldb, size_t ldc, int variant,
                     void* cuda_stream)
{
    if(!C_list || n_dst < 1 || n_dst > 1 + WS_MAX_EXTRA)
        return B200_SGEMM_INVALID_ARGUMENT;
    // like the drop-in entry, a table lookup (variant -1) may pre-transpose K-contiguous operands into the arena
    return run(layout_c, layout_a, layout_b, C_list[0], A, B, M, N, K, lda, ldb, ldc, variant, 1, nullptr, 0, variant < 0,
               static_cast<cudaStream_t>(cuda_stream), C_list + 1, n_dst - 1);
}

size_t b200_sgemm_workspace_bytes(int layout_c, int layout_a, int layout_b, size_t M, size_t N, size_t K, int variant,
                                  int split_k)
{
    if(M == 0 || N == 0 || K == 0 || bad_layout(layout_a) || bad_layout(layout_b) || bad_layout(layout_c)
       || variant >= KERNEL_VARIANTS)
        return 0;
    int v, want;
    choose(layout_a, layout_b, layout_c, M, N, K, variant, split_k, &v, &want);
    const bool stream = want == 0;
    int        splits, k_per;
    slice_k(K, kernel_variants[v].block_k, stream ? 1 : want, &splits, &k_per);
    if(splits > 1)
        return size_t(splits) * M * N * sizeof(float);
    // no split-K: the parking slots of schedule 1, when it applies on the current device (optional: with a smaller
    // or no workspace b200_sgemm_ex runs the round-robin schedule and computes the same bits)
    const HandoverPlan hand = plan_handover(kernel_variants[v], M, N, K, splits, stream,
                                            kernel_variants[v].pipeline >= 1 ? current_sm_count() : 0);
    return hand.use() ? (hand.slot_bytes + 255) / 256 * 256 + hand.flag_bytes : 0;
}

int b200_sgemm_stream_plan(int layout_c, int layout_a, int layout_b, size_t M, size_t N, size_t K, int variant,
                           int split_k, int sm_count, int* block_mnk, int* offsets, int* bounds, int capacity)
{
    if(M == 0 || N == 0 || K == 0 || bad_layout(layout_a) || bad_layout(layout_b) || bad_layout(layout_c)
       || variant >= KERNEL_VARIANTS || M > INT_MAX || N > INT_MAX || K > INT_MAX)
        return B200_SGEMM_INVALID_ARGUMENT;
    int v, want;
    choose(layout_a, layout_b, layout_c, M, N, K, variant, split_k, &v, &want);
    const KernelVariant& kv = kernel_variants[v];
    if(block_mnk)
    {
        block_mnk[0] = kv.block_m;
        block_mnk[1] = kv.block_n;
        block_mnk[2] = kv.block_k;
    }
    if(want != 0)
        return 0; // slices (or no split): the K cut points are the same for every tile
    const HandoverPlan hand = plan_handover(kv, M, N, K, 1, true, sm_count);
    if(hand.sched != 2)
        return 0;
    const int       grid_m = (int)((M + kv.block_m - 1) / kv.block_m), grid_n = (int)((N + kv.block_n - 1) / kv.block_n);
    const long long tiles  = (long long)grid_m * grid_n;
    const int       kts    = (int)((K + kv.block_k - 1) / kv.block_k);
    // pieces per tile, gathered by position in the kernel's tile order and written out by tile coordinates
    std::vector<std::vector<int>> cuts((size_t)tiles);
    for(long long pos = 0; pos < tiles; ++pos)
    {
        int tm = 0, tn = 0;
        switch(kv.raster)
        {
        case RASTER_GROUPED: map_tile<RASTER_GROUPED>((int)pos, grid_m, grid_n, tm, tn); break;
        case RASTER_HILBERT: map_tile<RASTER_HILBERT>((int)pos, grid_m, grid_n, tm, tn); break;
        default: map_tile<RASTER_ROW>((int)pos, grid_m, grid_n, tm, tn); break;
        }
        int       buf[64];
        const int n = ws_stream_cuts(tiles, kts, hand.ctas, pos, buf, 64);
        if(n > 64)
            return B200_SGEMM_UNSUPPORTED_SIZE;
        cuts[(size_t)tm * grid_n + tn].assign(buf, buf + n);
    }
    int total = 0;
    for(long long t = 0; t < tiles; ++t)
    {
        if(offsets && t < capacity)
            offsets[t] = total;
        for(int cut : cuts[(size_t)t])
        {
            if(bounds && total < capacity)
                bounds[total] = cut * kv.block_k;
            ++total;
        }
    }
    if(offsets && tiles < capacity)
        offsets[tiles] = total;
    return total > 0 ? total : 0;
}

int b200_sgemm_select_config(int layout_c, int layout_a, int layout_b, size_t M, size_t N, size_t K,
                             b200_sgemm_params* out, int* variant)
{
    if(M == 0 || N == 0 || K == 0 || bad_layout(layout_a) || bad_layout(layout_b) || bad_layout(layout_c))
        return B200_SGEMM_INVALID_ARGUMENT;
    int v, s, pre;
    choose(layout_a, layout_b, layout_c, M, N, K, -1, 0, &v, &s, &pre);
    if(out)
        fill_params(kernel_variants[v], s, pre, out);
    if(variant)
        *variant = v;
    return B200_SGEMM_OK;
}

int b200_sgemm_num_variants(void)
{
    return KERNEL_VARIANTS;
}

int b200_sgemm_get_variant(int variant, b200_sgemm_params* out)
{
    if(variant < 0 || variant >= KERNEL_VARIANTS || !out)
        return B200_SGEMM_INVALID_ARGUMENT;
    fill_params(kernel_variants[variant], 1, 0, out);
    return B200_SGEMM_OK;
}

int b200_sgemm_num_entries(void)
{
    return CONFIG_ENTRIES;
}

int b200_sgemm_get_entry(int index, size_t mnk[3], int layouts[3], int* variant, int* split_k)
{
    if(index < 0 || index >= CONFIG_ENTRIES)
        return B200_SGEMM_INVALID_ARGUMENT;
    const ConfigEntry& e = sorted_config_map[index];
    if(mnk)
    {
        mnk[0] = e.key.m;
        mnk[1] = e.key.n;
        mnk[2] = e.key.k;
    }
    if(layouts)
    {
        layouts[0] = e.key.layout_a;
        layouts[1] = e.key.layout_b;
        layouts[2] = e.key.layout_c;
    }
    if(variant)
        *variant = e.variant;
    if(split_k)
        *split_k = e.split_k;
    return B200_SGEMM_OK;
}

int b200_sgemm_get_entry_pretranspose(int index)
{
    if(index < 0 || index >= CONFIG_ENTRIES)
        return -1;
    return sorted_config_map[index].pretranspose;
}

int b200_sgemm_map_tile(int raster, int id, int grid_m, int grid_n, int* tile_m, int* tile_n)
{
    if(!tile_m || !tile_n || grid_m <= 0 || grid_n <= 0 || id < 0 || (long long)id >= (long long)grid_m * grid_n)
        return B200_SGEMM_INVALID_ARGUMENT;
    switch(raster)
    {
    case RASTER_ROW: map_tile<RASTER_ROW>(id, grid_m, grid_n, *tile_m, *tile_n); break;
    case RASTER_GROUPED: map_tile<RASTER_GROUPED>(id, grid_m, grid_n, *tile_m, *tile_n); break;
    case RASTER_HILBERT: map_tile<RASTER_HILBERT>(id, grid_m, grid_n, *tile_m, *tile_n); break;
    default: return B200_SGEMM_INVALID_ARGUMENT;
    }
    return B200_SGEMM_OK;
}

int b200_sgemm_has_kernel(int variant, int layout_index, int aligned)
{
    return lookup_kernel(variant, layout_index, aligned) != nullptr ? 1 : 0;
}

int b200_sgemm_select_in_table(const size_t* keys, size_t count, size_t M, size_t N, size_t K, int layout_a,
                               int layout_b, int layout_c)
{
    if(count == 0 || !keys)
        return -1;
    std::vector<ConfigEntry> map(count);
    for(size_t i = 0; i < count; ++i)
    {
        const size_t* r = keys + 6 * i;
        map[i]          = ConfigEntry{ConfigKey{r[0], r[1], r[2], (int)r[3], (int)r[4], (int)r[5]}, (int)i, 1};
    }
    return find_best_config(map.data(), count, ConfigKey{M, N, K, layout_a, layout_b, layout_c});
}

int b200_sgemm_fma_peak(int mode, int iterations, float* elapsed_ms, double* flops, void* cuda_stream)
{
    if((mode != 0 && mode != 1) || iterations <= 0 || !elapsed_ms || !flops)
        return B200_SGEMM_INVALID_ARGUMENT;
    cudaStream_t   stream = static_cast<cudaStream_t>(cuda_stream);
    int            device = 0;
    cudaDeviceProp prop;
    cudaError_t    e = cudaGetDevice(&device);
    if(e == cudaSuccess)
        e = cudaGetDeviceProperties(&prop, device);
    if(e != cudaSuccess)
        return (int)e;
    float* sink = nullptr;
    e           = cudaMalloc(&sink, sizeof(float));
    if(e != cudaSuccess)
        return (int)e;
    const int   blocks = prop.multiProcessorCount; // one CTA of 8 warps per SM, like the GEMM kernels' consumers
    cudaEvent_t t0, t1;
    cudaEventCreate(&t0);
    cudaEventCreate(&t1);
    auto launch = [&](int iters) {
        if(mode == 0)
            fma_peak_kernel<0><<<blocks, 256, 0, stream>>>(sink, iters, 1e-9f);
        else
            fma_peak_kernel<1><<<blocks, 256, 0, stream>>>(sink, iters, 1e-9f);
    };
    launch(iterations / 8 + 1); // warm-up
    cudaEventRecord(t0, stream);
    launch(iterations);
    cudaEventRecord(t1, stream);
    e = cudaEventSynchronize(t1);
    if(e == cudaSuccess)
        e = cudaEventElapsedTime(elapsed_ms, t0, t1);
    // 64 accumulators x 4 repeats x 2 flops per FMA per iteration per thread
    *flops = 2.0 * 64.0 * 4.0 * (double)iterations * 256.0 * (double)blocks;
    cudaEventDestroy(t0);
    cudaEventDestroy(t1);
    cudaFree(sink);
    return e == cudaSuccess ? B200_SGEMM_OK : (int)e;
}

int b200_sgemm_device_status(int* status)
{
    if(!status)
        return B200_SGEMM_INVALID_ARGUMENT;
    cudaError_t e = cudaDeviceSynchronize();
    if(e != cudaSuccess)
        return (int)e;
    int value = 0;
    e         = cudaMemcpyFromSymbol(&value, g_kernel_status, sizeof(int));
    if(e != cudaSuccess)
        return (int)e;
    if(value != 0)
    {
        const int zero = 0;
        e              = cudaMemcpyToSymbol(g_kernel_status, &zero, sizeof(int));
        if(e != cudaSuccess)
            return (int)e;
    }
    *status = value;
    return B200_SGEMM_OK;
}

int b200_sgemm_release_stream(void* cuda_stream)
{
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    int          device = 0;
    cudaError_t  e      = cudaGetDevice(&device);
    if(e != cudaSuccess)
        return (int)e;
    std::lock_guard<std::mutex> lock(g_arena_mutex);
    auto                        it = g_arenas.find(std::make_pair(device, stream));
    if(it == g_arenas.end())
        return B200_SGEMM_OK;
    if(it->second.ptr)
    {
        // work queued on the stream may still use the block
        e = cudaStreamSynchronize(stream);
        if(e != cudaSuccess)
            return (int)e;
        e = cudaFree(it->second.ptr);
    }
    g_arenas.erase(it);
    return (int)e;
}

int b200_sgemm_shutdown(void)
{
    std::lock_guard<std::mutex> lock(g_arena_mutex);
    cudaError_t                 first = cudaSuccess;
    int                         saved = 0;
    cudaGetDevice(&saved);
    for(auto& kv : g_arenas)
    {
        if(kv.second.ptr)
        {
            cudaSetDevice(kv.first.first);
            cudaError_t e = cudaFree(kv.second.ptr);
            if(e != cudaSuccess && first == cudaSuccess)
                first = e;
        }
    }
    g_arenas.clear();
    cudaSetDevice(saved);
    return first == cudaSuccess ? B200_SGEMM_OK : (int)first;
}

const char* b200_sgemm_status_string(int status)
{
    switch(status)
    {
    case B200_SGEMM_OK: return "ok";
    case B200_SGEMM_INVALID_ARGUMENT: return "invalid argument";
    case B200_SGEMM_NO_KERNEL: return "no kernel available for the requested configuration, layout and alignment";
    case B200_SGEMM_WORKSPACE_TOO_SMALL: return "split-K workspace missing or too small";
    case B200_SGEMM_UNSUPPORTED_SIZE: return "dimension exceeds the supported range";
    case B200_SGEMM_SCRATCH_LIMIT: return "split_k * M * N exceeds the built-in static scratch (B200_SGEMM_STATIC_SCRATCH_BYTES)";
    default: return status > 0 ? cudaGetErrorString(static_cast<cudaError_t>(status)) : "unknown status";
    }
}

} // extern "C"
