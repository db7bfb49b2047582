// b200_sgemm_route_*: tokens sorted by expert, and back with weights applied, and the gradients of both.
//
//   sort      slot s = t * top_k + j goes to row offsets[e] + (number of earlier slots of the same expert e)
//   dispatch  Xs[row(s)] = X[t]                        its gradient: combine without weights
//   combine   out[t]     = sum_j w[s] Y[row(s)]        its gradients: dY[row(s)] = w[s] dOut[t], dw[s] = <dOut[t], Y[row(s)]>
//
// sort is bound by latency: one kernel, one cluster, no workspace.  Each warp counts a contiguous range of slots in shared
// memory of its own (no atomics, so the order is the slots' own), the CTAs of the cluster exchange their totals through
// distributed shared memory, and each warp then places its slots.  The other three are bound by HBM and read and write
// every row once: a token's row stays in registers while it goes to its top_k rows, or while theirs are added to it.
#include "mx4_common.cuh"

#include <type_traits>

namespace
{
using namespace sgemm_b200;

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS   = SORT_THREADS / 32;
constexpr int SORT_CTAS    = 8; // of a cluster, at most
constexpr int MAX_EXPERTS  = 1024; // one thread each in the scan

struct SortArgs
{
    const int* ids;
    int*       offsets;
    int*       counts;
    int*       slot_row;
    int*       row_slot;
    int        slots, experts, align, rows, ctas, bits; // bits that tell experts and -1 apart
    int        warps, per_warp;                         // warps of a CTA that hold slots, and how many each
};

__device__ __forceinline__ int expert_of(const SortArgs& a, int slot)
{
    const int e = slot < a.slots ? __ldg(a.ids + slot) : -1;
    return (unsigned)e < (unsigned)a.experts ? e : -1;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_cluster_int(const int* p, int rank)
{
    uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
    int      v;
    asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__global__ void __launch_bounds__(SORT_THREADS, 1) route_sort_kernel(const __grid_constant__ SortArgs a)
{
    extern __shared__ int before[]; // [warps][experts]: slots of an expert in this CTA's earlier warps
    __shared__ int total[MAX_EXPERTS], start[MAX_EXPERTS], warp_sum[SORT_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = threadIdx.x;
    const int rank = a.ctas > 1 ? (int)(blockIdx.x % a.ctas) : 0;
    int*      mine = before + warp * a.experts;
    // the range of the last warps may lie behind the slots
    const long long begin = (long long)(rank * a.warps + warp) * a.per_warp;
    const int       count = warp < a.warps ? (int)max(0ll, min((long long)a.per_warp, a.slots - begin)) : 0;

    // f(expert, position in the range) for 32 slots at a time; the experts of four such batches are fetched together (one by one,
    // 32768 slots took 10.9 us)
    auto each_batch = [&](auto f) {
        for(int i0 = 0; i0 < count; i0 += 128)
        {
            int x[4];
#pragma unroll
            for(int b = 0; b < 4; ++b)
                x[b] = i0 + b * 32 + lane < count ? expert_of(a, (int)begin + i0 + b * 32 + lane) : -1;
#pragma unroll
            for(int b = 0; b < 4; ++b)
                if(i0 + b * 32 < count)
                    f(x[b], i0 + b * 32 + lane);
        }
    };

    if(warp < a.warps)
    {
        for(int i = lane; i < a.experts; i += 32)
            mine[i] = 0;
        __syncwarp();
        each_batch([&](int x, int) {
            if(x >= 0)
                atomicAdd(mine + x, 1); // of this warp alone, and a sum of ones: the order does not matter
        });
        __syncwarp();
    }
    // every row without a slot until one is placed there, which is behind the barriers below
    for(long long row = rank * SORT_THREADS + threadIdx.x; row < a.rows; row += a.ctas * SORT_THREADS)
        a.row_slot[row] = -1;
    __syncthreads();
    if(e < a.experts)
    {
        int sum = 0;
        for(int w0 = 0; w0 < a.warps; w0 += 8)
        {
            int n[8];
#pragma unroll
            for(int w = 0; w < 8; ++w)
                n[w] = w0 + w < a.warps ? before[(w0 + w) * a.experts + e] : 0;
#pragma unroll
            for(int w = 0; w < 8; ++w)
            {
                if(w0 + w < a.warps)
                    before[(w0 + w) * a.experts + e] = sum;
                sum += n[w];
            }
        }
        total[e] = sum;
    }
    if(a.ctas > 1)
        cluster_sync();
    int all = 0, earlier = 0;
    if(e < a.experts)
    {
        int n[SORT_CTAS]; // all in flight at once
#pragma unroll
        for(int r = 0; r < SORT_CTAS; ++r)
            n[r] = a.ctas == 1 ? (r == 0 ? total[e] : 0) : (r < a.ctas ? ld_cluster_int(total + e, r) : 0);
#pragma unroll
        for(int r = 0; r < SORT_CTAS; ++r)
        {
            earlier += r < rank ? n[r] : 0;
            all += n[r];
        }
    }
    // exclusive sum of the experts' rounded-up rows
    const int padded = (all + a.align - 1) / a.align * a.align;
    int       upto   = padded;
#pragma unroll
    for(int d = 1; d < 32; d <<= 1)
    {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        upto += lane >= d ? v : 0;
    }
    if(lane == 31)
        warp_sum[warp] = upto;
    __syncthreads();
    if(warp == 0)
    {
        int v = warp_sum[lane];
#pragma unroll
        for(int d = 1; d < 32; d <<= 1)
        {
            const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
            v += lane >= d ? u : 0;
        }
        warp_sum[lane] = v;
    }
    __syncthreads();
    const int first = upto - padded + (warp ? warp_sum[warp - 1] : 0);
    if(e < a.experts)
    {
        start[e] = first + earlier;
        if(rank == 0)
        {
            a.offsets[e] = first;
            a.counts[e]  = all;
            if(e == a.experts - 1)
                a.offsets[a.experts] = first + padded;
        }
    }
    __syncthreads();
    each_batch([&](int x, int i) {
        unsigned same = 0xFFFFFFFFu; // lanes with the same expert: those that agree in every bit (the match instruction is slower)
        for(int bit = 0; bit < a.bits; ++bit)
        {
            const bool     one = x >> bit & 1;
            const unsigned set = __ballot_sync(0xFFFFFFFFu, one);
            same &= one ? set : ~set;
        }
        const unsigned low  = same & ((1u << lane) - 1u);
        const int      slot = (int)begin + i, row = x >= 0 ? start[x] + mine[x] + __popc(low) : -1;
        __syncwarp();
        if(x >= 0 && low == 0)
            mine[x] += __popc(same);
        __syncwarp();
        if(i < count)
            a.slot_row[slot] = row;
        if(row >= 0)
            a.row_slot[row] = slot;
    });
    if(a.ctas > 1)
        cluster_sync(); // nobody leaves while its totals are being read
}

// ---- rows ----------------------------------------------------------------------------------------------------
constexpr int R_THREADS = 256;

// N elements of a row, loaded and stored at once: 16 bytes where base and pitch allow it, else one element
template<class T, int N>
struct Piece
{
    alignas(N * sizeof(T)) T v[N];
    __device__ __forceinline__ void load(const T* p)
    {
        if constexpr(N > 1)
            *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
        else
            v[0] = *p;
    }
    __device__ __forceinline__ void store(T* p) const
    {
        if constexpr(N > 1)
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
        else
            *p = v[0];
    }
};

struct RowArgs
{
    const void*  x;   // dispatch: X; combine: Y; backward: dOut
    const void*  y;   // backward: Y
    void*        out; // dispatch: Xs; combine: out; backward: dY
    float*       dw;
    const int*   slot_row;
    const float* weights;
    long long    ldx, ldy, ldo;
    int          tokens, top_k, width, rows;
    int          pieces; // pieces of a row, in units of a warp's step
};

// How a warp takes a token's row: UNROLL x 32 pieces of it, and (combine) ROWS of the slots' rows fetched at once.  Many tokens: 4
// pieces and one row, which leaves registers for many warps; few, where one warp's latency is all there is: 1 piece and 8 rows.
// Combine of 8192 tokens x 4 x 4096 BF16 took 51 us with (4, 1), 55 us with (2, 4), 72 us with (1, 8); of 64 tokens x 8
// 4.9 us with (4, 1), 3.1 us with (2, 4), 2.6 us with (1, 8).

__device__ __forceinline__ int row_of(const RowArgs& a, long long slot)
{
    const int r = __ldg(a.slot_row + slot);
    return (unsigned)r < (unsigned)a.rows ? r : -1;
}

template<class T, int N, int UNROLL>
__global__ void __launch_bounds__(R_THREADS) route_dispatch_kernel(const __grid_constant__ RowArgs a)
{
    const int       lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (R_THREADS / 32) + (threadIdx.x >> 5);
    const long long t    = unit / a.pieces;
    if(t >= a.tokens)
        return;
    const int c0 = ((int)(unit - t * a.pieces) * UNROLL * 32 + lane) * N;
    const T*  x  = static_cast<const T*>(a.x) + t * a.ldx;
    Piece<T, N> p[UNROLL];
#pragma unroll
    for(int u = 0; u < UNROLL; ++u)
        if(c0 + u * 32 * N < a.width)
            p[u].load(x + c0 + u * 32 * N);
    for(int j0 = 0; j0 < a.top_k; j0 += 32)
    {
        const int mine = j0 + lane < a.top_k ? row_of(a, t * a.top_k + j0 + lane) : -1;
        for(int j = 0; j < min(32, a.top_k - j0); ++j)
        {
            const int r = __shfl_sync(0xFFFFFFFFu, mine, j);
            if(r < 0)
                continue;
            T* to = static_cast<T*>(a.out) + r * a.ldo;
#pragma unroll
            for(int u = 0; u < UNROLL; ++u)
                if(c0 + u * 32 * N < a.width)
                    p[u].store(to + c0 + u * 32 * N);
        }
    }
}

template<class T, int N, int UNROLL, int ROWS>
__global__ void __launch_bounds__(R_THREADS) route_combine_kernel(const __grid_constant__ RowArgs a)
{
    const int       lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (R_THREADS / 32) + (threadIdx.x >> 5);
    const long long t    = unit / a.pieces;
    if(t >= a.tokens)
        return;
    const int c0 = ((int)(unit - t * a.pieces) * UNROLL * 32 + lane) * N;
    float     sum[UNROLL][N] = {};
    auto add = [&](const Piece<T, N>(&p)[UNROLL], float w) {
#pragma unroll
        for(int u = 0; u < UNROLL; ++u)
            if(c0 + u * 32 * N < a.width)
            {
#pragma unroll
                for(int i = 0; i < N; ++i)
                    sum[u][i] = fmaf(w, to_float(p[u].v[i]), sum[u][i]);
            }
    };
    auto fetch = [&](Piece<T, N>(&p)[UNROLL], int r) {
        const T* y = static_cast<const T*>(a.x) + r * a.ldx;
#pragma unroll
        for(int u = 0; u < UNROLL; ++u)
            if(c0 + u * 32 * N < a.width)
                p[u].load(y + c0 + u * 32 * N);
    };
    if constexpr(ROWS == 1)
    {
        for(int j = 0; j < a.top_k; ++j)
        {
            const int r = row_of(a, t * a.top_k + j);
            if(r < 0)
                continue;
            const float w = a.weights ? __ldg(a.weights + t * a.top_k + j) : 1.f;
            Piece<T, N> p[UNROLL];
            fetch(p, r);
            add(p, w);
        }
    }
    else
    {
        for(int j0 = 0; j0 < a.top_k; j0 += 32) // the rows and weights of 32 slots at once
        {
            const bool  slot   = j0 + lane < a.top_k;
            const int   mine   = slot ? row_of(a, t * a.top_k + j0 + lane) : -1;
            const float weight = slot && a.weights ? __ldg(a.weights + t * a.top_k + j0 + lane) : 1.f;
            const int   n      = min(32, a.top_k - j0);
            for(int j1 = 0; j1 < n; j1 += ROWS) // fetched together, added in order
            {
                int         r[ROWS];
                Piece<T, N> p[ROWS][UNROLL];
#pragma unroll
                for(int j = 0; j < ROWS; ++j)
                {
                    r[j] = j1 + j < n ? __shfl_sync(0xFFFFFFFFu, mine, j1 + j) : -1;
                    if(r[j] >= 0)
                        fetch(p[j], r[j]);
                }
#pragma unroll
                for(int j = 0; j < ROWS; ++j)
                {
                    const float w = __shfl_sync(0xFFFFFFFFu, weight, (j1 + j) & 31);
                    if(r[j] >= 0)
                        add(p[j], w);
                }
            }
        }
    }
    T* to = static_cast<T*>(a.out) + t * a.ldo;
#pragma unroll
    for(int u = 0; u < UNROLL; ++u)
        if(c0 + u * 32 * N < a.width)
        {
            Piece<T, N> p;
#pragma unroll
            for(int i = 0; i < N; ++i)
                p.v[i] = from_float<T>(sum[u][i]);
            p.store(to + c0 + u * 32 * N);
        }
}

constexpr int B_SLOTS = 4; // slots of a token whose sums are kept at once

// one CTA: one token; its row of dOut is read once per B_SLOTS slots
template<class T, int N>
__global__ void __launch_bounds__(R_THREADS) route_backward_kernel(const __grid_constant__ RowArgs a)
{
    __shared__ float part[R_THREADS / 32][B_SLOTS];
    const long long  t    = blockIdx.x;
    const T*         dout = static_cast<const T*>(a.x) + t * a.ldx;
    for(int j0 = 0; j0 < a.top_k; j0 += B_SLOTS)
    {
        const int n = min(B_SLOTS, a.top_k - j0);
        int   row[B_SLOTS];
        float w[B_SLOTS], dot[B_SLOTS];
#pragma unroll
        for(int j = 0; j < B_SLOTS; ++j)
        {
            row[j] = j < n ? row_of(a, t * a.top_k + j0 + j) : -1;
            w[j]   = j < n && a.weights ? __ldg(a.weights + t * a.top_k + j0 + j) : 1.f;
            dot[j] = 0.f;
        }
        for(int c = threadIdx.x * N; c < a.width; c += R_THREADS * N)
        {
            Piece<T, N> g, y[B_SLOTS];
            g.load(dout + c);
            if(a.dw)
            {
#pragma unroll
                for(int j = 0; j < B_SLOTS; ++j)
                    if(row[j] >= 0)
                        y[j].load(static_cast<const T*>(a.y) + row[j] * a.ldy + c);
            }
#pragma unroll
            for(int j = 0; j < B_SLOTS; ++j)
                if(row[j] >= 0)
                {
                    Piece<T, N> d;
#pragma unroll
                    for(int i = 0; i < N; ++i)
                    {
                        const float v = to_float(g.v[i]);
                        d.v[i]        = from_float<T>(w[j] * v);
                        if(a.dw)
                            dot[j] = fmaf(v, to_float(y[j].v[i]), dot[j]);
                    }
                    if(a.out)
                        d.store(static_cast<T*>(a.out) + row[j] * a.ldo + c);
                }
        }
        if(!a.dw)
            continue;
#pragma unroll
        for(int j = 0; j < B_SLOTS; ++j)
        {
#pragma unroll
            for(int d = 16; d; d >>= 1)
                dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], d);
            if((threadIdx.x & 31) == 0)
                part[threadIdx.x >> 5][j] = dot[j];
        }
        __syncthreads();
        if(threadIdx.x < n)
        {
            float sum = 0.f;
#pragma unroll
            for(int k = 0; k < R_THREADS / 32; ++k)
                sum += part[k][threadIdx.x];
            a.dw[t * a.top_k + j0 + threadIdx.x] = sum;
        }
        __syncthreads();
    }
}

// f(type, pieces per vector) where all rows start on 16 bytes and hold whole pieces, else element by element (8192 tokens x 4 BF16,
// dispatch / combine / its gradients: width 2048 28.5 / 29.9 / 54.3 us, width 2050 36.9 / 56.3 / 90.7)
template<class F>
int with_pieces(int type, bool vector, size_t width, F f)
{
    return with_type(type, [&](auto t) {
        using T         = decltype(t);
        constexpr int N = Vec16<T>::N;
        if(vector && width % N == 0)
            return f(t, std::integral_constant<int, N>());
        return f(t, std::integral_constant<int, 1>());
    });
}
bool rows_vector(int type, const void* p, size_t ld) { return !misaligned(p, 16) && ld * type_bytes(type) % 16 == 0; }

bool sizes_ok(size_t tokens, size_t top_k, size_t width, size_t rows)
{
    return tokens <= MAX_EXTENT && top_k <= MAX_EXTENT && tokens * top_k <= MAX_EXTENT && width <= MAX_EXTENT && rows <= MAX_EXTENT;
}
// CTAs for one warp per `unroll` x 32 pieces of n elements; 0: more than a grid holds
unsigned warp_grid(const RowArgs& a, int* pieces, int n, int unroll)
{
    const size_t per  = (size_t)unroll * 32 * n;
    *pieces           = (int)(((size_t)a.width + per - 1) / per);
    const size_t ctas = ((size_t)a.tokens * *pieces + R_THREADS / 32 - 1) / (R_THREADS / 32);
    return ctas > 0x7fffffffull ? 0u : (unsigned)ctas;
}
// f(grid, many), which launches, for the two ways of taking a row: `many` from one wave of 148 SMs x 8 CTAs on
template<class F>
int with_grid(RowArgs& a, int n, F f)
{
    unsigned   grid = warp_grid(a, &a.pieces, n, 4);
    const bool many = grid >= 148u * 8u || grid == 0;
    if(!many)
        grid = warp_grid(a, &a.pieces, n, 1);
    if(!grid)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    return f(grid, many);
}
} // namespace

extern "C" size_t b200_sgemm_route_capacity(size_t tokens, size_t top_k, size_t experts, size_t align)
{
    if(tokens == 0 || top_k == 0 || experts == 0 || align == 0 || tokens > MAX_EXTENT || top_k > MAX_EXTENT || experts > MAX_EXPERTS
       || align > MAX_EXTENT)
        return 0;
    const size_t slots = tokens * top_k, held = slots < experts ? slots : experts; // experts that can hold a slot
    return slots + held * (align - 1);
}

extern "C" int b200_sgemm_route_sort(const int* expert_ids, size_t tokens, size_t top_k, size_t experts, size_t align, int* offsets,
                                     int* counts, int* slot_row, int* row_slot, size_t rows, void* cuda_stream)
{
    if(!expert_ids || !offsets || !counts || !slot_row || !row_slot || tokens == 0 || top_k == 0 || experts == 0 || align == 0
       || misaligned(expert_ids, 4) || misaligned(offsets, 4) || misaligned(counts, 4) || misaligned(slot_row, 4)
       || misaligned(row_slot, 4))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(!sizes_ok(tokens, top_k, 1, rows) || experts > MAX_EXPERTS || align > MAX_EXTENT)
        return B200_SGEMM_UNSUPPORTED_SIZE;
    if(rows < b200_sgemm_route_capacity(tokens, top_k, experts, align))
        return B200_SGEMM_INVALID_ARGUMENT;
    SortArgs a;
    a.ids      = expert_ids;
    a.offsets  = offsets;
    a.counts   = counts;
    a.slot_row = slot_row;
    a.row_slot = row_slot;
    a.slots    = (int)(tokens * top_k);
    a.experts  = (int)experts;
    a.align    = (int)align;
    a.rows     = (int)rows;
    a.ctas     = a.slots <= 1024 ? 1 : (a.slots <= 4096 ? 4 : SORT_CTAS);
    a.bits = 1;
    while((1 << a.bits) <= a.experts)
        ++a.bits;
    const int per_cta = (a.slots + a.ctas - 1) / a.ctas;
    a.warps           = per_cta >= SORT_THREADS ? SORT_WARPS : (per_cta + 31) / 32;
    a.per_warp        = ((per_cta + a.warps - 1) / a.warps + 31) / 32 * 32;
    const size_t smem = (size_t)a.warps * experts * sizeof(int);
    if(smem > 48 * 1024 - sizeof(int) * (2 * MAX_EXPERTS + SORT_WARPS)) // beyond what every kernel may have
    {
        // always the most that a call can need: with this call's own size another thread's smaller one could take it back
        // between here and the launch
        constexpr int     most = SORT_WARPS * MAX_EXPERTS * (int)sizeof(int);
        const cudaError_t e    = cudaFuncSetAttribute(route_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if(e != cudaSuccess)
            return (int)e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned)a.ctas);
    cfg.blockDim           = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes   = smem;
    cfg.stream             = static_cast<cudaStream_t>(cuda_stream);
    cudaLaunchAttribute attr[1];
    attr[0].id               = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs                = attr;
    cfg.numAttrs             = a.ctas > 1 ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, route_sort_kernel, a);
}

extern "C" int b200_sgemm_route_dispatch(int type, const void* X, size_t tokens, size_t width, size_t ldx, const int* slot_row,
                                         size_t top_k, void* Xs, size_t rows, size_t lds, void* cuda_stream)
{
    if(!X || !slot_row || !Xs || tokens == 0 || width == 0 || top_k == 0 || rows == 0 || !type_ok(type))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(!sizes_ok(tokens, top_k, width, rows))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    ldx = ldx ? ldx : width;
    lds = lds ? lds : width;
    if(ldx < width || lds < width || misaligned(X, type_bytes(type)) || misaligned(Xs, type_bytes(type)) || misaligned(slot_row, 4))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(ldx > (size_t(1) << 30) || lds > (size_t(1) << 30))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    RowArgs a  = {};
    a.x        = X;
    a.out      = Xs;
    a.slot_row = slot_row;
    a.ldx      = (long long)ldx;
    a.ldo      = (long long)lds;
    a.tokens   = (int)tokens;
    a.top_k    = (int)top_k;
    a.width    = (int)width;
    a.rows     = (int)rows;
    return with_pieces(type, rows_vector(type, X, ldx) && rows_vector(type, Xs, lds), width, [&](auto t, auto n) {
        return with_grid(a, n(), [&](unsigned grid, bool many) {
            auto kernel = many ? route_dispatch_kernel<decltype(t), n(), 4> : route_dispatch_kernel<decltype(t), n(), 1>;
            return launch_kernel(kernel, grid, R_THREADS, static_cast<cudaStream_t>(cuda_stream), a);
        });
    });
}

extern "C" int b200_sgemm_route_combine(int type, const void* Y, size_t rows, size_t width, size_t ldy, const int* slot_row,
                                        size_t tokens, size_t top_k, const float* weights, void* out, size_t ldo, void* cuda_stream)
{
    if(!Y || !slot_row || !out || tokens == 0 || width == 0 || top_k == 0 || rows == 0 || !type_ok(type))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(!sizes_ok(tokens, top_k, width, rows))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    ldy = ldy ? ldy : width;
    ldo = ldo ? ldo : width;
    if(ldy < width || ldo < width || misaligned(Y, type_bytes(type)) || misaligned(out, type_bytes(type)) || misaligned(slot_row, 4)
       || misaligned(weights, 4))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(ldy > (size_t(1) << 30) || ldo > (size_t(1) << 30))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    RowArgs a  = {};
    a.x        = Y;
    a.out      = out;
    a.slot_row = slot_row;
    a.weights  = weights;
    a.ldx      = (long long)ldy;
    a.ldo      = (long long)ldo;
    a.tokens   = (int)tokens;
    a.top_k    = (int)top_k;
    a.width    = (int)width;
    a.rows     = (int)rows;
    return with_pieces(type, rows_vector(type, Y, ldy) && rows_vector(type, out, ldo), width, [&](auto t, auto n) {
        return with_grid(a, n(), [&](unsigned grid, bool many) {
            auto kernel = many ? route_combine_kernel<decltype(t), n(), 4, 1> : route_combine_kernel<decltype(t), n(), 1, 8>;
            return launch_kernel(kernel, grid, R_THREADS, static_cast<cudaStream_t>(cuda_stream), a);
        });
    });
}

extern "C" int b200_sgemm_route_combine_backward(int type, const void* d_out, size_t ldo, const void* Y, size_t rows, size_t width,
                                                 size_t ldy, const int* slot_row, size_t tokens, size_t top_k, const float* weights,
                                                 void* dY, size_t lddy, float* d_weights, void* cuda_stream)
{
    if(!d_out || !slot_row || (!dY && !d_weights) || (d_weights && !Y) || tokens == 0 || width == 0 || top_k == 0 || rows == 0
       || !type_ok(type))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(!sizes_ok(tokens, top_k, width, rows))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    ldo  = ldo ? ldo : width;
    ldy  = ldy ? ldy : width;
    lddy = lddy ? lddy : width;
    if(ldo < width || ldy < width || lddy < width || misaligned(d_out, type_bytes(type)) || misaligned(Y, type_bytes(type))
       || misaligned(dY, type_bytes(type)) || misaligned(slot_row, 4) || misaligned(weights, 4) || misaligned(d_weights, 4))
        return B200_SGEMM_INVALID_ARGUMENT;
    if(ldo > (size_t(1) << 30) || ldy > (size_t(1) << 30) || lddy > (size_t(1) << 30))
        return B200_SGEMM_UNSUPPORTED_SIZE;
    RowArgs a  = {};
    a.x        = d_out;
    a.y        = Y;
    a.out      = dY;
    a.dw       = d_weights;
    a.slot_row = slot_row;
    a.weights  = weights;
    a.ldx      = (long long)ldo;
    a.ldy      = (long long)ldy;
    a.ldo      = (long long)lddy;
    a.tokens   = (int)tokens;
    a.top_k    = (int)top_k;
    a.width    = (int)width;
    a.rows     = (int)rows;
    const bool vector = rows_vector(type, d_out, ldo) && (!d_weights || rows_vector(type, Y, ldy)) && (!dY || rows_vector(type, dY, lddy));
    return with_pieces(type, vector, width, [&](auto t, auto n) {
        return launch_kernel(route_backward_kernel<decltype(t), n()>, (unsigned)tokens, R_THREADS, static_cast<cudaStream_t>(cuda_stream), a);
    });
}
