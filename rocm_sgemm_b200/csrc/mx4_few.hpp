// The 4-bit product for a few rows on one side (mx4_few.cu).
#pragma once
#include <cstddef>
#include <cuda_runtime.h>

namespace sgemm_b200
{
// whether mx4_few takes the product: one or two rows against a matrix of which they cost less than the tensor core's set-up
// (measured: one row x 4096 x 4096 4.0 us against 7.0, x 16384 x 4096 11.1 us against 10.1; two rows 5.2 against 7.0, 17 against
// 10.2)
inline bool mx4_is_few(size_t few, size_t rows, size_t K)
{
    return few == 1 ? rows * K <= (size_t(1) << 25) : few == 2 && rows * K <= (size_t(1) << 24);
}

struct FewArgs
{
    const void*  codes;  // the long side: `rows` rows
    const void*  scales;
    const void*  codes_x; // the short side: `few` rows
    const void*  scales_x;
    const float* global;
    const float* global_x;
    void*        c;
    long long    ld_long, ld_few; // element strides of C along the two sides
    float        alpha;
    int          rows, few, K, type;
};

// status as b200_sgemm_mx4's
int mx4_few(int format, const FewArgs& a, int sms, cudaStream_t stream);
} // namespace sgemm_b200
