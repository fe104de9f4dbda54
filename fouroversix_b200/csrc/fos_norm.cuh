// What the norm's kernels share: their parameters, and the row's factor from exact squares.
#pragma once
#include "fos_common.cuh"

namespace fos {
namespace norm {

struct Params {
    const void *x, *residual, *weight;
    void *sum, *y;                        // h (with a residual only) and y
    float *amax;                          // raised to max |y|, or nullptr
    int64_t rows, cols, ld_x, ld_residual, ld_sum, ld_y;
    double eps, per_row;                  // per_row: 1 / cols
    int weight_fp32;
    float *amax_parts;                    // the largest |y| of every CTA, or nullptr
    uint8_t *codes, *sf;                  // MXFP4
    int64_t rows_p, cols_p;
    int sf_tiled, quarter;                // (quarter: static_4)
    float *amax_out;
};

// The square of a binary32 number that has at most 20 bits of mantissa, added to `acc` in binary64. The number is taken apart by
// hand (a conversion instruction runs at an eighth of this rate): its mantissa fits the upper word. Zero becomes 2^-127 this way,
// infinity and NaN become 2^128; the callers keep eps above the one and look for the others themselves.
__device__ __forceinline__ double add_square(double acc, float v) {
    const double d = __hiloint2double(static_cast<int>(((__float_as_uint(v) & 0x7fffffffu) >> 3) + 0x38000000u), 0);
    return __fma_rn(d, d, acc);
}
// The row's factor from the sum of its squares; `most` is the largest |h| as bits of a binary32 number.
__device__ __forceinline__ float row_factor(double sum, uint32_t most, const Params &p) {
    if (most >= 0x7f800000u) return most > 0x7f800000u ? __uint_as_float(0x7fc00000u) : 0.0f;
    return static_cast<float>(rsqrt(sum * p.per_row + p.eps));
}

// The same for a pair of 16-bit numbers whose signs have been cleared. A bf16 number's exponent and mantissa shift into place as they are.
template <typename T> __device__ __forceinline__ void add_squares(double &a, double &b, uint32_t pair) {
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = unpack2<T>(pair);
        a = add_square(a, f.x);
        b = add_square(b, f.y);
    } else {
        const double lo = __hiloint2double(static_cast<int>((pair & 0xffffu) * 8192u + 0x38000000u), 0);
        const double hi = __hiloint2double(static_cast<int>((pair >> 16) * 8192u + 0x38000000u), 0);
        a = __fma_rn(lo, lo, a);
        b = __fma_rn(hi, hi, b);
    }
}

template <typename T> __device__ __forceinline__ float round16(float v) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(__float2half_rn(v));
    else return __bfloat162float(__float2bfloat16_rn(v));
}
// A packed addition rounds once from the exact sum; so does adding in binary32 and rounding, for two 16-bit numbers.
template <typename T> __device__ __forceinline__ uint32_t add_pair(uint32_t a, uint32_t b) {
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const P r = __hadd2_rn(*reinterpret_cast<const P *>(&a), *reinterpret_cast<const P *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// The rows of x (and residual) packed to NVFP4 or IF4 in one launch, where the tensor is small enough for a cluster of 16 CTAs: see
// norm_quantize_small_kernel. p as for 16-byte accesses; codes, sf, rows_p, cols_p, sf_tiled and amax_out are set.
bool small_enough(int64_t rows, int64_t cols);
int quantize_small(const Params &p, int dtype, int format, int scale_rule, cudaStream_t stream, bool *launched);

}  // namespace norm
}  // namespace fos
