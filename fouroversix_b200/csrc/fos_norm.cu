// Root-mean-square norm with the residual's addition:
//     h = round16(x + residual)                 (h = x without a residual; h is the new residual stream)
//     f = 1 / sqrt(mean(h^2) + eps)
//     y = round16((h * f) * weight)             binary32 products, one rounding to 16 bits
// The mean is formed in binary64 and f rounded to binary32 from there: a square of a 16-bit number is exact in binary64, so
// f is the correctly rounded factor of the row but for a few in 2^28 cases, whatever the order of the sum - and with it every
// bit of y, which matters where y is packed to 4 bits and a value next to a border would fall to either side. A binary64
// addition per value costs the kernel nothing: it is bound by HBM (2 or 4 B in, 2 or 4 B out per value).
//
// norm_rows_kernel: G threads hold a row in registers, at most four chunks of 8 values each, and so read it once.
// What becomes of y: it is written, with the largest |y| of every CTA for the kernel that packs it; or, where no such number is needed,
// packed at once (MXFP4). (Packing y as it is formed again from h, two bytes written and read less per value, took the general
// quantize kernel 77 us for 8192 x 8192, and the one with a feed of its own takes 37 us from y in memory.) A decoding step's few rows are
// packed with the norm in one launch: norm_quantize_small_kernel, beside the kernel whose second half it shares.
// norm_any_kernel: rows that are longer, or that 16-byte loads cannot take: a CTA per row, in two passes.
#include "fos_mx.cuh"
#include "fos_norm.cuh"
#include "fos_tcgen05.cuh"

namespace fos {
namespace norm {
namespace {

constexpr int MAX_PARTS = AMAX_PARTS_WORDS;

constexpr int CHUNKS = 4;

// G threads per row; at least 256 threads in a CTA.
template <typename T, int G, bool RESIDUAL, bool MX>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_rows_kernel(const Params p) {
    constexpr int THREADS = G > 256 ? G : 256, ROWS = THREADS / G, WARPS = THREADS / 32;
    __shared__ double sums[WARPS];
    __shared__ uint32_t mosts[WARPS];
    __shared__ float factors[ROWS], maxima[WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = tid % G, slot = tid / G;
    const int cols = static_cast<int>(p.cols);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float y_max = 0.0f;
    if (MX && blockIdx.x == 0 && tid == 0) *p.amax_out = 1.0f;
    const int64_t last = MX ? p.rows_p : p.rows;                        // (the padding rows become zeros)
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * ROWS; r0 < last; r0 += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t row = r0 + slot;
        const bool live = row < p.rows;
        uint32_t h[CHUNKS][4];
        uint4 res[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = (c * G + g) * 8;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            res[c] = v;
            if (live && col < cols) {
                v = ld_16_stream(static_cast<const T *>(p.x) + row * p.ld_x + col);
                if constexpr (RESIDUAL) res[c] = ld_16_stream(static_cast<const T *>(p.residual) + row * p.ld_residual + col);
            }
            h[c][0] = v.x; h[c][1] = v.y; h[c][2] = v.z; h[c][3] = v.w;
        }
        double sum = 0.0, sum2 = 0.0;
        uint32_t most2 = 0u;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = (c * G + g) * 8;
            if (col >= cols) continue;
            if constexpr (RESIDUAL) {
                h[c][0] = add_pair<T>(h[c][0], res[c].x); h[c][1] = add_pair<T>(h[c][1], res[c].y);
                h[c][2] = add_pair<T>(h[c][2], res[c].z); h[c][3] = add_pair<T>(h[c][3], res[c].w);
                if (live) *reinterpret_cast<uint4 *>(static_cast<T *>(p.sum) + row * p.ld_sum + col) = make_uint4(h[c][0], h[c][1], h[c][2], h[c][3]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t bare = h[c][k] & 0x7fff7fffu;
                most2 = __vmaxu2(most2, bare);
                add_squares<T>(sum, sum2, bare);
            }
        }
        sum += sum2;
        most2 = max(most2 & 0xffffu, most2 >> 16);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        most2 = __reduce_max_sync(0xffffffffu, most2);
        uint32_t most = __float_as_uint(unpack2<T>(most2).x);
        float factor;
        if constexpr (G == 32) {
            factor = row_factor(sum, most, p);
        } else {
            // the row's first warp adds up and forms the factor for the others
            if (lane == 0) { sums[warp] = sum; mosts[warp] = most; }
            __syncthreads();
            if (g < 32) {
                constexpr int W = G / 32;
                sum = g < W ? sums[slot * W + g] : 0.0;
                most = g < W ? mosts[slot * W + g] : 0u;
#pragma unroll
                for (int o = W / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                most = __reduce_max_sync(0xffffffffu, most);
                if (g == 0) factors[slot] = row_factor(sum, most, p);
            }
            __syncthreads();
            factor = factors[slot];
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = (c * G + g) * 8;
            const bool inside = live && col < cols;
            if (!MX && !inside) continue;
            uint32_t out[4] = {0u, 0u, 0u, 0u};
            if (inside) {
                float w[8];
                if (p.weight_fp32) {
                    const uint4 a = ld_16(static_cast<const float *>(p.weight) + col), b = ld_16(static_cast<const float *>(p.weight) + col + 4);
                    w[0] = __uint_as_float(a.x); w[1] = __uint_as_float(a.y); w[2] = __uint_as_float(a.z); w[3] = __uint_as_float(a.w);
                    w[4] = __uint_as_float(b.x); w[5] = __uint_as_float(b.y); w[6] = __uint_as_float(b.z); w[7] = __uint_as_float(b.w);
                } else {
                    const uint4 a = ld_16(static_cast<const T *>(p.weight) + col);
                    const uint32_t words[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) { const float2 f = unpack2<T>(words[k]); w[2 * k] = f.x; w[2 * k + 1] = f.y; }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack2<T>(h[c][k]);
                    const float y0 = __fmul_rn(__fmul_rn(f.x, factor), w[2 * k]), y1 = __fmul_rn(__fmul_rn(f.y, factor), w[2 * k + 1]);
                    y_max = fmaxf(y_max, fmaxf(fabsf(y0), fabsf(y1)));         // (before it is rounded, which keeps the order)
                    out[k] = pack_pair<T>(y0, y1);
                }
            }
            if constexpr (MX) {
                // a block of 32 values is four neighbouring lanes'; the columns up to cols_p are written, zeros behind the last
                float v[8], block = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack2<T>(out[k]);
                    v[2 * k] = f.x; v[2 * k + 1] = f.y;
                    block = fmaxf(block, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
                block = fmaxf(block, __shfl_xor_sync(0xffffffffu, block, 1));
                block = fmaxf(block, __shfl_xor_sync(0xffffffffu, block, 2));
                float inv;
                const uint32_t e = mx_scale(block, p.quarter != 0, inv);
                if (row < p.rows_p && col < p.cols_p) {
                    float t[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) t[k] = __fadd_rn(__fmul_rn(v[k], inv), 0.0f);
                    *reinterpret_cast<uint32_t *>(p.codes + row * (p.cols_p >> 1) + (col >> 1)) = cvt_e2m1x8(t);
                    if ((g & 3) == 0) p.sf[sf_offset(row, col >> 5, p.cols_p >> 5, p.sf_tiled != 0)] = static_cast<uint8_t>(e);
                }
            } else {
                *reinterpret_cast<uint4 *>(static_cast<T *>(p.y) + row * p.ld_y + col) = make_uint4(out[0], out[1], out[2], out[3]);
            }
        }
    }
    if (!MX && (p.amax_parts || p.amax)) {
        y_max = round16<T>(y_max);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) y_max = fmaxf(y_max, __shfl_xor_sync(0xffffffffu, y_max, o));
        if (lane == 0) maxima[warp] = y_max;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < WARPS; ++w) y_max = fmaxf(y_max, maxima[w]);
            if (p.amax_parts) p.amax_parts[blockIdx.x] = y_max;
            else atomicMax(reinterpret_cast<unsigned *>(p.amax), __float_as_uint(y_max));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(512) norm_any_kernel(const Params p) {
    __shared__ double sums[16];
    __shared__ uint32_t mosts[16];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto value = [](const void *base, int64_t at) { return elem_to_float<T>(*reinterpret_cast<const T *>(static_cast<const T *>(base) + at)); };
    float y_max = 0.0f;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        double sum = 0.0;
        uint32_t most = 0u;
        for (int64_t c = tid; c < p.cols; c += 512) {
            float v = value(p.x, row * p.ld_x + c);
            if (p.residual) {
                v = round16<T>(__fadd_rn(v, value(p.residual, row * p.ld_residual + c)));
                if constexpr (std::is_same<T, __half>::value) static_cast<T *>(p.sum)[row * p.ld_sum + c] = __float2half_rn(v);
                else static_cast<T *>(p.sum)[row * p.ld_sum + c] = __float2bfloat16_rn(v);
            }
            sum = add_square(sum, v);
            most = max(most, __float_as_uint(v) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        __syncthreads();
        if (lane == 0) { sums[warp] = sum; mosts[warp] = most; }
        __syncthreads();
        sum = 0.0;
        most = 0u;
#pragma unroll
        for (int w = 0; w < 16; ++w) { sum += sums[w]; most = max(most, mosts[w]); }
        const float factor = row_factor(sum, most, p);
        // (each thread reads back only what it wrote itself)
        for (int64_t c = tid; c < p.cols; c += 512) {
            const float v = p.residual ? value(p.sum, row * p.ld_sum + c) : value(p.x, row * p.ld_x + c);
            const float w = p.weight_fp32 ? static_cast<const float *>(p.weight)[c] : value(p.weight, c);
            const float r = round16<T>(__fmul_rn(__fmul_rn(v, factor), w));
            y_max = fmaxf(y_max, fabsf(r));
            if constexpr (std::is_same<T, __half>::value) static_cast<T *>(p.y)[row * p.ld_y + c] = __float2half_rn(r);
            else static_cast<T *>(p.y)[row * p.ld_y + c] = __float2bfloat16_rn(r);
        }
    }
    if (p.amax) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) y_max = fmaxf(y_max, __shfl_xor_sync(0xffffffffu, y_max, o));
        if (lane == 0 && y_max > 0.0f) atomicMax(reinterpret_cast<unsigned *>(p.amax), __float_as_uint(y_max));
    }
}

template <typename T, int G, bool RESIDUAL, bool MX>
int launch_rows(const Params &p, int *ctas, cudaStream_t stream) {
    constexpr int THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
    int64_t grid = ((MX ? p.rows_p : p.rows) + ROWS - 1) / ROWS;
    const int64_t most = THREADS == 256 ? 148 * 6 : 148 * 2;
    static_assert(148 * 6 <= MAX_PARTS, "a part per CTA");
    if (grid > most) grid = most;
    *ctas = static_cast<int>(grid);
    FOS_CUDA_TRY(launch_dependent(norm_rows_kernel<T, G, RESIDUAL, MX>, dim3(static_cast<unsigned>(grid)), THREADS, 0, stream, p));
    return FOS_OK;
}

template <typename T, bool RESIDUAL, bool MX>
int launch_width(const Params &p, int *ctas, cudaStream_t stream) {
    if (p.cols <= 32 * 8 * CHUNKS) return launch_rows<T, 32, RESIDUAL, MX>(p, ctas, stream);
    if (p.cols <= 128 * 8 * CHUNKS) return launch_rows<T, 128, RESIDUAL, MX>(p, ctas, stream);
    if (p.cols <= 256 * 8 * CHUNKS) return launch_rows<T, 256, RESIDUAL, MX>(p, ctas, stream);
    return launch_rows<T, 1024, RESIDUAL, MX>(p, ctas, stream);
}

template <typename T, bool MX> int launch_out(const Params &p, int *ctas, cudaStream_t stream) {
    return p.residual ? launch_width<T, true, MX>(p, ctas, stream) : launch_width<T, false, MX>(p, ctas, stream);
}

// Whether norm_rows_kernel takes the rows: 16-byte loads and stores, rows that fit the registers of 1024 threads.
inline bool rows_fit(const Params &p) {
    auto aligned = [](const void *q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0; };
    return p.cols % 8 == 0 && p.cols <= 1024 * 8 * CHUNKS && aligned(p.x, p.ld_x) && aligned(p.weight, 0) && (!p.y || aligned(p.y, p.ld_y)) &&
           (!p.residual || (aligned(p.residual, p.ld_residual) && aligned(p.sum, p.ld_sum)));
}

template <typename T> int launch(const Params &p, cudaStream_t stream) {
    int ctas;
    if (rows_fit(p)) return launch_out<T, false>(p, &ctas, stream);
    const int64_t grid = p.rows < 148 * 4 ? p.rows : 148 * 4;
    FOS_CUDA_TRY(launch_dependent(norm_any_kernel<T>, dim3(static_cast<unsigned>(grid)), 512, 0, stream, p));
    return FOS_OK;
}

int check(const void *x, int dtype, int64_t rows, int64_t cols, int64_t ld_x, const void *residual, int64_t ld_residual, const void *weight,
          int weight_dtype, double eps, const void *sum, int64_t ld_sum) {
    if (!x || !weight || (residual && !sum)) return FOS_ERR_INVALID_ARGUMENT;
    if (dtype != FOS_BF16 && dtype != FOS_FP16) return FOS_ERR_INVALID_ARGUMENT;
    if (weight_dtype != dtype && weight_dtype != FOS_FP32) return FOS_ERR_INVALID_ARGUMENT;
    if (rows <= 0 || cols <= 0 || ld_x < cols || (residual && (ld_residual < cols || ld_sum < cols))) return FOS_ERR_INVALID_ARGUMENT;
    if (!(eps >= 1e-30)) return FOS_ERR_INVALID_ARGUMENT;
    if (cols > INT32_MAX) return FOS_ERR_TOO_LARGE;
    for (const void *q : {x, residual, residual ? sum : nullptr})
        if (reinterpret_cast<uintptr_t>(q) % 2) return FOS_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(weight) % (weight_dtype == FOS_FP32 ? 4 : 2)) return FOS_ERR_MISALIGNED;
    return FOS_OK;
}

}  // namespace
}  // namespace norm
}  // namespace fos

extern "C" int fos_rms_norm(const void *x, int dtype, int64_t rows, int64_t cols, int64_t ld_x, const void *residual, int64_t ld_residual,
                            const void *weight, int weight_dtype, double eps, void *sum, int64_t ld_sum, void *y, int64_t ld_y,
                            float *amax, void *stream_) {
    using namespace fos;
    int st = norm::check(x, dtype, rows, cols, ld_x, residual, ld_residual, weight, weight_dtype, eps, sum, ld_sum);
    if (st != FOS_OK) return st;
    if (!y || ld_y < cols) return FOS_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(y) % 2 || reinterpret_cast<uintptr_t>(amax) % 4) return FOS_ERR_MISALIGNED;
    if ((st = check_device()) != FOS_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (amax) FOS_CUDA_TRY(cudaMemsetAsync(amax, 0, sizeof(float), stream));
    norm::Params p{x, residual, weight, sum, y, amax, rows, cols, ld_x, ld_residual, ld_sum, ld_y, eps, 1.0 / static_cast<double>(cols),
                   weight_dtype == FOS_FP32};
    return dtype == FOS_BF16 ? norm::launch<__nv_bfloat16>(p, stream) : norm::launch<__half>(p, stream);
}

extern "C" int64_t fos_rms_norm_quantize_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || fos::norm::small_enough(rows, cols)) return 0;
    return fos::AMAX_PARTS_WORDS * 4 + rows * cols * 2;
}

extern "C" int fos_rms_norm_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int64_t ld_x, const void *residual,
                                     int64_t ld_residual, const void *weight, int weight_dtype, double eps, void *sum, int64_t ld_sum,
                                     int format, int scale_rule, int sf_layout, uint8_t *codes, uint8_t *sf, float *amax_out,
                                     void *workspace, int64_t workspace_bytes, void *stream_) {
    using namespace fos;
    int st = norm::check(x, dtype, rows, cols, ld_x, residual, ld_residual, weight, weight_dtype, eps, sum, ld_sum);
    if (st != FOS_OK) return st;
    if (!codes || !sf || !amax_out) return FOS_ERR_INVALID_ARGUMENT;
    if (format != FOS_NVFP4 && format != FOS_IF4 && format != FOS_MXFP4) return FOS_ERR_INVALID_ARGUMENT;
    if (scale_rule < FOS_RULE_STATIC_6 || scale_rule > FOS_RULE_ABS_MAX) return FOS_ERR_INVALID_ARGUMENT;
    if (sf_layout != FOS_SF_ROWMAJOR && sf_layout != FOS_SF_TILED) return FOS_ERR_INVALID_ARGUMENT;
    const bool is_static = scale_rule == FOS_RULE_STATIC_6 || scale_rule == FOS_RULE_STATIC_4;
    if ((format == FOS_IF4 && is_static) || (format == FOS_MXFP4 && !is_static)) return FOS_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(codes) % 8 || reinterpret_cast<uintptr_t>(amax_out) % 4) return FOS_ERR_MISALIGNED;
    norm::Params p{x, residual, weight, sum, nullptr, nullptr, rows, cols, ld_x, ld_residual, ld_sum, 0, eps, 1.0 / static_cast<double>(cols),
                   weight_dtype == FOS_FP32};
    if (!norm::rows_fit(p)) return FOS_ERR_UNSUPPORTED;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    int ctas = 0;
    p.codes = codes; p.sf = sf; p.amax_out = amax_out;
    p.rows_p = round_up64(rows, 128);
    p.cols_p = round_up64(cols, format == FOS_MXFP4 ? 128 : 64);
    p.sf_tiled = sf_layout == FOS_SF_TILED;
    if (format == FOS_MXFP4) {
        p.quarter = scale_rule == FOS_RULE_STATIC_4;
        if ((st = check_device()) != FOS_OK) return st;
        return dtype == FOS_BF16 ? norm::launch_out<__nv_bfloat16, true>(p, &ctas, stream) : norm::launch_out<__half, true>(p, &ctas, stream);
    }
    if (norm::small_enough(rows, cols)) {
        if ((st = check_device()) != FOS_OK) return st;
        bool launched = false;
        if ((st = norm::quantize_small(p, dtype, format, scale_rule, stream, &launched)) != FOS_OK) return st;
        return launched ? FOS_OK : FOS_ERR_UNSUPPORTED;
    }
    if (!workspace || workspace_bytes < fos_rms_norm_quantize_workspace_bytes(rows, cols)) return FOS_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(workspace) % 128) return FOS_ERR_MISALIGNED;
    if ((st = check_device()) != FOS_OK) return st;
    p.amax_parts = static_cast<float *>(workspace);
    p.y = p.amax_parts + AMAX_PARTS_WORDS;
    p.ld_y = cols;
    st = dtype == FOS_BF16 ? norm::launch_out<__nv_bfloat16, false>(p, &ctas, stream) : norm::launch_out<__half, false>(p, &ctas, stream);
    if (st != FOS_OK) return st;
    return quantize_with_parts(p.y, dtype, rows, cols, cols, format, scale_rule, sf_layout, p.amax_parts, ctas, codes, sf, amax_out, stream_);
}
