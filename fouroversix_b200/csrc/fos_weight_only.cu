// Products of 16-bit activations with packed 4-bit weights (weight-only quantization):
//     y[t, f] = alpha * sum_k x[t, k] * value(code[f, k]) * scale[f, k / block]  (+ bias[f])
// with alpha = amax / divisor(format, rule), in fp32 and rounded once to the output's type. For one weight, or for the rows
// of several groups with a weight each (the experts of a mixture-of-experts layer), fetched by index and without padding.
//
// The numbers that are multiplied are exact: an E2M1 value times an E4M3 scale has at most 6 significant bits, and an IF4
// block is taken 7 times as large (7 * value * scale on the float grid, 6 * int * scale on the integer grid: at most 9 bits),
// with 1 / 7 in alpha; fp16 holds both. MXFP4's scales are exact between 2^-23 and 2^13 (what lies outside goes the way of
// fp16: to zero or infinity, as in dequantize).
//
// few_rows_kernel (at most 16 rows at a time). What bounds it is the weight's way out of HBM, so every code is read once and
// goes straight from global memory to registers. A warp holds 16 features by 128 values of K: the A fragment of
// mma.m16n8k16, with the activations as B (8 rows of x per instruction). K may be permuted as one likes in a sum, so lane t of
// a quad takes 32 consecutive values of a row (one 16-byte load) and the instruction's k are four of each lane's.
// The codes become fp16 by one conversion and one multiplication per pair (measured on its own: 89 values per cycle and SM,
// where HBM delivers 41; expanding to bf16 by shifts and masks gave 48). So bf16 activations become fp16 too: a row's values
// are multiplied by the power of two that takes its largest to [2^14, 2^15). That is exact down to 2^-29 of the largest,
// and what is smaller is off by less than 2^-39 of it, where the fp32 sums are off by 2^-24. The factor goes into the epilogue.
// A projection has few tiles of 128 features, so K is split over the CTAs of a cluster, which add their sums through
// distributed shared memory in the order of K: no atomics, the same bits every time.
#include "fos_tcgen05.cuh"

namespace fos {
namespace {
namespace wo {

constexpr int TILE = 128;                 // features of a CTA: one row of scale tiles
constexpr int STEP = 128;                 // values of K per iteration of a warp
constexpr int THREADS = 256;
constexpr int DEPTH = 4;                  // iterations whose codes are on their way
constexpr int MAX_SPLIT = 8;

struct Params {
    const void *x;
    int64_t x_rows, x_ld, k;
    const int32_t *row_index;             // or nullptr: row r of the groups is row r of x
    const uint8_t *codes, *sf;            // of group 0
    const float *amax;                    // one per group; nullptr: 1
    float divisor;
    const int32_t *group_start, *group_rows;   // or nullptr: one group of all rows
    int num_groups;
    int64_t rows;                         // of the output
    const void *bias;                     // [n] of the output's type, or nullptr
    void *out;
    int out_dtype, vec;                   // vec: 16-byte loads of x
    int64_t ld_out, n, n_p, k_p;
    int sf_tiled, split;
};

// ---------------------------------------------------------------------------- weights to fp16

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Two E4M3 bytes -> two fp16.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {
    uint32_t r;
    asm("{ .reg .b16 h; cvt.u16.u32 h, %1; cvt.rn.f16x2.e4m3x2 %0, h; }" : "=r"(r) : "r"(two));
    return r;
}
// Eight E2M1 codes -> four pairs of fp16, pair j = values 2j, 2j + 1.
__device__ __forceinline__ void e2m1x8_to_h2(uint32_t w, uint32_t (&o)[4]) {
    asm("{ .reg .b8 a, b, c, d;\n"
        "mov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n"
        "cvt.rn.f16x2.e2m1x2 %3, d; }"
        : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(w));
}

// What an IF4 block's eight magnitudes are, looked up by the code's three low bits: low and high bytes of four each.
struct If4Table { uint32_t la, ha, lb, hb; bool ints; };
__device__ __forceinline__ If4Table if4_table(uint32_t s2, bool ints) {
    If4Table t;
    // 7 * {0, 1/2, 1, 3/2, 2, 3, 4, 6} or 6 * {0 .. 7}, fp16
    const uint32_t t01 = mul_h2(s2, ints ? 0x46000000u : 0x43000000u), t23 = mul_h2(s2, ints ? 0x4c804a00u : 0x49404700u);
    const uint32_t t45 = mul_h2(s2, ints ? 0x4f804e00u : 0x4d404b00u), t67 = mul_h2(s2, ints ? 0x51405080u : 0x51404f00u);
    t.la = __byte_perm(t01, t23, 0x6420); t.ha = __byte_perm(t01, t23, 0x7531);
    t.lb = __byte_perm(t45, t67, 0x6420); t.hb = __byte_perm(t45, t67, 0x7531);
    t.ints = ints;
    return t;
}
__device__ __forceinline__ void if4x8_to_h2(uint32_t w, const If4Table &t, uint32_t (&o)[4]) {
    const uint32_t sgn = (w >> 3) & 0x11111111u;
    // the magnitude of a two's-complement nibble n is (n ^ m) + sign with m = 15 where the sign is set; -8 does not occur
    const uint32_t mag = (t.ints ? (w ^ (sgn * 15u)) + sgn : w) & 0x77777777u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t sel = h ? mag >> 16 : mag, ss = h ? sgn >> 16 : sgn;
        const uint32_t lo = __byte_perm(t.la, t.lb, sel);
        const uint32_t hi = __byte_perm(t.ha, t.hb, sel) | __byte_perm(0x00008000u, 0u, ss);
        o[2 * h] = __byte_perm(lo, hi, 0x5140);
        o[2 * h + 1] = __byte_perm(lo, hi, 0x7362);
    }
}

// The scales of 32 consecutive values, as loaded (see load_scales), ready for the two halves of them.
template <int FMT> struct Scales {
    uint32_t s[2];                        // fp16 pairs (s, s)
    __device__ __forceinline__ explicit Scales(uint32_t raw) {
        if constexpr (FMT == FOS_MXFP4) {
            // E8M0 -> fp16 as a conversion of the binary32 value: infinite above 2^15, 0 below 2^-25, NaN for 255
            const float f = raw == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(raw << 23);
            const __half2 h = __float2half2_rn(f);
            s[0] = s[1] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const uint32_t both = e4m3x2_to_h2(FMT == FOS_IF4 ? raw & 0x7f7fu : raw);
            s[0] = __byte_perm(both, 0u, 0x1010);
            s[1] = __byte_perm(both, 0u, 0x3232);
        }
    }
};

// Thirty-two codes of a row (a 16-byte load) -> sixteen pairs of fp16 in their order.
template <int FMT>
__device__ __forceinline__ void expand32(const uint4 &c, uint32_t raw_scales, uint32_t (&o)[4][4]) {
    const Scales<FMT> sc(raw_scales);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    if constexpr (FMT == FOS_IF4) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const If4Table t = if4_table(sc.s[b], (raw_scales >> (8 * b + 7)) & 1u);
            if4x8_to_h2(w[2 * b], t, o[2 * b]);
            if4x8_to_h2(w[2 * b + 1], t, o[2 * b + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e2m1x8_to_h2(w[i], o[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = mul_h2(o[i][j], sc.s[i >> 1]);
        }
    }
}

// ---------------------------------------------------------------------------- activations

// The largest |x| of a bf16 row, as its bit pattern, gives the factor 2^(141 - e) that takes it to [2^14, 2^15), and the factor
// back. Both are normal numbers: e is taken as 15 at least (smaller values then stay below 2^14) and as 254 at most (a row with
// infinities or NaN has those in every sum anyway).
__device__ __forceinline__ uint32_t row_exponent(uint32_t max_bits) {
    const uint32_t e = max_bits >> 7;
    return e < 15u ? 15u : (e > 254u ? 254u : e);
}
__device__ __forceinline__ float row_factor(uint32_t e) { return __uint_as_float((268u - e) << 23); }
__device__ __forceinline__ float row_factor_back(uint32_t e) { return __uint_as_float((e - 14u) << 23); }

template <typename T> __device__ __forceinline__ uint32_t to_scaled_h2(uint32_t w, float factor) {
    if constexpr (std::is_same<T, __half>::value) {
        return w;
    } else {
        const float2 f = unpack2<T>(w);
        const __half2 h = __floats2half2_rn(f.x * factor, f.y * factor);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// Eight values of a row of x from column c on; zeros behind the last column.
__device__ __forceinline__ uint4 load_x8(const uint16_t *row, int64_t c, int64_t k, bool vec) {
    if (row == nullptr || c >= k) return make_uint4(0u, 0u, 0u, 0u);
    if (vec && c + 8 <= k) return ld_16(row + c);
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = c + i < k ? ld_b16(row + c + i) : 0u;
    return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}

__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void store_out(void *out, int dtype, int64_t at, float v) {
    if (dtype == FOS_BF16) static_cast<__nv_bfloat16 *>(out)[at] = __float2bfloat16_rn(v);
    else if (dtype == FOS_FP16) static_cast<__half *>(out)[at] = __float2half_rn(v);
    else static_cast<float *>(out)[at] = v;
}
__device__ __forceinline__ float load_bias(const void *bias, int dtype, int64_t at) {
    if (dtype == FOS_BF16) return __uint_as_float(ld_b16(static_cast<const uint16_t *>(bias) + at) << 16);
    if (dtype == FOS_FP16) return __half2float(__ushort_as_half(static_cast<unsigned short>(ld_b16(static_cast<const uint16_t *>(bias) + at))));
    return ld_float(static_cast<const float *>(bias) + at);
}

// The rows of a group: [first, first + count) of the output hold products, [first + count, end) belong to nobody and become zero.
// Whatever the two arrays say, nothing outside the output is touched.
struct GroupRange { int64_t first, count, end; };
__device__ __forceinline__ GroupRange group_range(const Params &p, int g) {
    if (!p.group_start) return {0, p.rows, p.rows};
    auto clamp = [](int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); };
    GroupRange r;
    r.first = clamp(ld_int(p.group_start + g), 0, p.rows);
    r.count = clamp(ld_int(p.group_rows + g), 0, p.rows - r.first);
    r.end = g + 1 < p.num_groups ? clamp(ld_int(p.group_start + g + 1), r.first + r.count, p.rows) : p.rows;
    return r;
}
// The row of x that row r of the output is made of, or nullptr for a row of zeros.
__device__ __forceinline__ const uint16_t *x_row(const Params &p, int64_t r) {
    const int64_t i = p.row_index ? static_cast<int64_t>(ld_int(p.row_index + r)) : r;
    return i >= 0 && i < p.x_rows ? static_cast<const uint16_t *>(p.x) + i * p.x_ld : nullptr;
}

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// ---------------------------------------------------------------------------- at most 8 * NT rows at a time

template <int NT> inline int few_rows_smem_bytes(int64_t k_p, int split) {
    const int64_t steps = (k_p + STEP - 1) / STEP, share = (steps + split - 1) / split;
    return static_cast<int>(share * STEP * 8 * NT * 2 + TILE * 8 * NT * 4);
}

template <typename T, int NT, int FMT>
__global__ void __launch_bounds__(THREADS, 2) few_rows_kernel(const Params p) {
    constexpr int MT = 8 * NT;
    constexpr bool SCALED = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t row_max[MT];
    float *sums = reinterpret_cast<float *>(smem);                    // [split][MT][TILE / split] of what the CTAs of a cluster sent here
    uint4 *xs = reinterpret_cast<uint4 *>(smem + TILE * MT * 4);      // [step][word][row][lane of the quad]: eight values each

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad_row = lane >> 2, t = lane & 3;
    const int split = p.split, part = static_cast<int>(blockIdx.x) % split;
    const int64_t tile = blockIdx.x / split;
    const int group = blockIdx.y;
    const int steps = static_cast<int>((p.k_p + STEP - 1) / STEP);
    const int it0 = static_cast<int>(static_cast<int64_t>(steps) * part / split);
    const int it1 = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / split);
    const int64_t n_cb = p.k_p / (FMT == FOS_MXFP4 ? 32 : 16);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const GroupRange range = group_range(p, group);

    // the fragment's row rho (0 .. 15) is row 4 * warp + rho % 4 + 32 * (rho / 4) of the tile: what the warp needs of the scale tiles
    // is then 64 consecutive bytes
    const int i = quad_row & 3, q = quad_row >> 2;
    const int64_t row_a = tile * TILE + 4 * warp + i + 32 * q, row_b = row_a + 64;
    const uint8_t *codes = p.codes + group * (p.n_p * (p.k_p / 2)), *sf = p.sf + group * (p.n_p * n_cb);
    const uint8_t *codes_a = codes + row_a * (p.k_p / 2) + t * 16, *codes_b = codes + row_b * (p.k_p / 2) + t * 16;

    uint4 ca[DEPTH], cb[DEPTH];
    uint32_t sa[DEPTH], sb[DEPTH];
    auto fetch = [&](int it, int u) {
        ca[u] = cb[u] = make_uint4(0u, 0u, 0u, 0u);
        sa[u] = sb[u] = 0u;
        if (it >= it1 || static_cast<int64_t>(it) * STEP + t * 32 >= p.k_p) return;     // (k_p may end in the middle of a step)
        ca[u] = ld_16_stream(codes_a + it * (STEP / 2));
        cb[u] = ld_16_stream(codes_b + it * (STEP / 2));
        if constexpr (FMT == FOS_MXFP4) {
            const int64_t col = static_cast<int64_t>(it) * 4 + t;
            sa[u] = ld_b8(sf + sf_offset(row_a, col, n_cb, p.sf_tiled));
            sb[u] = ld_b8(sf + sf_offset(row_b, col, n_cb, p.sf_tiled));
        } else {
            const int64_t col = static_cast<int64_t>(it) * 8 + 2 * t;
            sa[u] = ld_b16(sf + sf_offset(row_a, col, n_cb, p.sf_tiled));
            sb[u] = ld_b16(sf + sf_offset(row_b, col, n_cb, p.sf_tiled));
        }
    };

    const float alpha = p.amax ? __fdiv_rn(ld_float(p.amax + group), p.divisor) : 1.0f;
    const int64_t passes_from = static_cast<int64_t>(blockIdx.z) * MT, passes_by = static_cast<int64_t>(gridDim.z) * MT;
    for (int64_t r0 = passes_from; r0 < range.count; r0 += passes_by) {
        const int m = static_cast<int>(range.count - r0 < MT ? range.count - r0 : MT);
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) fetch(it0 + u, u);
        if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // nothing is read from `sums` any more

        // ---- the rows of x, this CTA's share of K, as fp16 in the order of the fragments
        const int per_row = m <= 1 ? THREADS : m <= 2 ? THREADS / 2 : m <= 4 ? THREADS / 4 : m <= 8 ? THREADS / 8 : THREADS / 16;
        const int n = tid / per_row, j0 = tid % per_row, chunks = (it1 - it0) * (STEP / 8);
        const uint16_t *row = n < m ? x_row(p, range.first + r0 + n) : nullptr;
        const int64_t c0 = static_cast<int64_t>(it0) * STEP;
        if constexpr (SCALED) {
            if (tid < MT) row_max[tid] = 0u;
            __syncthreads();
            uint32_t most = 0u;                                     // two 16-bit maxima of |x|'s bit patterns
            for (int j = j0; j < chunks; j += per_row) {
                const uint4 v = load_x8(row, c0 + j * 8, p.k, p.vec);
                most = __vmaxu2(__vmaxu2(most, v.x & 0x7fff7fffu), v.y & 0x7fff7fffu);
                most = __vmaxu2(__vmaxu2(most, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu);
            }
            most = max(most & 0xffffu, most >> 16);
            if (n < m && most) atomicMax(&row_max[n], most);
        }
        __syncthreads();                                           // (the last pass's fragments have been read, too)
        if (n < m) {
            const float factor = SCALED ? row_factor(row_exponent(row_max[n])) : 1.0f;
            for (int j = j0; j < chunks; j += per_row) {
                uint4 v = load_x8(row, c0 + j * 8, p.k, p.vec);
                v = make_uint4(to_scaled_h2<T>(v.x, factor), to_scaled_h2<T>(v.y, factor), to_scaled_h2<T>(v.z, factor), to_scaled_h2<T>(v.w, factor));
                // chunk j of the share: step j / 16, lane (j / 4) % 4 of the quad, word j % 4 of its sixteen bytes of codes
                xs[((j >> 4) * 4 + (j & 3)) * (MT * 4) + n * 4 + ((j >> 2) & 3)] = v;
            }
        }
        __syncthreads();

        // ---- the product
        float acc[NT][4];
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[a][r] = 0.0f;
        bool live[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) live[a] = 8 * a + quad_row < m;
        for (int base = it0; base < it1; base += DEPTH) {
#pragma unroll
            for (int u = 0; u < DEPTH; ++u) {
                const int it = base + u;
                if (it >= it1) break;
                uint32_t wa[4][4], wb[4][4];
                expand32<FMT>(ca[u], sa[u], wa);
                expand32<FMT>(cb[u], sb[u], wb);
                fetch(it + DEPTH, u);
                const uint4 *frag = xs + (it - it0) * (4 * MT * 4) + lane;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
#pragma unroll
                    for (int a = 0; a < NT; ++a) {
                        const uint4 b = live[a] ? frag[w * (MT * 4) + a * 32] : make_uint4(0u, 0u, 0u, 0u);
                        mma_m16n8k16(acc[a], wa[w][0], wb[w][0], wa[w][1], wb[w][1], b.x, b.y);
                        mma_m16n8k16(acc[a], wa[w][2], wb[w][2], wa[w][3], wb[w][3], b.z, b.w);
                    }
                }
            }
        }

        // ---- every CTA of the cluster gets the sums of its share of the tile's features
        const int share = TILE / split;
        const uint32_t sums_at = smem_u32(sums);
        if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
        for (int a = 0; a < NT; ++a) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int col = 8 * a + 2 * t + (r & 1), f = 4 * warp + i + 32 * (q + (r & 2));
                if (col >= m) continue;
                const float v = SCALED ? acc[a][r] * row_factor_back(row_exponent(row_max[col])) : acc[a][r];
                const int owner = f / share;
                const uint32_t at = sums_at + ((part * MT + col) * share + f - owner * share) * 4;
                if (split > 1) st_cluster_f32(map_to_cta(at, owner), v);
                else sums[col * TILE + f] = v;
            }
        }
        if (split > 1) cluster_sync_all();
        else __syncthreads();
        for (int e = tid; e < m * share; e += THREADS) {
            const int col = e / share, f = e - col * share;
            const int64_t feature = tile * TILE + part * share + f;
            if (feature >= p.n) continue;
            float sum = sums[col * share + f];
            for (int s = 1; s < split; ++s) sum += sums[(s * MT + col) * share + f];
            sum *= alpha;
            if (p.bias) sum += load_bias(p.bias, p.out_dtype, feature);
            store_out(p.out, p.out_dtype, (range.first + r0 + col) * p.ld_out + feature, sum);
        }
        if (split == 1) __syncthreads();
    }

    // ---- rows of no group: behind this group's, and before the first group's
    if (p.group_start && blockIdx.z == 0) {
        const int share = TILE / split;
        const int64_t f0 = tile * TILE + part * share;
        auto clear = [&](int64_t from, int64_t to) {
            for (int64_t e = tid; e < (to - from) * share; e += THREADS) {
                const int64_t r = from + e / share, f = f0 + e % share;
                if (f < p.n) store_out(p.out, p.out_dtype, r * p.ld_out + f, 0.0f);
            }
        };
        clear(range.first + range.count, range.end);
        if (group == 0) clear(0, range.first);
    }
}

// How many CTAs share a tile's K: as many as fill the SMs about twice over, while each keeps four steps, and more where the
// activations' share of K would not leave room for two CTAs on an SM.
inline int split_for(int64_t tiles, int64_t k_p, int rows_at_once, int sms) {
    const int64_t steps = (k_p + STEP - 1) / STEP;
    auto room = [&](int s) { return ((steps + s - 1) / s) * STEP * rows_at_once * 2 + TILE * rows_at_once * 4 <= 100 * 1024; };
    int split = 1;
    while (split < MAX_SPLIT && ((tiles * split * 2 <= 2 * sms + sms / 4 && steps / (split * 2) >= 4) || !room(split))) split *= 2;
    return split;
}

template <typename T, int NT, int FMT>
int launch_few_rows(const Params &p, unsigned grid_z, cudaStream_t stream) {
    auto kernel = few_rows_kernel<T, NT, FMT>;
    static OncePerDevice configured;      // per instantiation
    int dev = 0;
    FOS_CUDA_TRY(cudaGetDevice(&dev));
    FOS_CUDA_TRY(configured.run(dev, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024); }));
    const int smem = few_rows_smem_bytes<NT>(p.k_p, p.split);
    if (smem > 227 * 1024 - 1024) return FOS_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.n_p / TILE * p.split), static_cast<unsigned>(p.num_groups), grid_z);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(p.split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.split > 1 ? 2 : 1;
    FOS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
    return FOS_OK;
}

template <typename T, int NT>
int launch_few_rows_format(const Params &p, int format, unsigned grid_z, cudaStream_t stream) {
    if (format == FOS_NVFP4) return launch_few_rows<T, NT, FOS_NVFP4>(p, grid_z, stream);
    if (format == FOS_IF4) return launch_few_rows<T, NT, FOS_IF4>(p, grid_z, stream);
    return launch_few_rows<T, NT, FOS_MXFP4>(p, grid_z, stream);
}

int run(Params p, int x_dtype, int format, cudaStream_t stream) {
    int dev = 0, sms = 0;
    FOS_CUDA_TRY(cudaGetDevice(&dev));
    FOS_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // how the groups share the rows is known on the device only: twice the even share at once
    const int64_t at_once = p.group_start ? 2 * ((p.rows + p.num_groups - 1) / p.num_groups) : p.rows;
    const int mt = at_once <= 8 ? 8 : 16;
    p.split = split_for(p.n_p / TILE * (p.group_start ? (p.num_groups < p.rows ? p.num_groups : p.rows) : 1), p.k_p, mt, sms);
    int64_t z = p.group_start ? 1 : (p.rows + mt - 1) / mt;
    if (z > 65535) z = 65535;
    const unsigned grid_z = static_cast<unsigned>(z);
    if (x_dtype == FOS_BF16)
        return mt == 8 ? launch_few_rows_format<__nv_bfloat16, 1>(p, format, grid_z, stream) : launch_few_rows_format<__nv_bfloat16, 2>(p, format, grid_z, stream);
    return mt == 8 ? launch_few_rows_format<__half, 1>(p, format, grid_z, stream) : launch_few_rows_format<__half, 2>(p, format, grid_z, stream);
}

int check(const void *x, int x_dtype, int64_t x_rows, int64_t k, int64_t ld_x, const uint8_t *codes, const uint8_t *sf, const float *amax,
          int format, int rule, int sf_layout, int64_t n, int64_t n_p, int64_t k_p, int64_t rows, const void *out, int out_dtype, int64_t ld_out) {
    if (!x || !codes || !sf || !out) return FOS_ERR_INVALID_ARGUMENT;
    if (x_dtype != FOS_BF16 && x_dtype != FOS_FP16) return FOS_ERR_INVALID_ARGUMENT;
    if (out_dtype != FOS_BF16 && out_dtype != FOS_FP16 && out_dtype != FOS_FP32) return FOS_ERR_INVALID_ARGUMENT;
    if (format != FOS_NVFP4 && format != FOS_IF4 && format != FOS_MXFP4) return FOS_ERR_INVALID_ARGUMENT;
    if (format != FOS_MXFP4 && !amax) return FOS_ERR_INVALID_ARGUMENT;
    if (rule < FOS_RULE_STATIC_6 || rule > FOS_RULE_ABS_MAX) return FOS_ERR_INVALID_ARGUMENT;
    if (sf_layout != FOS_SF_ROWMAJOR && sf_layout != FOS_SF_TILED) return FOS_ERR_INVALID_ARGUMENT;
    if (rows <= 0 || x_rows <= 0 || k <= 0 || n <= 0 || ld_x < k || ld_out < n) return FOS_ERR_INVALID_ARGUMENT;
    if (n_p % 128 || n_p < n || k_p % (format == FOS_MXFP4 ? 128 : 64) || k_p < k) return FOS_ERR_INVALID_ARGUMENT;
    if (n_p > INT32_MAX / MAX_SPLIT || k_p > INT32_MAX / 8 || rows > INT32_MAX || x_rows > INT32_MAX) return FOS_ERR_TOO_LARGE;
    if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(sf) % 2 || reinterpret_cast<uintptr_t>(x) % 2) return FOS_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(out) % (out_dtype == FOS_FP32 ? 4 : 2)) return FOS_ERR_MISALIGNED;
    return FOS_OK;
}

// amax / divisor is what the packed numbers are multiplied with, in units of what the kernels multiply (IF4: seven times the values).
float divisor_for(int format, int rule, int unbiased) {
    if (format == FOS_MXFP4) return 1.0f;
    double d = dequant_divisor(format, rule);
    if (unbiased) d *= 16.0 / 17.0;
    return static_cast<float>(format == FOS_IF4 ? d * 7.0 : d);
}

}  // namespace wo
}  // namespace
}  // namespace fos

extern "C" int fos_weight_only_matmul(const void *x, int x_dtype, int64_t rows, int64_t k, int64_t ld_x, const uint8_t *w_codes,
                                      const uint8_t *w_sf, const float *w_amax, int format, int scale_rule, int unbiased, int sf_layout,
                                      int64_t n, int64_t n_p, int64_t k_p, const void *bias, void *out, int out_dtype, int64_t ld_out,
                                      void *stream) {
    using namespace fos;
    int st = wo::check(x, x_dtype, rows, k, ld_x, w_codes, w_sf, w_amax, format, scale_rule, sf_layout, n, n_p, k_p, rows, out, out_dtype, ld_out);
    if (st != FOS_OK) return st;
    if (reinterpret_cast<uintptr_t>(bias) % (out_dtype == FOS_FP32 ? 4 : 2)) return FOS_ERR_MISALIGNED;
    if ((st = check_device()) != FOS_OK) return st;
    wo::Params p{};
    p.x = x; p.x_rows = rows; p.x_ld = ld_x; p.k = k;
    p.codes = w_codes; p.sf = w_sf;
    p.amax = format == FOS_MXFP4 ? nullptr : w_amax;
    p.divisor = wo::divisor_for(format, scale_rule, unbiased);
    p.num_groups = 1; p.rows = rows;
    p.bias = bias; p.out = out; p.out_dtype = out_dtype; p.ld_out = ld_out;
    p.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x % 8 == 0;
    p.n = n; p.n_p = n_p; p.k_p = k_p; p.sf_tiled = sf_layout == FOS_SF_TILED;
    return wo::run(p, x_dtype, format, static_cast<cudaStream_t>(stream));
}

extern "C" int fos_weight_only_matmul_grouped(const void *x, int x_dtype, int64_t x_rows, int64_t k, int64_t ld_x, const int32_t *row_index,
                                              const uint8_t *w_codes, const uint8_t *w_sf, const float *w_amax, int format, int scale_rule,
                                              int sf_layout, const int32_t *group_start, const int32_t *group_rows, int num_groups,
                                              int64_t rows, int64_t n, int64_t n_p, int64_t k_p, void *out, int out_dtype, int64_t ld_out,
                                              void *stream) {
    using namespace fos;
    int st = wo::check(x, x_dtype, x_rows, k, ld_x, w_codes, w_sf, w_amax, format, scale_rule, sf_layout, n, n_p, k_p, rows, out, out_dtype, ld_out);
    if (st != FOS_OK) return st;
    if (!group_start || !group_rows || num_groups <= 0 || num_groups > 256) return FOS_ERR_INVALID_ARGUMENT;
    if ((st = check_device()) != FOS_OK) return st;
    wo::Params p{};
    p.x = x; p.x_rows = x_rows; p.x_ld = ld_x; p.k = k; p.row_index = row_index;
    p.codes = w_codes; p.sf = w_sf;
    p.amax = format == FOS_MXFP4 ? nullptr : w_amax;
    p.divisor = wo::divisor_for(format, scale_rule, 0);
    p.group_start = group_start; p.group_rows = group_rows; p.num_groups = num_groups; p.rows = rows;
    p.out = out; p.out_dtype = out_dtype; p.ld_out = ld_out;
    p.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x % 8 == 0;
    p.n = n; p.n_p = n_p; p.k_p = k_p; p.sf_tiled = sf_layout == FOS_SF_TILED;
    return wo::run(p, x_dtype, format, static_cast<cudaStream_t>(stream));
}
