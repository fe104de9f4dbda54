// Products of 16-bit activations with packed 4-bit weights (weight-only quantization):
//     y[t, f] = alpha * sum_k x[t, k] * value(code[f, k]) * scale[f, k / block]  (+ bias[f])
// with alpha = amax / divisor(format, rule), in fp32 and rounded once to the output's type. For one weight, or for the rows
// of several groups with a weight each (the experts of a mixture-of-experts layer), fetched by index and without padding.
//
// The numbers that are multiplied are exact: an E2M1 value times an E4M3 scale has at most 6 significant bits, and an IF4
// block is taken 7 times as large (7 * value * scale on the float grid, 6 * int * scale on the integer grid: at most 9 bits),
// with 1 / 7 in alpha; fp16 holds both. MXFP4's scales are exact between 2^-23 and 2^13; what lies outside goes the way of
// fp16, to zero or infinity, as in dequantize (tested over every scale).
//
// The codes become fp16 by one conversion and one multiplication per pair (measured on its own: 89 values per cycle and SM, where HBM
// delivers 41; expanding to bf16 by shifts and masks gave 48; the kernels here expand 10 to 23, so neither way is what bounds them). So bf16 activations become fp16 too: a row's values are
// multiplied by the power of two that takes its largest to [2^14, 2^15). That is exact down to 2^-29 of the largest, and what is
// smaller is off by less than 2^-39 of it, where the fp32 sums are off by 2^-24. The factor goes into the epilogue.
//
// Four kernels, chosen by gemm_choice:
//   few_rows_kernel   up to 16 rows at a time: mma.sync, every code read once
//   gemm_kernel       tiles of 128 features by 32 to 256 rows on one SM: tcgen05, the expanded weight in shared memory; its transpose too
//   gemm_pair_kernel  256 x 256 on two SMs
//   stream_kernel     128 x 128, the expanded weight in tensor memory, the stages of all tiles dealt out evenly
//
// few_rows_kernel. A warp holds 16 features by 128 values of K: the A fragment of mma.m16n8k16, with the activations as B (8 rows of x
// per instruction). K may be permuted as one likes in a sum, so lane t of a quad takes 32 consecutive values of a row (16 bytes)
// and the instruction's k are four of each lane's. A projection has few tiles of 128 features, so K is split over the CTAs of a
// cluster, which add their sums through distributed shared memory in the order of K: no atomics, the same bits every time.
// 1 x 4096 -> 4096 takes 6.7 us in a graph (its bytes 1.5), 1 x 8192 -> 10240 18.4 (7.3), 8 x 8192 -> 28672 47.7 (20.5). It issues some 190
// instructions per warp for its 1 KB of codes with one row of x, where HBM delivers that in 45 cycles, 180 issue slots of an SM: with every slot
// used it would be bound there. But 2.4 to 2.6 of 4 a cycle are used, by 33 to 42 % of the warps that an SM takes (registers, and the codes that wait
// in shared memory): what is left is the latency of a warp's own chain (codes, conversions, products). For small weights it is the way into the
// kernel: x, a barrier, the first codes, the exchange.
//
// Figures of rows of 32 experts, 2880 -> 5760, NVFP4 and bf16, are device times of graph replays: "even" 64 rows, two an expert, every weight read (299 MB);
// "drawn" 64 rows of which 23 experts have some.
#include "fos_pair.cuh"

namespace fos {
namespace {
namespace wo {

constexpr int TILE = 128;                 // features of a CTA: one row of scale tiles
constexpr int STEP = 128;                 // values of K per iteration of a warp
constexpr int THREADS = 256;
// Iterations whose codes are on their way. (Two leave room for another CTA on an SM where x's share is large, even rows 82.1 us instead of 83.7, drawn
// ones 66.4 instead of 68.6, but where it is small they cost more: 8 x 8192 -> 28672 53.7 instead of 47.7, 1 x 8192 -> 10240 20.1 instead of 18.4.)
constexpr int DEPTH = 3;
constexpr int MAX_SPLIT = 8;
constexpr int SMS = 148;                  // (a device with fewer works through the same shares)

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
    int held, held_log2;                  // few_rows_kernel: rows of x that shared memory has room for, a power of two, 8 * NT at most
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

// Thirty-two codes of a row (a 16-byte load), eight at a time: word w -> four pairs of fp16 in their order.
template <int FMT> struct Expand32 {
    Scales<FMT> sc;
    If4Table table[2];
    __device__ __forceinline__ explicit Expand32(uint32_t raw_scales) : sc(raw_scales) {
        if constexpr (FMT == FOS_IF4) {
            table[0] = if4_table(sc.s[0], (raw_scales >> 7) & 1u);
            table[1] = if4_table(sc.s[1], (raw_scales >> 15) & 1u);
        }
    }
    __device__ __forceinline__ void word(int w, uint32_t codes, uint32_t (&o)[4]) const {
        if constexpr (FMT == FOS_IF4) {
            if4x8_to_h2(codes, table[w >> 1], o);
        } else {
            e2m1x8_to_h2(codes, o);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = mul_h2(o[j], sc.s[w >> 1]);
        }
    }
};
__device__ __forceinline__ uint32_t word_of(const uint4 &v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

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

// The rows of a group: [first, first + count) of the output. Whatever the two arrays say, nothing outside the output is touched.
struct GroupRange { int64_t first, count; };
__device__ __forceinline__ GroupRange group_range(const Params &p, int g) {
    if (!p.group_start) return {0, p.rows};
    auto clamp = [](int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); };
    GroupRange r;
    r.first = clamp(ld_int(p.group_start + g), 0, p.rows);
    r.count = clamp(ld_int(p.group_rows + g), 0, p.rows - r.first);
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

constexpr int SLOT_BYTES = THREADS * 40;  // of a step: 32 codes of two rows and their scales per thread
constexpr int FEW_ROWS = 16, FEW_ROWS_SMEM = 226 * 1024;

inline int64_t few_rows_smem_bytes(int nt, int64_t k_p, int split, int held) {
    const int64_t steps = (k_p + STEP - 1) / STEP, share = (steps + split - 1) / split;
    return TILE * 8 * nt * 4 + DEPTH * SLOT_BYTES + share * STEP * held * 2;
}

__device__ __forceinline__ void copy_16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sts_16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ uint2 lds_8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}

// Sixteen bytes where `on`, else what was there.
__device__ __forceinline__ void lds_16_if(uint32_t on, uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("{ .reg .pred p;\n"
                 "setp.ne.b32 p, %4, 0;\n"
                 "@p ld.shared.v4.b32 {%0, %1, %2, %3}, [%5]; }"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]) : "r"(on), "r"(addr) : "memory");
}

template <typename T, int NT, int FMT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 4 : 3) few_rows_kernel(const Params p) {
    constexpr int MT = 8 * NT;
    constexpr bool SCALED = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t row_max[MT];
    float *sums = reinterpret_cast<float *>(smem);                    // [split][MT][TILE / split] of what the CTAs of a cluster sent here
    uint4 *xs = reinterpret_cast<uint4 *>(smem + TILE * MT * 4 + DEPTH * SLOT_BYTES);   // [step][word][row][lane of the quad]: eight values each

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad_row = lane >> 2, t = lane & 3;
    const int split = p.split, part = static_cast<int>(blockIdx.x) % split, held = p.held;
    const int64_t tile = blockIdx.x / split;
    const int steps = static_cast<int>((p.k_p + STEP - 1) / STEP);
    const int it0 = static_cast<int>(static_cast<int64_t>(steps) * part / split);
    const int share_steps = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / split) - it0;
    const int64_t n_cb = p.k_p / (FMT == FOS_MXFP4 ? 32 : 16);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int group = blockIdx.y;
    GroupRange range{0, 0};
    // The rows of nobody behind the CTA's group, and those before all groups, reach up to the first row that a group has, whatever the order of the
    // groups in the output (and where they overlap, too); a group without rows has no place. `mine`: a group per thread.
    __shared__ uint32_t behind_of[THREADS / 32], before_of[THREADS / 32];
    auto look_for_gaps = [&](const GroupRange &mine) {
        auto gap_end = [&](int64_t from) {
            const bool has = mine.count > 0 && mine.first + mine.count > from;
            return __reduce_min_sync(0xffffffffu, static_cast<uint32_t>(!has ? p.rows : mine.first > from ? mine.first : from));
        };
        const uint32_t behind = gap_end(range.first + range.count), before = gap_end(0);
        if (lane == 0) { behind_of[warp] = behind; before_of[warp] = before; }
    };
    if (p.num_groups <= p.rows) {
        range = group_range(p, group);
    } else {
        // More groups than rows: a CTA's group is the blockIdx.y-th of those that have rows. (The launch would otherwise be one of CTAs that
        // find nothing to do: 4 rows of 32 experts take 20.1 us this way instead of 34.0, 16 rows 46.2 instead of 51.9. With as many rows as
        // groups most CTAs have work, and looking for it costs what it saves: even rows 85.1 us instead of 83.7, drawn ones 68.4 instead of 68.6.)
        __shared__ uint32_t has_rows[THREADS / 32];
        __shared__ int found;
        __shared__ int64_t found_first, found_count;
        GroupRange mine{0, 0};
        if (tid < p.num_groups) mine = group_range(p, tid);
        const uint32_t ballot = __ballot_sync(0xffffffffu, mine.count > 0);
        if (lane == 0) has_rows[warp] = ballot;
        if (tid == 0) found = -1;
        __syncthreads();
        int rank = __popc(ballot & ((1u << lane) - 1u));
        for (int w = 0; w < warp; ++w) rank += __popc(has_rows[w]);
        if (mine.count > 0 && rank == static_cast<int>(blockIdx.y)) { found = tid; found_first = mine.first; found_count = mine.count; }
        __syncthreads();
        if (found < 0 && blockIdx.y > 0) return;
        group = found < 0 ? 0 : found;
        range.first = found < 0 ? 0 : found_first;
        range.count = found < 0 ? 0 : found_count;
        look_for_gaps(mine);
    }

    // the fragment's row rho (0 .. 15) is row 4 * warp + rho % 4 + 32 * (rho / 4) of the tile: what the warp needs of the scale tiles
    // is then 64 consecutive bytes
    const int i = quad_row & 3, q = quad_row >> 2;
    const int64_t row_a = tile * TILE + 4 * warp + i + 32 * q;                            // and row_a + 64
    const uint8_t *codes_a = p.codes + group * (p.n_p * (p.k_p / 2)) + row_a * (p.k_p / 2) + t * 16 + static_cast<int64_t>(it0) * (STEP / 2);
    const int64_t codes_b = 64 * (p.k_p / 2);                                             // from row_a to row_a + 64
    // a row's scales of a step: eight bytes of which a lane takes the word that holds its two (MXFP4: four bytes, one of which is its)
    const int sf_step = p.sf_tiled ? (FMT == FOS_MXFP4 ? 512 : 1024) : (FMT == FOS_MXFP4 ? 4 : 8);
    const int64_t sf_b = p.sf_tiled ? 8 : 64 * n_cb;
    const uint8_t *sf_a = p.sf + group * (p.n_p * n_cb) + sf_offset(row_a, FMT == FOS_MXFP4 ? 0 : 4 * (t >> 1), n_cb, p.sf_tiled) +
                          static_cast<int64_t>(it0) * sf_step;
    const int sf_shift = FMT == FOS_MXFP4 ? 8 * t : 16 * (t & 1);
    // (k_p may end in the middle of a step: two of a quad's lanes have a step less)
    const int missing = static_cast<int64_t>(it0 + share_steps) * STEP > p.k_p && t >= 2 ? 1 : 0;

    // A thread's codes wait in shared memory, in slots that it alone writes and reads: DEPTH - 1 steps are on their way without a
    // register held for them, and nobody has to be told.
    const uint32_t slots = smem_u32(smem) + TILE * MT * 4, my_codes = slots + tid * 16, my_scales = slots + THREADS * 32 + tid * 8;
    const uint8_t *next_codes = codes_a, *next_sf = sf_a;
    int to_fetch = 0, halves = 0;                                                         // steps still to be fetched; less those this lane has no part in
    auto fetch = [&](int slot) {
        if (to_fetch > halves) {
            copy_16(my_codes + slot * SLOT_BYTES, next_codes);
            copy_16(my_codes + slot * SLOT_BYTES + THREADS * 16, next_codes + codes_b);
            copy_4(my_scales + slot * SLOT_BYTES, next_sf);
            copy_4(my_scales + slot * SLOT_BYTES + 4, next_sf + sf_b);
            next_codes += STEP / 2;
            next_sf += sf_step;
        } else if (to_fetch > 0) {
            sts_16(my_codes + slot * SLOT_BYTES, 0u, 0u, 0u, 0u);
            sts_16(my_codes + slot * SLOT_BYTES + THREADS * 16, 0u, 0u, 0u, 0u);
            asm volatile("st.shared.v2.b32 [%0], {%1, %1};" ::"r"(my_scales + slot * SLOT_BYTES), "r"(0u) : "memory");
        }
        --to_fetch;
        copy_commit();
    };

    const float alpha = p.amax ? __fdiv_rn(ld_float(p.amax + group), p.divisor) : 1.0f;
    const int64_t passes_from = static_cast<int64_t>(blockIdx.z) * held, passes_by = static_cast<int64_t>(gridDim.z) * held;
    for (int64_t r0 = passes_from; r0 < range.count; r0 += passes_by) {
        const int m = static_cast<int>(range.count - r0 < held ? range.count - r0 : held);
        // the thread's row of x; (quads of lanes and rows vary fastest, so that the stores below meet no bank twice)
        const int n = (tid >> 2) & (held - 1);                     // (held is a power of two)
        const uint16_t *row = n < m ? x_row(p, range.first + r0 + n) : nullptr;
        next_codes = codes_a;
        next_sf = sf_a;
        to_fetch = share_steps;
        halves = missing;
#pragma unroll
        for (int u = 0; u < DEPTH - 1; ++u) fetch(u);
        // (this CTA runs, and nothing has been read from `sums` yet that could have to come first: .release would wait for the copies on their
        // way, 1 x 4096 -> 4096 7.45 us instead of 6.68)
        if (split > 1 && r0 == passes_from) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

        // ---- the rows of x, this CTA's share of K, as fp16 in the order of the fragments: all of it on its way at once (16 bytes
        // at a time, straight to where they belong), then the rows' maxima, then each thread turns its own chunks into fp16.
        // Word w of the share: word w % 4 of a lane's sixteen bytes of codes in step w / 4.
        const int words_at_once = THREADS / 4 >> p.held_log2, w0 = (tid >> 2) >> p.held_log2, words = share_steps * 4;
        const int64_t c0 = static_cast<int64_t>(it0) * STEP + t * 32;
        __syncthreads();                                           // (the last pass's fragments and maxima have been read)
        if (SCALED && tid < MT) row_max[tid] = 0u;
        if (n < m) {
            for (int w = w0; w < words; w += words_at_once) {
                uint4 *to = xs + w * (4 * held) + n * 4 + t;
                const int64_t c = c0 + (w >> 2) * STEP + (w & 3) * 8;
                if (row != nullptr && p.vec && c + 8 <= p.k)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(row + c) : "memory");
                else
                    *to = load_x8(row, c, p.k, p.vec);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if constexpr (SCALED) {
            __syncthreads();                                       // (row_max is zero)
            uint32_t most = 0u;                                     // two 16-bit maxima of |x|'s bit patterns
            if (n < m) {
#pragma unroll 4
                for (int w = w0; w < words; w += words_at_once) {
                    const uint4 v = xs[w * (4 * held) + n * 4 + t];
                    most = __vmaxu2(__vmaxu2(most, v.x & 0x7fff7fffu), v.y & 0x7fff7fffu);
                    most = __vmaxu2(__vmaxu2(most, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu);
                }
            }
            most = max(most & 0xffffu, most >> 16);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            if (t == 0 && n < m && most) atomicMax(&row_max[n], most);
            __syncthreads();
            if (n < m) {
                const float factor = row_factor(row_exponent(row_max[n]));
#pragma unroll 4
                for (int w = w0; w < words; w += words_at_once) {
                    uint4 *at = xs + w * (4 * held) + n * 4 + t;
                    const uint4 v = *at;
                    *at = make_uint4(to_scaled_h2<T>(v.x, factor), to_scaled_h2<T>(v.y, factor), to_scaled_h2<T>(v.z, factor), to_scaled_h2<T>(v.w, factor));
                }
            }
        }
        __syncthreads();

        // ---- the product (two sets of sums: an instruction need not wait for the one before it)
        float acc[NT][4], more[NT][4];
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[a][r] = more[a][r] = 0.0f;
        // rows beyond the last: their lanes' fragments are zero and stay so
        uint32_t b[NT][4], live[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            live[a] = 8 * a + quad_row < m;
            b[a][0] = b[a][1] = b[a][2] = b[a][3] = 0u;
        }
        uint32_t frag = smem_u32(xs) + lane * 16;
        const uint32_t word_bytes = held * 64;
        int left = share_steps;
#pragma unroll 1
        while (left > 0) {
#pragma unroll
            for (int u = 0; u < DEPTH; ++u) {
                if (left == 0) break;
                --left;
                fetch((u + DEPTH - 1) % DEPTH);
                copy_wait<DEPTH - 1>();
                const uint2 raw = lds_8(my_scales + u * SLOT_BYTES);
                const uint4 va = lds_16(my_codes + u * SLOT_BYTES), vb = lds_16(my_codes + u * SLOT_BYTES + THREADS * 16);
                constexpr uint32_t MASK = FMT == FOS_MXFP4 ? 0xffu : 0xffffu;
                const Expand32<FMT> ea((raw.x >> sf_shift) & MASK), eb((raw.y >> sf_shift) & MASK);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t wa[4], wb[4];
                    ea.word(w, word_of(va, w), wa);
                    eb.word(w, word_of(vb, w), wb);
#pragma unroll
                    for (int a = 0; a < NT; ++a) {
                        lds_16_if(live[a], frag + a * 512, b[a]);
                        mma_m16n8k16(acc[a], wa[0], wb[0], wa[1], wb[1], b[a][0], b[a][1]);
                        mma_m16n8k16(more[a], wa[2], wb[2], wa[3], wb[3], b[a][2], b[a][3]);
                    }
                    frag += word_bytes;
                }
            }
        }
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[a][r] += more[a][r];

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
        if (split == 1) {
            __syncthreads();
        } else if (r0 + passes_by < range.count) {
            // this pass's sums have been read: the peers' next ones, which are behind the wait, may overwrite them
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        }
    }

    // ---- rows of no group. (Looked for this late where a CTA's group is its own number: before the product, the code alone makes a call without
    // groups take 0.1 us more.)
    if (p.group_start && blockIdx.z == 0 && (range.count > 0 || blockIdx.y == 0)) {
        if (p.num_groups <= p.rows) look_for_gaps(tid < p.num_groups ? group_range(p, tid) : GroupRange{0, 0});
        __syncthreads();
        const int share = TILE / split;
        const int64_t f0 = tile * TILE + part * share;
        auto clear = [&](int64_t from, const uint32_t (&ends)[THREADS / 32]) {
            int64_t to = p.rows;
#pragma unroll
            for (int w = 0; w < THREADS / 32; ++w) to = ends[w] < to ? ends[w] : to;
            for (int64_t e = tid; e < (to - from) * share; e += THREADS) {
                const int64_t r = from + e / share, f = f0 + e % share;
                if (f < p.n) store_out(p.out, p.out_dtype, r * p.ld_out + f, 0.0f);
            }
        };
        if (range.count > 0) clear(range.first + range.count, behind_of);
        if (blockIdx.y == 0) clear(0, before_of);
    }
}

// ---------------------------------------------------------------------------- activations laid out for the tensor cores
//
// One CTA per row of the output: its row of x (fetched by index) as fp16, multiplied by the power of two that suits it, zeros up to
// the padded length; and the factor back. A row of no group gets a row of zeros in the output instead.
struct PackParams {
    Params p;
    int64_t inner, inner_p;               // values of a row, and padded
    int clear_cols;                       // of the output
    __half *packed;                       // [rows][inner_p]
    float *factor_back;                   // [rows]
    uint32_t *counters;                   // of stream_kernel, which runs next: set to zero
    int64_t num_counters;
};

template <int CTA> __device__ __forceinline__ void zero_counters(uint32_t *counters, int64_t count) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * CTA + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * CTA) counters[i] = 0u;
}
__global__ void __launch_bounds__(THREADS) zero_counters_kernel(uint32_t *counters, int64_t count) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    zero_counters<THREADS>(counters, count);
}

// A row of up to 16384 values stays in registers between its largest value and its conversion (32 x 14336: the product 27.8 us instead of
// 30.1). Up to 8192 of them, 256 threads are enough, and more rows are on their way on an SM.
constexpr int PACK_HELD = 4;
template <typename T, int PACK_THREADS>
__global__ void __launch_bounds__(PACK_THREADS) pack_rows_kernel(const PackParams q) {
    constexpr bool SCALED = std::is_same<T, __nv_bfloat16>::value;
    __shared__ uint32_t most_of_warp[PACK_THREADS / 32];
    const Params &p = q.p;
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    zero_counters<PACK_THREADS>(q.counters, q.num_counters);
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        if (p.group_start) {
            bool mine = false;
            if (tid < p.num_groups) {
                const GroupRange g = group_range(p, tid);
                mine = r >= g.first && r < g.first + g.count;
            }
            if (!__syncthreads_or(mine)) {
                for (int f = tid; f < q.clear_cols; f += PACK_THREADS) store_out(p.out, p.out_dtype, r * p.ld_out + f, 0.0f);
                continue;
            }
        }
        const uint16_t *row = x_row(p, r);
        uint4 held[PACK_HELD];
        uint32_t most = 0u;
        auto larger = [&](const uint4 &v) {
            most = __vmaxu2(__vmaxu2(most, v.x & 0x7fff7fffu), v.y & 0x7fff7fffu);
            most = __vmaxu2(__vmaxu2(most, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu);
        };
#pragma unroll
        for (int i = 0; i < PACK_HELD; ++i) held[i] = load_x8(row, (i * PACK_THREADS + tid) * 8, q.inner, p.vec);
        constexpr int64_t BEHIND = PACK_HELD * PACK_THREADS * 8;
        float factor = 1.0f;
        if constexpr (SCALED) {
#pragma unroll
            for (int i = 0; i < PACK_HELD; ++i) larger(held[i]);
            for (int64_t c = BEHIND + tid * 8; c < q.inner; c += PACK_THREADS * 8) larger(load_x8(row, c, q.inner, p.vec));
            most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
            __syncthreads();                                        // (the last row's maxima have been read)
            if ((tid & 31) == 0) most_of_warp[tid >> 5] = most;
            __syncthreads();
            most = __reduce_max_sync(0xffffffffu, most_of_warp[tid & (PACK_THREADS / 32 - 1)]);
            factor = row_factor(row_exponent(most));
        }
        if (tid == 0) q.factor_back[r] = SCALED ? row_factor_back(row_exponent(most)) : 1.0f;
        auto store = [&](int64_t c, const uint4 &v) {
            *reinterpret_cast<uint4 *>(q.packed + r * q.inner_p + c) =
                make_uint4(to_scaled_h2<T>(v.x, factor), to_scaled_h2<T>(v.y, factor), to_scaled_h2<T>(v.z, factor), to_scaled_h2<T>(v.w, factor));
        };
#pragma unroll
        for (int i = 0; i < PACK_HELD; ++i)
            if ((i * PACK_THREADS + tid) * 8 < q.inner_p) store((i * PACK_THREADS + tid) * 8, held[i]);
        for (int64_t c = BEHIND + tid * 8; c < q.inner_p; c += PACK_THREADS * 8) store(c, load_x8(row, c, q.inner, p.vec));
    }
}

// ---------------------------------------------------------------------------- many rows: tensor cores
//
// The weight is the M operand (128 features of a tile), up to 256 rows of x the N operand. The copy engine brings a stage's rows of x
// and its codes (32 bytes of 128 rows: 32 lanes loading them from as many lines themselves kept the L1 busy for 400 cycles); four
// warps expand the codes to fp16 and write them to shared memory in the swizzled order that the MMA reads, three other teams of four the next stages';
// one thread issues tcgen05.mma kind::f16; four warps drain one accumulator while the next tile fills the other. Expanding here, not in
// a pass of its own, keeps the weight at 4 bits until it is on the SM: a 128 x 64 tile is expanded once for up to 256 columns.
// TRANSPOSED multiplies with the weight's transpose (the input's gradient: dx = dy W): the features are then the weight's columns, the
// sum runs over its rows, and the expanded tile is the same rows of 128 bytes read as an M-major operand.
// K is split over a cluster as in few_rows_kernel where there are fewer tiles than SMs.
//   warp 0   copies      warp 1   MMAs      warps 2-17   expansion      warps 18-21   epilogue
constexpr int K_STAGE = 64, W_STAGE_BYTES = 128 * 128, CODE_STAGE_BYTES = 128 * 32;
constexpr int TEAMS = 4, TEAM_WARPS = 4, EXPAND_WARPS = TEAMS * TEAM_WARPS, EPILOGUE_WARPS = 4;
constexpr int GEMM_THREADS = 64 + 32 * (EXPAND_WARPS + EPILOGUE_WARPS);
constexpr int MAX_GROUPS = 256;
static_assert(MAX_GROUPS <= THREADS, "few_rows_kernel and pack_rows_kernel look at a group per thread");

template <int NT> struct GemmCfg {
    static constexpr int X_BYTES = NT * 128, STAGE_BYTES = W_STAGE_BYTES + X_BYTES;       // the codes of all stages lie behind
    static constexpr int STAGES = NT == 256 ? 4 : NT == 32 ? 8 : 6;
    static constexpr int TMEM = 2 * NT;                                 // 64 .. 512 columns: two accumulators
    static constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + CODE_STAGE_BYTES) + 1024 + 512;
    static_assert(STAGES >= TEAMS, "a stage for every team");
    static_assert(SMEM_BYTES + 3 * MAX_GROUPS * 4 + 64 <= 232448, "shared memory");
    static_assert(STAGES * STAGE_BYTES >= NT * 512, "the partial sums reuse the ring");
};

struct GemmParams {
    Params p;
    const float *factor_back;             // one per row of x, or nullptr
    int32_t *status;
    int64_t features;                     // of the output
    int f_tiles, steps;                   // tiles of 128 (pairs: 256) features, stages of 64 of the sum
    int code_row;                         // bytes of a row that a stage's copy of codes brings
    uint32_t *counters;                   // stream_kernel: how many CTAs have left their part of a tile, per 32 features of it; and
    float *parts;                         // two parts of a tile per CTA, [S_ROWS][128] each
    int64_t max_tiles;
};

// Where the groups' row tiles lie among the tiles of a launch.
struct GroupTables { int tiles[MAX_GROUPS + 1], first[MAX_GROUPS], count[MAX_GROUPS]; };

struct Tile { int group, feature0; int64_t row0, rows_left; };

// The tiles of a launch: `f_size` features by NT rows. One group: bands of tiles that share x and weight in L2. Groups: one after
// the other, their row tiles innermost.
template <int NT> struct TileMap {
    const Params &p;
    const GroupTables &g;
    int f_tiles, f_size, row_tiles;
    int64_t num_tiles;
    __device__ __forceinline__ TileMap(const GemmParams &q, const GroupTables &tables, int feature_size)
        : p(q.p), g(tables), f_tiles(q.f_tiles), f_size(feature_size) {
        row_tiles = p.group_start ? g.tiles[p.num_groups] : static_cast<int>((p.rows + NT - 1) / NT);
        num_tiles = static_cast<int64_t>(row_tiles) * f_tiles;
    }
    __device__ __forceinline__ Tile at(int64_t t) const {
        Tile r;
        if (!p.group_start) {
            int64_t fb, rb;
            tile_coords(t, f_tiles, row_tiles, fb, rb);
            r.group = 0;
            r.feature0 = static_cast<int>(fb) * f_size;
            r.row0 = rb * NT;
            r.rows_left = p.rows - r.row0;
        } else {
            int lo = 0, hi = p.num_groups - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (static_cast<int64_t>(g.tiles[mid]) * f_tiles <= t) lo = mid;
                else hi = mid - 1;
            }
            const int mine = g.tiles[lo + 1] - g.tiles[lo];
            const int64_t local = t - static_cast<int64_t>(g.tiles[lo]) * f_tiles;
            const int fb = static_cast<int>(local / mine), rb = static_cast<int>(local - static_cast<int64_t>(fb) * mine);
            r.group = lo;
            r.feature0 = fb * f_size;
            r.row0 = g.first[lo] + static_cast<int64_t>(rb) * NT;
            r.rows_left = g.count[lo] - rb * NT;
        }
        return r;
    }
};
// Fills the tables; every thread of the CTA, which synchronises before they are read.
template <int NT> __device__ __forceinline__ void fill_group_tables(const Params &p, GroupTables &g) {
    for (int i = threadIdx.x; i < p.num_groups; i += blockDim.x) {
        const GroupRange r = group_range(p, i);
        g.first[i] = static_cast<int>(r.first);
        g.count[i] = static_cast<int>(r.count);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int sum = 0;
        for (int i = 0; i < p.num_groups; ++i) {
            g.tiles[i] = sum;
            sum += (g.count[i] + NT - 1) / NT;
        }
        g.tiles[p.num_groups] = sum;
    }
}

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }\n"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }\n"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// One accumulator tile to the output: a lane's feature (`in_tile` of the tile), one row of x per column, so a warp stores 64 bytes of a
// row at a time. The rows' factors come 32 at a time, one per lane. `drained()` is called when the accumulator has been read.
template <typename OUT> __device__ __forceinline__ OUT round_to(float v) {
    if constexpr (std::is_same<OUT, __half>::value) return __float2half_rn(v);
    else if constexpr (std::is_same<OUT, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
    else return v;
}
template <typename OUT, typename Drained>
__device__ __forceinline__ void store_columns(const GemmParams &q, OUT *to, int64_t row0, int columns, bool f_ok, float alpha, float bias,
                                              uint32_t t_acc, Drained drained) {
    const int64_t ld = q.p.ld_out;
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int c = 0; c < columns; c += 32) {
        float factor = 1.0f;                                            // (a power of two, not to be multiplied into alpha: it may be tiny)
        if (q.factor_back && c + lane < columns) factor = ld_float(q.factor_back + row0 + c + lane);
        uint32_t v[32];
        tc_load_32cols_sync(t_acc + c, v);
        if (c + 32 >= columns) drained();
        if (c + 32 <= columns) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const OUT r = round_to<OUT>(__fmaf_rn(__uint_as_float(v[i]) * __shfl_sync(0xffffffffu, factor, i), alpha, bias));
                if (f_ok) to[i * ld] = r;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const OUT r = round_to<OUT>(__fmaf_rn(__uint_as_float(v[i]) * __shfl_sync(0xffffffffu, factor, i), alpha, bias));
                if (f_ok && c + i < columns) to[i * ld] = r;
            }
        }
        to += 32 * ld;
    }
}
template <int NT, typename Drained>
__device__ __forceinline__ void store_tile(const GemmParams &q, const Tile &at, int in_tile, uint32_t t_acc, Drained drained) {
    const Params &p = q.p;
    const int64_t feature = at.feature0 + in_tile;
    const bool f_ok = feature < q.features;
    const float alpha = p.amax ? __fdiv_rn(ld_float(p.amax + at.group), p.divisor) : 1.0f;
    const float bias = p.bias && f_ok ? load_bias(p.bias, p.out_dtype, feature) : 0.0f;
    const int columns = at.rows_left < NT ? static_cast<int>(at.rows_left) : NT;
    const int64_t first = at.row0 * p.ld_out + feature;
    if (p.out_dtype == FOS_BF16) store_columns(q, static_cast<__nv_bfloat16 *>(p.out) + first, at.row0, columns, f_ok, alpha, bias, t_acc, drained);
    else if (p.out_dtype == FOS_FP16) store_columns(q, static_cast<__half *>(p.out) + first, at.row0, columns, f_ok, alpha, bias, t_acc, drained);
    else store_columns(q, static_cast<float *>(p.out) + first, at.row0, columns, f_ok, alpha, bias, t_acc, drained);
}

// The copies of a stage: 128 rows by 32 bytes of codes, or 64 rows by 64 bytes of the transposed weight, and the rows of x.
template <bool TRANSPOSED>
__device__ __forceinline__ void copy_stage(const CUtensorMap *map_x, const CUtensorMap *map_codes, const GemmParams &q, const Tile &at, int64_t feature,
                                           int row0, int ks, uint32_t x_at, uint32_t codes_at, int x_bytes, uint32_t bar) {
    // (what lies outside is zero-filled and still counted)
    mbar_expect_tx(bar, x_bytes + (TRANSPOSED ? K_STAGE : TILE) * q.code_row);
    const int weight0 = static_cast<int>(at.group * q.p.n_p);
    if constexpr (TRANSPOSED) tma_load_2d(codes_at, map_codes, static_cast<int>(feature / 2), weight0 + ks * K_STAGE, bar);
    else tma_load_2d(codes_at, map_codes, ks * (K_STAGE / 2), weight0 + static_cast<int>(feature), bar);
    tma_load_2d(x_at, map_x, ks * 128, row0, bar);
}

// The expanding warps' work: a thread turns 64 codes of a row into 128 bytes of fp16 per stage, a team of four warps per stage and the
// other three teams on the next ones: what a stage costs a warp whatever its size (the wait, the fence, the arrival) comes a quarter as often.
// `wait(s, turn, parity)` returns when the stage's copies are complete (false: give up), `arrive(s)` (one lane of a warp) says that the
// warp's part is expanded. A barrier tells a phase from the next one only: where the teams take turns on a stage (six stages, four
// teams), a team that is early could take the copies before the last ones for its own. So the uses of a stage have two barriers in turn.
// (Waiting for the MMAs on the last use first cost 3 %: 4096 x 4096 -> 4096 fp16 129.9 us, this way 126.6.)
// The scales come straight from global memory, two stages ahead. feature_offset: of this CTA's 128 features.
template <int NT, bool TRANSPOSED, int FMT, int STAGES, int STAGE_BYTES, typename Wait, typename Arrive>
__device__ __forceinline__ void expand_stages(const GemmParams &q, const TileMap<NT> &map, int feature_offset, int64_t first_tile, int by_tiles,
                                              int ks0, int ks1, uint32_t smem_base, int thread, Wait wait, Arrive arrive) {
    constexpr int AHEAD = 2;
    const Params &p = q.p;
    const int e = thread & 127, team = thread >> 7, lane = thread & 31;
    const int r = TRANSPOSED ? e >> 1 : e, piece = TRANSPOSED ? e & 1 : 0;
    const int64_t n_cb = p.k_p / (FMT == FOS_MXFP4 ? 32 : 16);
    const uint32_t to_row = smem_base + piece * 8192 + r * 128 + (r & 7) * 16, from_row = smem_base + STAGES * STAGE_BYTES + r * q.code_row + (q.code_row > 32 ? piece * 32 : 0);
    const int per_tile = ks1 - ks0;
    const int64_t my_tiles = map.num_tiles > first_tile ? (map.num_tiles - first_tile + by_tiles - 1) / by_tiles : 0;
    int64_t left = (my_tiles * per_tile + TEAMS - 1 - team) / TEAMS, to_fetch = left;     // stages of this team
    // (the teams are an even number: within a tile a team's stages are all even or all odd, and the scales advance by a constant)
    constexpr int PER_ROW = FMT == FOS_MXFP4 ? 2 : 4;                   // scales of 64 values
    const int64_t sf_two = TRANSPOSED ? 128 * n_cb : (p.sf_tiled ? PER_ROW * 256 : PER_ROW * 2), sf_step = TEAMS / 2 * sf_two;
    const int64_t sf_odd = TRANSPOSED ? (p.sf_tiled ? 8 : 64 * n_cb) : (p.sf_tiled && FMT != FOS_MXFP4 ? 512 : PER_ROW);
    int64_t f_tile = first_tile - by_tiles;
    int f_ks = ks1 + team;
    const uint8_t *f_sf = nullptr;                                      // nullptr: outside the weight, zeros
    uint32_t scale[AHEAD];
    auto fetch = [&](int u) {
        if (to_fetch == 0) return;
        --to_fetch;
        if (f_ks >= ks1) {
            do {
                f_ks -= per_tile;
                f_tile += by_tiles;
            } while (f_ks >= ks1);
            const Tile at = map.at(f_tile);
            const int64_t feature = at.feature0 + feature_offset;
            const int64_t row = TRANSPOSED ? r : feature + r, col = TRANSPOSED ? feature + piece * 64 : 0;
            f_sf = p.sf + at.group * (p.n_p * n_cb) + sf_offset(row, col / (FMT == FOS_MXFP4 ? 32 : 16), n_cb, p.sf_tiled) +
                   (f_ks >> 1) * sf_two + ((f_ks & 1) ? sf_odd : 0);
            // (a tile may reach beyond the weight: the second 128 rows of a pair's, or the last 64 of 128 columns)
            if (TRANSPOSED ? col >= p.k_p : feature >= p.n_p) f_sf = nullptr;
        }
        scale[u] = 0u;
        if (f_sf != nullptr) {
            scale[u] = FMT == FOS_MXFP4 ? ld_b16(f_sf) : ld_b32(f_sf);
            f_sf += sf_step;
        }
        f_ks += TEAMS;
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(u);
    int s = team;
    uint32_t turn = 0, ph = 0;
    bool ok = true;
    while (left > 0 && ok) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (left == 0) break;
            --left;
            ok = wait(s, turn, ph);
            if (!ok) break;
            const uint32_t from = from_row + s * CODE_STAGE_BYTES, to = to_row + s * STAGE_BYTES;      // (rows are 128 bytes and aligned)
            const uint4 code[2] = {lds_16(from), lds_16(from + 16)};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const Expand32<FMT> ex(FMT == FOS_MXFP4 ? (scale[u] >> (8 * half)) & 0xffu : (scale[u] >> (16 * half)) & 0xffffu);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t h[4];
                    ex.word(w, word_of(code[half], w), h);
                    sts_16(to ^ ((4 * half + w) * 16), h[0], h[1], h[2], h[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive(s);
            fetch(u);
            s += TEAMS;
            if (s >= STAGES) {
                s -= STAGES;
                ph ^= turn;
                turn ^= 1u;
            }
        }
    }
}

template <int NT, bool TRANSPOSED, int FMT>
__global__ void __launch_bounds__(GEMM_THREADS, 1) gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes,
                                                               const GemmParams q) {
    using C = GemmCfg<NT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ GroupTables groups;
    const Params &p = q.p;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_gen + C::STAGES * (C::STAGE_BYTES + CODE_STAGE_BYTES));
    // a stage's way: copied (loaded), expanded (ready), multiplied (empty)
    const uint32_t loaded = smem_u32(bars), ready = loaded + 16 * C::STAGES, empty = ready + 8 * C::STAGES;      // loaded: two in turn
    const uint32_t acc_full = empty + 8 * C::STAGES, acc_empty = acc_full + 16, drain = acc_empty + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 4 * C::STAGES + 5);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(loaded + 8 * s, 1);
            mbar_init(loaded + 8 * (s + C::STAGES), 1);
            mbar_init(ready + 8 * s, TEAM_WARPS);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full + 8 * a, 1);
            mbar_init(acc_empty + 8 * a, EPILOGUE_WARPS);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // (the codes and whatever the caller wrote before the rows were packed, too: nothing is read before this)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (p.group_start) fill_group_tables<NT>(p, groups);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int split = p.split, part = static_cast<int>(blockIdx.x) % split;
    const int first_tile = static_cast<int>(blockIdx.x) / split, by_tiles = static_cast<int>(gridDim.x) / split;
    const TileMap<NT> map(q, groups, TILE);
    const int64_t num_tiles = map.num_tiles;
    const int ks0 = static_cast<int>(static_cast<int64_t>(q.steps) * part / split), ks1 = static_cast<int>(static_cast<int64_t>(q.steps) * (part + 1) / split);

    if (warp == 0) {
        // ------------------------------------------------------------------ copies
        const bool issue = elect_one();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int64_t t = first_tile; t < num_tiles && ok; t += by_tiles) {
            const Tile at = map.at(t);
            for (int ks = ks0; ks < ks1; ++ks) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ph ^ 1u, abort_flag, q.status, 1));
                if (!ok) break;
                if (issue)
                    copy_stage<TRANSPOSED>(&map_x, &map_codes, q, at, at.feature0, static_cast<int>(at.row0), ks,
                                           smem_base + s * C::STAGE_BYTES + W_STAGE_BYTES,
                                           smem_base + C::STAGES * C::STAGE_BYTES + s * CODE_STAGE_BYTES, C::X_BYTES, loaded + 8 * (s + ph * C::STAGES));
                __syncwarp();
                if (++s == C::STAGES) { s = 0; ph ^= 1u; }
            }
        }
        if (!ok) {
            const unsigned long long t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMAs
        const bool issue = elect_one();
        // fp32 accumulators, both operands fp16, the weight M-major where it is transposed; N >> 3 in [17, 23), M >> 4 in [24, 29)
        constexpr uint32_t idesc = (1u << 4) | (TRANSPOSED ? 1u << 15 : 0u) | (static_cast<uint32_t>(NT >> 3) << 17) | (8u << 24);
        int s = 0;
        uint32_t ph = 0, tile_i = 0;
        bool ok = true;
        for (int64_t t = first_tile; t < num_tiles && ok; t += by_tiles, ++tile_i) {
            const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
            ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + 8 * acc, acc_ph ^ 1u, abort_flag, q.status, 3));
            if (!ok) break;
            tc_fence_after();
            for (int ks = ks0; ks < ks1; ++ks) {
                ok = __all_sync(0xffffffffu, mbar_wait(ready + 8 * s, ph, abort_flag, q.status, 2));
                if (!ok) break;
                tc_fence_after();
                const uint32_t stage = smem_base + s * C::STAGE_BYTES;
                // K-major: rows of 128 bytes, groups of 8 rows 1024 bytes apart. M-major: 64 features to a row of 128 bytes, groups of 8
                // rows of the sum 1024 bytes apart, the second 64 features 8 KB behind
                const uint64_t w_desc = smem_desc(stage, TRANSPOSED ? 8192 : 16, 1024, 2), x_desc = smem_desc(stage + W_STAGE_BYTES, 16, 1024, 2);
                if (issue) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_f16(tmem_base + acc * NT, w_desc + (TRANSPOSED ? 128 : 2) * j, x_desc + 2 * j, idesc, (ks > ks0 || j > 0) ? 1u : 0u);
                    tc_commit(empty + 8 * s);
                }
                __syncwarp();
                if (++s == C::STAGES) { s = 0; ph ^= 1u; }
            }
            if (ok && issue) tc_commit(acc_full + 8 * acc);
        }
        if (!ok) {
            // giving up: the MMAs already issued must have finished before tensor memory is released
            if (issue) tc_commit(drain);
            __syncwarp();
            const long long t0 = clock64();
            while (!mbar_try_wait(drain, 0) && clock64() - t0 < 20000000ll) {}   // about 10 ms
        }
    } else if (warp < 2 + EXPAND_WARPS) {
        // ------------------------------------------------------------------ expansion
        expand_stages<NT, TRANSPOSED, FMT, C::STAGES, C::STAGE_BYTES>(
            q, map, 0, first_tile, by_tiles, ks0, ks1, smem_base, threadIdx.x - 64,
            [&](int s, uint32_t turn, uint32_t parity) {
                return __all_sync(0xffffffffu, mbar_wait(loaded + 8 * (s + turn * C::STAGES), parity, abort_flag, q.status, 6));
            },
            [&](int s) { mbar_arrive(ready + 8 * s); });
    }

    // ---------------------------------------------------------------------- epilogue
    const int quad = warp & 3, in_tile = quad * 32 + lane;
    const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    auto put = [&](const Tile &at, float alpha, float bias, int64_t row, float v) {
        if (q.factor_back) v *= ld_float(q.factor_back + row);
        v *= alpha;
        store_out(p.out, p.out_dtype, row * p.ld_out + at.feature0 + in_tile, p.bias ? v + bias : v);
    };
    if (split == 1 && warp >= 2 + EXPAND_WARPS) {
        uint32_t tile_i = 0;
        bool ok = true;
        for (int64_t t = first_tile; t < num_tiles && ok; t += by_tiles, ++tile_i) {
            const Tile at = map.at(t);
            const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * acc, acc_ph, abort_flag, q.status, 4));
            if (!ok) break;
            tc_fence_after();
            store_tile<NT>(q, at, in_tile, t_acc + acc * NT, [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty + 8 * acc);
            });
        }
    }
    if (split > 1) {
        // one tile per cluster: its CTAs exchange their sums, each adding up a share of the rows in the order of K
        const Tile at = map.at(first_tile);
        const int mine = NT / split;
        bool ok = true;
        __syncwarp();
        if (warp >= 2 + EXPAND_WARPS) {
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, abort_flag, q.status, 4));
            tc_fence_after();
        }
        cluster_sync_all();       // every CTA's MMAs are done: its ring may take sums
        if (warp >= 2 + EXPAND_WARPS && ok) {
#pragma unroll 1
            for (int c = 0; c < NT; c += 32) {
                uint32_t v[32];
                tc_load_32cols_sync(t_acc + c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int col = c + i, owner = col / mine;
                    st_cluster_f32(map_to_cta(smem_base + ((part * mine + col - owner * mine) * TILE + in_tile) * 4, owner), __uint_as_float(v[i]));
                }
            }
        }
        cluster_sync_all();
        if (warp >= 2 + EXPAND_WARPS && ok && at.feature0 + in_tile < q.features) {
            const float alpha = p.amax ? __fdiv_rn(ld_float(p.amax + at.group), p.divisor) : 1.0f;
            const float bias = p.bias ? load_bias(p.bias, p.out_dtype, at.feature0 + in_tile) : 0.0f;
            for (int c = 0; c < mine; ++c) {
                if (part * mine + c >= at.rows_left) break;
                float sum = lds_f32(smem_base + (c * TILE + in_tile) * 4);
                for (int k = 1; k < split; ++k) sum += lds_f32(smem_base + ((k * mine + c) * TILE + in_tile) * 4);
                put(at, alpha, bias, at.row0 + part * mine + c, sum);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM) : "memory");
    }
}

// ---------------------------------------------------------------------------- the weight's bytes first: tensor cores, weight in tensor memory
//
// For rows so few that the expansion counts, not the MMAs. In gemm_kernel an expanded stage goes through shared memory, 16 KB in and 16 KB
// out to the tensor cores for 4 KB of codes: at 128 bytes a cycle that alone takes 256 cycles of the 400 that a stage takes. Here
// a thread expands the 128 codes of its row into registers and stores them to tensor memory, from where the MMA takes its A operand (a
// lane is a feature, a 32-bit column two values of K): shared memory sees the codes and x only.
// The launch's stages, tile after tile, are dealt out evenly (10240 features are 80 tiles, which would keep 80 of 148 SMs busy):
// a CTA's share may begin and end within a tile. Such parts go to memory, and whoever leaves the last of a tile's (for its 32
// features) adds them up in the order of K: nobody waits for another CTA, and the sums do not depend on who is last.
// The kernel in front is pack_rows_kernel or zero_counters_kernel, which let this one start only when whatever ran before them is
// complete: the weight's way into shared memory begins at once, and only x, the factors and the counters wait.
// 16 x 8192 -> 28672 54 us (few_rows_kernel 76), 64 rows 62 (gemm_kernel 89), 512 x 8192 -> 10240 95 (131). A stage takes 700 cycles whatever of it is left
// out (MMAs but one, the conversions, the copies of x, HBM), so none of these bounds it. Nor does the way into tensor memory: stores alone go at 750 (four
// warps that wait for each) to 1000 bytes a cycle, 32 KB in 33 to 44 cycles. What does was not isolated. A team has one slot, so its chain, from the MMAs on the
// slot's last use over wait, expansion, store and arrival to the next MMAs, does not overlap itself: four teams, 2800 cycles each.
//   warp 0   copies      warp 1   MMAs      warps 2-17   expansion, four teams of four      warps 18-21   epilogue
constexpr int S_ROWS = 128, S_STAGE = 128, S_BOX = 64;                   // rows of a tile; values of K of a stage; rows of a copy
constexpr int S_X_BYTES = 2 * S_ROWS * 128, S_CODE_BYTES = TILE * (S_STAGE / 2), S_STAGE_BYTES = S_X_BYTES + S_CODE_BYTES, S_STAGES = 5;
constexpr int S_SLOTS = TEAMS, S_SLOT_COLS = S_STAGE / 2;               // of tensor memory, one for each team's stage
constexpr int S_BARRIERS = 2 * S_STAGES + S_SLOTS + 5, S_SMEM_BYTES = S_STAGES * S_STAGE_BYTES + 1024 + 512;
static_assert(S_STAGES >= TEAMS, "see expand_to_tmem");
static_assert(2 * S_ROWS + S_SLOTS * S_SLOT_COLS <= TMEM_COLS, "tensor memory");
static_assert(S_BARRIERS * 8 + 8 <= 512 && S_SMEM_BYTES + sizeof(GroupTables) + 64 <= 232448, "shared memory");

// The eight MMAs of a stage: 128 values of K, 8 columns of tensor memory and 32 bytes of x's rows (of two halves of 64 values) each.
__device__ __forceinline__ void mma_stage_from_tmem(uint32_t d_tmem, uint32_t a_tmem, uint32_t x_lo, uint32_t x_hi, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        asm volatile(
            "{ .reg .pred p;\n"
            ".reg .b64 x;\n"
            "setp.ne.b32 p, %5, 0;\n"
            "mov.b64 x, {%2, %3};\n"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], x, %4, p; }\n"
            ::"r"(d_tmem), "r"(a_tmem + 8 * j), "r"(x_lo + (j / 4) * (S_ROWS * 128 / 16) + 2 * (j % 4)), "r"(x_hi), "r"(idesc), "r"(j == 0 ? accumulate : 1u) : "memory");
    }
}

// The CTAs' shares of `total` stages: CTA c has [first(c), first(c + 1)).
struct Shares {
    int64_t total;
    int ctas;
    __device__ __forceinline__ int64_t first(int c) const { return total * c / ctas; }
    __device__ __forceinline__ int owner(int64_t u) const { return static_cast<int>(((u + 1) * ctas + total - 1) / total) - 1; }
};

// Where a walk over a share stands: a tile, and the stage within it.
__device__ __forceinline__ int rows_of(const Tile &at) { return at.rows_left < S_ROWS ? static_cast<int>(at.rows_left) : S_ROWS; }

struct Walk {
    const TileMap<S_ROWS> &map;
    int steps, ks;
    int64_t tile;
    Tile at;
    __device__ __forceinline__ Walk(const TileMap<S_ROWS> &m, int steps_, int64_t u) : map(m), steps(steps_), ks(static_cast<int>(u % steps_)), tile(u / steps_) {}
    __device__ __forceinline__ void look() { at = map.at(tile); }
    __device__ __forceinline__ void advance(int by) {
        ks += by;
        if (ks < steps) return;
        do { ks -= steps; ++tile; } while (ks >= steps);
        if (tile < map.num_tiles) look();
    }
};

template <int FMT>
__device__ __forceinline__ void expand_to_tmem(const GemmParams &q, const TileMap<S_ROWS> &map, int64_t u0, int64_t u1, uint32_t smem_base, uint32_t slots,
                                               uint32_t loaded, uint32_t ready, uint32_t empty, volatile int *abort_flag) {
    constexpr int AHEAD = 3;
    const Params &p = q.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = (warp - 2) / TEAM_WARPS, r = (warp & 3) * 32 + lane;
    const int64_t n_cb = p.k_p / (FMT == FOS_MXFP4 ? 32 : 16);
    const int sf_step = p.sf_tiled ? (FMT == FOS_MXFP4 ? 512 : 1024) : (FMT == FOS_MXFP4 ? 4 : 8), sf_second = p.sf_tiled ? 512 : 4;
    const uint32_t slot = slots + (static_cast<uint32_t>((warp & 3) * 32) << 16) + team * S_SLOT_COLS;
    const uint32_t codes_at = smem_base + S_X_BYTES + r * 64, turn = (r >> 1) & 3;          // (rows of 64 bytes, swizzled)
    int64_t left = (u1 - u0 + TEAMS - 1 - team) / TEAMS, to_fetch = left;
    Walk walk(map, q.steps, u0 + team);
    if (left > 0) walk.look();
    const uint8_t *f_sf = nullptr;
    int64_t f_tile = -1;
    uint32_t scale[AHEAD][2];
    auto fetch = [&](int u) {
        if (to_fetch == 0) return;
        --to_fetch;
        if (walk.tile != f_tile) {
            f_tile = walk.tile;
            f_sf = p.sf + walk.at.group * (p.n_p * n_cb) + sf_offset(walk.at.feature0 + r, 0, n_cb, p.sf_tiled);
        }
        const uint8_t *sf = f_sf + static_cast<int64_t>(walk.ks) * sf_step;
        scale[u][0] = ld_b32(sf);
        if constexpr (FMT != FOS_MXFP4) scale[u][1] = static_cast<int64_t>(walk.ks) * S_STAGE + 64 < p.k_p ? ld_b32(sf + sf_second) : 0u;
        walk.advance(TEAMS);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(u);
    int s = team, before = 0;
    uint32_t ph = 0, before_ph = 0;
    bool again = false, ok = true;
    while (left > 0 && ok) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (left == 0) break;
            --left;
            // First the MMAs that last read the team's slot. They come behind those on the stage's last copies, which the wait for the next
            // ones must not take for its own where the teams take turns on a stage (see expand_stages). (That stage's copies were
            // seen, so the MMAs one round before it are complete: no barrier is more than a phase away from the one waited for.)
            if (again) ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * before, before_ph, abort_flag, q.status, 8));
            ok = ok && __all_sync(0xffffffffu, mbar_wait(loaded + 8 * s, ph, abort_flag, q.status, 6));
            if (!ok) break;
            tc_fence_after();
            const uint32_t from = codes_at + s * S_STAGE_BYTES;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint4 code[2] = {lds_16(from + ((2 * half) ^ turn) * 16), lds_16(from + ((2 * half + 1) ^ turn) * 16)};
                uint32_t h[32];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Expand32<FMT> ex(FMT == FOS_MXFP4 ? (scale[u][0] >> (16 * half + 8 * c)) & 0xffu : (scale[u][half] >> (16 * c)) & 0xffffu);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t o[4];
                        ex.word(w, word_of(code[c], w), o);
#pragma unroll
                        for (int j = 0; j < 4; ++j) h[16 * c + 4 * w + j] = o[j];
                    }
                }
                tc_store_cols<32>(slot + half * 32, h);
            }
            tc_wait_store();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ready + 8 * team);
            fetch(u);
            again = true;
            before = s;
            before_ph = ph;
            s += TEAMS;
            if (s >= S_STAGES) { s -= S_STAGES; ph ^= 1u; }
        }
    }
}

template <typename OUT>
__device__ __forceinline__ void store_joined(const GemmParams &q, OUT *to, const Tile &at, int in_tile, int columns, bool f_ok, float alpha, float bias,
                                             const Shares &shares, int64_t tile) {
    const int64_t begin = tile * q.steps;
    const int first = shares.owner(begin), last = shares.owner(begin + q.steps - 1), lane = threadIdx.x & 31;
    // (a CTA whose share begins in this tile left it as its first part)
    auto part = [&](int c) { return q.parts + ((2 * c + (shares.first(c) < begin ? 1 : 0)) * static_cast<int64_t>(S_ROWS) * TILE + in_tile); };
#pragma unroll 1
    for (int c0 = 0; c0 < columns; c0 += 16) {
        // (two parts' loads on their way at once)
        float sum[16], next[16];
        auto load = [&](int c, float (&v)[16]) {
            const float *from = part(c) + c0 * TILE;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = c <= last && c0 + i < columns ? __ldcg(from + i * TILE) : 0.0f;
        };
        load(first, sum);
        load(first + 1, next);
        for (int c = first + 1; c <= last; ++c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[i] += next[i];
            load(c + 1, next);
        }
        float factor = 1.0f;
        if (q.factor_back && c0 + (lane & 15) < columns) factor = ld_float(q.factor_back + at.row0 + c0 + (lane & 15));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const OUT r = round_to<OUT>(__fmaf_rn(sum[i] * __shfl_sync(0xffffffffu, factor, i), alpha, bias));
            if (c0 + i < columns && f_ok) to[(c0 + i) * q.p.ld_out] = r;
        }
    }
}

template <int FMT>
__global__ void __launch_bounds__(GEMM_THREADS, 1) stream_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes,
                                                                 const GemmParams q) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ GroupTables groups;
    const Params &p = q.p;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_raw + (smem_base - smem_u32(smem_raw)) + S_STAGES * S_STAGE_BYTES);
    const uint32_t loaded = smem_u32(bars), empty = loaded + 8 * S_STAGES, ready = empty + 8 * S_STAGES;
    const uint32_t acc_full = ready + 8 * S_SLOTS, acc_empty = acc_full + 16, drain = acc_empty + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + S_BARRIERS);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S_STAGES; ++s) {
            mbar_init(loaded + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < S_SLOTS; ++s) mbar_init(ready + 8 * s, TEAM_WARPS);
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full + 8 * a, 1);
            mbar_init(acc_empty + 8 * a, EPILOGUE_WARPS);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (p.group_start) fill_group_tables<S_ROWS>(p, groups);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot, slots = tmem_base + 2 * S_ROWS;

    TileMap<S_ROWS> map(q, groups, TILE);
    if (map.num_tiles > q.max_tiles) map.num_tiles = q.max_tiles;          // (groups that overlap: there are counters for so many only)
    const int64_t stages = map.num_tiles * q.steps;
    const Shares shares{stages, static_cast<int>(stages < gridDim.x ? stages : gridDim.x)};      // (nobody's share is empty)
    const bool mine = static_cast<int>(blockIdx.x) < shares.ctas;
    const int64_t u0 = mine ? shares.first(blockIdx.x) : 0, u1 = mine ? shares.first(blockIdx.x + 1) : 0;

    if (warp == 0) {
        // ------------------------------------------------------------------ copies
        const bool issue = elect_one();
        auto boxes = [](const Walk &w) { return static_cast<int>(rows_of(w.at) + S_BOX - 1) / S_BOX; };
        auto codes = [&](const Walk &w, int s) {
            if (!issue) return;
            // (what lies outside is zero-filled and still counted)
            mbar_expect_tx(loaded + 8 * s, S_CODE_BYTES + 2 * boxes(w) * S_BOX * 128);
            tma_load_2d(smem_base + s * S_STAGE_BYTES + S_X_BYTES, &map_codes, w.ks * (S_STAGE / 2),
                        static_cast<int>(w.at.group * p.n_p) + w.at.feature0, loaded + 8 * s);
        };
        auto rows = [&](const Walk &w, int s) {
            if (!issue) return;
            const uint32_t to = smem_base + s * S_STAGE_BYTES;
            for (int b = boxes(w) - 1; b >= 0; --b) {
                const int row = static_cast<int>(w.at.row0) + b * S_BOX;
                tma_load_2d(to + b * S_BOX * 128, &map_x, w.ks * 256, row, loaded + 8 * s);
                tma_load_2d(to + (S_ROWS + b * S_BOX) * 128, &map_x, w.ks * 256 + 128, row, loaded + 8 * s);
            }
        };
        const int ahead = static_cast<int>(u1 - u0 < S_STAGES ? u1 - u0 : S_STAGES);
        Walk walk(map, q.steps, u0);
        if (ahead > 0) walk.look();
        for (int s = 0; s < ahead; ++s, walk.advance(1)) codes(walk, s);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        Walk behind(map, q.steps, u0);
        if (ahead > 0) behind.look();
        for (int s = 0; s < ahead; ++s, behind.advance(1)) rows(behind, s);
        __syncwarp();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int64_t u = u0 + S_STAGES; u < u1; ++u, walk.advance(1)) {
            ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ph, abort_flag, q.status, 1));
            if (!ok) break;
            codes(walk, s);
            rows(walk, s);
            __syncwarp();
            if (++s == S_STAGES) { s = 0; ph ^= 1u; }
        }
        if (!ok) {
            const unsigned long long t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMAs
        // (elected where it is asked for: the compiler then knows that the branch is the warp's and keeps the operands in uniform registers)
        constexpr uint32_t IDESC = (1u << 4) | (8u << 24);
        const uint64_t x_desc = smem_desc(smem_base, 16, 1024, 2);
        const uint32_t x_lo = static_cast<uint32_t>(x_desc), x_hi = static_cast<uint32_t>(x_desc >> 32);
        int s = 0, slot = 0;
        uint32_t slot_ph = 0, tile_i = 0;
        bool ok = true;
        for (int64_t u = u0; u < u1 && ok; ++tile_i) {
            const int64_t tile_end = (u / q.steps + 1) * q.steps, end = tile_end < u1 ? tile_end : u1;
            const uint32_t acc = tile_i % 2, acc_ph = (tile_i / 2) & 1u;
            const uint32_t idesc = IDESC | (static_cast<uint32_t>(rows_of(map.at(u / q.steps)) + 15) / 16 * 2 << 17);   // N: the tile's rows, rounded up to 16
            ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + 8 * acc, acc_ph ^ 1u, abort_flag, q.status, 3));
            if (!ok) break;
            tc_fence_after();
            for (bool first = true; u < end; ++u, first = false) {
                ok = __all_sync(0xffffffffu, mbar_wait(ready + 8 * slot, slot_ph, abort_flag, q.status, 2));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    mma_stage_from_tmem(tmem_base + acc * S_ROWS, slots + slot * S_SLOT_COLS, x_lo + s * (S_STAGE_BYTES / 16), x_hi, idesc, first ? 0u : 1u);
                    tc_commit(empty + 8 * s);
                }
                __syncwarp();
                if (++s == S_STAGES) s = 0;
                if (++slot == S_SLOTS) { slot = 0; slot_ph ^= 1u; }
            }
            if (ok && elect_one()) tc_commit(acc_full + 8 * acc);
        }
        if (!ok) {
            // giving up: the MMAs already issued must have finished before tensor memory is released
            if (elect_one()) tc_commit(drain);
            __syncwarp();
            const long long t0 = clock64();
            while (!mbar_try_wait(drain, 0) && clock64() - t0 < 20000000ll) {}   // about 10 ms
        }
    } else if (warp < 2 + EXPAND_WARPS) {
        expand_to_tmem<FMT>(q, map, u0, u1, smem_base, slots, loaded, ready, empty, abort_flag);
    } else {
        // ------------------------------------------------------------------ epilogue
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int quad = warp & 3, in_tile = quad * 32 + lane;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
        uint32_t tile_i = 0;
        bool ok = true;
        for (int64_t u = u0; u < u1; ++tile_i) {
            const int64_t tile = u / q.steps, begin = tile * q.steps, end = begin + q.steps < u1 ? begin + q.steps : u1;
            const Tile at = map.at(tile);
            const uint32_t acc = tile_i % 2, acc_ph = (tile_i / 2) & 1u, t_acc = t_lane + acc * S_ROWS;
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * acc, acc_ph, abort_flag, q.status, 4));
            if (!ok) break;
            tc_fence_after();
            auto drained = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty + 8 * acc);
            };
            if (u == begin && end == begin + q.steps) {
                store_tile<S_ROWS>(q, at, in_tile, t_acc, drained);
            } else {
                const int columns = rows_of(at);
                float *to = q.parts + ((2 * static_cast<int64_t>(blockIdx.x) + (u == u0 ? 0 : 1)) * S_ROWS * TILE + in_tile);
#pragma unroll 1
                for (int c = 0; c < columns; c += 32) {
                    uint32_t v[32];
                    tc_load_32cols_sync(t_acc + c, v);
                    if (c + 32 >= columns) drained();
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + i < columns) to[(c + i) * TILE] = __uint_as_float(v[i]);
                }
                // the warp's 32 features are its own: whoever comes last adds up
                __threadfence();
                __syncwarp();
                const int parts = shares.owner(begin + q.steps - 1) - shares.owner(begin) + 1;
                uint32_t came = 0u;
                if (lane == 0) came = atomicAdd(q.counters + tile * 4 + quad, 1u);
                came = __shfl_sync(0xffffffffu, came, 0);
                if (static_cast<int>(came) == parts - 1) {
                    __threadfence();
                    const int64_t feature = at.feature0 + in_tile;
                    const bool f_ok = feature < q.features;
                    const float alpha = p.amax ? __fdiv_rn(ld_float(p.amax + at.group), p.divisor) : 1.0f;
                    const float bias = p.bias && f_ok ? load_bias(p.bias, p.out_dtype, feature) : 0.0f;
                    const int64_t out = at.row0 * p.ld_out + feature;
                    if (p.out_dtype == FOS_BF16)
                        store_joined(q, static_cast<__nv_bfloat16 *>(p.out) + out, at, in_tile, columns, f_ok, alpha, bias, shares, tile);
                    else if (p.out_dtype == FOS_FP16)
                        store_joined(q, static_cast<__half *>(p.out) + out, at, in_tile, columns, f_ok, alpha, bias, shares, tile);
                    else
                        store_joined(q, static_cast<float *>(p.out) + out, at, in_tile, columns, f_ok, alpha, bias, shares, tile);
                }
            }
            u = end;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------- many rows: tensor cores, CTA pairs
//
// The same with cta_group::2 MMAs: two SMs compute 256 features by 256 rows, each expanding its own 128 features and fetching 128 of
// the rows. A stage of 512 cycles of MMA then moves 64 KB through each SM's shared memory (expanded weight and rows in, both out
// to the tensor cores) where the kernel above moves 96 KB, which takes it 768 cycles at 128 bytes a cycle.
constexpr int PAIR_STAGES = 6, PAIR_STAGE_BYTES = W_STAGE_BYTES + 128 * 128;
constexpr int PAIR_SMEM_BYTES = PAIR_STAGES * (PAIR_STAGE_BYTES + CODE_STAGE_BYTES) + 1024 + 256;       // (barriers: 240)
static_assert(PAIR_SMEM_BYTES + sizeof(GroupTables) <= 232448, "shared memory");

// A wait for arrivals from both CTAs, behind which the tensor cores read both CTAs' shared memory.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int *abort_flag, int32_t *status, int where) {
    const long long t0 = clock64();
#pragma unroll 1
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i) {
            uint32_t done;
            asm volatile(
                "{ .reg .pred p;\n"
                "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n"
                "selp.u32 %0, 1, 0, p; }\n"
                : "=r"(done) : "r"(bar), "r"(parity), "r"(POLL_SUSPEND_NS) : "memory");
            if (done) return true;
        }
        if (*abort_flag) {
            atomicOr(&g_wait_roles, 1u << (where & 31));
            return false;
        }
        if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
            *abort_flag = 1;
            if (status) atomicCAS(status, 0, where);
            atomicOr(&g_wait_roles, 1u << (where & 31));
            return false;
        }
    }
}

template <bool TRANSPOSED, int FMT>
__global__ void __launch_bounds__(GEMM_THREADS, 1) gemm_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes,
                                                                    const GemmParams q) {
    constexpr int NT = 256;
    extern __shared__ uint8_t smem_raw[];
    __shared__ GroupTables groups;
    const Params &p = q.p;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_gen + PAIR_STAGES * (PAIR_STAGE_BYTES + CODE_STAGE_BYTES));
    const uint32_t loaded = smem_u32(bars), ready = loaded + 16 * PAIR_STAGES;          // loaded: two in turn; ready: both CTAs', used in the leader
    const uint32_t empty = ready + 8 * PAIR_STAGES, acc_full = empty + 8 * PAIR_STAGES;
    const uint32_t acc_empty = acc_full + 16, drain = acc_empty + 16;   // acc_empty: used in the leader
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 4 * PAIR_STAGES + 5);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < PAIR_STAGES; ++s) {
            mbar_init(loaded + 8 * s, 1);
            mbar_init(loaded + 8 * (s + PAIR_STAGES), 1);
            mbar_init(ready + 8 * s, 2 * TEAM_WARPS);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full + 8 * a, 1);
            mbar_init(acc_empty + 8 * a, 2 * EPILOGUE_WARPS);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (p.group_start) fill_group_tables<NT>(p, groups);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();            // both CTAs have initialised their barriers and tensor memory
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const TileMap<NT> map(q, groups, 2 * TILE);
    const int64_t num_tiles = map.num_tiles;
    const int first_tile = static_cast<int>(blockIdx.x) >> 1, by_tiles = static_cast<int>(gridDim.x) >> 1, steps = q.steps;
    const uint32_t leader_ready = map_to_cta(ready, 0);

    if (warp == 0) {
        // ------------------------------------------------------------------ copies (both CTAs, each its own)
        const bool issue = elect_one();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int64_t t = first_tile; t < num_tiles && ok; t += by_tiles) {
            const Tile at = map.at(t);
            const int row0 = static_cast<int>(at.row0) + static_cast<int>(rank) * 128;
            const int64_t feature = at.feature0 + static_cast<int>(rank) * TILE;
            for (int ks = 0; ks < steps; ++ks) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ph ^ 1u, abort_flag, q.status, 1));
                if (!ok) break;
                if (issue)
                    copy_stage<TRANSPOSED>(&map_x, &map_codes, q, at, feature, row0, ks, smem_base + s * PAIR_STAGE_BYTES + W_STAGE_BYTES,
                                           smem_base + PAIR_STAGES * PAIR_STAGE_BYTES + s * CODE_STAGE_BYTES, 128 * 128, loaded + 8 * (s + ph * PAIR_STAGES));
                __syncwarp();
                if (++s == PAIR_STAGES) { s = 0; ph ^= 1u; }
            }
        }
        // the leader's last releases arrive in both CTAs' shared memory: stay until they have
        for (int i = 0; i < PAIR_STAGES && ok; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ph ^ 1u, abort_flag, q.status, 7));
            if (++s == PAIR_STAGES) { s = 0; ph ^= 1u; }
        }
        if (!ok) {
            const unsigned long long t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
    } else if (warp == 1 && leader) {
        // ------------------------------------------------------------------ MMAs, for both CTAs
        const bool issue = elect_one();
        constexpr uint32_t idesc = (1u << 4) | (TRANSPOSED ? 1u << 15 : 0u) | (static_cast<uint32_t>(NT >> 3) << 17) | (16u << 24);
        int s = 0;
        uint32_t ph = 0, tile_i = 0;
        bool ok = true;
        for (int64_t t = first_tile; t < num_tiles && ok; t += by_tiles, ++tile_i) {
            const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
            ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + 8 * acc, acc_ph ^ 1u, abort_flag, q.status, 3));
            if (!ok) break;
            tc_fence_after();
            for (int ks = 0; ks < steps; ++ks) {
                ok = __all_sync(0xffffffffu, mbar_wait_cluster(ready + 8 * s, ph, abort_flag, q.status, 2));
                if (!ok) break;
                tc_fence_after();
                const uint32_t stage = smem_base + s * PAIR_STAGE_BYTES;
                const uint64_t w_desc = smem_desc(stage, TRANSPOSED ? 8192 : 16, 1024, 2), x_desc = smem_desc(stage + W_STAGE_BYTES, 16, 1024, 2);
                if (issue) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_f16_pair(tmem_base + acc * NT, w_desc + (TRANSPOSED ? 128 : 2) * j, x_desc + 2 * j, idesc, (ks > 0 || j > 0) ? 1u : 0u);
                    tc_commit_pair(empty + 8 * s);
                }
                __syncwarp();
                if (++s == PAIR_STAGES) { s = 0; ph ^= 1u; }
            }
            if (ok && issue) tc_commit_pair(acc_full + 8 * acc);
        }
        if (!ok) {
            // giving up: the MMAs already issued must have finished before tensor memory is released
            if (issue) pair::tc_commit_pair_local(drain);
            __syncwarp();
            const long long t0 = clock64();
            while (!mbar_try_wait(drain, 0) && clock64() - t0 < 20000000ll) {}   // about 10 ms
        }
    } else if (warp >= 2 && warp < 2 + EXPAND_WARPS) {
        // ------------------------------------------------------------------ expansion (both CTAs)
        expand_stages<NT, TRANSPOSED, FMT, PAIR_STAGES, PAIR_STAGE_BYTES>(
            q, map, static_cast<int>(rank) * TILE, first_tile, by_tiles, 0, steps, smem_base, threadIdx.x - 64,
            [&](int s, uint32_t turn, uint32_t parity) {
                return __all_sync(0xffffffffu, mbar_wait(loaded + 8 * (s + turn * PAIR_STAGES), parity, abort_flag, q.status, 6));
            },
            [&](int s) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_ready + 8 * s) : "memory"); });
    } else if (warp >= 2 + EXPAND_WARPS) {
        // ------------------------------------------------------------------ epilogue (both CTAs)
        const int quad = warp & 3, in_tile = static_cast<int>(rank) * TILE + quad * 32 + lane;
        const uint32_t leader_acc_empty = map_to_cta(acc_empty, 0);
        uint32_t tile_i = 0;
        bool ok = true;
        for (int64_t t = first_tile; t < num_tiles && ok; t += by_tiles, ++tile_i) {
            const Tile at = map.at(t);
            const uint32_t acc = tile_i & 1u, acc_ph = (tile_i >> 1) & 1u;
            if (lane == 0) ok = mbar_wait_poll(acc_full + 8 * acc, acc_ph, abort_flag, q.status, 4);
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
            if (!ok) break;
            tc_fence_after();
            store_tile<NT>(q, at, in_tile, tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * NT, [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(leader_acc_empty + 8 * acc);
            });
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();            // nobody leaves while the peer may still touch this CTA's memory
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// How many CTAs share a tile's K: as many as keep four steps each and do not come to more than six per SM and a fifth of one (a last round that is
// all but empty costs less than CTAs twice as long: 8 x 8192 -> 28672 takes 47.7 us with 896 CTAs, 48.8 with 448). Split 1 / 2 / 4 / 8, us:
// 1 x 8192 -> 10240 24.1 / 19.7 / 20.1 / 18.4; 16 x 14336 -> 4096 - / - / 19.7 / 18.8; 8 x 8192 -> 28672 59.6 / 49.2 / 47.8 / 48.5. More where
// the activations' share of K would not leave room for two CTAs on an SM.
inline int split_for(int64_t tiles, int64_t k_p, int nt, int held) {
    const int64_t steps = (k_p + STEP - 1) / STEP;
    int split = 1;
    while (split < MAX_SPLIT && ((tiles * split * 2 <= 6 * SMS + SMS / 5 && steps / (split * 2) >= 4) || few_rows_smem_bytes(nt, k_p, split, held) > 100 * 1024)) split *= 2;
    return split;
}

template <typename T, int NT, int FMT>
int launch_few_rows(const Params &p, unsigned grid_z, cudaStream_t stream) {
    auto kernel = few_rows_kernel<T, NT, FMT>;
    static OncePerDevice configured;      // per instantiation
    int dev = 0;
    FOS_CUDA_TRY(cudaGetDevice(&dev));
    FOS_CUDA_TRY(configured.run(dev, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_ROWS_SMEM); }));
    const int64_t smem = few_rows_smem_bytes(NT, p.k_p, p.split, p.held);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.n_p / TILE * p.split), static_cast<unsigned>(p.num_groups < p.rows ? p.num_groups : p.rows), grid_z);
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

// How the groups share the rows is known on the device only: twice the even share is taken to be a group's rows at once.
inline int64_t rows_at_once(int64_t rows, int num_groups, bool grouped) { return grouped ? 2 * ((rows + num_groups - 1) / num_groups) : rows; }

// The rows that few_rows_kernel has instructions for (mt) and room for, and the CTAs that share a tile's K.
struct FewRowsShape { int mt, held_log2, split; };
inline FewRowsShape few_rows_shape(int64_t rows, int num_groups, bool grouped, int64_t n_p, int64_t k_p) {
    const int64_t at_once = rows_at_once(rows, num_groups, grouped);
    FewRowsShape s{at_once <= 8 ? 8 : 16, at_once <= 8 ? 3 : 4, 1};
    // (groups: with room for four rows instead of eight more CTAs fit onto an SM, even rows 71.9 us instead of 83.7, but drawn ones take 73.4
    // instead of 68.6 and 64 rows of four of the experts 79.8 instead of 41.7: an expert with more rows than there is room for is read again)
    while (!grouped && s.held_log2 > 0 && at_once <= 1 << (s.held_log2 - 1)) --s.held_log2;
    s.split = split_for(n_p / TILE * (grouped ? (num_groups < rows ? num_groups : rows) : 1), k_p, s.mt / 8, 1 << s.held_log2);
    return s;
}

int run_few_rows(Params p, int x_dtype, int format, cudaStream_t stream) {
    const FewRowsShape shape = few_rows_shape(p.rows, p.num_groups, p.group_start != nullptr, p.n_p, p.k_p);
    const int mt = shape.mt;
    p.held_log2 = shape.held_log2;
    p.held = 1 << p.held_log2;
    p.split = shape.split;
    int64_t z = p.group_start ? 1 : (p.rows + mt - 1) / mt;
    if (z > 65535) z = 65535;
    const unsigned grid_z = static_cast<unsigned>(z);
    if (x_dtype == FOS_BF16)
        return mt == 8 ? launch_few_rows_format<__nv_bfloat16, 1>(p, format, grid_z, stream) : launch_few_rows_format<__nv_bfloat16, 2>(p, format, grid_z, stream);
    return mt == 8 ? launch_few_rows_format<__half, 1>(p, format, grid_z, stream) : launch_few_rows_format<__half, 2>(p, format, grid_z, stream);
}

// The kernel, its tile width and the split of K, by the cycles they take. Fitted to measured times (fp16, us, measured / the formula at 1.9 GHz):
//   gemm_kernel     a stage 3.9 a column, 520 at least; 13000 a call; a split 4000 more for the exchange of the sums
//                   (32 x 8192 -> 10240 41.6 / 41.9, 32 x 14336 -> 4096 24.3 / 24.3, 333 x 2880 -> 5000 20.1 / 19.2)
//   gemm_pair_kernel  850 a stage, 16000 a call (512 x 8192 -> 10240 124 / 123; it is never far from the power limit, so the clock is lower)
//   stream_kernel   a stage 700 (see there) and 2 a column, 20000 a call, and what joining the parts of a tile takes: 1200 per part and 16
//                   columns, one after the other
//                   (16 x 8192 -> 10240 26.4 / 25.7, 512 x 8192 -> 10240 90 / 88, 64 x 8192 -> 28672 59 / 57)
//   few_rows_kernel, 9 to 16 rows   9500, and one for 1 KB of the weights (16 x 8192 -> 10240 29.2 / 29.2, -> 28672 67 / 74; 256 rows of 32 experts
//                   2880 -> 5760 140 / 155, where stream_kernel takes 120); up to eight rows take 0.6, which is what stream_kernel takes
//                   for the bytes alone
enum class Kernel { few_rows, single, pair, stream };
struct GemmChoice { Kernel kernel; int nt, split; };
inline GemmChoice gemm_choice(int64_t rows, int num_groups, bool grouped, bool transposed, int64_t features, int64_t inner_p) {
    const int64_t f_tiles = (features + TILE - 1) / TILE, steps = inner_p / K_STAGE, at_once = rows_at_once(rows, num_groups, grouped);
    const bool few = !transposed && at_once <= FEW_ROWS && few_rows_smem_bytes(at_once <= 8 ? 1 : 2, inner_p, MAX_SPLIT, at_once <= 8 ? 8 : 16) <= FEW_ROWS_SMEM;
    if (few && at_once <= 8) return {Kernel::few_rows, 0, 1};
    const int64_t in_use = !grouped ? 1 : num_groups < rows ? num_groups : rows;       // groups
    GemmChoice best{Kernel::single, 32, 1};
    double least = 1e300;
    auto row_tiles = [&](int nt) {        // of groups: as if each had half a tile too much, and one at least
        const double some = static_cast<double>(rows) / nt + 0.5 * in_use;
        return grouped ? (some > in_use ? some : static_cast<double>(in_use)) : static_cast<double>((rows + nt - 1) / nt);
    };
    auto consider = [&](GemmChoice c, double cycles) {
        if (cycles < least) {
            least = cycles;
            best = c;
        }
    };
    for (int nt : {32, 64, 128, 256}) {
        const double tiles = row_tiles(nt) * f_tiles, stage = 3.9 * nt > 520 ? 3.9 * nt : 520;
        for (int split : {1, 2, 4, 8}) {
            if (split > 1 && (grouped || tiles * split > (split < 4 ? SMS : SMS - SMS / 8) || steps / split < 4)) break;
            const double rounds = split > 1 ? 1.0 : __builtin_ceil(tiles / SMS);
            consider({Kernel::single, nt, split}, rounds * __builtin_ceil(static_cast<double>(steps) / split) * stage + 13000.0 + (split > 1 ? 4000.0 : 0.0));
        }
    }
    const double pairs = row_tiles(256) * ((f_tiles + 1) / 2);
    consider({Kernel::pair, 256, 1}, __builtin_ceil(pairs / (SMS / 2)) * steps * 850.0 + 16000.0);
    if (!transposed && inner_p >= S_STAGE) {
        const double s_steps = static_cast<double>((inner_p + S_STAGE - 1) / S_STAGE), share = row_tiles(S_ROWS) * f_tiles * s_steps / SMS;
        const int64_t high = ((grouped ? at_once : rows) + 15) / 16 * 16;
        const double columns = high < S_ROWS ? static_cast<double>(high) : S_ROWS;
        consider({Kernel::stream, S_ROWS, 1}, share * (700.0 + 2.0 * columns) + 20000.0 + 1200.0 * columns / 16 * (1.0 + s_steps / share));
    }
    if (few) consider({Kernel::few_rows, 0, 1}, 9500.0 + 0.55 * in_use * features / 1024 * inner_p);
    return best;
}

inline int make_rows_map(CUtensorMap *map, const void *base, int64_t rows, int64_t row_bytes, int64_t stride_bytes, int box_bytes, int box_rows, bool swizzled) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return FOS_ERR_CUDA;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride_bytes)};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(box_bytes), static_cast<cuuint32_t>(box_rows)};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    swizzled && box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : swizzled && box_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FOS_OK : FOS_ERR_CUDA;
}

template <int NT, bool TRANSPOSED, int FMT>
int launch_gemm(const CUtensorMap &map, const CUtensorMap &map_codes, const GemmParams &q, unsigned grid, cudaStream_t stream) {
    auto kernel = gemm_kernel<NT, TRANSPOSED, FMT>;
    static OncePerDevice configured;      // per instantiation
    int dev = 0;
    FOS_CUDA_TRY(cudaGetDevice(&dev));
    FOS_CUDA_TRY(configured.run(dev, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GemmCfg<NT>::SMEM_BYTES); }));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(GEMM_THREADS);
    cfg.dynamicSmemBytes = GemmCfg<NT>::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(q.p.split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = q.p.split > 1 ? 2 : 1;
    FOS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map, map_codes, q));
    return FOS_OK;
}
template <bool TRANSPOSED, int FMT>
int launch_gemm_width(int nt, const CUtensorMap &map, const CUtensorMap &map_codes, const GemmParams &q, unsigned grid, cudaStream_t stream) {
    if (nt == 32) return launch_gemm<32, TRANSPOSED, FMT>(map, map_codes, q, grid, stream);
    if (nt == 64) return launch_gemm<64, TRANSPOSED, FMT>(map, map_codes, q, grid, stream);
    if (nt == 128) return launch_gemm<128, TRANSPOSED, FMT>(map, map_codes, q, grid, stream);
    return launch_gemm<256, TRANSPOSED, FMT>(map, map_codes, q, grid, stream);
}
template <bool TRANSPOSED>
int launch_gemm_format(int format, int nt, const CUtensorMap &map, const CUtensorMap &map_codes, const GemmParams &q, unsigned grid, cudaStream_t stream) {
    if (format == FOS_NVFP4) return launch_gemm_width<TRANSPOSED, FOS_NVFP4>(nt, map, map_codes, q, grid, stream);
    if (format == FOS_IF4) return launch_gemm_width<TRANSPOSED, FOS_IF4>(nt, map, map_codes, q, grid, stream);
    return launch_gemm_width<TRANSPOSED, FOS_MXFP4>(nt, map, map_codes, q, grid, stream);
}

template <bool TRANSPOSED>
int launch_pair_format(int format, const CUtensorMap &map, const CUtensorMap &map_codes, const GemmParams &q, int64_t tiles, cudaStream_t stream) {
    if (format == FOS_NVFP4) return pair::launch<gemm_pair_kernel<TRANSPOSED, FOS_NVFP4>>(GEMM_THREADS, PAIR_SMEM_BYTES, tiles, 0, stream, map, map_codes, q);
    if (format == FOS_IF4) return pair::launch<gemm_pair_kernel<TRANSPOSED, FOS_IF4>>(GEMM_THREADS, PAIR_SMEM_BYTES, tiles, 0, stream, map, map_codes, q);
    return pair::launch<gemm_pair_kernel<TRANSPOSED, FOS_MXFP4>>(GEMM_THREADS, PAIR_SMEM_BYTES, tiles, 0, stream, map, map_codes, q);
}

template <int FMT> int launch_stream(const CUtensorMap &map, const CUtensorMap &map_codes, const GemmParams &q, unsigned grid, cudaStream_t stream) {
    auto kernel = stream_kernel<FMT>;
    static OncePerDevice configured;      // per instantiation
    int dev = 0;
    FOS_CUDA_TRY(cudaGetDevice(&dev));
    FOS_CUDA_TRY(configured.run(dev, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S_SMEM_BYTES); }));
    FOS_CUDA_TRY(launch_dependent(kernel, dim3(grid), GEMM_THREADS, S_SMEM_BYTES, stream, map, map_codes, q));
    return FOS_OK;
}

// What a call keeps in its workspace: x as fp16, the rows' factors, and for stream_kernel the tiles' counters and parts.
struct Workspace {
    int64_t factors, counters, parts, bytes, max_tiles;
    Workspace(const GemmChoice &choice, int64_t rows, int64_t inner_p, int64_t features, int num_groups, bool grouped) {
        factors = round_up64(rows * inner_p * 2, 256);
        counters = factors + round_up64(rows * 4, 256);
        parts = bytes = counters;
        max_tiles = 0;
        if (choice.kernel != Kernel::stream) return;
        const int64_t f_tiles = (features + TILE - 1) / TILE;
        max_tiles = (grouped ? rows / choice.nt + (num_groups < rows ? num_groups : rows) : (rows + choice.nt - 1) / choice.nt) * f_tiles;
        parts = counters + round_up64(max_tiles * 16, 256);
        bytes = parts + 2 * static_cast<int64_t>(SMS) * choice.nt * TILE * 4;
    }
};

// x may be read by the copy engine as it is: fp16 rows that start on 16 bytes, one after the other, as long as a copied row at least.
inline bool reads_x_itself(const Params &p, int x_dtype, int64_t inner) {
    return x_dtype == FOS_FP16 && p.vec && !p.group_start && !p.row_index && inner >= K_STAGE;
}

int run_gemm(Params p, const GemmChoice &choice, int x_dtype, int format, bool transposed, void *workspace, int64_t workspace_bytes, int32_t *status, cudaStream_t stream) {
    const int64_t inner = transposed ? p.n : p.k, inner_p = transposed ? p.n_p : p.k_p, features = transposed ? p.k : p.n;
    const int64_t features_p = transposed ? p.k_p : p.n_p;
    const bool grouped = p.group_start != nullptr;
    const Workspace at(choice, p.rows, inner_p, features_p, p.num_groups, grouped);
    if (!workspace || workspace_bytes < at.bytes) return FOS_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return FOS_ERR_MISALIGNED;
    uint8_t *work = static_cast<uint8_t *>(workspace);
    const bool pair = choice.kernel == Kernel::pair, streams = choice.kernel == Kernel::stream;
    GemmParams q{};
    q.features = features;
    q.steps = static_cast<int>(streams ? (inner_p + S_STAGE - 1) / S_STAGE : inner_p / K_STAGE);
    const int f_size = pair ? 2 * TILE : TILE, box = streams ? S_BOX : pair ? 128 : choice.nt;
    q.f_tiles = static_cast<int>((features + f_size - 1) / f_size);
    q.max_tiles = at.max_tiles;
    q.counters = reinterpret_cast<uint32_t *>(work + at.counters);
    q.parts = reinterpret_cast<float *>(work + at.parts);
    p.split = choice.split;
    CUtensorMap map, map_codes;
    int st;
    // encoding a tensor map wants a current context, which a thread that has launched nothing yet (autograd's) may not have
    int dev = 0;
    FOS_CUDA_TRY(cudaGetDevice(&dev));
    FOS_CUDA_TRY(cudaSetDevice(dev));
    // (a copied row is no longer than the tensor's: a weight of 64 columns has rows of 32 bytes)
    q.code_row = streams || (transposed && p.k_p >= 128) ? 64 : 32;
    if ((st = make_rows_map(&map_codes, p.codes, p.num_groups * p.n_p, p.k_p / 2, p.k_p / 2, q.code_row, transposed ? K_STAGE : TILE, streams)) != FOS_OK) return st;
    if (reads_x_itself(p, x_dtype, inner)) {
        if ((st = make_rows_map(&map, p.x, p.rows, inner * 2, p.x_ld * 2, 128, box, true)) != FOS_OK) return st;
        if (streams)
            FOS_CUDA_TRY(launch_dependent(zero_counters_kernel, dim3(static_cast<unsigned>(at.max_tiles * 4 < 16 * THREADS ? (at.max_tiles * 4 + THREADS - 1) / THREADS : 16)), THREADS, 0, stream,
                                          q.counters, at.max_tiles * 4));
    } else {
        PackParams k{p, inner, inner_p, static_cast<int>(features), reinterpret_cast<__half *>(work), reinterpret_cast<float *>(work + at.factors), q.counters,
                     at.max_tiles * 4};
        const bool wide = inner_p > PACK_HELD * 256 * 8;
        const int64_t most = SMS * (wide ? 4 : 10);
        const dim3 grid(static_cast<unsigned>(p.rows < most ? p.rows : most));
        auto pack = [&](auto kernel, unsigned threads) { return launch_dependent(kernel, grid, threads, 0, stream, k); };
        if (x_dtype == FOS_BF16) FOS_CUDA_TRY(wide ? pack(pack_rows_kernel<__nv_bfloat16, 512>, 512) : pack(pack_rows_kernel<__nv_bfloat16, 256>, 256));
        else FOS_CUDA_TRY(wide ? pack(pack_rows_kernel<__half, 512>, 512) : pack(pack_rows_kernel<__half, 256>, 256));
        q.factor_back = k.factor_back;
        if ((st = make_rows_map(&map, workspace, p.rows, inner_p * 2, inner_p * 2, 128, box, true)) != FOS_OK) return st;
    }
    if (status) {
        FOS_CUDA_TRY(cudaMemsetAsync(status, 0, sizeof(int32_t), stream));
    } else {
        FOS_CUDA_TRY(wait_failures_ptr(&status));   // the library's sticky word
    }
    q.status = status;
    q.p = p;
    const int64_t tiles = grouped ? INT32_MAX : (p.rows + choice.nt - 1) / choice.nt * q.f_tiles;
    if (streams) {
        const int64_t stages = tiles * q.steps;
        const unsigned grid = static_cast<unsigned>(stages < SMS ? stages : SMS);
        if (format == FOS_NVFP4) return launch_stream<FOS_NVFP4>(map, map_codes, q, grid, stream);
        if (format == FOS_IF4) return launch_stream<FOS_IF4>(map, map_codes, q, grid, stream);
        return launch_stream<FOS_MXFP4>(map, map_codes, q, grid, stream);
    }
    if (pair) return transposed ? launch_pair_format<true>(format, map, map_codes, q, tiles, stream) : launch_pair_format<false>(format, map, map_codes, q, tiles, stream);
    const unsigned grid = static_cast<unsigned>(choice.split > 1 ? tiles * choice.split : tiles < SMS ? tiles : SMS);
    return transposed ? launch_gemm_format<true>(format, choice.nt, map, map_codes, q, grid, stream) : launch_gemm_format<false>(format, choice.nt, map, map_codes, q, grid, stream);
}

int run(const Params &p, int x_dtype, int format, bool transposed, void *workspace, int64_t workspace_bytes, int32_t *status, cudaStream_t stream) {
    const GemmChoice choice = gemm_choice(p.rows, p.num_groups, p.group_start != nullptr, transposed, transposed ? p.k_p : p.n_p, transposed ? p.n_p : p.k_p);
    if (choice.kernel == Kernel::few_rows) {
        if (status) FOS_CUDA_TRY(cudaMemsetAsync(status, 0, sizeof(int32_t), stream));      // (no wait there can give up)
        return run_few_rows(p, x_dtype, format, stream);
    }
    return run_gemm(p, choice, x_dtype, format, transposed, workspace, workspace_bytes, status, stream);
}

int check(const void *x, int x_dtype, int64_t x_rows, const uint8_t *codes, const uint8_t *sf, const float *amax, int format, int rule,
          int sf_layout, int64_t n, int64_t k, int64_t n_p, int64_t k_p, int64_t rows, const void *out, int out_dtype, const int32_t *status) {
    if (!x || !codes || !sf || !out) return FOS_ERR_INVALID_ARGUMENT;
    if (x_dtype != FOS_BF16 && x_dtype != FOS_FP16) return FOS_ERR_INVALID_ARGUMENT;
    if (out_dtype != FOS_BF16 && out_dtype != FOS_FP16 && out_dtype != FOS_FP32) return FOS_ERR_INVALID_ARGUMENT;
    if (format != FOS_NVFP4 && format != FOS_IF4 && format != FOS_MXFP4) return FOS_ERR_INVALID_ARGUMENT;
    if (format != FOS_MXFP4 && !amax) return FOS_ERR_INVALID_ARGUMENT;
    if (rule < FOS_RULE_STATIC_6 || rule > FOS_RULE_ABS_MAX) return FOS_ERR_INVALID_ARGUMENT;
    if (sf_layout != FOS_SF_ROWMAJOR && sf_layout != FOS_SF_TILED) return FOS_ERR_INVALID_ARGUMENT;
    if (rows <= 0 || x_rows <= 0 || k <= 0 || n <= 0) return FOS_ERR_INVALID_ARGUMENT;
    if (n_p % 128 || n_p < n || k_p % (format == FOS_MXFP4 ? 128 : 64) || k_p < k) return FOS_ERR_INVALID_ARGUMENT;
    // (row tiles and features are counted in 32 bits, coordinates of the copy engine too)
    if (n_p > INT32_MAX / MAX_SPLIT || k_p > INT32_MAX / 8 || rows > INT32_MAX - 512 || x_rows > INT32_MAX) return FOS_ERR_TOO_LARGE;
    if (reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(sf) % 4 || reinterpret_cast<uintptr_t>(x) % 2) return FOS_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(out) % (out_dtype == FOS_FP32 ? 4 : 2)) return FOS_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(amax) % 4 || reinterpret_cast<uintptr_t>(status) % 4) return FOS_ERR_MISALIGNED;
    return FOS_OK;
}

// amax / divisor is what the packed numbers are multiplied with, in units of what the kernels multiply (IF4: seven times the values).
float divisor_for(int format, int rule, int unbiased) {
    if (format == FOS_MXFP4) return 1.0f;
    double d = dequant_divisor(format, rule);
    if (unbiased) d *= 16.0 / 17.0;
    return static_cast<float>(format == FOS_IF4 ? d * 7.0 : d);
}

Params params(const void *x, int64_t x_rows, int64_t k, int64_t ld_x, const uint8_t *codes, const uint8_t *sf, const float *amax, int format,
              int rule, int unbiased, int sf_layout, int64_t n, int64_t n_p, int64_t k_p, int64_t rows, void *out, int out_dtype, int64_t ld_out) {
    Params p{};
    p.x = x; p.x_rows = x_rows; p.x_ld = ld_x; p.k = k;
    p.codes = codes; p.sf = sf;
    p.amax = format == FOS_MXFP4 ? nullptr : amax;
    p.divisor = divisor_for(format, rule, unbiased);
    p.num_groups = 1; p.rows = rows;
    p.out = out; p.out_dtype = out_dtype; p.ld_out = ld_out;
    p.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x % 8 == 0;
    p.n = n; p.n_p = n_p; p.k_p = k_p; p.sf_tiled = sf_layout == FOS_SF_TILED;
    p.split = 1;
    return p;
}

}  // namespace wo
}  // namespace
}  // namespace fos

cudaError_t fos::weight_only_wait_failures(int32_t *host_value) { return fos::read_wait_failures(host_value); }
cudaError_t fos::weight_only_wait_roles(uint32_t *host_value) { return fos::read_wait_roles(host_value); }

extern "C" int64_t fos_weight_only_workspace_bytes(int64_t rows, int64_t n_p, int64_t k_p, int num_groups, int transposed) {
    using namespace fos::wo;
    if (rows <= 0 || n_p <= 0 || k_p <= 0 || num_groups < 0) return 0;
    const bool grouped = num_groups > 0;
    const int64_t inner_p = transposed ? n_p : k_p, features_p = transposed ? k_p : n_p;
    const GemmChoice choice = gemm_choice(rows, num_groups, grouped, transposed != 0, features_p, inner_p);
    return choice.kernel == Kernel::few_rows ? 0 : Workspace(choice, rows, inner_p, features_p, num_groups, grouped).bytes;
}

extern "C" int fos_weight_only_kernel(int64_t rows, int64_t n_p, int64_t k_p, int num_groups, int transposed, int *k_split) {
    using namespace fos::wo;
    if (rows <= 0 || n_p <= 0 || n_p % 128 || k_p <= 0 || k_p % 64 || num_groups < 0 || num_groups > MAX_GROUPS || (transposed && num_groups > 0))
        return FOS_ERR_INVALID_ARGUMENT;
    const bool grouped = num_groups > 0;
    const GemmChoice choice = gemm_choice(rows, num_groups, grouped, transposed != 0, transposed ? k_p : n_p, transposed ? n_p : k_p);
    const bool few = choice.kernel == Kernel::few_rows;
    if (k_split) *k_split = few ? few_rows_shape(rows, grouped ? num_groups : 1, grouped, n_p, k_p).split : choice.split;
    return few ? 1 : choice.kernel == Kernel::pair ? 2 : choice.kernel == Kernel::stream ? 3 : choice.nt;
}

extern "C" int fos_weight_only_matmul(const void *x, int x_dtype, int64_t rows, int64_t k, int64_t ld_x, const uint8_t *w_codes,
                                      const uint8_t *w_sf, const float *w_amax, int format, int scale_rule, int unbiased, int sf_layout,
                                      int64_t n, int64_t n_p, int64_t k_p, const void *bias, void *out, int out_dtype, int64_t ld_out,
                                      void *workspace, int64_t workspace_bytes, int32_t *status, void *stream) {
    using namespace fos;
    if (ld_x < k || ld_out < n) return FOS_ERR_INVALID_ARGUMENT;
    int st = wo::check(x, x_dtype, rows, w_codes, w_sf, w_amax, format, scale_rule, sf_layout, n, k, n_p, k_p, rows, out, out_dtype, status);
    if (st != FOS_OK) return st;
    if (reinterpret_cast<uintptr_t>(bias) % (out_dtype == FOS_FP32 ? 4 : 2)) return FOS_ERR_MISALIGNED;
    if ((st = check_device()) != FOS_OK) return st;
    wo::Params p = wo::params(x, rows, k, ld_x, w_codes, w_sf, w_amax, format, scale_rule, unbiased, sf_layout, n, n_p, k_p, rows, out, out_dtype, ld_out);
    p.bias = bias;
    return wo::run(p, x_dtype, format, false, workspace, workspace_bytes, status, static_cast<cudaStream_t>(stream));
}

extern "C" int fos_weight_only_matmul_dgrad(const void *dy, int dtype, int64_t rows, int64_t n, int64_t ld_dy, const uint8_t *w_codes,
                                            const uint8_t *w_sf, const float *w_amax, int format, int scale_rule, int unbiased, int sf_layout,
                                            int64_t k, int64_t n_p, int64_t k_p, void *dx, int out_dtype, int64_t ld_dx, void *workspace,
                                            int64_t workspace_bytes, int32_t *status, void *stream) {
    using namespace fos;
    if (ld_dy < n || ld_dx < k) return FOS_ERR_INVALID_ARGUMENT;
    int st = wo::check(dy, dtype, rows, w_codes, w_sf, w_amax, format, scale_rule, sf_layout, n, k, n_p, k_p, rows, dx, out_dtype, status);
    if (st != FOS_OK) return st;
    if ((st = check_device()) != FOS_OK) return st;
    wo::Params p = wo::params(dy, rows, k, ld_dy, w_codes, w_sf, w_amax, format, scale_rule, unbiased, sf_layout, n, n_p, k_p, rows, dx, out_dtype, ld_dx);
    return wo::run(p, dtype, format, true, workspace, workspace_bytes, status, static_cast<cudaStream_t>(stream));
}

extern "C" int fos_weight_only_matmul_grouped(const void *x, int x_dtype, int64_t x_rows, int64_t k, int64_t ld_x, const int32_t *row_index,
                                              const uint8_t *w_codes, const uint8_t *w_sf, const float *w_amax, int format, int scale_rule,
                                              int sf_layout, const int32_t *group_start, const int32_t *group_rows, int num_groups,
                                              int64_t rows, int64_t n, int64_t n_p, int64_t k_p, void *out, int out_dtype, int64_t ld_out,
                                              void *workspace, int64_t workspace_bytes, int32_t *status, void *stream) {
    using namespace fos;
    if (ld_x < k || ld_out < n) return FOS_ERR_INVALID_ARGUMENT;
    int st = wo::check(x, x_dtype, x_rows, w_codes, w_sf, w_amax, format, scale_rule, sf_layout, n, k, n_p, k_p, rows, out, out_dtype, status);
    if (st != FOS_OK) return st;
    if (!group_start || !group_rows || num_groups <= 0 || num_groups > wo::MAX_GROUPS) return FOS_ERR_INVALID_ARGUMENT;
    if (n_p > INT32_MAX / num_groups) return FOS_ERR_TOO_LARGE;         // (the copy engine counts their rows in 32 bits)
    for (const int32_t *table : {row_index, group_start, group_rows})
        if (reinterpret_cast<uintptr_t>(table) % 4) return FOS_ERR_MISALIGNED;
    if ((st = check_device()) != FOS_OK) return st;
    wo::Params p = wo::params(x, x_rows, k, ld_x, w_codes, w_sf, w_amax, format, scale_rule, 0, sf_layout, n, n_p, k_p, rows, out, out_dtype, ld_out);
    p.row_index = row_index;
    p.group_start = group_start; p.group_rows = group_rows; p.num_groups = num_groups;
    return wo::run(p, x_dtype, format, false, workspace, workspace_bytes, status, static_cast<cudaStream_t>(stream));
}
