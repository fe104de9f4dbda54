// The scale of an MXFP4 block, shared by the quantize kernel and the norm that packs (sm_100a).
#pragma once

#include "fos_common.cuh"

namespace fos {
namespace {

// Scale byte of a block with maximum `bmax` and the factor 2^(127-e) that divides by the scale.
__device__ __forceinline__ uint32_t mx_scale(float bmax, bool quarter, float &inv) {
    const float hp = quarter ? bmax * 0.25f : div6_exact(bmax);
    const uint32_t bits = __float_as_uint(hp);
    uint32_t e = (bits >> 23) & 0xffu;
    if (bits & 0x7fffffu) e = (e + 1u) & 0xffu;
    // 2^(127-e): a normal number up to e = 253, the subnormal 2^-127 for e = 254; an all-zero
    // block (e = 0) quantizes to zeros whatever the factor
    inv = e == 0u ? 0.0f : __uint_as_float(e < 254u ? (254u - e) << 23 : 0x00400000u);
    return e;
}

}  // namespace
}  // namespace fos
