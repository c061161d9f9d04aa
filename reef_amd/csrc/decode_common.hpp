// What the attention kernels over the int8 decode cache share (gfx950): the keys of a step,
// operand conversions and loads.
#pragma once

#include "reef_common.hpp"

namespace reef {

constexpr int kBlockKeys = 64;  // keys per inner step (4 pages)

// int8 x 16 (one 16-byte word) -> two fp16 x 8 operands, exactly. After the XOR a
// byte holds u = b + 128; a byte permute puts each u under the exponent byte 0x64,
// which reads as the fp16 1024 + u, and subtracting 1152 leaves b. Five
// instructions per 4 values.
__device__ __forceinline__ void int8x16_to_f16(i32x4 w, f16x8 &lo, f16x8 &hi) {
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = (uint32_t)w[j] ^ 0x80808080u;
        const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
        const f16x2 c = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
        f16x8 &dst = j < 2 ? lo : hi;
        const int e = 4 * (j & 1);
        dst[e] = a[0];
        dst[e + 1] = a[1];
        dst[e + 2] = c[0];
        dst[e + 3] = c[1];
    }
}

// A vector load of the streamed cache; NT marks it non-temporal (read once: a
// contiguous cache is not re-read within a step, and keeping it out of the caches
// measured faster there).
template <bool NT, typename V>
__device__ __forceinline__ V load_stream(const V *p) {
    return NT ? __builtin_nontemporal_load(p) : *p;
}

// The values of a row's 16 lanes, on every lane of the row (DPP row_newbcast). As shuffles
// through LDS the 16 index registers made the paged kernel spill inside its key loop (ragged
// paged decode of 128 sequences: 44.1 us, 41.0 this way).
template <int R = 0>
__device__ __forceinline__ void row_lanes(float x, float (&out)[16]) {
    out[R] = __int_as_float(
        __builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + R, 0xf, 0xf, true));
    if constexpr (R < 15) row_lanes<R + 1>(x, out);
}

}  // namespace reef
