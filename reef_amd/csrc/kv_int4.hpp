// The 4-bit KV cache's codes (gfx950): c in [-7, 7] held as the nibble c + 8. A key row's byte
// j holds channel j (low nibble) and channel j + D/2 (high); of a value channel's 16 tokens,
// 8 bytes, token t is nibble kv_nibble(t), low nibbles first.
#pragma once

#include "reef_common.hpp"

namespace reef {

typedef int32_t i32x2 __attribute__((ext_vector_type(2)));

constexpr float kInt4Max = 7.0f;
constexpr int kInt4Zero = 8;

__host__ __device__ constexpr int kv_nibble(int t) { return 8 * (t / 8) + t % 8 / 2 + 4 * (t % 2); }
// The token whose code is nibble n.
__host__ __device__ constexpr int kv_nibble_token(int n) { return 8 * (n / 8) + 2 * (n % 4) + n % 8 / 4; }

// The low or high nibbles of a word's bytes, each in a byte: codes + 8.
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w) { return w & 0x0f0f0f0fu; }
__device__ __forceinline__ uint32_t high_nibbles(uint32_t w) { return (w >> 4) & 0x0f0f0f0fu; }

// Bytes holding codes + 8 as int8 codes: with bit 7 set no byte's subtraction borrows from the
// next, and clearing it by XOR leaves each difference modulo 256.
__device__ __forceinline__ uint32_t nibbles_to_int8(uint32_t u) {
    return ((u | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
}

// One half (4 bytes, 8 tokens) of a value channel as fp16 in token order, exactly. Under the
// exponent of 1024 a nibble in bits 0-3 reads as 1024 + u, one in bits 4-7 as 1024 + 16 u;
// tokens 2i and 2i + 1 lie 16 bits apart, so one mask takes both. Nine instructions for eight
// values (the empty asm keeps mask and exponent in registers, where one instruction takes both;
// as literals they cost one each: 64 more a block of decode at head_dim 128, which has about 440).
__device__ __forceinline__ f16x8 int4x8_to_f16(uint32_t w) {
    const f16x2 low = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    const f16x2 high = {(_Float16)-72.0f, (_Float16)-72.0f};
    const f16x2 part = {(_Float16)0.0625f, (_Float16)0.0625f};
    uint32_t lower = 0x000f000fu, upper = 0x00f000f0u, exponent = 0x64006400u;
    asm("" : "+s"(lower), "+s"(upper));
    asm("" : "+v"(exponent));
    const uint32_t s = w >> 8;
    const uint32_t u[4] = {(w & lower) | exponent, (w & upper) | exponent, (s & lower) | exponent,
                           (s & upper) | exponent};
    f16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 x = __builtin_bit_cast(f16x2, u[i]);
        const f16x2 y = i & 1 ? __builtin_elementwise_fma(x, part, high) : x + low;
        r[2 * i] = y[0];
        r[2 * i + 1] = y[1];
    }
    return r;
}

}  // namespace reef
