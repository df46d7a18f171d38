// kv4.cuh — the 4-bit KV cache format (alpaca_kv4_cache): row addressing and decoding shared by the kernels.
//
// A head row of d channels is d/32 blocks of 32 channels. Block b has a 16-bit header: the f16 bits of its step with
// the low 4 mantissa bits replaced by the zero point z, so the step has 7 significant bits, and
//     value = (code - z) * step,  code, z in 0..15.
// |code - z| <= 15 is 4 bits and the step 7, so every value is exact in f16 (denormal steps are multiples of 2^-20):
// kernels may hold decoded values as f16 MMA operands without rounding.
// The codes are 32-bit words of eight, channel 32 b + 8 t + n in nibble n of word t * (d/32) + b (t = 0..3): the words
// that lane t of a quad needs from all blocks are one contiguous load.
#pragma once

#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace alpaca {

constexpr uint32_t kKv4StepMask = 0xFFF0u;   // header bits of the step
constexpr uint32_t kKv4NanHeader = 0x7E00u;  // a block that held a NaN or an infinity: every value reads as NaN
constexpr float kKv4MaxStep = 4352.f;        // largest 7-bit step with 15 * step below the f16 maximum (0x6C40)

// Device-side view of alpaca_kv4_cache.
struct Kv4View {
    uint8_t* k_codes;
    uint8_t* v_codes;
    uint16_t* k_scales;
    uint16_t* v_scales;
    int64_t code_head_stride, code_unit_stride;    // bytes
    int64_t scale_head_stride, scale_unit_stride;  // 16-bit elements
    const int* block_table;  // null: unit s is sequence s
    int rows, max_blocks, pool_blocks;
};

inline Kv4View kv4_view(const alpaca_kv4_cache& c) {
    Kv4View v;
    v.k_codes = static_cast<uint8_t*>(c.k_codes);
    v.v_codes = static_cast<uint8_t*>(c.v_codes);
    v.k_scales = static_cast<uint16_t*>(c.k_scales);
    v.v_scales = static_cast<uint16_t*>(c.v_scales);
    v.code_head_stride = c.code_head_stride;
    v.code_unit_stride = c.code_unit_stride;
    v.scale_head_stride = c.scale_head_stride;
    v.scale_unit_stride = c.scale_unit_stride;
    v.block_table = c.block_table;
    v.rows = c.rows;
    v.max_blocks = c.max_blocks;
    v.pool_blocks = c.pool_blocks;
    return v;
}

// Unit and row within it of cache row `row` of sequence `seq`. False (and the device error word raised) when the row
// lies outside the cache or the table entry outside the pool.
__device__ __forceinline__ bool kv4_locate(const Kv4View& c, int seq, int row, unsigned* err, int64_t& unit, int& r) {
    if (!c.block_table) {
        unit = seq;
        r = row;
        if (row >= 0 && row < c.rows) return true;
        atomicOr(err, kDevErrBadIndex);
        return false;
    }
    const int b = row >= 0 ? row / c.rows : -1;
    const int blk = (b >= 0 && b < c.max_blocks) ? c.block_table[static_cast<int64_t>(seq) * c.max_blocks + b] : -1;
    if (blk < 0 || blk >= c.pool_blocks) {
        atomicOr(err, kDevErrBadIndex);
        return false;
    }
    unit = blk;
    r = row - b * c.rows;
    return true;
}

__device__ __forceinline__ uint32_t kv4_and_or(uint32_t x, uint32_t mask, uint32_t bits) {  // (x & mask) | bits
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
    return r;
}

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }

// A block's (step, zero point) as f16 pairs for two decodes side by side: .x / .y from headers h0 / h1.
//   step, and 1024 + zero   for codes in bits 0-3 of each half  (0x6400 | c      = 1024 + c)
//   step / 16, 1024 + 16 z  for codes in bits 4-7               (0x6400 | c << 4 = 1024 + 16 c)
// Both are exact: the step has 7 significant bits and is a multiple of 2^-20.
struct Kv4Pair {
    __half2 d, z, d16, z16;
};
__device__ __forceinline__ Kv4Pair kv4_pair(uint32_t h) {  // h: header of the low half | header of the high half << 16
    Kv4Pair p;
    p.d = as_half2(h & 0xFFF0FFF0u);
    p.z = as_half2(kv4_and_or(h, 0x000F000Fu, 0x64006400u));
    p.d16 = __hmul2(p.d, as_half2(0x2C002C00u));  // * 2^-4
    p.z16 = as_half2(kv4_and_or(h << 4, 0x00F000F0u, 0x64006400u));
    return p;
}
// (code - z) * step of the codes in bits 0-3 / bits 4-7 of each half of x: two exact f16 operations.
__device__ __forceinline__ uint32_t kv4_lo(uint32_t x, const Kv4Pair& p) {
    return as_u32(__hmul2(__hsub2(as_half2(kv4_and_or(x, 0x000F000Fu, 0x64006400u)), p.z), p.d));
}
__device__ __forceinline__ uint32_t kv4_hi(uint32_t x, const Kv4Pair& p) {
    return as_u32(__hmul2(__hsub2(as_half2(kv4_and_or(x, 0x00F000F0u, 0x64006400u)), p.z16), p.d16));
}

// The eight values of one word in channel order, as four f16 pairs.
__device__ __forceinline__ uint4 kv4_word_values(uint32_t w, uint32_t header) {
    const Kv4Pair p = kv4_pair(header * 0x10001u);
    const uint32_t p04 = kv4_lo(w, p), p15 = kv4_hi(w, p), p26 = kv4_lo(w >> 8, p), p37 = kv4_hi(w >> 8, p);
    return make_uint4(__byte_perm(p04, p15, 0x5410), __byte_perm(p26, p37, 0x5410), __byte_perm(p04, p15, 0x7632),
                      __byte_perm(p26, p37, 0x7632));
}

// A block's quantiser.
struct Kv4Block {
    uint32_t header;
    float step, inv;  // inv = 1 / step, correctly rounded; both 0 where every code is 0
    int bias;         // zero point less the bits of 1.5 * 2^23
    bool wide;        // the step is saturated: values may lie beyond the codes
};

// From the block's extremes lo <= 0 <= hi (NaN when it held one): the smallest step of 7 significant bits that is
// >= (hi - lo) / 15, and the zero point. Every finite value is then within half a step of a code, up to the saturation of
// the step at kKv4MaxStep.
__device__ __forceinline__ Kv4Block kv4_block(float lo, float hi) {
    Kv4Block b;
    b.step = b.inv = 0.f;
    b.bias = 0;
    b.wide = false;
    b.header = kKv4NanHeader;
    if (!(hi <= FLT_MAX && lo >= -FLT_MAX)) return b;
    const float span = hi - lo, s0 = span * (1.f / 15.f);
    const float s = __fmaf_rn(__fmaf_rn(-s0, 15.f, span), 1.f / 15.f, s0);  // span / 15 (as in kv4_code_pair); NaN past f32
    b.wide = !(s < kKv4MaxStep);
    const uint32_t bits = (static_cast<uint32_t>(__half_as_ushort(__float2half_ru(fminf(s, kKv4MaxStep)))) + 15u) & kKv4StepMask;
    b.header = bits;
    if (bits == 0) return b;
    b.step = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
    b.inv = __frcp_rn(b.step);
    const float z0 = -fmaxf(lo, -32.f * kKv4MaxStep) * b.inv;
    const float z = __fmaf_rn(__fmaf_rn(-z0, b.step, -fmaxf(lo, -32.f * kKv4MaxStep)), b.inv, z0);
    const int zero = min(__float_as_int(__fadd_rn(z, 12582912.f)) - 0x4B400000, 15);
    b.header = bits | static_cast<uint32_t>(zero);
    b.bias = zero - 0x4B400000;
    return b;
}

// clamp(round(x / step) + zero, 0, 15) of two values, the quotient as f32 division rounds it: from the correctly rounded
// reciprocal, one residual step gives the correctly rounded quotient (Markstein, "Computation of elementary functions on the
// IBM RISC System/6000 processor", 1990). Adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low bits.
__device__ __forceinline__ uint32_t kv4_code_pair(float2 x, const Kv4Block& b) {  // second code in bits 4-7
    const float2 inv = make_float2(b.inv, b.inv), minus_step = make_float2(-b.step, -b.step);
    const float2 q = __fmul2_rn(x, inv);
    const float2 m = __fadd2_rn(__ffma2_rn(__ffma2_rn(q, minus_step, x), inv, q), make_float2(12582912.f, 12582912.f));
    return static_cast<uint32_t>(__vimin_s32_relu(__float_as_int(m.x) + b.bias, 15)) +
           16u * static_cast<uint32_t>(__vimin_s32_relu(__float_as_int(m.y) + b.bias, 15));
}

}  // namespace alpaca
