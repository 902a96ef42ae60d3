// The packed form of a matrix in microscaled 4-bit floating point (MXFP4, the OCP microscaling format), and its values.
//
// Along K a matrix is cut into blocks of 32.  A block has one scale S = 2^(s - 127) with a byte s (255: the block is NaN) and
// 32 elements of 4 bits, a sign and the magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6 (e2m1).
//
// The packed form, as every kernel reads it: [row tiles of 128][K chunks of 128][MX_CHUNK bytes].  A chunk holds four
// pieces, one for each block, of 128 rows x 16 bytes of codes, then 512 bytes of scales: row r's four in one word at
// (r % 32) * 16 + (r / 32) * 4.  Nibble j of a 4-byte word of codes is element 2 j for j < 4 and 2 (j - 4) + 1 after that, so
// that one shift and one mask give two neighbours in the two halves of a word.  A row's codes of a block are 16 bytes in one
// piece and a tile's rows lie side by side: what an 8 x 16-byte core matrix of a tcgen05 operand is, and a chunk is one
// copy.  The scales lie as tcgen05.cp takes them to tensor memory.
#pragma once

#include "common.cuh"

#define MX_ROWS 128
#define MX_CODES 8192
#define MX_CHUNK 8704
#define MX_DEVICES 64

// The current device's index, for what a launcher asks or sets once on each (a function's attributes are a device's own); -1: none.
static inline int mx_device() {
    int device;
    return cudaGetDevice(&device) == cudaSuccess && device < MX_DEVICES ? device : -1;
}

__device__ __forceinline__ long mx_scale_at(int r) { return MX_CODES + (r & 31) * 16 + (r >> 5) * 4; }
__device__ __forceinline__ float mx_scale(int s) {          // 2^(s - 127)
    return s == 255 ? CUDART_NAN_F : (s == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)s << 23));
}
// A code in float, without its block's scale: sign and magnitude put where a float of exponent 2^-126 has them, a subnormal for the
// magnitudes 0 and 0.5, and multiplied by 2^126, exactly.
__device__ __forceinline__ float mx_value(uint32_t code) {
    return __uint_as_float(((code & 8u) << 28) | ((code & 7u) << 22)) * 8.507059173023462e37f;
}
__device__ __forceinline__ uint32_t mx_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// A word of 8 codes as 4 pairs of bfloat16, element 2 i in the low half of w[i]: sign and magnitude of nibbles i and 4 + i where
// a bfloat16 of exponent 2^-126 has them (the magnitudes 0 and 0.5 are subnormal), times m1.  A product with two powers of two puts
// a nibble in both places at once.
__device__ __forceinline__ void mx_pairs(uint32_t q, uint32_t m1, uint32_t* w) {
    constexpr uint32_t PLACES = 0x81C081C0u, NIBBLE = 0x000F000Fu;
    w[0] = mx_mul(((q & NIBBLE) * 0x1040u) & PLACES, m1);
    w[1] = mx_mul(((q & (NIBBLE << 4)) * 0x104u) & PLACES, m1);
    w[2] = mx_mul((((q >> 8) & NIBBLE) * 0x1040u) & PLACES, m1);
    w[3] = mx_mul((((q >> 8) & (NIBBLE << 4)) * 0x104u) & PLACES, m1);
}
__device__ __forceinline__ uint32_t mx_both(uint32_t h) { return h | h << 16; }
// The factors of a block with scale byte s: m1 = 2^(s - 1), both halves alike; where that has no bfloat16 (s > 128: a block whose
// largest magnitude is 4 or more) m1 is 2^127 and m2 the rest, else 1.
__device__ __forceinline__ uint32_t mx_factor(uint32_t s) { return (s + 126u) * 0x00800080u; }
__device__ __forceinline__ uint32_t mx_factor_large(uint32_t s) { return mx_both(s == 255 ? 0x7FC0u : (min(s, 128u) + 126u) << 7); }
__device__ __forceinline__ uint32_t mx_factor_rest(uint32_t s) { return mx_both(s == 255 || s <= 128 ? 0x3F80u : (s - 1) << 7); }
// A block of a row, 16 bytes of codes with scale byte s, as 16 pairs: exactly the values.
__device__ __forceinline__ void mx_block(const uint4 q, uint32_t m1, uint32_t* w) {
    mx_pairs(q.x, m1, w);
    mx_pairs(q.y, m1, w + 4);
    mx_pairs(q.z, m1, w + 8);
    mx_pairs(q.w, m1, w + 12);
}
__device__ __forceinline__ void mx_block_large(const uint4 q, uint32_t s, uint32_t* w) {
    mx_block(q, mx_factor_large(s), w);
    const uint32_t m2 = mx_factor_rest(s);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = mx_mul(w[i], m2);
}
