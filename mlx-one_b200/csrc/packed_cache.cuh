// The format of a key/value cache held in 4 bits.
//
//   [pages, kv_heads, page_size / 16, 2, part bytes]
//
// units of 16 tokens of one key head: the keys' part, then the values' part, one after the other, so that
// a unit is one run of memory. A part is 16 * HD / 2 bytes of codes, then 16 words for each group of a
// token's values (64 values, 32 where the head size is no multiple of 64): step in the low half, lowest
// value in the high half, both bfloat16. A value is lowest + step * code.
//
// The codes lie as the lanes of a warp need them for the 16 x 16 operand of mma.m16n8k16, so that a lane
// gets all its codes of a unit by 16-byte loads and needs no transposing: the dimensions are cut into blocks
// of 64 (the last of 32 where 32 are left) with n = 4 (or 2) runs of 16, a block is 32 lanes x n words. The
// eight codes of word s of lane (r = lane / 4, c = lane % 4), by bits:
//
//   bits      keys: key, dimension in run s    values: key, dimension in run s
//   0..3      r      2c                        2c       r
//   4..7      r      2c + 8                    2c       r + 8
//   8..11     r + 8  2c                        2c + 8   r
//   12..15    r + 8  2c + 8                    2c + 8   r + 8
//   16..31    the same with 2c + 1             the same with 2c + 1
//
// (word >> 4 i) & 0x000f000f is thus one operand register's pair of codes, and 0x43004300 on top of it makes
// the bfloat16 numbers 128 + code. A byte belongs to one token: tokens of a unit can be written one by one.
// The word of token k of a group lies at place 2 (k % 8) + k / 8: a lane finds those of tokens r and r + 8 by
// one 8-byte load.
#pragma once

#include "common.cuh"

template <int HD>
struct Packed {
    static_assert(HD % 32 == 0 && HD >= 32 && HD <= 128, "heads of 32, 64, 96 or 128 values");
    static constexpr int GROUP = HD % 64 == 0 ? 64 : 32;
    static constexpr int GROUPS = HD / GROUP;
    static constexpr int RUNS = HD / 16;
    static constexpr int CODES = 8 * HD;                    // bytes of a part
    static constexpr int PART = CODES + 64 * GROUPS;
    static constexpr int UNIT = 2 * PART;                   // a multiple of 128 bytes

    // words of a lane in the block of dimensions that run s lies in, and where that block begins
    __host__ __device__ static constexpr int block_runs(int s) {
        return RUNS - (s & ~3) < 4 ? RUNS - (s & ~3) : 4;
    }
    __host__ __device__ static constexpr int word_at(int lane, int s) {
        return (s >> 2) * 512 + 4 * (lane * block_runs(s) + (s & 3));
    }
    // the byte of (key, dimension e of run s): codes of e and e + 8 share it (e < 8)
    __host__ __device__ static constexpr int key_byte(int key, int s, int e) {
        return word_at(4 * (key & 7) + (e >> 1), s) + (key >> 3) + 2 * (e & 1);
    }
    __host__ __device__ static constexpr int value_byte(int key, int s, int e) {
        return word_at(4 * e + ((key & 7) >> 1), s) + (key >> 3) + 2 * (key & 1);
    }
    __host__ __device__ static constexpr int scale_at(int key, int group) {
        return CODES + 64 * group + 4 * (2 * (key & 7) + (key >> 3));
    }
};

__device__ __forceinline__ float packed_step(uint32_t word) { return __uint_as_float(word << 16); }
__device__ __forceinline__ float packed_lowest(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

// 2^(to - floor(log2 x)) for x > 0, and its inverse; x is taken for 2^-113 at least
__device__ __forceinline__ float power_towards(float x, int to, float& inverse) {
    const int exponent = max((int)(__float_as_uint(x) >> 23 & 255u), 14);
    inverse = __uint_as_float((uint32_t)(exponent - to) << 23);
    return __uint_as_float((uint32_t)(254 - (exponent - to)) << 23);
}

#define MLXONE_PACKED_DIMS(CALL)                                                                  \
    switch (head_dim) {                                                                           \
        case 32: CALL(32); break;                                                                 \
        case 64: CALL(64); break;                                                                 \
        case 96: CALL(96); break;                                                                 \
        case 128: CALL(128); break;                                                               \
        default:                                                                                  \
            mlxone_set_error("a cache of 4 bits takes heads of 32, 64, 96 or 128 values, not %d", \
                             head_dim);                                                           \
            return 1;                                                                             \
    }
