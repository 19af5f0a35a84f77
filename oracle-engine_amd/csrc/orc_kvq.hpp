// The layout of a cache in fewer bits, shared by orc_kvq.hip (write, read
// back) and orc_attn_kvq.hip (attention).
//
// A cache is [sequence][kv head][ctx / 64] blocks of 64 positions; a block is
// its codes, then (8 and 4 bits) its scale bytes, in the order in which
// v_mfma_f32_16x16x32_f16 takes operands: every wave load is 1 KB in a row and
// no value crosses lanes on its way into a product. "Lane" is the one that
// holds the value: c = lane % 16, g = lane / 16.
//   K operand (16 keys x 32 dims): c = key % 16, the lane's head dims are the
//   hd / 4 in a row from g hd / 4.
//     fp16:   [tile = key / 16][dim / 8][lane][8 halves]
//     8 bits: [tile][dim / 16][lane][16 bytes]
//     4 bits: [tile][lane][hd / 8 bytes]: byte b = dim b, and dim b + hd / 8 in the high half
//     scales: [group of 32 dims][key % 16][tile]
//   V operand (16 dims x 32 keys): c = dim % 16, the lane's keys of step s are
//   s 32 + q 16 + g 4 + i in the order (q, i), which is the order in which the
//   scores' product leaves them.
//     fp16:   [dim / 16][s][lane][(q, i): 8 halves]
//     8 bits: [dim / 16][lane][(s, q, i): 16 bytes]
//     4 bits: [dim / 32][lane][(s, q, i): 16 bytes], dim / 16 odd in the high half
//     scales: [group of 32 dims][g][(s, q, i)]
//
// A scale byte b is the fp16 number with the bits b << 7 (5 exponent bits, 3 of
// the mantissa), and the value of a code is code x scale / 16. A product of 7
// (or 3) bits and 4 bits is an fp16 number exactly, so the matrix cores read
// the very values that the cache stands for; a finer scale would have cost a
// rounding of each value or a multiplication per score and group.
#pragma once
#include "orc_internal.hpp"

namespace orc {

typedef _Float16 kq_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 kq_h2 __attribute__((ext_vector_type(2)));
typedef float kq_f4 __attribute__((ext_vector_type(4)));
typedef float kq_f2 __attribute__((ext_vector_type(2)));

constexpr int kKvBlock = 64;  // positions of a block
constexpr int kKvGroup = 32;  // head dims of a scale
constexpr float kKvMax = 4064.f;  // largest magnitude of an 8 or 4 bit value: 127 x 512 / 16

constexpr int kvq_bits(int type) { return type == ORC_F16 ? 16 : type == ORC_KV_Q8 ? 8 : 4; }
constexpr int kvq_levels(int type) { return type == ORC_KV_Q8 ? 127 : 7; }
constexpr int kvq_code_bytes(int type, int hd) { return kKvBlock * hd * kvq_bits(type) / 8; }
constexpr int kvq_block_bytes(int type, int hd) {
    return kvq_code_bytes(type, hd) + (type == ORC_F16 ? 0 : kKvBlock * (hd / kKvGroup));
}
inline bool kvq_type_ok(int type) { return type == ORC_F16 || type == ORC_KV_Q8 || type == ORC_KV_Q4; }

// Where position p (0..63 of its block) and head dim d lie in a block: byte of
// the code (4 bits: high = the upper half of it), byte of the scale.
struct KvqAt {
    int code, scale;
    bool high;
};
template <int TY, int HD> __device__ __forceinline__ KvqAt kvq_at_k(int p, int d) {
    constexpr int L = HD / 4;
    const int tile = p >> 4, lane = (d / L) * 16 + (p & 15), e = d % L;
    KvqAt r{0, kvq_code_bytes(TY, HD) + (d / kKvGroup) * 64 + (p & 15) * 4 + tile, false};
    if (TY == ORC_F16) r.code = tile * 32 * HD + (e / 8) * 1024 + lane * 16 + (e % 8) * 2;
    else if (TY == ORC_KV_Q8) r.code = tile * 16 * HD + (e / 16) * 1024 + lane * 16 + e % 16;
    else {
        r.code = tile * 8 * HD + lane * (L / 2) + e % (L / 2);
        r.high = e >= L / 2;
    }
    return r;
}
template <int TY, int HD> __device__ __forceinline__ KvqAt kvq_at_v(int p, int d) {
    const int g = (p & 15) >> 2, slot = (p >> 5) * 8 + ((p >> 4) & 1) * 4 + (p & 3), lane = g * 16 + (d & 15), dt = d >> 4;
    KvqAt r{0, kvq_code_bytes(TY, HD) + (d / kKvGroup) * 64 + g * 16 + slot, false};
    if (TY == ORC_F16) r.code = dt * 2048 + (slot / 8) * 1024 + lane * 16 + (slot % 8) * 2;
    else if (TY == ORC_KV_Q8) r.code = dt * 1024 + lane * 16 + slot;
    else {
        r.code = (dt >> 1) * 1024 + lane * 16 + slot;
        r.high = dt & 1;
    }
    return r;
}

__device__ __forceinline__ float kvq_scale(uint32_t byte) { return h2f(byte << 7); }

// First own row of a sequence's new tokens; -1 (an idle sequence) where it lies outside [0, end).
__device__ __forceinline__ int kvq_start(const int32_t* d_pos, int seq, int pos_off, int end) {
    const int64_t p = (int64_t)(d_pos ? d_pos[seq] : 0) + pos_off;
    return p < 0 || p >= end ? -1 : (int)p;
}

// Division of a non-negative int by one that the host knows: a product and a shift instead of the 40 instructions of a
// quotient of two registers, which stood between a workgroup's start and its first load.
struct KvqDiv {
    uint32_t mul;  // 2^(31 + shift) / d rounded down, and 1
    int shift, d;
    __device__ __forceinline__ int operator()(int n) const {
        return d == 1 ? n : (int)(__umulhi((uint32_t)n << 1, mul) >> shift);
    }
};
inline KvqDiv kvq_div(int d) {
    KvqDiv r{0, 0, d > 1 ? d : 1};
    while (((int64_t)1 << r.shift) < r.d) ++r.shift;
    if (r.d > 1) r.mul = (uint32_t)((((uint64_t)1 << (31 + r.shift)) / r.d) + 1);
    return r;
}

}  // namespace orc
