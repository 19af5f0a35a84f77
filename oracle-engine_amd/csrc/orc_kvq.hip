// A KV cache in fewer bits (gfx950): the rotary table with scaled frequencies,
// the write of new tokens' K and V (rotary positions, quantisation, the
// cache's layout) and the read-back to fp32 rows. Layout and formats:
// orc_kvq.hpp; attention over such caches: orc_attn_kvq.hip. No counterpart in
// the reference, whose cache is fp32 and whose rotation is the rotate-half of
// core/ops.cpp:440-485.
#include "orc_kvq.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace orc {

// ── rotary table ─────────────────────────────────────────────────────────────
struct RopeFreqs {
    double f[64];  // angle of one position, per pair
};

// (cos, sin) of pos f_i times the table's factor, formed in 64 bits: an angle of 2^17 radians has 2^-7 left of a
// 24-bit mantissa, and sums of rounded angles drift with the position. A thread takes one pair at `steps` rows, `rows`
// apart: the sine and cosine of the first row's angle and of the step's, then one complex product per row (their error,
// 2^-52 a row, stays 2^20 below the result's last place), a tenth of the work of a sine for every entry, which bound the
// table (131072 x 64 pairs: 25.6 us; so 12.2 us, 5.5 TB/s). Neighbouring threads hold neighbouring pairs, so a workgroup
// writes rows in a row.
__global__ __launch_bounds__(256) void k_rope_table(float2* out, int64_t pos0, int64_t n, int pairs, int rows, int steps,
                                                    RopeFreqs fr, double mul) {
    const int r = threadIdx.x / pairs, i = threadIdx.x - r * pairs;
    if (r >= rows) return;
    int64_t p = (int64_t)blockIdx.x * rows * steps + r;
    double s, c, ds, dc;
    sincos((double)(pos0 + p) * fr.f[i], &s, &c);
    sincos((double)rows * fr.f[i], &ds, &dc);
    s *= mul;
    c *= mul;
    for (int k = 0; k < steps && p < n; ++k, p += rows) {
        out[p * pairs + i] = make_float2((float)c, (float)s);
        const double t = c * dc - s * ds;
        s = s * dc + c * ds;
        c = t;
    }
}

// ── quantisation ─────────────────────────────────────────────────────────────
// Scale byte of a group whose largest magnitude is amax (finite, clamped to
// kKvMax): the smallest scale D with M D >= 16 amax. M D is exact in fp32 (11
// significant bits), so the candidate from the rounded quotient is corrected
// by comparing products; no border depends on a rounding.
template <int M> __device__ __forceinline__ uint32_t kvq_scale_byte(float amax) {
    const float t = amax * 16.f;
    const float y = t * (1.f / M);
    int b;
    if (y < 6.103515625e-5f) b = (int)ceilf(y * 131072.f);  // below 2^-14: steps of 2^-17
    else b = (int)((__builtin_bit_cast(uint32_t, y) + 0xFFFFFu) >> 20) - (112 << 3);
    while (b > 0 && kvq_scale(b - 1) * M >= t) --b;
    while (kvq_scale(b) * M < t) ++b;
    return b;
}

// Code of x (biased to be positive): nearest multiple of the scale, ties to
// the even one. The correctly rounded quotient of a 24-bit and a 4-bit number
// is a tie only where the exact one is.
template <int M> __device__ __forceinline__ uint32_t kvq_code(float x, float D) {
    const float q = D > 0.f ? rintf(x * 16.f / D) : 0.f;
    return (uint32_t)((int)q + M + 1);
}

struct StoreArgs {
    const float* qkv;
    int ldqkv, n_seq, n_tok, n_heads, n_kv, layout, rot;
    const float2* rope;
    int64_t rope_off;
    const int32_t* d_pos;
    int pos_off;
    float* q;
    int ldq;
    uint8_t *kc, *vc;
    int ctx;
    KvqDiv by_vecs, by_tok, by_heads;  // by_heads: what of a token's q vectors one wave or set of threads takes
};

// Rotated value d of the head vector x. The products of two fp32 numbers are
// exact in 64 bits, so the fp32 result is the correctly rounded one and the
// codes behind it do not depend on how a compiler contracts the sum.
__device__ __forceinline__ float kvq_rotated(const float* x, int d, int layout, int rot, const float2* cs) {
    if (d >= rot) return x[d];
    const int half = rot >> 1;
    int a, b;
    bool first;
    if (layout == ORC_ROPE_HALF) {
        first = d < half;
        a = first ? d : d - half;
        b = a + half;
    } else {
        first = !(d & 1);
        a = d & ~1;
        b = a + 1;
    }
    const float2 c = cs[layout == ORC_ROPE_HALF ? a : a >> 1];
    const double va = x[a], vb = x[b], co = c.x, si = c.y;
    return (float)(first ? va * co - vb * si : va * si + vb * co);
}

// A few tokens a sequence: one wave per head vector, q heads are rotated, K
// heads rotated and quantised, V heads quantised. A scale group is 32 lanes; a
// row's codes are bytes (K: pieces of 16) all over its block. Bound by latency:
// 3.1 us for one token, 4.2 us for 61 of 32/8 heads.
template <int TY, int HD> __global__ __launch_bounds__(256) void k_kvq_store(StoreArgs a) {
    const int lane = threadIdx.x & 63;
    const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = a.by_vecs(unit);
    if (row >= a.n_seq * a.n_tok) return;
    const int h = unit - row * a.by_vecs.d, seq = a.by_tok(row), t = row - seq * a.n_tok;
    const int start = kvq_start(a.d_pos, seq, a.pos_off, a.ctx);
    if (start < 0 || start + (int64_t)t >= a.ctx) return;
    const int p = start + t;
    const float* x = a.qkv + (int64_t)row * a.ldqkv + (size_t)h * HD;
    const float2* cs = a.rope + (a.rope_off + p) * (a.rot >> 1);
    const bool is_v = h >= a.n_heads + a.n_kv;
    constexpr int E = HD / 64;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = kvq_rotated(x, lane + 64 * e, a.layout, is_v ? 0 : a.rot, cs);
    if (h < a.n_heads) {
        float* q = a.q + (int64_t)row * a.ldq + (size_t)h * HD;
#pragma unroll
        for (int e = 0; e < E; ++e) q[lane + 64 * e] = v[e];
        return;
    }
    const int kv = is_v ? h - a.n_heads - a.n_kv : h - a.n_heads;
    uint8_t* blk = (is_v ? a.vc : a.kc) +
                   (((size_t)seq * a.n_kv + kv) * (a.ctx / kKvBlock) + p / kKvBlock) * kvq_block_bytes(TY, HD);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane + 64 * e;
        const KvqAt at = is_v ? kvq_at_v<TY, HD>(p & 63, d) : kvq_at_k<TY, HD>(p & 63, d);
        if constexpr (TY == ORC_F16) {
            float y = v[e];
            if (fabsf(y) < __builtin_inff()) y = fminf(fmaxf(y, -65504.f), 65504.f);
            *(_Float16*)(blk + at.code) = (_Float16)y;
        } else {
            constexpr int M = kvq_levels(TY);
            const bool fin = fabsf(v[e]) < __builtin_inff();
            const float y = fin ? fminf(fmaxf(v[e], -kKvMax), kKvMax) : 0.f;
            float mx = fabsf(y);
#pragma unroll
            for (int s = 16; s; s >>= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 32));
            const uint64_t bad = __ballot(!fin);
            const uint32_t byte = kvq_scale_byte<M>(mx), code = kvq_code<M>(y, kvq_scale(byte));
            if ((lane & 31) == 0) blk[at.scale] = (uint32_t)(bad >> (lane & 32)) ? 0xFF : byte;
            if constexpr (TY == ORC_KV_Q8) blk[at.code] = code;
            else {  // the lane with the low half writes both: K's partner is hd / 8 dims on, V's 16
                const uint32_t other = __shfl_xor(code, 16, 64);
                const uint32_t k64 = HD == 64 ? __shfl_xor(code, 8, 64) : other;
                if (!at.high) blk[at.code] = code | (is_v ? other : k64) << 4;
            }
        }
    }
}

// Prompts: a workgroup per 64-position block of one kv head's K or V, and workgroups of q vectors behind them.
// K: a thread takes HD / 8 dims of one key and the ones HD / 2 further on, a rotate-half pair's two sides, so that the
// row is read once; its codes are whole 16 or 8 byte pieces of the block, stored in order. V: rows go through LDS,
// since a stored piece is one dim of 16 keys; pieces that hold rows of other calls are written byte by byte. 4001 tokens
// of 32/8 heads of 128: 39 us, 4.3 TB/s (a wave per head vector: 87 us); from 16 tokens on, fewer fill no block's pieces.
constexpr int kStoreBlocks = 16;  // tokens of a sequence from which on a call takes whole blocks
enum { kRotHalf, kRotPairs, kRotAny };  // whole heads half-split; pairs (2 i, 2 i + 1), or nothing rotated; the rest

template <int TY, int HD> struct StoreLds {
    float x[64][HD + 1];
    float d[64][HD / 32 + 1];
};

__device__ __forceinline__ float kvq_clamp(float v, float lim, bool& bad) {
    bad |= !(fabsf(v) < __builtin_inff());
    return fminf(fmaxf(v, -lim), lim);  // of a NaN: lim, in a group that is marked
}
__device__ __forceinline__ _Float16 kvq_half(float y) {
    if (fabsf(y) < __builtin_inff()) y = fminf(fmaxf(y, -65504.f), 65504.f);
    return (_Float16)y;
}

template <int TY, int HD>
__device__ __forceinline__ void kvq_store_k(const StoreArgs& a, int mode, int seq, int kv, int start, int64_t b) {
    constexpr int P = HD / 8, L = HD / 4;
    const int lane = threadIdx.x & 63, tile = threadIdx.x >> 6, c = lane & 15, u = lane >> 4;
    const int64_t p = b * kKvBlock + tile * 16 + c, t = p - start;
    const bool live = t >= 0 && t < a.n_tok;
    float v[2][P] = {};
    if (live) {
        const float* x = a.qkv + ((int64_t)seq * a.n_tok + t) * a.ldqkv + (size_t)(a.n_heads + kv) * HD;
        const float2* cs = a.rope + (a.rope_off + p) * (a.rot >> 1);
        if (mode == kRotAny) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < P; ++e) v[h][e] = kvq_rotated(x, h * (HD / 2) + u * P + e, ORC_ROPE_HALF, a.rot, cs);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < P; e += 4) {
                    const kq_f4 w = *(const kq_f4*)(x + h * (HD / 2) + u * P + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[h][e + k] = w[k];
                }
            if (mode == kRotHalf) {
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    const float2 r = cs[u * P + e];
                    const double va = v[0][e], vb = v[1][e], co = r.x, si = r.y;
                    v[0][e] = (float)(va * co - vb * si);
                    v[1][e] = (float)(va * si + vb * co);
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < P; e += 2) {
                        const int d = h * (HD / 2) + u * P + e;
                        if (d < a.rot) {
                            const float2 r = cs[d >> 1];
                            const double va = v[h][e], vb = v[h][e + 1], co = r.x, si = r.y;
                            v[h][e] = (float)(va * co - vb * si);
                            v[h][e + 1] = (float)(va * si + vb * co);
                        }
                    }
            }
        }
    }
    uint8_t* blk = a.kc + (((size_t)seq * a.n_kv + kv) * (a.ctx / kKvBlock) + b) * kvq_block_bytes(TY, HD);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int d0 = h * (HD / 2) + u * P, g = d0 / L, e0 = d0 % L;  // the operand's lane group, and where in its dims
        if constexpr (TY == ORC_F16) {
#pragma unroll
            for (int e = 0; e < P; e += 8) {
                kq_h8 y;
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = kvq_half(v[h][e + k]);
                if (live) *(kq_h8*)(blk + tile * 32 * HD + (e0 + e) / 8 * 1024 + (g * 16 + c) * 16) = y;
            }
        } else {
            constexpr int M = kvq_levels(TY);
            bool bad = false;
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                v[h][e] = kvq_clamp(v[h][e], kKvMax, bad);
                mx = fmaxf(mx, fabsf(v[h][e]));
            }
            int any = bad;
#pragma unroll
            for (int s = 16; s < 16 * (kKvGroup / P); s *= 2) {  // the threads of a scale group
                mx = fmaxf(mx, __shfl_xor(mx, s, 64));
                any |= __shfl_xor(any, s, 64);
            }
            const uint32_t byte = kvq_scale_byte<M>(mx);
            const float D = kvq_scale(byte);
            if (live && d0 % kKvGroup == 0)
                blk[kvq_code_bytes(TY, HD) + d0 / kKvGroup * 64 + c * 4 + tile] = any ? 0xFF : byte;
            uint32_t w[P / 4];
#pragma unroll
            for (int e = 0; e < P / 4; ++e) {
                w[e] = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) w[e] |= kvq_code<M>(v[h][e * 4 + k], D) << (8 * k);
            }
            if constexpr (TY == ORC_KV_Q8) {
                uint8_t* at = blk + tile * 16 * HD + (g * 16 + c) * 16;
                if (live) {
                    if constexpr (HD == 128) *(u32x4*)(at + e0 / 16 * 1024) = u32x4{w[0], w[1], w[2], w[3]};
                    else *(u32x2*)(at + e0) = u32x2{w[0], w[1]};
                }
            } else {  // the next thread group holds the upper halves
#pragma unroll
                for (int e = 0; e < P / 4; ++e) w[e] |= __shfl_xor(w[e], 16, 64) << 4;
                uint8_t* at = blk + tile * 8 * HD + (g * 16 + c) * (L / 2);
                if (live && !(u & 1)) {
                    if constexpr (HD == 128) *(u32x4*)at = u32x4{w[0], w[1], w[2], w[3]};
                    else *(u32x2*)at = u32x2{w[0], w[1]};
                }
            }
        }
    }
}

template <int TY, int HD>
__device__ __forceinline__ void kvq_store_v(const StoreArgs& a, int seq, int kv, int start, int64_t b, StoreLds<TY, HD>& sh) {
    const int tid = threadIdx.x;
    const int64_t t0 = b * kKvBlock - start;  // token of the block's first row
    const float* x = a.qkv + (int64_t)seq * a.n_tok * a.ldqkv + (size_t)(a.n_heads + a.n_kv + kv) * HD;
    for (int it = tid; it < 64 * HD / 4; it += 256) {
        const int r = it / (HD / 4), d = it % (HD / 4) * 4;
        kq_f4 v = {0.f, 0.f, 0.f, 0.f};
        if (t0 + r >= 0 && t0 + r < a.n_tok) v = *(const kq_f4*)(x + (t0 + r) * a.ldqkv + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) sh.x[r][d + k] = v[k];
    }
    __syncthreads();
    uint8_t* blk = a.vc + (((size_t)seq * a.n_kv + kv) * (a.ctx / kKvBlock) + b) * kvq_block_bytes(TY, HD);
    constexpr int M = kvq_levels(TY);
    if constexpr (TY != ORC_F16) {
        for (int it = tid; it < 64 * (HD / 32); it += 256) {
            const int r = it & 63, grp = it >> 6;
            bool bad = false;
            float mx = 0.f;
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, fabsf(kvq_clamp(sh.x[r][grp * 32 + e], kKvMax, bad)));
            const uint32_t byte = kvq_scale_byte<M>(mx);
            sh.d[r][grp] = kvq_scale(byte);
            if (t0 + r >= 0 && t0 + r < a.n_tok) {
                const int slot = (r >> 5) * 8 + ((r >> 4) & 1) * 4 + (r & 3);
                blk[kvq_code_bytes(TY, HD) + grp * 64 + ((r & 15) >> 2) * 16 + slot] = bad ? 0xFF : byte;
            }
        }
        __syncthreads();
    }
    constexpr int kUnits = TY == ORC_KV_Q4 ? HD * 2 : HD * 4;  // (dim or pair of dims, lane group)
    for (int it = tid; it < kUnits; it += 256) {
        const int lane = it & 63, dt = (it >> 6) * (TY == ORC_KV_Q4 ? 2 : 1), g = lane >> 4, d = dt * 16 + (lane & 15);
        bool all = true;
#pragma unroll
        for (int q = 0; q < 4; ++q) all &= t0 + q * 16 + g * 4 >= 0 && t0 + q * 16 + g * 4 + 3 < a.n_tok;
        if constexpr (TY == ORC_F16) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                kq_h8 y;
                _Float16* at = (_Float16*)(blk + dt * 2048 + s * 1024 + lane * 16);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = kvq_half(sh.x[s * 32 + (e >> 2) * 16 + g * 4 + (e & 3)][d]);
                if (all) *(kq_h8*)at = y;
                else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int64_t t = t0 + s * 32 + (e >> 2) * 16 + g * 4 + (e & 3);
                        if (t >= 0 && t < a.n_tok) at[e] = y[e];
                    }
                }
            }
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = (e >> 3) * 32 + ((e >> 2) & 1) * 16 + g * 4 + (e & 3);
                bool bad = false;
                uint32_t u = kvq_code<M>(kvq_clamp(sh.x[r][d], kKvMax, bad), sh.d[r][d >> 5]);
                if constexpr (TY == ORC_KV_Q4) u |= kvq_code<M>(kvq_clamp(sh.x[r][d + 16], kKvMax, bad), sh.d[r][d >> 5]) << 4;
                w[e >> 2] = (e & 3) ? w[e >> 2] | u << (8 * (e & 3)) : u;
            }
            uint8_t* at = blk + (TY == ORC_KV_Q4 ? dt >> 1 : dt) * 1024 + lane * 16;
            if (all) *(u32x4*)at = u32x4{w[0], w[1], w[2], w[3]};
            else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int64_t t = t0 + (e >> 3) * 32 + ((e >> 2) & 1) * 16 + g * 4 + (e & 3);
                    if (t >= 0 && t < a.n_tok) at[e] = w[e >> 2] >> (8 * (e & 3));
                }
            }
        }
    }
}

// Eight values of each of up to four q vectors of a token a thread: four and the four HD / 2 further on, or eight in a
// row, whose pairs' table entries serve all four.
constexpr int kQHeads = 4;
template <int HD> __device__ __forceinline__ void kvq_store_q(const StoreArgs& a, int mode, int w) {
    constexpr int N = HD / 8;
    const int part = threadIdx.x % N, unit = w * (256 / N) + threadIdx.x / N, row = a.by_heads(unit);
    if (row >= a.n_seq * a.n_tok) return;
    const int h0 = unit - row * a.by_heads.d, seq = a.by_tok(row), start = kvq_start(a.d_pos, seq, a.pos_off, a.ctx);
    const int64_t p = (int64_t)start + (row - seq * a.n_tok);
    if (start < 0 || p >= a.ctx) return;
    const int d0 = mode == kRotPairs ? part * 8 : part * 4, d1 = mode == kRotPairs ? d0 + 4 : d0 + HD / 2;
    const float* x = a.qkv + (int64_t)row * a.ldqkv;
    float* q = a.q + (int64_t)row * a.ldq;
    const float2* cs = a.rope + (a.rope_off + p) * (a.rot >> 1) + (mode == kRotPairs ? d0 >> 1 : d0);
    float2 r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = mode == kRotHalf || d0 + 2 * e < a.rot ? cs[e] : make_float2(1.f, 0.f);
    kq_f4 v0[kQHeads], v1[kQHeads];
#pragma unroll
    for (int u = 0; u < kQHeads; ++u) {
        const int h = min(h0 + u * a.by_heads.d, a.n_heads - 1);
        v0[u] = *(const kq_f4*)(x + (size_t)h * HD + d0);
        v1[u] = *(const kq_f4*)(x + (size_t)h * HD + d1);
    }
#pragma unroll
    for (int u = 0; u < kQHeads; ++u) {
        const int h = h0 + u * a.by_heads.d;
        if (h >= a.n_heads) break;
        if (mode == kRotHalf) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double va = v0[u][e], vb = v1[u][e], co = r[e].x, si = r[e].y;
                v0[u][e] = (float)(va * co - vb * si);
                v1[u][e] = (float)(va * si + vb * co);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kq_f4& v = e < 2 ? v0[u] : v1[u];
                const double va = v[e % 2 * 2], vb = v[e % 2 * 2 + 1], co = r[e].x, si = r[e].y;
                if (d0 + 2 * e < a.rot) {
                    v[e % 2 * 2] = (float)(va * co - vb * si);
                    v[e % 2 * 2 + 1] = (float)(va * si + vb * co);
                }
            }
        }
        *(kq_f4*)(q + (size_t)h * HD + d0) = v0[u];
        *(kq_f4*)(q + (size_t)h * HD + d1) = v1[u];
    }
}

// Grid: blocks_kv workgroups of K and V blocks (nblk a sequence and head), then q. kRotAny's q vectors, whose pairs lie
// anywhere in the head, take a wave each as in k_kvq_store.
template <int TY, int HD>
__global__ __launch_bounds__(256) void k_kvq_store_blocks(StoreArgs a, int mode, KvqDiv by_nblk, KvqDiv by_kv2, int blocks_kv) {
    __shared__ StoreLds<TY, HD> sh;
    int w = blockIdx.x;
    if (w < blocks_kv) {
        const int v = by_nblk(w), bi = w - v * by_nblk.d, seq = by_kv2(v), kv2 = v - seq * by_kv2.d;
        const int start = kvq_start(a.d_pos, seq, a.pos_off, a.ctx);
        const int64_t b = start / kKvBlock + (int64_t)bi;
        if (start < 0 || b >= a.ctx / kKvBlock || b * kKvBlock >= (int64_t)start + a.n_tok) return;
        if (kv2 < a.n_kv) kvq_store_k<TY, HD>(a, mode, seq, kv2, start, b);
        else kvq_store_v<TY, HD>(a, seq, kv2 - a.n_kv, start, b, sh);
        return;
    }
    w -= blocks_kv;
    if (mode != kRotAny) {
        kvq_store_q<HD>(a, mode, w);
        return;
    }
    const int lane = threadIdx.x & 63, hv = w * 4 + (threadIdx.x >> 6), row = a.by_heads(hv);
    if (row >= a.n_seq * a.n_tok) return;
    const int h = hv - row * a.by_heads.d, seq = a.by_tok(row), start = kvq_start(a.d_pos, seq, a.pos_off, a.ctx);
    const int64_t p = (int64_t)start + (row - seq * a.n_tok);
    if (start < 0 || p >= a.ctx) return;
    const float* x = a.qkv + (int64_t)row * a.ldqkv + (size_t)h * HD;
    float* q = a.q + (int64_t)row * a.ldq + (size_t)h * HD;
    float v[HD / 64];
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) v[e] = kvq_rotated(x, lane + 64 * e, a.layout, a.rot, a.rope + (a.rope_off + p) * (a.rot >> 1));
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) q[lane + 64 * e] = v[e];
}

// ── read-back ────────────────────────────────────────────────────────────────
// A few rows: a thread per value.
template <int TY, int HD> __global__ __launch_bounds__(256) void k_kvq_load(const uint8_t* kc, const uint8_t* vc,
                                                                            int n_kv, int ctx, const int32_t* d_pos,
                                                                            int pos_off, int n, float* ko, float* vo) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(t % HD);
    const int64_t j = t / HD;
    if (j >= n) return;
    const int seq = blockIdx.y / n_kv;
    const bool is_v = blockIdx.z == (ko ? 1 : 0);
    const int64_t p = (int64_t)(d_pos ? d_pos[seq] : 0) + pos_off + j;
    float y = 0.f;
    if (p >= 0 && p < ctx) {
        const uint8_t* blk = (is_v ? vc : kc) + ((size_t)blockIdx.y * (ctx / kKvBlock) + p / kKvBlock) * kvq_block_bytes(TY, HD);
        const int q = (int)(p & 63);
        const KvqAt at = is_v ? kvq_at_v<TY, HD>(q, d) : kvq_at_k<TY, HD>(q, d);
        if constexpr (TY == ORC_F16) y = (float)*(const _Float16*)(blk + at.code);
        else {
            int u = blk[at.code];
            if constexpr (TY == ORC_KV_Q4) u = at.high ? u >> 4 : u & 15;
            y = (float)(u - kvq_levels(TY) - 1) * kvq_scale(blk[at.scale]) * 0.0625f;
        }
    }
    (is_v ? vo : ko)[((size_t)blockIdx.y * n + j) * HD + d] = y;
}

// Many rows: a workgroup per 64-position block of one head's K or V. Codes are loaded as the whole pieces they are
// stored in, values turned into rows in LDS, and rows stored in order. 32768 rows of 4 heads of 128, 8 bits: 32 us, 5.3
// TB/s (a thread per value: 98 us).
template <int TY, int HD> __global__ __launch_bounds__(256) void k_kvq_load_blocks(const uint8_t* kc, const uint8_t* vc,
                                                                                   int n_kv, int ctx, const int32_t* d_pos,
                                                                                   int pos_off, int n, float* ko, float* vo) {
    constexpr int BB = kvq_block_bytes(TY, HD), CB = kvq_code_bytes(TY, HD), L = HD / 4;
    __shared__ float sh[kKvBlock][HD + 4];
    const int tid = threadIdx.x, seq = blockIdx.y / n_kv;
    const bool is_v = blockIdx.z == (ko ? 1 : 0);
    const int64_t start = (int64_t)(d_pos ? d_pos[seq] : 0) + pos_off, b = (start >> 6) + blockIdx.x;
    const int64_t j0 = b * kKvBlock - start;  // output row of the block's first one
    if (j0 >= n) return;
    float* out = (is_v ? vo : ko) + (size_t)blockIdx.y * n * HD;
    const bool in = b >= 0 && b < ctx / kKvBlock;
    if (in) {
        const uint8_t* blk = (is_v ? vc : kc) + ((size_t)blockIdx.y * (ctx / kKvBlock) + b) * BB;
        const int lane = tid & 63, c = lane & 15, g = lane >> 4;
        constexpr float bias = kvq_levels(TY) + 1;
        if (!is_v) {  // a wave takes a tile of 16 keys
            const int tile = tid >> 6;
            float s = 0.f;
            if constexpr (TY != ORC_F16) s = kvq_scale(blk[CB + (g * L / kKvGroup) * 64 + c * 4 + tile]) * 0.0625f;
            float* row = &sh[tile * 16 + c][g * L];
            constexpr int kP = TY == ORC_F16 ? 8 : L < 16 ? L : 16;  // values of a piece (4 bits: all)
            if constexpr (TY == ORC_F16) {
#pragma unroll
                for (int e = 0; e < L; e += kP) {
                    const kq_h8 h = *(const kq_h8*)(blk + tile * 32 * HD + e / 8 * 1024 + lane * 16);
#pragma unroll
                    for (int k = 0; k < 8; k += 4) *(kq_f4*)(row + e + k) = kq_f4{(float)h[k], (float)h[k + 1], (float)h[k + 2], (float)h[k + 3]};
                }
            } else if constexpr (TY == ORC_KV_Q8) {
#pragma unroll
                for (int e = 0; e < L; e += 16) {
                    const u32x4 w = *(const u32x4*)(blk + tile * 16 * HD + e / 16 * 1024 + lane * 16);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *(kq_f4*)(row + e + k * 4) = kq_f4{(ubyte_f(w[k], 0) - bias) * s, (ubyte_f(w[k], 1) - bias) * s,
                                                           (ubyte_f(w[k], 2) - bias) * s, (ubyte_f(w[k], 3) - bias) * s};
                }
            } else {
                const uint8_t* at = blk + tile * 8 * HD + lane * (L / 2);
#pragma unroll
                for (int k = 0; k < L / 8; ++k) {
                    const uint32_t w = *(const uint32_t*)(at + k * 4), lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
                    *(kq_f4*)(row + k * 4) = kq_f4{(ubyte_f(lo, 0) - bias) * s, (ubyte_f(lo, 1) - bias) * s,
                                                   (ubyte_f(lo, 2) - bias) * s, (ubyte_f(lo, 3) - bias) * s};
                    *(kq_f4*)(row + L / 2 + k * 4) = kq_f4{(ubyte_f(hi, 0) - bias) * s, (ubyte_f(hi, 1) - bias) * s,
                                                           (ubyte_f(hi, 2) - bias) * s, (ubyte_f(hi, 3) - bias) * s};
                }
            }
        } else {  // a wave takes every fourth dim tile
            for (int dt = tid >> 6; dt < HD / 16; dt += 4) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {  // (step, half): four keys
                    float v[4];
                    if constexpr (TY == ORC_F16) {
                        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
                        const h4 h = *(const h4*)(blk + dt * 2048 + (q >> 1) * 1024 + lane * 16 + (q & 1) * 8);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (float)h[i];
                    } else {
                        uint32_t w = *(const uint32_t*)(blk + (TY == ORC_KV_Q4 ? dt >> 1 : dt) * 1024 + lane * 16 + q * 4);
                        if constexpr (TY == ORC_KV_Q4) w = (w >> (dt & 1) * 4) & 0x0F0F0F0Fu;
                        const uint32_t s = *(const uint32_t*)(blk + CB + (dt >> 1) * 64 + g * 16 + q * 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (ubyte_f(w, i) - bias) * (kvq_scale((s >> (8 * i)) & 0xFF) * 0.0625f);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) sh[q * 16 + g * 4 + i][dt * 16 + c] = v[i];
                }
            }
        }
    }
    __syncthreads();
    for (int it = tid; it < kKvBlock * HD / 4; it += 256) {
        const int r = it / (HD / 4), d = it % (HD / 4) * 4;
        if (j0 + r < 0 || j0 + r >= n) continue;
        kq_f4 y = {0.f, 0.f, 0.f, 0.f};
        if (in) y = *(const kq_f4*)&sh[r][d];
        *(kq_f4*)(out + (j0 + r) * HD + d) = y;
    }
}

}  // namespace orc

using namespace orc;

extern "C" size_t orc_kvq_bytes(int type, int n_seq, int n_kv, int ctx, int head_dim) {
    if (!kvq_type_ok(type) || (head_dim != 64 && head_dim != 128) || n_seq < 1 || n_kv < 1 || ctx < 1 || ctx % kKvBlock)
        return 0;
    size_t bytes = (size_t)n_seq * n_kv;  // below 2^62
    if (__builtin_mul_overflow(bytes, (size_t)(ctx / kKvBlock) * kvq_block_bytes(type, head_dim), &bytes)) return 0;
    return bytes;
}

extern "C" int orc_rope_table(float* d_rope, int pos0, int n_pos, int rot_dim, double base,
                              const orc_rope_scaling* sc, orc_stream_t s) {
    if (!initialized()) return set_error(ORC_E_NOINIT, "orc_init not called");
    const int kind = sc ? sc->kind : ORC_ROPE_PLAIN;
    if (pos0 < 0 || n_pos < 0 || (int64_t)pos0 + n_pos > 0x7fffffff || rot_dim < 2 || rot_dim > 128 || rot_dim % 2 ||
        !(base > 1.0) || !std::isfinite(base) || (n_pos && (!d_rope || ((uintptr_t)d_rope & 7))))
        return set_error(ORC_E_INVALID, "rope_table: bad args (an even rot_dim of 2..128, base above 1)");
    if (kind < ORC_ROPE_PLAIN || kind > ORC_ROPE_YARN) return set_error(ORC_E_INVALID, "rope_table: no such scaling");
    RopeFreqs fr{};
    const double tau = 6.283185307179586476925;
    double mul = 1.0;
    if (kind != ORC_ROPE_PLAIN) {
        if (!(sc->factor >= 1.f) || !std::isfinite(sc->factor))
            return set_error(ORC_E_INVALID, "rope_table: the scaling's factor must be 1 or more");
        if (kind != ORC_ROPE_LINEAR && (sc->orig_ctx < 1 || !(sc->low > 0.f) || !(sc->high > sc->low) || !std::isfinite(sc->high)))
            return set_error(ORC_E_INVALID, "rope_table: the scaling needs orig_ctx >= 1 and 0 < low < high");
        if (!(sc->mscale >= 0.f) || !std::isfinite(sc->mscale))
            return set_error(ORC_E_INVALID, "rope_table: mscale must be 0 (the default) or positive");
    }
    double lo = 0, hi = 0;
    if (kind == ORC_ROPE_YARN) {
        // pair index at which a frequency makes `turns` turns over the original context
        auto pair_of = [&](double turns) { return rot_dim * std::log(sc->orig_ctx / (tau * turns)) / (2 * std::log(base)); };
        lo = std::max(0.0, std::floor(pair_of(sc->high)));
        hi = std::min(rot_dim - 1.0, std::ceil(pair_of(sc->low)));
        mul = sc->mscale > 0.f ? sc->mscale : 0.1 * std::log((double)sc->factor) + 1.0;
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (kind == ORC_ROPE_LINEAR) f /= sc->factor;
        else if (kind == ORC_ROPE_BANDS) {
            const double turns = sc->orig_ctx * f / tau;
            const double keep = std::clamp((turns - sc->low) / ((double)sc->high - sc->low), 0.0, 1.0);
            f = keep * f + (1 - keep) * f / sc->factor;
        } else if (kind == ORC_ROPE_YARN) {
            const double slow = std::clamp((i - lo) / std::max(hi - lo, 0.001), 0.0, 1.0);
            f = (1 - slow) * f + slow * f / sc->factor;
        }
        fr.f[i] = f;
    }
    if (!n_pos) return ORC_OK;
    const int pairs = rot_dim / 2, rows = 256 / pairs;
    // 16 rows a thread where that still makes two workgroups for every CU, else 4
    const int steps = n_pos / (rows * 16) >= 512 ? 16 : 4;
    const int64_t blocks = ((int64_t)n_pos + rows * steps - 1) / (rows * steps);
    if (blocks > 0xffffff00ll / 256) return set_error(ORC_E_INVALID, "rope_table: too many positions");
    hipLaunchKernelGGL(k_rope_table, dim3((unsigned)blocks), dim3(256), 0, resolve_stream(s), (float2*)d_rope, (int64_t)pos0,
                       (int64_t)n_pos, pairs, rows, steps, fr, mul);
    ORC_LAUNCH_CHECK();
    return ORC_OK;
}

extern "C" int orc_kvq_store(int type, const float* d_qkv, int ldqkv, int n_seq, int n_tok, int n_heads, int n_kv,
                             int head_dim, int rope_layout, int rot_dim, const float* d_rope, int rope_off,
                             const int32_t* d_pos, int pos_off, float* d_q, int ldq, void* d_kc, void* d_vc, int ctx,
                             orc_stream_t s) {
    if (!initialized()) return set_error(ORC_E_NOINIT, "orc_init not called");
    if (!kvq_type_ok(type)) return set_error(ORC_E_UNSUPPORTED, "kvq_store: cache types are F16, KV_Q8 and KV_Q4");
    if (head_dim != 64 && head_dim != 128) return set_error(ORC_E_UNSUPPORTED, "kvq_store: head_dim must be 64 or 128");
    const int64_t vecs = (int64_t)n_heads + 2 * (int64_t)n_kv;
    if (n_seq < 0 || n_tok < 0 || n_heads < 1 || n_kv < 1 || ldqkv < vecs * head_dim || ldq < (int64_t)n_heads * head_dim ||
        ldqkv % 4 || ldq % 4 || (rope_layout != ORC_ROPE_HALF && rope_layout != ORC_ROPE_PAIRS) || rot_dim < 0 ||
        rot_dim > head_dim || rot_dim % 2 || rope_off < 0 || ctx < 1 || ctx % kKvBlock)
        return set_error(ORC_E_INVALID, "kvq_store: bad args (ctx a multiple of 64, rows a multiple of 4 floats)");
    if (!n_seq || !n_tok) return ORC_OK;
    if (!d_qkv || !d_q || !d_kc || !d_vc || (rot_dim && !d_rope) || ((uintptr_t)d_qkv & 15) || ((uintptr_t)d_q & 15) ||
        ((uintptr_t)d_kc & 15) || ((uintptr_t)d_vc & 15) || ((uintptr_t)d_rope & 7))
        return set_error(ORC_E_INVALID, "kvq_store: null or misaligned pointer");
    if (d_q == d_qkv && ldq != ldqkv) return set_error(ORC_E_INVALID, "kvq_store: q in place needs ldq = ldqkv");
    if (!d_pos && (pos_off < 0 || (int64_t)pos_off + n_tok > ctx))
        return set_error(ORC_E_INVALID, "kvq_store: positions must fit the cache");
    const int64_t rows = (int64_t)n_seq * n_tok;
    if (rows > 0x7fffffff) return set_error(ORC_E_INVALID, "kvq_store: too many rows");
    const int64_t blocks = (rows * vecs + 3) / 4;
    if (n_tok < kStoreBlocks && blocks > 0xffffff00ll / 256) return set_error(ORC_E_INVALID, "kvq_store: too many rows");
    StoreArgs a{d_qkv, ldqkv, n_seq, n_tok, n_heads, n_kv, rope_layout, rot_dim, (const float2*)d_rope, rope_off,
                      d_pos, pos_off, d_q, ldq, (uint8_t*)d_kc, (uint8_t*)d_vc, ctx, kvq_div((int)vecs), kvq_div(n_tok),
                      kvq_div(n_heads)};
    const hipStream_t st = resolve_stream(s);
    auto each = [&](auto f) {  // f of (type, head size)
        using std::integral_constant;
        auto with = [&](auto ty) { head_dim == 64 ? f(ty, integral_constant<int, 64>()) : f(ty, integral_constant<int, 128>()); };
        if (type == ORC_F16) with(integral_constant<int, ORC_F16>());
        else if (type == ORC_KV_Q8) with(integral_constant<int, ORC_KV_Q8>());
        else with(integral_constant<int, ORC_KV_Q4>());
    };
    if (n_tok < kStoreBlocks)
        each([&](auto ty, auto hd) {
            hipLaunchKernelGGL((k_kvq_store<decltype(ty)::value, decltype(hd)::value>), dim3((unsigned)blocks), dim3(256), 0, st, a);
        });
    else {
        const int mode = rope_layout == ORC_ROPE_PAIRS || !rot_dim ? kRotPairs : rot_dim == head_dim ? kRotHalf : kRotAny;
        const int nblk = (int)(((int64_t)n_tok + 2 * kKvBlock - 2) / kKvBlock);  // blocks that n_tok rows may touch
        if (mode != kRotAny) a.by_heads = kvq_div((n_heads + kQHeads - 1) / kQHeads);
        const int64_t kv = (int64_t)n_seq * 2 * n_kv * nblk, q = rows * a.by_heads.d;
        const int64_t all = kv + (mode == kRotAny ? (q + 3) / 4 : (q * (head_dim / 8) + 255) / 256);
        if (all > 0xffffff00ll / 256) return set_error(ORC_E_INVALID, "kvq_store: too many rows");
        each([&](auto ty, auto hd) {
            hipLaunchKernelGGL((k_kvq_store_blocks<decltype(ty)::value, decltype(hd)::value>), dim3((unsigned)all), dim3(256), 0, st,
                               a, mode, kvq_div(nblk), kvq_div(2 * n_kv), (int)kv);
        });
    }
    ORC_LAUNCH_CHECK();
    return ORC_OK;
}

extern "C" int orc_kvq_load(int type, const void* d_kc, const void* d_vc, int n_seq, int n_kv, int head_dim, int ctx,
                            const int32_t* d_pos, int pos_off, int n, float* d_k, float* d_v, orc_stream_t s) {
    if (!initialized()) return set_error(ORC_E_NOINIT, "orc_init not called");
    if (!kvq_type_ok(type)) return set_error(ORC_E_UNSUPPORTED, "kvq_load: cache types are F16, KV_Q8 and KV_Q4");
    if (head_dim != 64 && head_dim != 128) return set_error(ORC_E_UNSUPPORTED, "kvq_load: head_dim must be 64 or 128");
    if (n_seq < 0 || n_kv < 1 || n < 0 || ctx < 1 || ctx % kKvBlock)
        return set_error(ORC_E_INVALID, "kvq_load: bad args (ctx a multiple of 64)");
    if (!d_kc != !d_k || !d_vc != !d_v) return set_error(ORC_E_INVALID, "kvq_load: a cache and its rows come together");
    if (((uintptr_t)d_kc | (uintptr_t)d_vc | (uintptr_t)d_k | (uintptr_t)d_v) & 15)
        return set_error(ORC_E_INVALID, "kvq_load: misaligned pointer");
    if (!d_pos && (pos_off < 0 || (int64_t)pos_off + n > ctx))
        return set_error(ORC_E_INVALID, "kvq_load: rows must lie in the cache");
    const int z = (d_k ? 1 : 0) + (d_v ? 1 : 0);
    if (!n_seq || !n || !z) return ORC_OK;
    if ((int64_t)n_seq * n_kv > 65535) return set_error(ORC_E_INVALID, "kvq_load: more than 65535 sequence heads");
    const bool many = n >= kStoreBlocks;
    const int64_t blocks = many ? ((int64_t)n + 2 * kKvBlock - 2) / kKvBlock : ((int64_t)n * head_dim + 255) / 256;
    if (blocks > 0xffffff00ll / 256) return set_error(ORC_E_INVALID, "kvq_load: too many rows");
    const dim3 grid((unsigned)blocks, (unsigned)(n_seq * n_kv), (unsigned)z);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, resolve_stream(s), (const uint8_t*)d_kc, (const uint8_t*)d_vc, n_kv,
                           ctx, d_pos, pos_off, n, d_k, d_v);
    };
    auto with = [&](auto ty) {
        constexpr int T = decltype(ty)::value;
        if (many) head_dim == 64 ? go(k_kvq_load_blocks<T, 64>) : go(k_kvq_load_blocks<T, 128>);
        else head_dim == 64 ? go(k_kvq_load<T, 64>) : go(k_kvq_load<T, 128>);
    };
    if (type == ORC_F16) with(std::integral_constant<int, ORC_F16>());
    else if (type == ORC_KV_Q8) with(std::integral_constant<int, ORC_KV_Q8>());
    else with(std::integral_constant<int, ORC_KV_Q4>());
    ORC_LAUNCH_CHECK();
    return ORC_OK;
}
