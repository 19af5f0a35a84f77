// A KV cache in fewer bits (gfx950): the rotary table with scaled frequencies,
// the write of new tokens' K and V (rotary positions, quantisation, the
// cache's layout) and the read-back to fp32 rows. Layout and formats:
// orc_kvq.hpp; attention over such caches: orc_attn_kvq.hip. No counterpart in
// the reference, whose cache is fp32 and whose rotation is the rotate-half of
// core/ops.cpp:440-485.
#include "orc_kvq.hpp"

#include <algorithm>
#include <cmath>

namespace orc {

// ── rotary table ─────────────────────────────────────────────────────────────
struct RopeFreqs {
    double f[64];  // angle of one position, per pair
};

// (cos, sin) of pos f_i times the table's factor, formed in 64 bits: an angle
// of 2^17 radians has 2^-7 left of a 24-bit mantissa, and sums of rounded
// angles drift with the position.
__global__ __launch_bounds__(256) void k_rope_table(float2* out, int64_t pos0, int64_t n, int pairs, RopeFreqs fr,
                                                    double mul) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= n * pairs) return;
    const int64_t p = t / pairs;
    double s, c;
    sincos((double)(pos0 + p) * fr.f[t - p * pairs], &s, &c);
    out[t] = make_float2((float)(c * mul), (float)(s * mul));
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

// One wave per head vector: q heads are rotated, K heads rotated and
// quantised, V heads quantised. A scale group is 32 lanes.
template <int TY, int HD> __global__ __launch_bounds__(256) void k_kvq_store(StoreArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int vecs = a.n_heads + 2 * a.n_kv;
    const int64_t row = unit / vecs;
    if (row >= (int64_t)a.n_seq * a.n_tok) return;
    const int h = (int)(unit - row * vecs), seq = (int)(row / a.n_tok), t = (int)(row - (int64_t)seq * a.n_tok);
    const int start = kvq_start(a.d_pos, seq, a.pos_off, a.ctx);
    if (start < 0 || start + (int64_t)t >= a.ctx) return;
    const int p = start + t;
    const float* x = a.qkv + row * a.ldqkv + (size_t)h * HD;
    const float2* cs = a.rope + (a.rope_off + p) * (a.rot >> 1);
    const bool is_v = h >= a.n_heads + a.n_kv;
    constexpr int E = HD / 64;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = kvq_rotated(x, lane + 64 * e, a.layout, is_v ? 0 : a.rot, cs);
    if (h < a.n_heads) {
        float* q = a.q + row * a.ldq + (size_t)h * HD;
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

// ── read-back ────────────────────────────────────────────────────────────────
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

}  // namespace orc

using namespace orc;

extern "C" size_t orc_kvq_bytes(int type, int n_seq, int n_kv, int ctx, int head_dim) {
    if (!kvq_type_ok(type) || (head_dim != 64 && head_dim != 128) || n_seq < 1 || n_kv < 1 || ctx < 1 || ctx % kKvBlock)
        return 0;
    return (size_t)n_seq * n_kv * (ctx / kKvBlock) * kvq_block_bytes(type, head_dim);
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
    const int64_t total = (int64_t)n_pos * (rot_dim / 2);
    if (total > 0xffffff00ll) return set_error(ORC_E_INVALID, "rope_table: more than 2^32 pairs");
    hipLaunchKernelGGL(k_rope_table, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, resolve_stream(s),
                       (float2*)d_rope, (int64_t)pos0, (int64_t)n_pos, rot_dim / 2, fr, mul);
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
    const int64_t blocks = ((int64_t)n_seq * n_tok * vecs + 3) / 4;
    if (blocks > 0xffffff00ll / 256) return set_error(ORC_E_INVALID, "kvq_store: too many rows");
    const StoreArgs a{d_qkv, ldqkv, n_seq, n_tok, n_heads, n_kv, rope_layout, rot_dim, (const float2*)d_rope, rope_off,
                      d_pos, pos_off, d_q, ldq, (uint8_t*)d_kc, (uint8_t*)d_vc, ctx};
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, resolve_stream(s), a); };
    if (head_dim == 64)
        type == ORC_F16 ? go(k_kvq_store<ORC_F16, 64>) : type == ORC_KV_Q8 ? go(k_kvq_store<ORC_KV_Q8, 64>) : go(k_kvq_store<ORC_KV_Q4, 64>);
    else
        type == ORC_F16 ? go(k_kvq_store<ORC_F16, 128>) : type == ORC_KV_Q8 ? go(k_kvq_store<ORC_KV_Q8, 128>) : go(k_kvq_store<ORC_KV_Q4, 128>);
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
    const int64_t blocks = ((int64_t)n * head_dim + 255) / 256;
    if (blocks > 0xffffff00ll / 256) return set_error(ORC_E_INVALID, "kvq_load: too many rows");
    if ((int64_t)n_seq * n_kv > 65535) return set_error(ORC_E_INVALID, "kvq_load: more than 65535 sequence heads");
    const dim3 grid((unsigned)blocks, (unsigned)(n_seq * n_kv), (unsigned)z);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, resolve_stream(s), (const uint8_t*)d_kc, (const uint8_t*)d_vc, n_kv,
                           ctx, d_pos, pos_off, n, d_k, d_v);
    };
    if (head_dim == 64)
        type == ORC_F16 ? go(k_kvq_load<ORC_F16, 64>) : type == ORC_KV_Q8 ? go(k_kvq_load<ORC_KV_Q8, 64>) : go(k_kvq_load<ORC_KV_Q4, 64>);
    else
        type == ORC_F16 ? go(k_kvq_load<ORC_F16, 128>) : type == ORC_KV_Q8 ? go(k_kvq_load<ORC_KV_Q8, 128>) : go(k_kvq_load<ORC_KV_Q4, 128>);
    ORC_LAUNCH_CHECK();
    return ORC_OK;
}
