// Attention over caches in fewer bits (gfx950): n_seq sequences of n_tok new
// tokens over a prefix that all share and rows of their own (orc_attn_kvq).
// The cache's layout and values: orc_kvq.hpp.
//
// Scores are formed transposed, S^T = K Q^T, so a lane holds one query row's
// scores of 16 of a block's 64 keys, a row's softmax needs two exchanges
// between lane groups for its maximum and none for the weights, and the
// weights are already the second operand of O^T = V^T P^T. q and the weights are
// two fp16 halves (22 bits), K and V fp16 numbers as stored: every product is
// exact.
// Sums: the matrix cores round toward minus infinity, so each block's products
// start from zero and are added up in fp32 on the vector ALUs, and every other
// block's weights are negated, so that what is left of that drift cancels.
// The weights carry 2^15 (they cancel against their sum), which keeps both
// halves normal fp16 numbers down to weights of 2^-29.
// How the work is cut (ka_plan): the rows of one kv head, tokens times the
// query heads of its group, in tiles of 16 or 32 (k_attn_kvq: the waves share
// out the keys), 64 or 128 (k_attn_kvq_tile: the waves share the keys'
// operands); the keys in chunks where the tiles alone leave CUs idle, merged by
// k_attn_kvq_merge. With a shared prefix its jobs take the rows of all
// sequences, so the prefix is read once per row tile and not per sequence, and
// the own rows are chunks of their own in the same launch (k_attn_kvq_both).
// Bounds: few rows are bound by latency (a launch's first load is 1 us away, a
// block of 64 keys takes a wave 1.2 us alone) or by the cache's bytes (64
// sequences of 4000 rows, 8 kv heads of 128, 8 bits: 5.5 TB/s), many rows by
// the matrix and vector instructions together, which hardly overlap on this
// card (a 16x16x32 product and four fp32 multiply-adds, four waves a SIMD:
// 11.7 ns against 8.7 and 4.4 alone).
#include "orc_kvq.hpp"

#include <algorithm>
#include <type_traits>

namespace orc {

struct KaArgs {
    const float* q;
    int ldq, n_seq, n_tok, n_heads, n_kv, group;
    const uint8_t *pk, *pv, *kc, *vc;
    int prefix, pctx, ctx;
    const int32_t* d_pos;
    int pos_off, limit;
    float* out;
    int ldo;
    float* part_o;   // [slot][row][hd], row = token n_heads + head
    float2* part_ml; // [slot][row] (maximum, sum)
    int n_rows;      // n_seq n_tok n_heads
    // jobs: prefix ones (shared form only), then own ones
    int shared, tiles_p, cp, tiles_o, co;
    int jobs_p, jobs_o;
    KvqDiv by_group, by_kv, by_tiles_p, by_cp, by_tiles_o, by_co, by_heads, by_tok;
};

// Blocks [b0, b1) of chunk c of n chunks over nb blocks.
__device__ __forceinline__ void ka_chunk(int nb, const KvqDiv& n, int c, int& b0, int& b1) {
    const int per = n(nb + n.d - 1);
    b0 = min(nb, c * per);
    b1 = min(nb, b0 + per);
}

// What a workgroup has to do: rows [r0, r1) of kv head `kv` (row = token G +
// head in its group, tokens of all sequences in a row), key blocks [b0, b1) of
// the prefix's nbp blocks and then the own ones of sequence seq.
struct KaJob {
    int kv, seq, r0, r1, b0, b1, slot, start, len;
};

// The rows, from the grid alone.
__device__ __forceinline__ bool ka_rows(const KaArgs& a, int m_p, int m_o, KaJob& j) {
    // Every XCD takes an eighth of the prefix jobs, then an eighth of the own ones, each in order: the row tiles of one
    // chunk, which read the same keys, share its L2.
    const int per_p = (a.jobs_p + 7) / 8, per_o = (a.jobs_o + 7) / 8, x = blockIdx.x & 7, i = blockIdx.x >> 3;
    const bool pre = i < per_p;
    const int w = pre ? x * per_p + i : x * per_o + i - per_p;
    if (w >= (pre ? a.jobs_p : a.jobs_o)) return false;
    if (pre) {
        const int t = a.by_tiles_p(w), tile = w - t * a.tiles_p;
        j.kv = a.by_cp(t);
        j.slot = t - j.kv * a.cp;
        j.seq = -1;
        j.r0 = tile * m_p;
        j.r1 = min(j.r0 + m_p, a.n_seq * a.n_tok * a.group);
        return true;
    }
    // The longest rows first, every other 32 of them the other way round: an XCD's 32 CUs take workgroups in turn, and
    // so each gets long and short ones.
    const int t = a.by_tiles_o(w);
    int tile = w - t * a.tiles_o;
    if ((tile & 32) && (tile | 31) < a.tiles_o) tile ^= 31;
    tile = a.tiles_o - 1 - tile;
    const int sk = a.by_co(t), rows = a.n_tok * a.group;
    j.slot = a.cp + t - sk * a.co;
    j.seq = a.by_kv(sk);
    j.kv = sk - j.seq * a.n_kv;
    j.r0 = j.seq * rows + tile * m_o;
    j.r1 = min(j.r0 + m_o, (j.seq + 1) * rows);
    return true;
}

// The keys, which may depend on a position in device memory.
__device__ __forceinline__ void ka_keys(const KaArgs& a, KaJob& j) {
    const int nbp = (a.prefix + kKvBlock - 1) / kKvBlock;
    if (j.seq < 0) {
        j.start = j.len = 0;
        ka_chunk(nbp, a.by_cp, j.slot, j.b0, j.b1);
        return;
    }
    j.start = kvq_start(a.d_pos, j.seq, a.pos_off, a.limit);
    j.len = j.start < 0 ? 0 : (int)min((int64_t)j.start + a.n_tok, (int64_t)a.limit);
    const int first = a.shared ? nbp : 0;
    const int nb = j.len ? nbp - first + (j.len + kKvBlock - 1) / kKvBlock : 0;
    ka_chunk(nb, a.by_co, j.slot - a.cp, j.b0, j.b1);
    j.b0 += first;
    j.b1 += first;
    // nothing behind the tile's last token
    const int last = min(j.start + a.by_group(j.r1 - 1) - j.seq * a.n_tok, j.len - 1);
    if (j.len) j.b1 = min(j.b1, nbp + last / kKvBlock + 1);
}

// ── operands ─────────────────────────────────────────────────────────────────
// Bytes u of w (codes plus a bias) times their scales as fp16: 0x6400 | u is
// 1024 + u.
__device__ __forceinline__ void ka_cvt4(uint32_t w, kq_h2 s01, kq_h2 s23, _Float16 bias, kq_h2& o01, kq_h2& o23) {
    const kq_h2 b = {bias, bias};
    o01 = (__builtin_bit_cast(kq_h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - b) * s01;
    o23 = (__builtin_bit_cast(kq_h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - b) * s23;
}
__device__ __forceinline__ kq_h8 ka_join(kq_h2 a, kq_h2 b, kq_h2 c, kq_h2 d) {
    return kq_h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

template <int TY> constexpr float ka_bias() { return 1024.f + kvq_levels(TY) + 1; }

// One key tile's raw K bytes of a lane, and its operands.
template <int TY, int HD> struct KaK {
    static constexpr int kN = TY == ORC_F16 ? HD / 32 : TY == ORC_KV_Q8 ? HD / 64 : 1;
    u32x4 r[kN];
    __device__ __forceinline__ void load(const uint8_t* blk, int tile, int lane) {
        const uint8_t* p = blk + tile * (16 * HD * kvq_bits(TY) / 8);
        if constexpr (TY == ORC_KV_Q4 && HD == 64) {
            const u32x2 v = *(const u32x2*)(p + lane * 8);
            r[0].x = v.x;
            r[0].y = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i) r[i] = *(const u32x4*)(p + i * 1024 + lane * 16);
        }
    }
    // operand of dims j 8 .. j 8 + 7 of the lane; sc: the tile's scale twice
    __device__ __forceinline__ kq_h8 op(int j, kq_h2 sc) const {
        if constexpr (TY == ORC_F16) return __builtin_bit_cast(kq_h8, r[j]);
        else {
            uint32_t w0, w1;
            if constexpr (TY == ORC_KV_Q8) {
                w0 = r[j / 2][(j & 1) * 2];
                w1 = r[j / 2][(j & 1) * 2 + 1];
            } else {
                constexpr int half = HD / 64;  // steps in the low halves
                const int i = j % half * 2, sh = j / half * 4;
                w0 = (r[0][i] >> sh) & 0x0F0F0F0Fu;
                w1 = (r[0][i + 1] >> sh) & 0x0F0F0F0Fu;
            }
            kq_h2 o[4];
            ka_cvt4(w0, sc, sc, (_Float16)ka_bias<TY>(), o[0], o[1]);
            ka_cvt4(w1, sc, sc, (_Float16)ka_bias<TY>(), o[2], o[3]);
            return ka_join(o[0], o[1], o[2], o[3]);
        }
    }
};

// Scale of tile T from the dword of the lane's key and group.
__device__ __forceinline__ kq_h2 ka_scale_k(uint32_t w, int T) {
    return __builtin_bit_cast(kq_h2, __builtin_amdgcn_perm(0u, w, 0x000C000Cu | (T << 8) | (T << 24)) >> 1);
}
// Scales of bytes e, e + 1 of w; sign 0x80008000 negates them.
__device__ __forceinline__ kq_h2 ka_scale_v(uint32_t w, int e, uint32_t sign = 0) {
    return __builtin_bit_cast(kq_h2, __builtin_amdgcn_perm(0u, w, 0x000C000Cu | (e << 8) | ((e + 1) << 24)) >> 1 ^ sign);
}

// ── infinities and NaN in V rows that only some of a tile's rows see ─────────
// A product of the matrix cores takes every row through every key, and 0 times a NaN is one. In the blocks where a call's
// own tokens see different numbers of keys, such values are taken out of V and noted, as a 64-bit mask of the block's
// keys for each head dim, and the rows that do see them are made NaN at the end.
__device__ __forceinline__ bool ka_odd_scales(uint32_t w) {  // a scale byte of all exponent bits among the four?
    const uint32_t x = ~w & 0xF8F8F8F8u;
    return (x - 0x01010101u) & ~x & 0x80808080u;
}
__device__ __forceinline__ bool ka_odd_halves(uint32_t w) {
    return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
}
// Which of the 16 bytes of sc are odd (bit e: byte e); those become 0 (a scale of 0).
__device__ __forceinline__ uint32_t ka_take_scales(u32x4& sc) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if ((sc[e >> 2] & (0xF8u << (8 * (e & 3)))) == 0xF8u << (8 * (e & 3))) {
            m |= 1u << e;
            sc[e >> 2] &= ~(0xFFu << (8 * (e & 3)));
        }
    return m;
}
// The same for the 16 halves of a dim, v0 and v1 (32 keys each).
__device__ __forceinline__ uint32_t ka_take_halves(u32x4& v0, u32x4& v1) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        u32x4& v = e < 8 ? v0 : v1;
        const int w = (e & 7) >> 1, sh = (e & 1) * 16;
        if ((v[w] & (0x7C00u << sh)) == 0x7C00u << sh) {
            m |= 1u << e;
            v[w] &= ~(0xFFFFu << sh);
        }
    }
    return m;
}
// The lane groups' bits (s, q, i) of a dim as a mask of keys s 32 + q 16 + g 4 + i.
__device__ __forceinline__ void ka_note(uint64_t* list, int dim, uint32_t m, int g) {
    uint32_t lo = ((m & 15) | (m >> 4 & 15) << 16) << (g * 4), hi = ((m >> 8 & 15) | (m >> 12 & 15) << 16) << (g * 4);
#pragma unroll
    for (int d = 16; d < 64; d *= 2) {
        lo |= __shfl_xor(lo, d, 64);
        hi |= __shfl_xor(hi, d, 64);
    }
    if (g == 0) list[dim] = (uint64_t)hi << 32 | lo;
}
// Four dims' values of a row that sees n of the block's keys: NaN where it sees an odd one.
__device__ __forceinline__ void ka_spoil(kq_f4& o, const uint64_t* list, int n) {
    const uint64_t sees = n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (list[i] & sees) o[i] = __builtin_nanf("");
}
// What the workgroup's NW waves noted of up to N blocks (a tile of 128 tokens ends in up to three).
template <int HD, int N, int NW> struct KaOdd {
    uint64_t list[N][HD];
    int any[N][NW];
};

// V bytes of one dim tile (both tiles of a pair for 4 bits) of a lane.
template <int TY, int HD> struct KaV {
    static constexpr int kN = TY == ORC_F16 ? HD / 8 : TY == ORC_KV_Q8 ? HD / 16 : HD / 32;
    u32x4 r[kN];
    u32x4 sc[TY == ORC_F16 ? 1 : HD / 32];
    __device__ __forceinline__ void load(const uint8_t* blk, int lane) {
#pragma unroll
        for (int i = 0; i < kN; ++i) r[i] = *(const u32x4*)(blk + i * 1024 + lane * 16);
        if constexpr (TY != ORC_F16) {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
                sc[i] = *(const u32x4*)(blk + kvq_code_bytes(TY, HD) + i * 64 + (lane >> 4) * 16);
        }
    }
    // Makes each register group one whole value here. Without it the compiler (ROCm 7.2) took parts of them for
    // temporaries between keep() and the products, where the next block's load is conditional: wrong results.
    __device__ __forceinline__ void pin() {
#pragma unroll
        for (int i = 0; i < kN; ++i) asm volatile("" : "+v"(r[i]));
        if constexpr (TY != ORC_F16) {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) asm volatile("" : "+v"(sc[i]));
        }
    }
    // The rows from key `n` of the block on count as zeros (0 times whatever they hold would not): the bytes'
    // scales, or the halves themselves.
    __device__ __forceinline__ void keep(int n, int lane) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = min(max(n - (s * 32 + q * 16 + (lane >> 4) * 4), 0), 4);
                if constexpr (TY == ORC_F16) {
                    const uint32_t m0 = k >= 2 ? ~0u : k ? 0xFFFFu : 0u, m1 = k >= 4 ? ~0u : k == 3 ? 0xFFFFu : 0u;
#pragma unroll
                    for (int dt = 0; dt < HD / 16; ++dt) {
                        r[dt * 2 + s][q * 2] &= m0;
                        r[dt * 2 + s][q * 2 + 1] &= m1;
                    }
                } else {
                    const uint32_t m = k >= 4 ? ~0u : (1u << (8 * k)) - 1u;
#pragma unroll
                    for (int g = 0; g < HD / 32; ++g) sc[g][s * 2 + q] &= m;
                }
            }
    }
    __device__ __forceinline__ bool odd() const {
        bool any = false;
        if constexpr (TY == ORC_F16) {
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) any |= ka_odd_halves(r[i][w]);
        } else {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) any |= ka_odd_scales(sc[i][w]);
        }
        return any;
    }
    __device__ __forceinline__ void take(uint64_t* list, int lane) {
        const int c = lane & 15, g = lane >> 4;
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) {
            uint32_t m;
            if constexpr (TY == ORC_F16) m = ka_take_halves(r[dt * 2], r[dt * 2 + 1]);
            else {
                if (dt & 1) continue;
                m = ka_take_scales(sc[dt / 2]);
                ka_note(list, (dt + 1) * 16 + c, m, g);
            }
            ka_note(list, dt * 16 + c, m, g);
        }
    }
    // operand of dim tile dt and the 32 keys of step s
    __device__ __forceinline__ kq_h8 op(int dt, int s) const {
        if constexpr (TY == ORC_F16) return __builtin_bit_cast(kq_h8, r[dt * 2 + s]);
        else {
            uint32_t w0, w1;
            if constexpr (TY == ORC_KV_Q8) {
                w0 = r[dt][s * 2];
                w1 = r[dt][s * 2 + 1];
            } else {
                w0 = (r[dt / 2][s * 2] >> (dt & 1) * 4) & 0x0F0F0F0Fu;
                w1 = (r[dt / 2][s * 2 + 1] >> (dt & 1) * 4) & 0x0F0F0F0Fu;
            }
            const uint32_t s0 = sc[dt / 2][s * 2], s1 = sc[dt / 2][s * 2 + 1];
            kq_h2 o[4];
            ka_cvt4(w0, ka_scale_v(s0, 0), ka_scale_v(s0, 2), (_Float16)ka_bias<TY>(), o[0], o[1]);
            ka_cvt4(w1, ka_scale_v(s1, 0), ka_scale_v(s1, 2), (_Float16)ka_bias<TY>(), o[2], o[3]);
            return ka_join(o[0], o[1], o[2], o[3]);
        }
    }
};

// Larger of two by v_maximum3_f32: takes the matrix cores' results as they come, which v_max_f32 does not (a move each
// to quiet what might be a signalling NaN), and hands a NaN on.
__device__ __forceinline__ float ka_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Two fp16 halves of a and b. `minus` is -1 where the compiler does not see it, so that the rest is one v_fma_mix_f32
// (which widens its fp16 factor) instead of a conversion and a subtraction.
__device__ __forceinline__ uint32_t ka_split(float a, float b, float minus, uint32_t& lo) {
    const kq_h2 hi = __builtin_convertvector((kq_f2){a, b}, kq_h2);
    const kq_f2 rest = {__builtin_fmaf((float)hi.x, minus, a), __builtin_fmaf((float)hi.y, minus, b)};
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, kq_h2));
    return __builtin_bit_cast(uint32_t, hi);
}
__device__ __forceinline__ float ka_minus() {
    float m = -1.f;
    asm("" : "+s"(m));
    return m;
}

// A query row as operands: its head dims (hd / 4 per lane group) times a power
// of two that brings the largest below 2^15, in two halves; f turns its scores into powers of two.
template <int HD> struct KaRaw {
    kq_f4 v[HD / 16];
    __device__ __forceinline__ void load(const float* p, int g) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) v[i] = *(const kq_f4*)(p + g * (HD / 4) + i * 4);
    }
};
template <int TY, int HD> struct KaQ {
    kq_h8 hi[HD / 32], lo[HD / 32];
    __device__ __forceinline__ void split(const KaRaw<HD>& x, float& f) {
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x.v[i][e]));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        int ex = 0;
        if (mx > 0.f && mx < __builtin_inff()) (void)frexpf(mx, &ex);
        ex = max(-96, min(15 - ex, 120));
        f = ldexpf(1.4426950408889634f / (HD == 64 ? 8.f : 11.313708498984761f) * (TY == ORC_F16 ? 1.f : 0.0625f), -ex);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                h[e] = ka_split(ldexpf(x.v[j * 2 + e / 2][e % 2 * 2], ex), ldexpf(x.v[j * 2 + e / 2][e % 2 * 2 + 1], ex), -1.f, l[e]);
            hi[j] = __builtin_bit_cast(kq_h8, u32x4{h[0], h[1], h[2], h[3]});
            lo[j] = __builtin_bit_cast(kq_h8, u32x4{l[0], l[1], l[2], l[3]});
        }
    }
};

__device__ __forceinline__ kq_f4 ka_mfma(kq_h8 a, kq_h8 b, kq_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Running softmax of a row (per lane; the four lanes of a row agree on m and c, each sums its own keys).
struct KaRow {
    float m = -__builtin_inff(), l = 0.f;
    float c = 15.f;  // 15 less the reference that the weights are formed against
    __device__ __forceinline__ float largest(const kq_f4 (&s)[4]) const {
        float mx = ka_max(ka_max(s[0][0], s[0][1]), s[0][2]);
        mx = ka_max(ka_max(mx, s[0][3]), s[1][0]);
        mx = ka_max(ka_max(mx, s[1][1]), s[1][2]);
        mx = ka_max(ka_max(mx, s[1][3]), s[2][0]);
        mx = ka_max(ka_max(mx, s[2][1]), s[2][2]);
        mx = ka_max(ka_max(mx, s[2][3]), s[3][0]);
        mx = ka_max(ka_max(mx, s[3][1]), s[3][2]);
        return ka_max(mx, s[3][3]);
    }
    // A new reference for the row whose lanes' largest score is mx; returns what the sums so far are scaled by.
    __device__ __forceinline__ float raise(float mx) {
        mx = ka_max(ka_max(mx, __shfl_xor(mx, 16, 64)), __shfl_xor(mx, 32, 64));
        mx = ka_max(mx, __shfl_xor(mx, 48, 64));
        const float mn = ka_max(m, mx), ref = mn == -__builtin_inff() ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        c = 15.f - ref;
        l *= alpha;
        return alpha;
    }
    // Scores -> weights times 2^15, in two halves (SIGN: and the sign bit)
    template <bool SIGN>
    __device__ __forceinline__ void weigh(const kq_f4 (&s)[4], float f, float minus, uint32_t sign, u32x4 (&hi)[2], u32x4 (&lo)[2]) {
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], f, c));
                sum += p[i];
            }
            uint32_t l0, l1, h0 = ka_split(p[0], p[1], minus, l0), h1 = ka_split(p[2], p[3], minus, l1);
            if (SIGN) h0 ^= sign, h1 ^= sign, l0 ^= sign, l1 ^= sign;
            hi[t / 2][(t & 1) * 2] = h0;
            hi[t / 2][(t & 1) * 2 + 1] = h1;
            lo[t / 2][(t & 1) * 2] = l0;
            lo[t / 2][(t & 1) * 2 + 1] = l1;
        }
        l += sum;
    }
};

// The weights of a block's 64 keys (16 a lane) for RT row tiles; beta: less what the sums so far are scaled by. The
// reference is a maximum seen before; it is raised, for all of the wave's rows, only when some score passes its row's
// by so much (7/8) that a weight could pass fp16's range: after the first blocks hardly ever, and neither the exchanges
// between lanes nor the scaling's exponential are on the way from the scores to the weights.
template <bool SIGN, int RT>
__device__ __forceinline__ void ka_weights(const kq_f4 (&s)[RT][4], const float (&f)[RT], float minus, uint32_t sign,
                                           KaRow (&st)[RT], u32x4 (&hi)[RT][2], u32x4 (&lo)[RT][2], float (&beta)[RT]) {
    float mx[RT];
    bool over = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        mx[r] = st[r].largest(s[r]) * f[r];
        over |= !(mx[r] <= st[r].m + 0.875f);
        beta[r] = -1.f;
    }
    // (two row tiles: always, which costs less there than two stretches of code that cannot be interleaved)
    if (RT > 1 || __ballot(over)) {
#pragma unroll
        for (int r = 0; r < RT; ++r) beta[r] = -st[r].raise(mx[r]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) st[r].template weigh<SIGN>(s[r], f[r], minus, sign, hi[r], lo[r]);
}

// A job's key blocks by one number, the prefix's and then the own ones, so that block b's keys start at 64 b and the
// own ones at 64 nbp: where their bytes are, how many of them there are, how many own ones a token sees.
template <int BB> struct KaKeys {
    const uint8_t *pk, *pv, *ok, *ov;
    int nbp, end_p, end_o, first;
    __device__ __forceinline__ KaKeys(const KaArgs& a, const KaJob& j) {
        nbp = (a.prefix + kKvBlock - 1) / kKvBlock;
        const size_t pre = (size_t)j.kv * (a.pctx / kKvBlock) * BB;
        // (from block nbp on)
        const size_t own = (((size_t)max(j.seq, 0) * a.n_kv + j.kv) * (a.ctx / kKvBlock) - nbp) * BB;
        pk = a.pk + pre;
        pv = a.pv + pre;
        ok = a.kc + own;
        ov = a.vc + own;
        end_p = a.prefix;
        end_o = nbp * kKvBlock + j.len;
        first = nbp * kKvBlock + (j.seq < 0 ? 0 : j.start + 1 - j.seq * a.n_tok);
    }
    __device__ __forceinline__ const uint8_t* k(int b) const { return (b < nbp ? pk : ok) + (size_t)b * BB; }
    __device__ __forceinline__ const uint8_t* v(int b) const { return (b < nbp ? pv : ov) + (size_t)b * BB; }
    __device__ __forceinline__ int limit(int b) const { return (b < nbp ? end_p : end_o) - b * kKvBlock; }  // keys from b's first
    __device__ __forceinline__ int sees(int tok) const { return min(first + tok, end_o); }  // end of the keys a token sees
};

// ── few rows: the waves share out the keys ───────────────────────────────────
// A workgroup takes 16 RT rows; its NW waves take every NW-th key block each,
// straight from memory to operands, and join their sums at the end. The loads
// of a wave are whole KB in a row, and no key is read twice. Decode of 64
// sequences at 4000 (32/8 heads of 128): 8 bits 99 us, 5.5 TB/s; fp16, 32 of
// them, 90 us, 5.8 TB/s; 4 bits 71 us, 4.0 TB/s (there the conversions take as
// long as the bytes). One token at 300: 6.2 us, most of it latency.
template <int HD, int RT, int NW> struct KaStreamLds {
    float o[NW][16 * RT][HD + 4];
    float2 ml[NW][16 * RT];
    KaOdd<HD, 2, NW> odd;
};

template <int TY, int HD, int RT, int NW>
__device__ __forceinline__ void ka_stream(const KaArgs& a, KaJob j, KaStreamLds<HD, RT, NW>& sh) {
    constexpr int DT = HD / 16, KS = HD / 32, BB = kvq_block_bytes(TY, HD), M = 16 * RT;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    KaRaw<HD> raw[RT];  // asked for before the position that the keys depend on is there
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = min(j.r0 + r * 16 + c, j.r1 - 1), tok = a.by_group(row), hg = row - tok * a.group;
        raw[r].load(a.q + (int64_t)tok * a.ldq + (size_t)(j.kv * a.group + hg) * HD, g);
    }
    ka_keys(a, j);
    const bool direct = a.cp + a.co == 1;
    if (j.b0 >= j.b1 && !direct) return;
    const KaKeys<BB> keys(a, j);
    const int least = keys.sees(a.by_group(j.r0)), most = keys.sees(a.by_group(j.r1 - 1));  // what the first and last row see
    if (lane < 2) sh.odd.any[lane][wave] = 0;
    KaK<TY, HD> kr[4] = {};
    KaV<TY, HD> vr = {};
    uint32_t ks = 0;
    auto load_k = [&](int b) {
        const uint8_t* kb = keys.k(b);
#pragma unroll
        for (int t = 0; t < 4; ++t) kr[t].load(kb, t, lane);
        if constexpr (TY != ORC_F16) ks = *(const uint32_t*)(kb + kvq_code_bytes(TY, HD) + ((HD == 128 ? g : g >> 1) * 16 + c) * 4);
    };
    auto load_v = [&](int b) { vr.load(keys.v(b), lane); };
    // One row tile: a block's bytes are on their way while q is split and while the block before it is worked on. Two
    // row tiles, or 128 fp16 dims (128 registers of bytes), leave no registers for that, and both together none for V
    // before K is done with.
    constexpr bool kWide = TY == ORC_F16 && HD == 128, kAhead = RT == 1 && !kWide, kLateV = RT > 1 && kWide;
    if (kAhead && j.b0 + wave < j.b1) {
        load_k(j.b0 + wave);
        load_v(j.b0 + wave);
    }
    KaQ<TY, HD> q[RT];
    float f[RT];
    KaRow st[RT];
    int vis[RT];  // end of the keys that the lane's query row sees
    kq_f4 o[RT][DT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int tok = a.by_group(min(j.r0 + r * 16 + c, j.r1 - 1));
        q[r].split(raw[r], f[r]);
        vis[r] = keys.sees(tok);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] = kq_f4{0.f, 0.f, 0.f, 0.f};
    }
    const float minus = ka_minus();
    float sgn = 1.f;
    for (int b = j.b0 + wave; b < j.b1; b += NW) {
        const bool pre = b < keys.nbp;
        if (!kAhead) {
            load_k(b);
            if (!kLateV) load_v(b);
        }
        const int key0 = b * kKvBlock, lim = keys.limit(b);
        kq_f4 s[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            kq_h2 sc = {};
            if constexpr (TY != ORC_F16) sc = ka_scale_k(ks, t);
            kq_h8 k[KS];
#pragma unroll
            for (int i = 0; i < KS; ++i) k[i] = kr[t].op(i, sc);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                kq_f4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < KS; ++i) z = ka_mfma(k[i], q[r].lo[i], z);
#pragma unroll
                for (int i = 0; i < KS; ++i) z = ka_mfma(k[i], q[r].hi[i], z);
                s[r][t] = z;
            }
        }
        if (kAhead && b + NW < j.b1) load_k(b + NW);
        if (kLateV) load_v(b);
        if (lim < kKvBlock || (!pre && least - key0 < kKvBlock)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int n = pre ? lim : min(lim, vis[r] - key0);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (t * 16 + g * 4 + i >= n) s[r][t][i] = -__builtin_inff();
            }
        }
        if (lim < kKvBlock) vr.keep(lim, lane);
        vr.pin();
        if (!pre && least < most && least - key0 < kKvBlock && __ballot(vr.odd())) {
            vr.take(sh.odd.list[b - (least >> 6)], lane);
            if (lane == 0) sh.odd.any[b - (least >> 6)][wave] = 1;
            vr.pin();
        }
        sgn = -sgn;
        const uint32_t sign = sgn < 0.f ? 0x80008000u : 0u;
        u32x4 ph[RT][2], pl[RT][2];
        float beta[RT];
        ka_weights<true>(s, f, minus, sign, st, ph, pl, beta);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const kq_h8 v0 = vr.op(d, 0), v1 = vr.op(d, 1);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                kq_f4 z = {0.f, 0.f, 0.f, 0.f};
                z = ka_mfma(v0, __builtin_bit_cast(kq_h8, pl[r][0]), z);
                z = ka_mfma(v1, __builtin_bit_cast(kq_h8, pl[r][1]), z);
                z = ka_mfma(v0, __builtin_bit_cast(kq_h8, ph[r][0]), z);
                z = ka_mfma(v1, __builtin_bit_cast(kq_h8, ph[r][1]), z);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[r][d][i] = __builtin_fmaf(o[r][d][i], beta[r], z[i]);
            }
        }
        if (kAhead && b + NW < j.b1) load_v(b + NW);
    }
    // join the waves' sums
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        float l = st[r].l;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        st[r].l = l;
        if (g == 0) sh.ml[wave][r * 16 + c] = make_float2(st[r].m, l);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        float mm = sh.ml[0][r * 16 + c].x;
#pragma unroll
        for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sh.ml[w][r * 16 + c].x);
        const float e = st[r].l == 0.f ? 0.f : __builtin_amdgcn_exp2f(st[r].m - mm) * sgn;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sh.o[wave][r * 16 + c][d * 16 + g * 4 + i] = st[r].l == 0.f ? 0.f : o[r][d][i] * e;
    }
    __syncthreads();
    for (int it = tid; it < M * (HD / 4); it += 64 * NW) {
        const int rr = it / (HD / 4), d = it % (HD / 4) * 4, row = j.r0 + rr;
        if (row >= j.r1) continue;
        float mm = sh.ml[0][rr].x, l = 0.f;
#pragma unroll
        for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sh.ml[w][rr].x);
        kq_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 ml = sh.ml[w][rr];
            if (ml.y != 0.f) l += ml.y * __builtin_amdgcn_exp2f(ml.x - mm);
            v += *(const kq_f4*)&sh.o[w][rr][d];
        }
        const int tok = a.by_group(row), head = j.kv * a.group + (row - tok * a.group);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            int any = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) any |= sh.odd.any[n][w];
            if (any) ka_spoil(v, sh.odd.list[n] + d, keys.sees(tok) - (((least >> 6) + n) << 6));
        }
        if (direct) {
            const bool live = j.start >= 0 && j.start + (int64_t)(tok - j.seq * a.n_tok) < a.limit;
            const float inv = (TY == ORC_F16 ? 1.f : 0.0625f) / l;
            kq_f4 y = {0.f, 0.f, 0.f, 0.f};
            if (live && l != 0.f) y = v * inv;
            *(kq_f4*)(a.out + (int64_t)tok * a.ldo + (size_t)head * HD + d) = y;
        } else {
            const size_t at = (size_t)j.slot * a.n_rows + (size_t)tok * a.n_heads + head;
            *(kq_f4*)(a.part_o + at * HD + d) = v;
            if (d == 0) a.part_ml[at] = make_float2(mm, l);
        }
    }
}

// ── many rows: the waves share the keys' operands ────────────────────────────
// A workgroup takes 64 RT rows, 16 RT a wave, through every key block of its
// chunk. Each wave turns a quarter of the block into operands in LDS (two
// buffers, one barrier per block), the next block's bytes are on their way
// meanwhile: the conversion costs a quarter of what it would in each wave, and
// an operand read serves 2 RT products. KG = 2: two such groups of waves take
// alternate blocks of one row tile and join their sums in LDS, where the rows
// are too few to fill the card (500 tokens, 32/8 heads of 128: 28 -> 16 us; at
// 2000 tokens it would cost 82 -> 94). RT = 2 shares more (4000 tokens: 286 ->
// 237 us), RT = 1 spreads a prompt over more CUs (2047 tokens of 64-wide heads:
// 56 -> 47). 48 x 4 tokens over a 32 K prompt: 179 us, 1030 TFLOP/s of products
// with both halves, against 1156 of an 8192 x 8192 x 8192 library product.
// Forming the next block's scores beside this block's weights was 2-8 % slower,
// with and without an interleaving asked of the compiler.
template <int TY, int HD> struct KaStage {
    static constexpr int DW = HD / 64;  // dim tiles of V a wave stages
    KaK<TY, HD> k;
    uint32_t ks;
    u32x4 v[TY == ORC_F16 ? DW * 2 : TY == ORC_KV_Q8 ? DW : 1], vs;
    __device__ __forceinline__ void load(const uint8_t* kb, const uint8_t* vb, int wave, int lane) {
        const int c = lane & 15, g = lane >> 4;
        k.load(kb, wave, lane);
        if constexpr (TY == ORC_F16) {
#pragma unroll
            for (int i = 0; i < DW * 2; ++i) v[i] = *(const u32x4*)(vb + (wave * DW * 2 + i) * 1024 + lane * 16);
        } else {
            ks = *(const uint32_t*)(kb + kvq_code_bytes(TY, HD) + ((HD == 128 ? g : g >> 1) * 16 + c) * 4);
            vs = *(const u32x4*)(vb + kvq_code_bytes(TY, HD) + (wave * DW >> 1) * 64 + g * 16);
            if constexpr (TY == ORC_KV_Q8) {
#pragma unroll
                for (int i = 0; i < DW; ++i) v[i] = *(const u32x4*)(vb + (wave * DW + i) * 1024 + lane * 16);
            } else
                v[0] = *(const u32x4*)(vb + (wave * DW >> 1) * 1024 + lane * 16);
        }
    }
    __device__ __forceinline__ void keep(int n, int lane) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int m = min(max(n - (s * 32 + q * 16 + (lane >> 4) * 4), 0), 4);
                if constexpr (TY == ORC_F16) {
                    const uint32_t m0 = m >= 2 ? ~0u : m ? 0xFFFFu : 0u, m1 = m >= 4 ? ~0u : m == 3 ? 0xFFFFu : 0u;
#pragma unroll
                    for (int i = 0; i < DW; ++i) {
                        v[i * 2 + s][q * 2] &= m0;
                        v[i * 2 + s][q * 2 + 1] &= m1;
                    }
                } else
                    vs[s * 2 + q] &= m >= 4 ? ~0u : (1u << (8 * m)) - 1u;
            }
    }
    __device__ __forceinline__ bool odd() const {
        bool any = false;
        if constexpr (TY == ORC_F16) {
#pragma unroll
            for (int i = 0; i < DW * 2; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) any |= ka_odd_halves(v[i][w]);
        } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) any |= ka_odd_scales(vs[w]);
        }
        return any;
    }
    __device__ __forceinline__ void take(uint64_t* list, int wave, int lane) {
        const int c = lane & 15, g = lane >> 4;
        if constexpr (TY == ORC_F16) {
#pragma unroll
            for (int i = 0; i < DW; ++i) ka_note(list, (wave * DW + i) * 16 + c, ka_take_halves(v[i * 2], v[i * 2 + 1]), g);
        } else {
            const uint32_t m = ka_take_scales(vs);
#pragma unroll
            for (int i = 0; i < DW; ++i) ka_note(list, (wave * DW + i) * 16 + c, m, g);
        }
    }
    // sign: 0x80008000 negates the block's V
    __device__ __forceinline__ void put(uint8_t* kt, uint8_t* vt, int wave, int lane, uint32_t sign) const {
        kq_h2 sc = {};
        if constexpr (TY != ORC_F16) sc = ka_scale_k(ks, wave);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) *(kq_h8*)(kt + (wave * (HD / 32) + i) * 1024 + lane * 16) = k.op(i, sc);
#pragma unroll
        for (int i = 0; i < DW; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                kq_h8 o;
                if constexpr (TY == ORC_F16) o = __builtin_bit_cast(kq_h8, v[i * 2 + s] ^ sign);
                else {
                    const int sh = TY == ORC_KV_Q4 ? ((wave * DW + i) & 1) * 4 : 0;
                    const u32x4& r = v[TY == ORC_KV_Q8 ? i : 0];
                    uint32_t w0 = r[s * 2] >> sh, w1 = r[s * 2 + 1] >> sh;
                    if constexpr (TY == ORC_KV_Q4) {
                        w0 &= 0x0F0F0F0Fu;
                        w1 &= 0x0F0F0F0Fu;
                    }
                    kq_h2 q[4];
                    ka_cvt4(w0, ka_scale_v(vs[s * 2], 0, sign), ka_scale_v(vs[s * 2], 2, sign), (_Float16)ka_bias<TY>(), q[0], q[1]);
                    ka_cvt4(w1, ka_scale_v(vs[s * 2 + 1], 0, sign), ka_scale_v(vs[s * 2 + 1], 2, sign), (_Float16)ka_bias<TY>(), q[2], q[3]);
                    o = ka_join(q[0], q[1], q[2], q[3]);
                }
                *(kq_h8*)(vt + ((wave * DW + i) * 2 + s) * 1024 + lane * 16) = o;
            }
    }
};

template <int HD, int RT, int KG> struct KaTileLds {
    union {
        uint8_t t[KG][2][2][kKvBlock * HD * 2];  // [key group][buffer][K, V]
        struct {                                 // the second key group's sums
            float o[HD / 16][KG == 1 ? 1 : 4 * RT * 64 * 4];  // [dim tile][wave, row tile, lane, dim]
            float2 ml[KG == 1 ? 1 : 4 * RT * 64];
        } join;
    };
    KaOdd<HD, 3, 4 * KG> odd;
};

template <int TY, int HD, int RT, int KG>
__device__ __forceinline__ void ka_tile(const KaArgs& a, KaJob j, KaTileLds<HD, RT, KG>& sh) {
    constexpr int DT = HD / 16, KS = HD / 32, BB = kvq_block_bytes(TY, HD);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3, kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 8), c = lane & 15, g = lane >> 4;
    const int w0 = j.r0 + wave * 16 * RT;  // the wave's first row
    KaRaw<HD> raw[RT];  // asked for before the position that the keys depend on is there
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = min(w0 + r * 16 + c, j.r1 - 1), tok = a.by_group(row), hg = row - tok * a.group;
        raw[r].load(a.q + (int64_t)tok * a.ldq + (size_t)(j.kv * a.group + hg) * HD, g);
    }
    ka_keys(a, j);
    const bool direct = a.cp + a.co == 1;
    if (j.b0 >= j.b1 && !direct) return;
    const KaKeys<BB> keys(a, j);
    // ends of the keys that the wave's first and last row see
    const int least = keys.sees(a.by_group(w0)), most = keys.sees(a.by_group(min(w0 + 16 * RT, j.r1) - 1));
    const bool rows = w0 < j.r1;
    // keys that not all of the tile's rows see lie behind this one
    const int tile_least = keys.sees(a.by_group(j.r0)), apart = j.seq < 0 || tile_least == keys.sees(a.by_group(j.r1 - 1)) ? 0x7fffffff : tile_least;
    if (lane < 3) sh.odd.any[lane][kg * 4 + wave] = 0;
    KaStage<TY, HD> sg = {};
    auto load = [&](int b) { sg.load(keys.k(b), keys.v(b), wave, lane); };
    auto put = [&](int b, int buf) {
        const int lim = keys.limit(b);
        if (lim < kKvBlock) sg.keep(lim, lane);
        if (b >= keys.nbp && (b + 1) * kKvBlock > apart) {
            uint64_t* list = sh.odd.list[b - (apart >> 6)];
            if (__ballot(sg.odd())) {
                sg.take(list, wave, lane);
                if (lane == 0) sh.odd.any[b - (apart >> 6)][kg * 4 + wave] = 1;
            } else if (lane < HD / 4) list[wave * (HD / 4) + lane] = 0;
        }
        sg.put(sh.t[kg][buf][0], sh.t[kg][buf][1], wave, lane, buf ? 0u : 0x80008000u);
    };
    const float minus = ka_minus();
    float sgn = 1.f;
    const int bg = j.b0 + kg;  // the key group's first block; it takes every KG-th
    if (bg < j.b1) load(bg);  // on its way while q is split
    KaQ<TY, HD> q[RT];
    float f[RT];
    KaRow st[RT];
    int vis[RT];
    kq_f4 o[RT][DT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int tok = a.by_group(min(w0 + r * 16 + c, j.r1 - 1));
        q[r].split(raw[r], f[r]);
        vis[r] = keys.sees(tok);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] = kq_f4{0.f, 0.f, 0.f, 0.f};
    }
    if (bg < j.b1) {
        put(bg, 0);
        load(min(bg + KG, j.b1 - 1));
    }
    __syncthreads();
    for (int b = bg, cur = 0; b < j.b1 + kg; b += KG, cur ^= 1) {  // every group as many rounds as the first
        const bool pre = b < keys.nbp;
        const int key0 = b * kKvBlock, lim = keys.limit(b);
        const uint8_t *kt = sh.t[kg][cur][0] + lane * 16, *vt = sh.t[kg][cur][1] + lane * 16;
        if (rows && b < j.b1 && (pre || key0 < most)) {
            sgn = cur ? 1.f : -1.f;
            kq_f4 s[RT][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int r = 0; r < RT; ++r) s[r][t] = kq_f4{0.f, 0.f, 0.f, 0.f};
                kq_h8 k[KS];
#pragma unroll
                for (int i = 0; i < KS; ++i) k[i] = *(const kq_h8*)(kt + (t * KS + i) * 1024);
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int r = 0; r < RT; ++r) s[r][t] = ka_mfma(k[i], q[r].lo[i], s[r][t]);
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int r = 0; r < RT; ++r) s[r][t] = ka_mfma(k[i], q[r].hi[i], s[r][t]);
            }
            if (lim < kKvBlock || (!pre && least - key0 < kKvBlock)) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int n = pre ? lim : min(lim, vis[r] - key0);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t * 16 + g * 4 + i >= n) s[r][t][i] = -__builtin_inff();
                }
            }
            u32x4 ph[RT][2], pl[RT][2];
            float beta[RT];
            ka_weights<false>(s, f, minus, 0u, st, ph, pl, beta);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const kq_h8 v0 = *(const kq_h8*)(vt + d * 2048), v1 = *(const kq_h8*)(vt + d * 2048 + 1024);
                kq_f4 z[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) z[r] = ka_mfma(v0, __builtin_bit_cast(kq_h8, pl[r][0]), kq_f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int r = 0; r < RT; ++r) z[r] = ka_mfma(v1, __builtin_bit_cast(kq_h8, pl[r][1]), z[r]);
#pragma unroll
                for (int r = 0; r < RT; ++r) z[r] = ka_mfma(v0, __builtin_bit_cast(kq_h8, ph[r][0]), z[r]);
#pragma unroll
                for (int r = 0; r < RT; ++r) z[r] = ka_mfma(v1, __builtin_bit_cast(kq_h8, ph[r][1]), z[r]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[r][d][i] = __builtin_fmaf(o[r][d][i], beta[r], z[r][i]);
            }
        }
        // the next block into the other buffer (read last before the barrier that ended the block before this one)
        if (b + KG < j.b1) {
            put(b + KG, cur ^ 1);
            load(min(b + 2 * KG, j.b1 - 1));
        }
        __syncthreads();
    }
    if constexpr (KG == 2) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
            if (kg) {
                sh.join.ml[(wave * RT + r) * 64 + lane] = make_float2(st[r].m, st[r].l);
#pragma unroll
                for (int d = 0; d < DT; ++d) *(kq_f4*)&sh.join.o[d][((wave * RT + r) * 64 + lane) * 4] = o[r][d] * sgn;
            }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float2 ml = sh.join.ml[(wave * RT + r) * 64 + lane];
            const float mm = ka_max(st[r].m, ml.x), ref = mm == -__builtin_inff() ? 0.f : mm;
            const float e0 = __builtin_amdgcn_exp2f(st[r].m - ref), e1 = __builtin_amdgcn_exp2f(ml.x - ref);
            st[r].m = mm;
            st[r].l = st[r].l * e0 + ml.y * e1;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[r][d] = o[r][d] * (e0 * sgn) + *(const kq_f4*)&sh.join.o[d][((wave * RT + r) * 64 + lane) * 4] * e1;
        }
        sgn = 1.f;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        float l = st[r].l;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        const int row = w0 + r * 16 + c;
        if (row >= j.r1) continue;
        const int tok = a.by_group(row), head = j.kv * a.group + (row - tok * a.group);
        if (apart != 0x7fffffff)
            for (int n = 0; n < 3; ++n) {
                int any = 0;
#pragma unroll
                for (int w = 0; w < 4 * KG; ++w) any |= sh.odd.any[n][w];
                if (!any) continue;
#pragma unroll
                for (int d = 0; d < DT; ++d) ka_spoil(o[r][d], sh.odd.list[n] + d * 16 + g * 4, vis[r] - (((apart >> 6) + n) << 6));
            }
        if (direct) {
            const bool live = j.start >= 0 && j.start + (int64_t)(tok - j.seq * a.n_tok) < a.limit && l != 0.f;
            const float inv = sgn * (TY == ORC_F16 ? 1.f : 0.0625f) / l;
            float* out = a.out + (int64_t)tok * a.ldo + (size_t)head * HD + g * 4;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                kq_f4 y = {0.f, 0.f, 0.f, 0.f};
                if (live) y = o[r][d] * inv;
                *(kq_f4*)(out + d * 16) = y;
            }
        } else {
            const size_t at = (size_t)j.slot * a.n_rows + (size_t)tok * a.n_heads + head;
#pragma unroll
            for (int d = 0; d < DT; ++d) *(kq_f4*)(a.part_o + at * HD + d * 16 + g * 4) = o[r][d] * sgn;
            if (g == 0) a.part_ml[at] = make_float2(st[r].m, l);
        }
    }
}

// ── kernels ──────────────────────────────────────────────────────────────────
template <int TY, int HD, int RT> __global__ __launch_bounds__(256) void k_attn_kvq(KaArgs a) {
    __shared__ __attribute__((aligned(16))) KaStreamLds<HD, RT, 4> sh;
    KaJob j;
    if (ka_rows(a, 16 * RT, 16 * RT, j)) ka_stream<TY, HD, RT, 4>(a, j, sh);
}

template <int TY, int HD, int RT, int KG> __global__ __launch_bounds__(256 * KG, 2) void k_attn_kvq_tile(KaArgs a) {
    __shared__ __attribute__((aligned(16))) KaTileLds<HD, RT, KG> sh;
    KaJob j;
    if (ka_rows(a, 64 * RT, 64 * RT, j)) ka_tile<TY, HD, RT, KG>(a, j, sh);
}

// Prefix jobs of many rows and own jobs of few in one launch: the own ones fill the CUs that the prefix leaves idle.
template <int TY, int HD, int RP, int RO> __global__ __launch_bounds__(256, 2) void k_attn_kvq_both(KaArgs a) {
    __shared__ __attribute__((aligned(16))) union {
        KaTileLds<HD, RP, 1> t;
        KaStreamLds<HD, RO, 4> s;
    } sh;
    KaJob j;
    if (!ka_rows(a, 64 * RP, 16 * RO, j)) return;
    if (j.seq < 0) ka_tile<TY, HD, RP, 1>(a, j, sh.t);
    else ka_stream<TY, HD, RO, 4>(a, j, sh.s);
}

// ── the chunks' partial sums ─────────────────────────────────────────────────
// out = sum over chunks of 2^(m_c - max) O_c over the same of l_c, W waves a
// row: the lanes form the chunks' weights side by side, then each wave adds
// every W-th chunk. Bound by two latencies, the sums' and, asked for with them,
// the rows': 4.4 us for 252 rows of 44 chunks.
constexpr int kKaSlots = 1024;
template <int HD, int W> __global__ __launch_bounds__(256) void k_attn_kvq_merge(KaArgs a, float unit) {
    constexpr int R = 4 / W, E = HD / 64, N = W == 1 ? 16 : kKaSlots;  // rows of a workgroup
    __shared__ float wt[R][N];
    __shared__ float acc[W][HD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = wave / W;
    const int64_t row = (int64_t)blockIdx.x * R + sub;
    const bool some = row < a.n_rows;
    const int tok = some ? a.by_heads((int)row) : 0, head = some ? (int)row - tok * a.n_heads : 0, seq = a.by_tok(tok);
    const int n = a.cp + a.co;
    // the first chunks' sums and rows are asked for before the position is there; what an unwritten chunk holds is dropped
    const float* po = a.part_o + (size_t)(some ? row : 0) * HD + lane * E;
    const float2* pm = a.part_ml + (some ? row : 0);
    const size_t step = (size_t)a.n_rows * HD;
    float2 ml[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) ml[u] = pm[(size_t)min(lane + u * 64, n - 1) * a.n_rows];
    constexpr int U = 8;
    float x[U][E];
    auto ask = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < E; ++i) x[u][i] = po[(size_t)min(c0 + u * W, n - 1) * step + i];
    };
    ask(wave % W);
    const int start = kvq_start(a.d_pos, seq, a.pos_off, a.limit);
    const bool live = some && start >= 0 && start + (int64_t)(tok - seq * a.n_tok) < a.limit;
    float v[E] = {};
    float l = 0.f;
    if (live) {
        const int len = (int)min((int64_t)start + a.n_tok, (int64_t)a.limit);
        const int nbp = (a.prefix + kKvBlock - 1) / kKvBlock, first = a.shared ? nbp : 0;
        const int nb = nbp - first + (len + kKvBlock - 1) / kKvBlock;
        const int last = nbp - first + (start + tok - seq * a.n_tok) / kKvBlock;  // the row's last block
        float m = -__builtin_inff();
        auto get = [&](int c) {  // (maximum, sum) of chunk c; (-inf, 0) where it holds nothing of the row
            int b0, b1;
            if (c < a.cp) ka_chunk(nbp, a.by_cp, c, b0, b1);
            else ka_chunk(nb, a.by_co, c - a.cp, b0, b1);
            if (c >= n || b0 >= b1 || (c >= a.cp && b0 > last)) return make_float2(-__builtin_inff(), 0.f);
            return c < 64 ? ml[0] : c < 128 ? ml[1] : pm[(size_t)c * a.n_rows];
        };
        for (int c = lane; c < n; c += 64) m = fmaxf(m, get(c).x);
#pragma unroll
        for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        for (int c = lane; c < n; c += 64) {
            const float2 y = get(c);
            const float e = y.y == 0.f ? -1.f : __builtin_amdgcn_exp2f(y.x - m);  // -1: nothing of the row
            if (y.y != 0.f) l += e * y.y;
            if (W == 1 || wave == 0) wt[sub][c] = e;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d, 64);
    }
    __syncthreads();
    if (live) {
        for (int c0 = wave % W; c0 < n; c0 += W * U) {
            if (c0 >= W) ask(c0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float e = c0 + u * W < n ? wt[sub][c0 + u * W] : -1.f;
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] += e < 0.f ? 0.f : e * x[u][i];
            }
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int i = 0; i < E; ++i) acc[wave][lane * E + i] = v[i];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < W; ++w)
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += acc[w][lane * E + i];
    }
    if (!some) return;
    float* out = a.out + (int64_t)tok * a.ldo + (size_t)head * HD + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) out[i] = l == 0.f ? 0.f : v[i] * (unit / l);
}

// ── host ─────────────────────────────────────────────────────────────────────
struct KaPlan {
    bool shared;
    int m_p, m_o;  // rows of a workgroup: 16 or 32 (the waves share out the keys), 64 or 128 (they share the operands)
    int kg;        // key groups of the 64-row workgroups: 4 waves each
    int tiles_p, cp, tiles_o, co;
    size_t rows;
    int slots() const { return cp + co; }
    size_t bytes(int hd) const { return slots() > 1 ? (size_t)slots() * rows * (4 * (size_t)hd + 8) : 0; }
};

static int ka_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Chunks of nb key blocks for `base` workgroups' worth of row tiles: at most `most` workgroups, and `least` blocks each
// or more, all of a length but the last; one where `one` blocks are no more work than a second launch.
static int ka_chunks(int64_t base, int nb, int64_t most, int one, int least) {
    if (nb <= one) return 1;
    const int n = (int)std::max<int64_t>(1, std::min<int64_t>(most / base, (nb + least - 1) / least));
    return ka_div(nb, ka_div(nb, n));
}

static KaPlan ka_plan(int n_seq, int n_tok, int n_heads, int n_kv, int hd, int prefix_len, int pos_limit) {
    KaPlan p{};
    const int64_t group = n_heads / n_kv, rows_o = n_tok * group, rows_p = n_seq * rows_o;
    p.rows = (size_t)n_seq * n_tok * n_heads;
    const int nbp = ka_div(prefix_len, kKvBlock), nbo = ka_div(pos_limit, kKvBlock);
    // with this many rows each, sequences gain nothing from common tiles
    p.shared = prefix_len > 0 && n_seq > 1 && rows_o < 128;
    p.kg = 1;
    if (p.shared) {
        p.m_p = rows_p <= 16 ? 16 : rows_p <= 32 ? 32 : n_kv * (int64_t)ka_div(rows_p, 128) * (nbp / 8) >= 384 ? 128 : 64;
        p.m_o = p.m_p <= 32 ? p.m_p : rows_o <= 16 ? 16 : rows_o <= 32 ? 32 : p.m_p;
    } else {
        // 128 rows share more work, 64 spread over more CUs: a prompt's first rows, which see few keys, want many
        // workgroups to even out; rows behind a long context can have theirs by chunks of 8 blocks and more
        const int64_t base = (int64_t)n_seq * n_kv * ka_div(rows_o, 128);
        const bool many = 4 * (int64_t)n_tok > (int64_t)prefix_len + pos_limit ? base >= (hd == 64 ? 1024 : 640)
                                                                               : base * ((nbp + nbo) / 8) >= 384;
        p.m_o = rows_o <= 16 ? 16 : rows_o <= 32 ? 32 : many ? 128 : 64;
        if (p.m_o == 64 && (int64_t)n_seq * n_kv * ka_div(rows_o, 64) * ka_div(nbp + nbo, 4) < 2048) p.kg = 2;
    }
    p.tiles_o = ka_div(rows_o, p.m_o);
    // Workgroups that fill the card: two a CU where tiles are multiplied, one where K and V stream past few rows (a
    // second adds no bandwidth but partial sums: 32000 tokens, 32/8 heads of 128, 8 bits: 23.9 us with 512, 19.3 with
    // 256; 16 sequences x 4 tokens of 4000, 28/4 heads: 33.6 and 27.7; but 512 tokens after 7500: 135 and 178).
    const int64_t base_o = (int64_t)n_seq * n_kv * p.tiles_o, fill = 512 / p.kg;
    // Few blocks stay one chunk, for the merge is a launch: up to two for each wave (8 blocks, 8 bits: 8.3 us against 9.9;
    // 12: 10.2 against 9.8; at 64 dims 12: 7.6 against 8.6) or three for each group of waves that share operands (9
    // tokens at 300 and 500, 28/4 heads: 12.1 against 12.6, and 15.2 against 12.9). Beyond, two a chunk or more (5 tokens
    // at 1000: 14.0 us with 4, 12.0 with 2).
    p.co = ka_chunks(base_o, p.shared ? nbo : nbp + nbo, p.m_o <= 32 ? 256 : fill, p.m_o > 32 ? 3 * p.kg : hd == 64 ? 12 : 8, 2);
    if (p.shared) {
        p.tiles_p = ka_div(rows_p, p.m_p);
        const int64_t base_p = (int64_t)n_kv * p.tiles_p;
        // short prefix chunks share the card with the own jobs; beside long ones those are done in passing
        const bool lng = nbp * base_p >= 16 * fill;
        // (2 blocks or more a chunk, 4 where the own jobs fill the card: 16 sequences after 1000 tokens, 28/4 heads of 128:
        // 15.2 us with 4, 13.5 with 2; 64 after 500, 32/8 heads: 20.3 and 21.7)
        p.cp = ka_chunks(base_p, nbp, lng ? fill : std::max<int64_t>(fill / 2, fill - base_o * p.co), 4,
                         base_o * p.co >= fill ? 4 : 2);
    }
    return p;
}

template <int TY, int HD> static void ka_launch(const KaPlan& p, const KaArgs& a, hipStream_t s) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(8 * ((unsigned)(a.jobs_p + 7) / 8 + (unsigned)(a.jobs_o + 7) / 8)), dim3(256 * p.kg), 0, s, a);
    };
    if (!p.shared || p.m_p == p.m_o) {
        if (p.m_o == 16) go(k_attn_kvq<TY, HD, 1>);
        else if (p.m_o == 32) go(k_attn_kvq<TY, HD, 2>);
        else if (p.m_o == 64) p.kg == 1 ? go(k_attn_kvq_tile<TY, HD, 1, 1>) : go(k_attn_kvq_tile<TY, HD, 1, 2>);
        else go(k_attn_kvq_tile<TY, HD, 2, 1>);
    } else if (p.m_p == 64) p.m_o == 16 ? go(k_attn_kvq_both<TY, HD, 1, 1>) : go(k_attn_kvq_both<TY, HD, 1, 2>);
    else p.m_o == 16 ? go(k_attn_kvq_both<TY, HD, 2, 1>) : go(k_attn_kvq_both<TY, HD, 2, 2>);
}

}  // namespace orc

using namespace orc;

static bool ka_shape_ok(int n_seq, int n_tok, int n_heads, int n_kv, int prefix_len, int pos_limit) {
    return n_seq >= 1 && n_tok >= 1 && n_heads >= 1 && n_kv >= 1 && n_heads % n_kv == 0 && prefix_len >= 0 && pos_limit >= 1 &&
           (int64_t)n_seq * n_tok <= 0x7fffffff / n_heads && (int64_t)prefix_len + pos_limit + n_tok <= 0x7fffff00;
}

extern "C" size_t orc_attn_kvq_workspace(int n_seq, int n_tok, int n_heads, int n_kv, int head_dim, int prefix_len,
                                         int pos_limit) {
    if ((head_dim != 64 && head_dim != 128) || !ka_shape_ok(n_seq, n_tok, n_heads, n_kv, prefix_len, pos_limit)) return 0;
    return ka_plan(n_seq, n_tok, n_heads, n_kv, head_dim, prefix_len, pos_limit).bytes(head_dim);
}

extern "C" int orc_attn_kvq(int type, const float* d_q, int ldq, int n_seq, int n_tok, int n_heads, int n_kv,
                            int head_dim, const void* d_pk, const void* d_pv, int prefix_len, int prefix_ctx,
                            const void* d_kc, const void* d_vc, int ctx, const int32_t* d_pos, int pos_off,
                            int pos_limit, float* d_out, int ldo, void* d_work, orc_stream_t s) {
    if (!initialized()) return set_error(ORC_E_NOINIT, "orc_init not called");
    if (!kvq_type_ok(type)) return set_error(ORC_E_UNSUPPORTED, "attn_kvq: cache types are F16, KV_Q8 and KV_Q4");
    if (head_dim != 64 && head_dim != 128) return set_error(ORC_E_UNSUPPORTED, "attn_kvq: head_dim must be 64 or 128");
    if (n_seq < 0 || n_tok < 0) return set_error(ORC_E_INVALID, "attn_kvq: bad args");
    if (!n_seq || !n_tok) return ORC_OK;
    if (!ka_shape_ok(n_seq, n_tok, n_heads, n_kv, prefix_len, pos_limit) || ctx % kKvBlock || pos_limit > ctx ||
        prefix_len > prefix_ctx || prefix_ctx % kKvBlock || ldq < (int64_t)n_heads * head_dim ||
        ldo < (int64_t)n_heads * head_dim || ldq % 4 || ldo % 4)
        return set_error(ORC_E_INVALID, "attn_kvq: bad args (heads a multiple of the kv heads, 1 <= pos_limit <= ctx, "
                                        "prefix_len <= prefix_ctx, contexts multiples of 64)");
    if (!d_pos && (pos_off < 0 || (int64_t)pos_off + n_tok > pos_limit))
        return set_error(ORC_E_INVALID, "attn_kvq: positions must lie below pos_limit");
    const KaPlan p = ka_plan(n_seq, n_tok, n_heads, n_kv, head_dim, prefix_len, pos_limit);
    const size_t bytes = p.bytes(head_dim);
    if (!d_q || !d_out || !d_kc || !d_vc || (prefix_len && (!d_pk || !d_pv)) || (bytes && !d_work) ||
        (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_kc | (uintptr_t)d_vc | (uintptr_t)d_pk | (uintptr_t)d_pv |
          (uintptr_t)d_work) & 15))
        return set_error(ORC_E_INVALID, "attn_kvq: null or misaligned pointer");
    const int64_t jobs_p = (int64_t)n_kv * p.cp * p.tiles_p, jobs_o = (int64_t)n_seq * n_kv * p.co * p.tiles_o;
    if (jobs_p + jobs_o > 0xffffff00ll / 256 - 16 || (p.slots() > 1 && p.rows > 4 * (0xffffff00ull / 256))) return set_error(ORC_E_INVALID, "attn_kvq: too many rows");
    KaArgs a{d_q, ldq, n_seq, n_tok, n_heads, n_kv, n_heads / n_kv, (const uint8_t*)d_pk, (const uint8_t*)d_pv,
             (const uint8_t*)d_kc, (const uint8_t*)d_vc, prefix_len, prefix_ctx, ctx, d_pos, pos_off, pos_limit, d_out,
             ldo, nullptr, nullptr, (int)p.rows, p.shared, p.tiles_p, p.cp, p.tiles_o, p.co, (int)jobs_p, (int)jobs_o,
             kvq_div(n_heads / n_kv), kvq_div(n_kv), kvq_div(p.tiles_p), kvq_div(p.cp), kvq_div(p.tiles_o), kvq_div(p.co),
             kvq_div(n_heads), kvq_div(n_tok)};
    if (bytes) {
        a.part_o = (float*)d_work;
        a.part_ml = (float2*)((uint8_t*)d_work + (size_t)p.slots() * p.rows * head_dim * 4);
    }
    const hipStream_t st = resolve_stream(s);
    auto go = [&](auto ty) {
        constexpr int T = decltype(ty)::value;
        head_dim == 64 ? ka_launch<T, 64>(p, a, st) : ka_launch<T, 128>(p, a, st);
    };
    if (type == ORC_F16) go(std::integral_constant<int, ORC_F16>());
    else if (type == ORC_KV_Q8) go(std::integral_constant<int, ORC_KV_Q8>());
    else go(std::integral_constant<int, ORC_KV_Q4>());
    ORC_LAUNCH_CHECK();
    if (p.slots() > 1) {
        const float unit = type == ORC_F16 ? 1.f : 0.0625f;
        auto merge = [&](auto kernel, int rows) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)ka_div((int64_t)p.rows, rows)), dim3(256), 0, st, a, unit);
        };
        if (p.slots() <= 16) head_dim == 64 ? merge(k_attn_kvq_merge<64, 1>, 4) : merge(k_attn_kvq_merge<128, 1>, 4);
        else head_dim == 64 ? merge(k_attn_kvq_merge<64, 4>, 1) : merge(k_attn_kvq_merge<128, 4>, 1);
        ORC_LAUNCH_CHECK();
    }
    return ORC_OK;
}
