// The 8-bit cache, trees of drafted tokens: norm_rope_kv, kv_read, atencion_mx8 (and atencion_arbol on 8-bit caches), kv_ramal.
//
// 8-bit blocks ("mx8"): 32 channels of one token's head share a power of two, value = q 2^(x - 133), q within +-127 held as
// the byte q + 128, x the smallest byte for which the block's largest magnitude times 2^(133 - x) is below 127.5 (so that q,
// rounded half to even, is off by at most half a step); x = 255: a value of the block was not finite, and all of it is NaN.
// (The blocks of OCP's MXINT8, with the scale one step up where the standard's own would saturate.)  With scales that are
// powers of two, q 2^(x - E) is an f16 operand of the matrix cores without rounding: neither scores nor probabilities have to
// be multiplied by the scales of blocks, which scales of any value (Q8_0's) would need, once per score and block of the key
// and twice per probability and block of the value.
//
// Layout, R slots (the rows rounded up to 32): the K cache holds the bytes of each head's tiles of 32 slots, [nkv][R / 32],
// a tile [slot / 16][c / 64][c % 64 / 16][slot % 16][c % 16], then the scales [nkv][R][hd / 32]; the V cache likewise, a tile
// [i][g][n][e][j] with channel c = hd / 16 n + 2 i + e and slot 16 (j / 4) + 4 g + j % 4, then the scales
// [nkv][R / 32][hd / 32][g][j].  These are the orders in which the lanes of a wavefront take a tile: every load is 1 KB.
#include "qp_ints.h"

typedef uint16_t us2 __attribute__((ext_vector_type(2)));
typedef uint16_t us4 __attribute__((ext_vector_type(4)));

// ====================================================================================== the blocks
constexpr uint32_t MX_NAN = 255;
QP_DEV uint32_t mx_slots(uint32_t rows) { return (rows + 31) & ~31u; }
// The scale byte of a block whose largest magnitude is m (NaN and infinities: MX_NAN).
QP_DEV uint32_t mx_scale(float m) {
    const uint32_t b = __float_as_uint(m), e = b >> 23, f = b & 0x7fffffu;
    if (e == 255) return MX_NAN;
    return e ? e + (f >= 0x7f0000u ? 1u : 0u) : (f >= 0x7f8000u ? 1u : 0u);
}
// The byte of v in a block of scale x.
QP_DEV uint32_t mx_byte(float v, uint32_t x) {
    if (x == MX_NAN) return 128;
    return (uint32_t)((int)__builtin_rintf(__builtin_ldexpf(v, 133 - (int)x)) + 128);
}
QP_DEV float mx_value(uint32_t byte, uint32_t x) {
    if (x == MX_NAN) return __builtin_nanf("");
    return __builtin_ldexpf((float)((int)byte - 128), (int)x - 133);
}
// Where a K or V cache holds channel c of slot s of head h (bytes from its start), and that block's scale.
QP_DEV uint64_t mx_k_at(uint32_t h, uint32_t s, uint32_t c, uint32_t R, uint32_t hd) {
    return ((uint64_t)h * R + (s & ~31u)) * hd + ((((s >> 4) & 1) * (hd >> 6) + (c >> 6)) * 4 + ((c >> 4) & 3)) * 256 +
           (s & 15) * 16 + (c & 15);
}
QP_DEV uint64_t mx_kx_at(uint32_t h, uint32_t s, uint32_t b, uint32_t R, uint32_t hd, uint32_t nkv) {
    return (uint64_t)nkv * R * hd + ((uint64_t)h * R + s) * (hd >> 5) + b;
}
QP_DEV uint64_t mx_v_at(uint32_t h, uint32_t s, uint32_t c, uint32_t R, uint32_t hd) {
    const uint32_t dt = hd >> 4, n = c / dt, d = c % dt;
    return ((uint64_t)h * R + (s & ~31u)) * hd + (d >> 1) * 1024 + (((s >> 2) & 3) * 16 + n) * 16 + (d & 1) * 8 +
           ((s >> 4) & 1) * 4 + (s & 3);
}
QP_DEV uint64_t mx_vx_at(uint32_t h, uint32_t s, uint32_t b, uint32_t R, uint32_t hd, uint32_t nkv) {
    return (uint64_t)nkv * R * hd + ((uint64_t)h * R + (s & ~31u)) * (hd >> 5) + b * 32 + ((s >> 2) & 3) * 8 +
           ((s >> 4) & 1) * 4 + (s & 3);
}

// ====================================================================================== norm, rotation and store
// Sine and cosine of x, reduced in 64 bits so that far positions keep theirs, then the polynomials of sincos2.
QP_DEV void sincos_far(float x, float& sn_out, float& cs_out) {
    const double xd = (double)x, k = __builtin_rint(xd * 0.63661977236758134308);
    const float r = (float)__builtin_fma(k, -6.123233995736766e-17, __builtin_fma(k, -1.5707963267948966, xd));
    const float r2 = r * r;
    const float sn = r + (r * r2) * (-1.6666654611e-1f + r2 * (8.3321608736e-3f + r2 * -1.9515295891e-4f));
    const float cs = (1.0f - 0.5f * r2) +
                     (r2 * r2) * (4.166664568298827e-2f + r2 * (-1.388731625493765e-3f + r2 * 2.443315711809948e-5f));
    const uint32_t q = (uint32_t)(int64_t)k & 3u;
    const float a = q & 1 ? cs : sn, b = q & 1 ? sn : cs;
    sn_out = q & 2 ? -a : a;
    cs_out = q == 1 || q == 2 ? -b : b;
}

// One wavefront (hd = 128) or half of one (hd = 64) per token and head of q, k or v; grid (T, ceil((nh + 2 nkv) / heads per
// workgroup)).  A lane takes the two elements of a pair, norms and rotates them, then (through LDS where pairs are not
// neighbours) two neighbouring channels, which it stores.
KERNEL __launch_bounds__(256) void qp_norm_rope_kv(QpRopeKvArgs a) {
    __shared__ float row_s[4][128];
    const uint32_t t = blockIdx.x, hl = a.hd >> 1;             // lanes per head
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (hl - 1);
    const uint32_t per = 256 / hl, head = blockIdx.y * per + threadIdx.x / hl;
    if (t >= paso_T(a.paso)) return;
    const uint32_t nq = a.nh, nall = a.nh + 2 * a.nkv;
    const bool on = head < nall, isq = head < nq, isv = head >= nq + a.nkv;
    const uint32_t h = isq ? head : isv ? head - nq - a.nkv : head - nq;
    const uint64_t src = (isq ? a.q : isv ? a.v : a.k) + 4ull * (((uint64_t)t * (isq ? a.nh : a.nkv) + h) * a.hd);
    const uint32_t half = a.nrot >> 1;
    const bool apart = a.neox && !isv;                          // pairs (j, j + nrot / 2)
    const uint32_t i0 = apart && l < half ? l : 2 * l, i1 = apart && l < half ? l + half : 2 * l + 1;
    float x0 = on ? gload<float>(src + 4 * i0) : 0.0f, x1 = on ? gload<float>(src + 4 * i1) : 0.0f;
    const uint64_t w = isv ? 0 : isq ? a.qnorm : a.knorm;
    float ss = x0 * x0 + x1 * x1;
    ss += bfly_f<0>(ss, lane);
    ss += bfly_f<1>(ss, lane);
    ss += bfly_f<2>(ss, lane);
    ss += bfly_f<3>(ss, lane);
    ss += bfly_f<4>(ss, lane);
    if (hl == 64) ss += bfly_f<5>(ss, lane);
    if (w) {
        const float inv = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
        x0 = (x0 * inv) * gload<float>(w + 4 * i0);
        x1 = (x1 * inv) * gload<float>(w + 4 * i1);
    }
    if (!isv && l < half) {
        const uint32_t pos = a.pos ? cptr<uint32_t>(a.pos)[t] : paso_pos(a.paso) + t;
        float sn, cs;
        sincos_far(((float)pos * a.esc) * gload<float>(a.freq + 4 * l), sn, cs);
        const float r0 = x0 * cs - x1 * sn, r1 = x0 * sn + x1 * cs;
        x0 = r0;
        x1 = r1;
    }
    if (a.neox) {  // back to neighbouring channels
        float* row = row_s[wave] + (lane - l) * 2;
        row[i0] = x0;
        row[i1] = x1;
        __builtin_amdgcn_wave_barrier();
        x0 = row[2 * l];
        x1 = row[2 * l + 1];
    }
    // the largest magnitude of 32 channels (16 lanes; a NaN's or an infinity's bits lie above all others)
    uint32_t m = max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu);
    m = max(m, bfly<0>(m, lane));
    m = max(m, bfly<1>(m, lane));
    m = max(m, bfly<2>(m, lane));
    m = max(m, bfly<3>(m, lane));
    if (!on) return;
    const uint32_t c = 2 * l;
    if (isq) {
        gstore<float2>(a.qo + 4ull * (((uint64_t)t * a.nh + h) * a.hd + c), make_float2(x0, x1));
        return;
    }
    uint32_t slot = paso_pos(a.paso) + t;
    if (a.cap) slot %= a.cap;
    if (slot >= a.rows) return;
    const uint32_t kvd = a.nkv * a.hd, ch = h * a.hd + c, R = mx_slots(a.rows);
    if (a.fmt == 0) {
        gstore<float2>((isv ? a.vc : a.kc) + 4 * ((uint64_t)slot * kvd + ch), make_float2(x0, x1));
    } else if (a.fmt == 1) {
        if (isv) {
            mptr<uint16_t>(a.vc)[vt_index(slot, kvd, ch)] = f2h(x0);
            mptr<uint16_t>(a.vc)[vt_index(slot, kvd, ch + 1)] = f2h(x1);
        } else {
            gstore<uint32_t>(a.kc + 2 * ((uint64_t)slot * kvd + ch), (uint32_t)f2h(x0) | ((uint32_t)f2h(x1) << 16));
        }
    } else {
        const uint32_t x = mx_scale(__uint_as_float(m)), b0 = mx_byte(x0, x), b1 = mx_byte(x1, x);
        if (isv) {
            mptr<uint8_t>(a.vc)[mx_v_at(h, slot, c, R, a.hd)] = (uint8_t)b0;
            mptr<uint8_t>(a.vc)[mx_v_at(h, slot, c + 1, R, a.hd)] = (uint8_t)b1;
            if ((l & 15) == 0) mptr<uint8_t>(a.vc)[mx_vx_at(h, slot, l >> 4, R, a.hd, a.nkv)] = (uint8_t)x;
        } else {
            gstore<uint16_t>(a.kc + mx_k_at(h, slot, c, R, a.hd), (uint16_t)(b0 | (b1 << 8)));
            if ((l & 15) == 0) mptr<uint8_t>(a.kc)[mx_kx_at(h, slot, l >> 4, R, a.hd, a.nkv)] = (uint8_t)x;
        }
    }
}

// ====================================================================================== reading back
// Rows of positions p0 .. p0 + n - 1 as f32 or f16 [n][nkv hd]: a thread takes two channels of K and of V.
KERNEL __launch_bounds__(256) void qp_kv_read(QpKvReadArgs a) {
    const uint32_t kvd = a.nkv * a.hd, R = mx_slots(a.rows);
    const uint64_t total = (uint64_t)a.n * (kvd >> 1);
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t t = (uint32_t)(i / (kvd >> 1)), ch = 2 * (uint32_t)(i % (kvd >> 1)), h = ch / a.hd, c = ch % a.hd;
        uint32_t s = a.p0 + t;
        if (a.cap) s %= a.cap;
        float k0, k1, v0, v1;
        if (a.fmt == 0) {
            const float2 k = gload<float2>(a.kc + 4 * ((uint64_t)s * kvd + ch)), v = gload<float2>(a.vc + 4 * ((uint64_t)s * kvd + ch));
            k0 = k.x, k1 = k.y, v0 = v.x, v1 = v.y;
        } else if (a.fmt == 1) {
            const uint32_t k = gload<uint32_t>(a.kc + 2 * ((uint64_t)s * kvd + ch));
            k0 = h2f(k), k1 = h2f(k >> 16);
            v0 = h2f(cptr<uint16_t>(a.vc)[vt_index(s, kvd, ch)]);
            v1 = h2f(cptr<uint16_t>(a.vc)[vt_index(s, kvd, ch + 1)]);
        } else {
            const uint32_t k = gload<uint16_t>(a.kc + mx_k_at(h, s, c, R, a.hd));
            const uint32_t kx = cptr<uint8_t>(a.kc)[mx_kx_at(h, s, c >> 5, R, a.hd, a.nkv)];
            const uint32_t vx = cptr<uint8_t>(a.vc)[mx_vx_at(h, s, c >> 5, R, a.hd, a.nkv)];
            k0 = mx_value(k & 255, kx), k1 = mx_value(k >> 8, kx);
            v0 = mx_value(cptr<uint8_t>(a.vc)[mx_v_at(h, s, c, R, a.hd)], vx);
            v1 = mx_value(cptr<uint8_t>(a.vc)[mx_v_at(h, s, c + 1, R, a.hd)], vx);
        }
        const uint64_t o = (uint64_t)t * kvd + ch;
        if (a.out == 0) {
            gstore<float2>(a.k + 4 * o, make_float2(k0, k1));
            gstore<float2>(a.v + 4 * o, make_float2(v0, v1));
        } else {
            gstore<uint32_t>(a.k + 2 * o, (uint32_t)f2h(k0) | ((uint32_t)f2h(k1) << 16));
            gstore<uint32_t>(a.v + 2 * o, (uint32_t)f2h(v0) | ((uint32_t)f2h(v1) << 16));
        }
    }
}

// ====================================================================================== the accepted path
// Slot of position pos0 + i <- slot of position pos0 + idx[i], i = 0 .. n - 1, in every cache of the list.  A thread has a
// piece of the row (16, 2 or 1 bytes that stay together in every slot) of one cache and moves it through all n rows, eight at
// a time: their loads, then their stores.  idx increases, so idx[i] >= i, and a store only reaches slots whose rows have been
// taken.
template <class U>
QP_DEV void ramal_piece(const QpRamalArgs& a, uint64_t base, uint64_t (*at)(const QpRamalArgs&, uint32_t, uint32_t), uint32_t u) {
    const uint32_t pos0 = paso_pos(a.paso), T = paso_T(a.paso);
    for (uint32_t i0 = 0; i0 < a.n; i0 += 8) {
        U v[8];
        uint32_t ok = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i0 + i >= a.n) break;
            const uint32_t j = cptr<uint32_t>(a.idx)[i0 + i];
            uint32_t s = pos0 + j, d = pos0 + i0 + i;
            if (a.cap) s %= a.cap, d %= a.cap;
            if (j >= T || s >= a.rows || d >= a.rows || s == d) continue;
            v[i] = gload<U>(base + at(a, u, s));
            ok |= 1u << i;
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            uint32_t d = pos0 + i0 + i;
            if (a.cap) d %= a.cap;
            if (ok >> i & 1) gstore<U>(base + at(a, u, d), v[i]);
        }
    }
}
// grid (pieces / 256, 2 caches): cache 2 i is layer i's K, 2 i + 1 its V
KERNEL __launch_bounds__(256) void qp_kv_ramal(QpRamalArgs a) {
    const uint32_t u = blockIdx.x * 256 + threadIdx.x, kvd = a.nkv * a.hd;
    const bool isv = blockIdx.y & 1;
    const uint64_t base = a.cache[blockIdx.y];
    if (a.fmt == 0) {
        if (u < kvd / 4)
            ramal_piece<float4>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return 4ull * s * (b.nkv * b.hd) + 16 * p; }, u);
    } else if (a.fmt == 1 && !isv) {
        if (u < kvd / 8)
            ramal_piece<float4>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return 2ull * s * (b.nkv * b.hd) + 16 * p; }, u);
    } else if (a.fmt == 1) {
        if (u < kvd)
            ramal_piece<uint16_t>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return 2 * vt_index(s, b.nkv * b.hd, p); }, u);
    } else if (!isv) {
        if (u < kvd / 16)
            ramal_piece<float4>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return mx_k_at(16 * p / b.hd, s, 16 * p % b.hd, mx_slots(b.rows), b.hd); }, u);
        else if (u < kvd / 16 + kvd / 32)
            ramal_piece<uint8_t>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return mx_kx_at(32 * p / b.hd, s, 32 * p % b.hd / 32, mx_slots(b.rows), b.hd, b.nkv); }, u - kvd / 16);
    } else {
        if (u < kvd)
            ramal_piece<uint8_t>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return mx_v_at(p / b.hd, s, p % b.hd, mx_slots(b.rows), b.hd); }, u);
        else if (u < kvd + kvd / 32)
            ramal_piece<uint8_t>(a, base, [](const QpRamalArgs& b, uint32_t p, uint32_t s) -> uint64_t {
                return mx_vx_at(32 * p / b.hd, s, 32 * p % b.hd / 32, mx_slots(b.rows), b.hd, b.nkv); }, u - kvd);
    }
}

// ====================================================================================== attention
QP_DEV f32x4 mx_mfma(h8 a, h8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
QP_DEV f32x4 mx_mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

constexpr float MX_LOG2E = 1.4426950408889634f;

// A workgroup takes 16 RG (query, head) rows of one KV head and a share of the key tiles, dealt to its four wavefronts, each
// with a softmax state of its own; they meet in LDS.  Scores are S^T = K Q^T and outputs O^T += V^T P^T with
// v_mfma_f32_16x16x32_f16; queries and probabilities are f16 high and low parts (22 bits) below a power of two, keys and
// values q 2^(x - E + 5) with one E of the wavefront each (16 times its first tile's largest), exact and normal for
// x - E = -19 .. 0.  A wavefront takes its remaining tiles with the f32 matrix instruction (an eighth of the rate) where that
// does not hold: a block of a tile lies outside that range, or a query's element is not 0 and below 2^-20 of its row's
// largest (its part would lose bits), or not finite.  So no row loses bits to a key that it does not see.
template <int HD, int RG, bool TREE>
QP_DEV void attn_mx8_body(const QpAttnArgs& a) {
    constexpr int CC = HD / 64, KS = HD / 32, DT = HD / 16, NB = HD / 32;
    extern __shared__ float4 mx_lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n16 = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t T = min(paso_T(a.paso), a.tcov), pos0 = paso_pos(a.paso);
    const uint32_t G = a.nh / a.nkv, kvh = blockIdx.x, nrow = T * G;
    // (long prompts: the blocks with the most keys first)
    const uint32_t r0 = (TREE ? blockIdx.y : gridDim.y - 1 - blockIdx.y) * (16 * RG);
    if (r0 >= nrow) return;
    const uint32_t t_lo = r0 / G, t_hi = (min(r0 + 16 * RG, nrow) - 1) / G;
    const uint32_t R = mx_slots(a.rows);
    // ---- the rows' queries
    h8 qh[RG][KS], ql[RG][KS];
    int qe[RG], lim[RG], low[RG];  // keys low < key <= lim
    uint64_t mrow[RG];             // TREE: the row's mask words
    bool alike = true;             // the lane's queries fit the f16 parts
    auto q_at = [&](int r) __attribute__((always_inline)) {
        const uint32_t rc = min(r0 + r * 16 + n16, nrow - 1);
        return a.q + 4 * (((uint64_t)(rc / G) * a.nh + kvh * G + rc % G) * HD + 16 * g);
    };
#pragma unroll
    for (int r = 0; r < RG; r++) {
        const uint32_t t = min(r0 + r * 16 + n16, nrow - 1) / G;
        const uint64_t at = q_at(r);
        float v[KS][8], mine = 0.0f, least = 3.4e38f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const float4 x = gload<float4>(at + (s >> 1) * 256 + (s & 1) * 32), y = gload<float4>(at + (s >> 1) * 256 + (s & 1) * 32 + 16);
            const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float u = fabsf(w[i]);
                v[s][i] = w[i];
                mine = fmaxf(mine, u);
                alike = alike & (u < __builtin_inff());  // (a NaN neither)
                least = fminf(least, u == 0.0f ? 3.4e38f : u);
            }
        }
        float all = fmaxf(mine, bfly_f<4>(mine, lane));
        all = fmaxf(all, bfly_f<5>(all, lane));
        const int e = max((int)((__float_as_uint(all) >> 23) & 255) - 127, -110);
        alike = alike & (least >= all * 0x1p-20f);
        qe[r] = e;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x = __builtin_ldexpf(v[s][i], 14 - e);  // below 2^15
                qh[r][s][i] = (_Float16)x;
                ql[r][s][i] = (_Float16)(x - (float)qh[r][s][i]);
            }
        uint32_t p = pos0 + t;
        if constexpr (TREE) {
            if (a.where) p = min(max(cptr<uint32_t>(a.where)[t], pos0), pos0 + T - 1);
            mrow[r] = a.mask + 4ull * t * a.mw;
        }
        lim[r] = (int)p;
        low[r] = a.swa && p >= a.swa ? (int)(p - a.swa) : -1;
    }
    // ---- the key tiles: keys kbeg .. kend in slots first .. (ring: then 0 ..), whole tiles of 32 slots
    const uint32_t last = TREE ? T - 1 : t_hi, early = TREE ? 0 : t_lo;
    const uint32_t kend = a.cap ? pos0 + last + 1 : min(pos0 + last + 1, a.rows);
    const uint32_t kbeg = a.swa && pos0 + early + 1 > a.swa ? min(pos0 + early + 1 - a.swa, kend) : 0;
    const uint32_t first = a.cap ? kbeg % a.cap : kbeg, nkey = a.cap ? min(kend - kbeg, a.cap) : kend - kbeg;
    const uint32_t end_a = a.cap ? min(first + nkey, a.cap) : first + nkey, end_b = first + nkey - end_a;
    const uint32_t ta = nkey ? (end_a + 31) / 32 - first / 32 : 0, nt = ta + (end_b + 31) / 32;
    const uint32_t per = (nt + a.nsplit - 1) / a.nsplit, i0 = blockIdx.z * per, i1 = min(nt, i0 + per);
    const uint64_t planes = (uint64_t)a.nkv * R * HD, hk = (uint64_t)kvh * R * HD, hx = planes + (uint64_t)kvh * R * NB;
    const __amdgpu_buffer_rsrc_t kr = kq_rsrc(a.kc + hk, (uint64_t)R * HD), vr = kq_rsrc(a.vc + hk, (uint64_t)R * HD);
    const __amdgpu_buffer_rsrc_t kxr = kq_rsrc(a.kc + hx, (uint64_t)R * NB), vxr = kq_rsrc(a.vc + hx, (uint64_t)R * NB);

    u32x4 kw[2][CC], vw[DT / 2];
    uint32_t kx[2], vx[2];  // the scales of the lane's key of each half, and of its 8 values' keys
    struct Tile { uint32_t slot, lo, hi; int off; };  // slots lo .. hi of it hold keys slot + off
    auto tile = [&](uint32_t i) __attribute__((always_inline)) {
        Tile t;
        if (i < ta) t = {(first / 32 + i) * 32, first, end_a, (int)(kbeg - first)};
        else t = {(i - ta) * 32, 0, end_b, (int)(kbeg + a.cap - first)};
        return t;
    };
    auto load_k = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t s = tile(i).slot, o = i < i1 ? s * HD + lane * 16 : QP_NOOFF;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t x = i < i1 ? (s + h * 16 + n16) * NB : QP_NOOFF;
            if constexpr (NB == 4) kx[h] = __builtin_amdgcn_raw_buffer_load_b32(kxr, x, 0, 0);
            else kx[h] = __builtin_amdgcn_raw_buffer_load_b16(kxr, x, 0, 0);
#pragma unroll
            for (int c = 0; c < CC; c++) kw[h][c] = __builtin_amdgcn_raw_buffer_load_b128(kr, o, (h * CC + c) * 1024, 0);
        }
    };
    auto load_v = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t s = tile(i).slot, o = i < i1 ? s * HD + lane * 16 : QP_NOOFF;
        const uint32_t x = i < i1 ? s * NB + (n16 * DT / 32) * 32 + g * 8 : QP_NOOFF;
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(vxr, x, 0, 0);
        vx[0] = w[0];
        vx[1] = w[1];
#pragma unroll
        for (int c = 0; c < DT / 2; c++) vw[c] = __builtin_amdgcn_raw_buffer_load_b128(vr, o, c * 1024, 0);
    };
    // slot k of the tile holds a key
    auto held = [&](const Tile& t, uint32_t k) __attribute__((always_inline)) { return t.slot + k >= t.lo && t.slot + k < t.hi; };
    // bits of the mask for the tile's 32 slots (drafted tokens only)
    auto drafted = [&](const Tile& t, int r) __attribute__((always_inline)) -> uint32_t {
        if constexpr (!TREE) return 0;
        const int j = (int)t.slot + t.off - (int)pos0, w = j >> 5, sh = j & 31;
        const uint32_t b0 = w >= 0 && w < (int)a.mw ? gload<uint32_t>(mrow[r] + 4ull * (uint32_t)w) : 0;
        const uint32_t b1 = w + 1 >= 0 && w + 1 < (int)a.mw ? gload<uint32_t>(mrow[r] + 4ull * (uint32_t)(w + 1)) : 0;
        return (uint32_t)((((uint64_t)b1 << 32) | b0) >> sh);
    };
    // row r sees the key in slot k of the tile
    auto sees = [&](const Tile& t, int r, uint32_t k, uint32_t bits) __attribute__((always_inline)) {
        const int key = (int)(t.slot + k) + t.off;
        if constexpr (TREE) return held(t, k) & (key < (int)pos0 ? key > low[r] : ((bits >> k) & 1) != 0);
        else return held(t, k) & (key <= lim[r]) & (key > low[r]);
    };
    // all slots hold keys that every row of the block sees
    auto all_see = [&](const Tile& t) __attribute__((always_inline)) {
        const int k0 = (int)t.slot + t.off;
        return t.slot >= t.lo && t.slot + 32 <= t.hi && k0 + 31 <= (int)(pos0 + t_lo) - (TREE ? (int)t_lo + 1 : 0) &&
               (!a.swa || k0 > (int)(pos0 + (TREE ? T - 1 : t_hi)) - (int)a.swa);
    };

    f32x4 o[RG][DT];
    float m[RG], l[RG], p[RG][8], corr[RG], cs[RG];
    int ek = -1, ev = -1;  // E of the keys and values, or -1: only zeros so far
#pragma unroll
    for (int r = 0; r < RG; r++) {
        m[r] = -3.0e38f;
        l[r] = 0.0f;
        cs[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[r][d] = f32x4{0, 0, 0, 0};
    }
    // softmax of the lane's 8 keys of each of its rows: scores s times c in units of log2
    auto softmax = [&](const Tile& t, bool whole, const f32x4 (&s)[RG][2], const float (&c)[RG]) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t bits = TREE && !whole ? drafted(t, r) : 0;
            float x[8], mx = -3.0e38f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = s[r][j >> 2][j & 3] * c[r];
                if (!whole) x[j] = sees(t, r, (j >> 2) * 16 + 4 * g + (j & 3), bits) ? x[j] : -__builtin_inff();
                mx = fmaxf(mx, x[j]);
            }
            mx = fmaxf(mx, bfly_f<4>(mx, lane));
            mx = fmaxf(mx, bfly_f<5>(mx, lane));
            const float mn = fmaxf(m[r], mx);
            corr[r] = __builtin_amdgcn_exp2f(m[r] - mn);
            m[r] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[r][j] = __builtin_amdgcn_exp2f(x[j] - mn);
                sum += p[r][j];
            }
            l[r] = l[r] * corr[r] + sum;
        }
    };
    auto rescale = [&]() __attribute__((always_inline)) {
        bool same = true;
#pragma unroll
        for (int r = 0; r < RG; r++) same = same && corr[r] == 1.0f;
        if (__all(same)) return;
#pragma unroll
        for (int r = 0; r < RG; r++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[r][d][x] *= corr[r];
    };
    // the scales of slots without a key: 0 (they may hold anything)
    auto clear = [&](const Tile& t) __attribute__((always_inline)) {
        if (t.slot >= t.lo && t.slot + 32 <= t.hi) return;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            kx[h] = held(t, h * 16 + n16) ? kx[h] : 0;
#pragma unroll
            for (int j = 0; j < 4; j++) vx[h] &= held(t, h * 16 + 4 * g + j) ? 0xffffffffu : ~(255u << (8 * j));
        }
    };
    // A value that is not finite reaches the rows that see its key, and no others: their channels become NaN here (the
    // lane's own, which are of one block), the scale 0.
    auto poison = [&](const Tile& t) __attribute__((always_inline)) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) bad |= ((vx[i] >> (8 * j)) & 255) == MX_NAN ? 1u : 0u;
        if (!__any(bad != 0)) return;
        const uint64_t xs = a.vc + hx + (uint64_t)t.slot * NB + (DT * 4 * g / 32) * 32;
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t bits = drafted(t, r);
            bool nan = false;
            for (uint32_t i = 0; i < 32; i++) {  // byte i: lane group i / 8, value i % 8
                const uint32_t k = ((i >> 2) & 1) * 16 + 4 * (i >> 3) + (i & 3);
                nan |= sees(t, r, k, bits) && gload<uint8_t>(xs + i) == MX_NAN;
            }
            if (nan)
#pragma unroll
                for (int d = 0; d < DT; d++) o[r][d] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (((vx[i] >> (8 * j)) & 255) == MX_NAN) vx[i] &= ~(255u << (8 * j));
    };
    // E for scales up to the lanes' b: 4 above the largest; -1: all 0
    auto widest = [&](int b) __attribute__((always_inline)) {
        const int x = (int)__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_max_v(b == (int)MX_NAN ? 0.0f : (float)b, lane))));
        return x ? min(x + 4, 254) : -1;
    };
    auto pair = [&](uint32_t w, int i) __attribute__((always_inline)) {  // bytes 2 i and 2 i + 1 of w
        return __builtin_bit_cast(us2, __builtin_amdgcn_perm(0u, w, i ? 0x0c030c02u : 0x0c010c00u));
    };
    // two bytes q + 128 of w (sel) as f16 times the scales s, off = -1152 s
    auto unpack = [&](uint32_t w, uint32_t sel, h2 s, h2 off) __attribute__((always_inline)) {
        return __builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(0x64646464u, w, sel)), s, off);
    };
    const h2 k1152 = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    uint32_t i = i0 + wave;
    load_k(i);
    load_v(i);
    if (__all(alike)) {
        for (; i < i1; i += 4) {
            const Tile t = tile(i);
            const bool whole = all_see(t);
            clear(t);
            if (!whole) poison(t);
            us2 hi = {0, 0}, lo = {0xffff, 0xffff};  // the largest scale, and the smallest that is not 0, less 1
            auto note = [&](us2 b) __attribute__((always_inline)) {
                hi = __builtin_elementwise_max(hi, b);
                lo = __builtin_elementwise_min(lo, (us2)(b - us2{1, 1}));
            };
            note(pair(kx[0], 0)), note(pair(kx[1], 0));
            if constexpr (NB == 4) note(pair(kx[0], 1)), note(pair(kx[1], 1));
            const int khi = max(hi[0], hi[1]), klo = min(lo[0], lo[1]);
            hi = us2{0, 0}, lo = us2{0xffff, 0xffff};
#pragma unroll
            for (int c = 0; c < 4; c++) note(pair(vx[c >> 1], c & 1));
            const int vhi = max(hi[0], hi[1]), vlo = min(lo[0], lo[1]);
            // the wavefront's E: from its first tile that is not all zeros
            if (ek < 0 && (ek = widest(khi)) >= 0) {
#pragma unroll
                for (int r = 0; r < RG; r++) cs[r] = __builtin_ldexpf(a.scale * MX_LOG2E, ek - 138 + qe[r] - 14);
            }
            if (ev < 0) ev = widest(vhi);
            if (!__all(khi <= max(ek, 0) && klo + 1 >= ek - 19 && vhi <= max(ev, 0) && vlo + 1 >= ev - 19)) break;
            // ---- S^T = K Q^T
            const us2 bk = {(uint16_t)max(ek - 20, 0), (uint16_t)max(ek - 20, 0)};  // (exponent 20: 2^5)
            const us2 dk = {(uint16_t)max(20 - max(ek, 0), 0), (uint16_t)max(20 - max(ek, 0), 0)};
            f32x4 s[RG][2];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < CC; c++) {
                    const uint32_t at = 2 * c + (g >> 1);
                    const us2 b = __builtin_bit_cast(us2, __builtin_amdgcn_perm(0u, kx[h], 0x0c000c00u | at | (at << 16)));
                    const h2 sc = __builtin_bit_cast(h2, (us2)((__builtin_elementwise_sub_sat(b, bk) + dk) << us2{10, 10}));
                    const h2 off = sc * k1152;
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        h8 k;
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const h2 v = unpack(kw[h][c][2 * x + (y >> 1)], y & 1 ? 0x04030402u : 0x04010400u, sc, off);
                            k[2 * y] = v[0];
                            k[2 * y + 1] = v[1];
                        }
#pragma unroll
                        for (int r = 0; r < RG; r++) {
                            s[r][h] = mx_mfma(k, qh[r][2 * c + x], c + x ? s[r][h] : f32x4{0, 0, 0, 0});
                            s[r][h] = mx_mfma(k, ql[r][2 * c + x], s[r][h]);
                        }
                    }
                }
            load_k(i + 4);
            softmax(t, whole, s, cs);
            rescale();
            // ---- O^T += V^T P^T
            h8 ph[RG], pl[RG];
#pragma unroll
            for (int r = 0; r < RG; r++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = p[r][j] * 0x1p15f;  // (so that small probabilities keep their low parts)
                    ph[r][j] = (_Float16)x;
                    pl[r][j] = (_Float16)(x - (float)ph[r][j]);
                }
            const us2 bv = {(uint16_t)max(ev - 20, 0), (uint16_t)max(ev - 20, 0)};
            const us2 dv = {(uint16_t)max(20 - max(ev, 0), 0), (uint16_t)max(20 - max(ev, 0), 0)};
            h2 sv[4], ov[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                sv[c] = __builtin_bit_cast(h2, (us2)((__builtin_elementwise_sub_sat(pair(vx[c >> 1], c & 1), bv) + dv) << us2{10, 10}));
                ov[c] = sv[c] * k1152;
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                h8 v;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const h2 u = unpack(vw[d >> 1][2 * (d & 1) + (y >> 1)], y & 1 ? 0x04030402u : 0x04010400u, sv[y], ov[y]);
                    v[2 * y] = u[0];
                    v[2 * y + 1] = u[1];
                }
#pragma unroll
                for (int r = 0; r < RG; r++) {
                    o[r][d] = mx_mfma(v, ph[r], o[r][d]);
                    o[r][d] = mx_mfma(v, pl[r], o[r][d]);
                }
            }
            load_v(i + 4);
        }
    }
    int back = max(ev, 0) - 153;  // o times 2^back: the outputs
    if (i < i1) {  // the other tiles in f32
#pragma unroll
        for (int r = 0; r < RG; r++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[r][d][x] = __builtin_ldexpf(o[r][d][x], back);
        back = 0;
        float c[RG];
#pragma unroll
        for (int r = 0; r < RG; r++) c[r] = a.scale * MX_LOG2E;
        for (; i < i1; i += 4) {
            const Tile t = tile(i);
            const bool whole = all_see(t);
            clear(t);
            if (!whole) poison(t);
            f32x4 s[RG][2];
#pragma unroll
            for (int r = 0; r < RG; r++) {
                const uint64_t at = q_at(r);
                s[r][0] = s[r][1] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int cc = 0; cc < CC; cc++)
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const float q = gload<float>(at + cc * 256 + 4 * x);
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            s[r][h] = mx_mfma(mx_value((kw[h][cc][x >> 2] >> (8 * (x & 3))) & 255, (kx[h] >> (8 * (2 * cc + (g >> 1)))) & 255), q, s[r][h]);
                    }
            }
            load_k(i + 4);
            softmax(t, whole, s, c);
            rescale();
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float v = mx_value((vw[d >> 1][2 * (d & 1) + (j >> 2)] >> (8 * (j & 3))) & 255, (vx[j >> 2] >> (8 * (j & 3))) & 255);
#pragma unroll
                    for (int r = 0; r < RG; r++) o[r][d] = mx_mfma(v, p[r][j], o[r][d]);
                }
            load_v(i + 4);
        }
    }
    // ---- the four wavefronts' states meet: [wave][row][HD + 4], then [wave][row] (m, l)
    constexpr int LD = HD + 4;
    float* ol = reinterpret_cast<float*>(mx_lds);
    float* ml = ol + 4 * RG * 16 * LD;
#pragma unroll
    for (int r = 0; r < RG; r++) {
        float lt = l[r];
        lt += bfly_f<4>(lt, lane);
        lt += bfly_f<5>(lt, lane);
        const uint32_t at = wave * RG * 16 + r * 16 + n16;
        if (g == 0) {
            ml[2 * at] = m[r];
            ml[2 * at + 1] = lt;
        }
        // dimensions DT * (4 g + x) + d of the row
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int d = 0; d < DT; d += 4)
                *reinterpret_cast<float4*>(ol + at * LD + DT * (4 * g + x) + d) =
                    make_float4(__builtin_ldexpf(o[r][d][x], back), __builtin_ldexpf(o[r][d + 1][x], back),
                                __builtin_ldexpf(o[r][d + 2][x], back), __builtin_ldexpf(o[r][d + 3][x], back));
    }
    __syncthreads();
    for (uint32_t k = tid; k < RG * 16 * (HD / 4); k += 256) {
        const uint32_t lr = k / (HD / 4), c = k % (HD / 4), row = r0 + lr;
        if (row >= nrow) continue;
        float M = -3.0e38f;
#pragma unroll
        for (int w = 0; w < 4; w++) M = fmaxf(M, ml[2 * (w * RG * 16 + lr)]);
        float L = 0.0f;
        float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const uint32_t at = w * RG * 16 + lr;
            const float lw = ml[2 * at + 1];
            if (lw != 0.0f) {
                const float f = __builtin_amdgcn_exp2f(ml[2 * at] - M);
                const float4 v = *reinterpret_cast<const float4*>(ol + at * LD + 4 * c);
                L += lw * f;
                s = make_float4(s.x + v.x * f, s.y + v.y * f, s.z + v.z * f, s.w + v.w * f);
            }
        }
        const uint32_t t = row / G, h = kvh * G + row % G;
        const uint64_t at = (uint64_t)t * a.nh + h;
        if (a.nsplit == 1) {
            const float4 z = L == 0.0f ? make_float4(0, 0, 0, 0) : make_float4(s.x / L, s.y / L, s.z / L, s.w / L);
            gstore<float4>(a.o + 4 * (at * HD + 4 * c), z);
        } else {
            gstore<float4>(a.part_o + 4 * ((at * a.nsplit + blockIdx.z) * HD + 4 * c), s);
            if (c == 0) gstore<float2>(a.part_ml + 8 * (at * a.nsplit + blockIdx.z), make_float2(M, L));
        }
    }
}

#define ATTN_MX8(HD, NAME, TREE)                                                                                      \
    KERNEL __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void qp_attn_mx8_h##HD##_##NAME##_r1(       \
        QpAttnArgs a) { attn_mx8_body<HD, 1, TREE>(a); }                                                              \
    KERNEL __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void qp_attn_mx8_h##HD##_##NAME##_r2(       \
        QpAttnArgs a) { attn_mx8_body<HD, 2, TREE>(a); }
ATTN_MX8(64, causal, false) ATTN_MX8(128, causal, false) ATTN_MX8(64, tree, true) ATTN_MX8(128, tree, true)

// The shares' partial states of each (query, head) row -> o, in their order: grid rows, hd threads (at most 64 shares).
// A row that no share saw a key of is 0.
KERNEL __launch_bounds__(128) void qp_attn_mx8_comb(QpAttnArgs a) {
    __shared__ float wt[64], den;
    const uint32_t t = blockIdx.x / a.nh, d = threadIdx.x, ns = a.nsplit;
    if (t >= paso_T(a.paso)) return;
    const uint64_t row = blockIdx.x, po = a.part_o + 4 * (row * ns * a.hd + d);
    float v[8];
#pragma unroll
    for (uint32_t s = 0; s < 8; s++) v[s] = s < ns ? gload<float>(po + 4ull * s * a.hd) : 0.0f;
    if (d < 64) {
        const float2 ml = d < ns ? gload<float2>(a.part_ml + 8 * (row * ns + d)) : make_float2(-3.0e38f, 0.0f);
        const float M = wave_max_v(ml.x, d), f = ml.y != 0.0f ? __builtin_amdgcn_exp2f(ml.x - M) : -1.0f;
        wt[d] = f;
        const float L = wave_sum_v(ml.y != 0.0f ? ml.y * f : 0.0f, d);
        if (d == 0) den = L;
    }
    __syncthreads();
    float o = 0.0f;
    for (uint32_t s0 = 0; s0 < ns; s0 += 8) {
#pragma unroll
        for (uint32_t s = 0; s < 8; s++)
            if (s0 + s < ns && wt[s0 + s] != -1.0f) o += v[s] * wt[s0 + s];
#pragma unroll
        for (uint32_t s = 0; s < 8; s++) v[s] = s0 + 8 + s < ns ? gload<float>(po + 4ull * (s0 + 8 + s) * a.hd) : 0.0f;
    }
    gstore<float>(a.o + 4 * (row * a.hd + d), den == 0.0f ? 0.0f : o / den);
}
