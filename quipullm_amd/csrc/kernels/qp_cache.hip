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

// 1 / sqrt(y) for y >= 0: the instruction (off by a step, and no subnormal y) and a step of Newton's, since a value next to the
// border of two bytes of a block may fall to either side for any error
QP_DEV float rsqrt_any(float y) {
    const bool tiny = y < 0x1p-100f;
    const float z = tiny ? y * 0x1p100f : y, r = __builtin_amdgcn_rsqf(z), n = fmaf(0.5f * r, fmaf(-z * r, r, 1.0f), r);
    const float s = z > 0.0f && z < __builtin_inff() ? n : r;
    return tiny ? s * 0x1p50f : s;
}

// A wavefront has one token (hd = 128) or two (hd = 64) of N heads of q, of k or of v, which share the token's angles; grid
// (ceil(T / tokens), ceil(groups of N heads / 4)).  A lane takes the two elements of a pair, norms and rotates them, then
// (through LDS where pairs are not neighbours) two neighbouring channels, which it stores.  With a token's 48 heads one by one
// it is bound by the latency of its loads (T = 1, 8B shape: 2.7 us); with many tokens it was by the instructions for each head
// (2048 tokens of 32 + 2 x 4 heads of 128: 30.4 us), hence the kind of head and the addresses in scalar registers and the angles
// once for four heads: 17.7 us, 4.2 TB/s.
template <int HD, int N>
QP_DEV void norm_rope_kv_body(const QpRopeKvArgs& a) {
    __shared__ float row_s[4][N][128];
    constexpr uint32_t HL = HD / 2, TW = 128 / HD;              // lanes per head, tokens of a wavefront
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & (HL - 1);
    const uint32_t nq = a.nh, gq = (nq + N - 1) / N, gk = (a.nkv + N - 1) / N, group = blockIdx.y * 4 + wave;
    if (group >= gq + 2 * gk) return;
    const bool isq = group < gq, isv = group >= gq + gk;
    const uint32_t h0 = (isq ? group : isv ? group - gq - gk : group - gq) * N, nx = isq ? nq : a.nkv;
    const uint32_t t0 = blockIdx.x * TW, t = t0 + lane / HL, half = isv ? 0 : a.nrot >> 1;
    const bool apart = a.neox && l < half;                      // pairs (j, j + nrot / 2)
    const uint32_t i0 = apart ? l : 2 * l, i1 = apart ? l + half : 2 * l + 1, row0 = lane / HL * nx * HD;
    const uint64_t in = (isq ? a.q : isv ? a.v : a.k) + 4 * ((uint64_t)t0 * nx + h0) * HD;
    const bool covered = t < a.tcov;
    float x0[N], x1[N];
#pragma unroll
    for (int n = 0; n < N; n++) {  // (the loads are of the call's T rows, whatever the Paso says)
        const bool on = covered && h0 + n < nx;
        x0[n] = on ? gload<float>(in + n * HD * 4 + (row0 + i0) * 4) : 0.0f;
        x1[n] = on ? gload<float>(in + n * HD * 4 + (row0 + i1) * 4) : 0.0f;
    }
    const uint64_t w = isv ? 0 : isq ? a.qnorm : a.knorm;
    const float w0 = w ? gload<float>(w + 4 * i0) : 1.0f, w1 = w ? gload<float>(w + 4 * i1) : 1.0f;
    const float freq = l < half ? gload<float>(a.freq + 4 * l) : 0.0f;
    const uint2 paso = gload<uint2>(a.paso);
    const uint32_t T = min(__builtin_amdgcn_readfirstlane(paso.x), a.tcov), pos0 = __builtin_amdgcn_readfirstlane(paso.y);
    const uint32_t pos = a.pos && covered ? cptr<uint32_t>(a.pos)[t] : pos0 + t;
    if (t0 >= T) return;
    if (w) {
        float ss[N];
#pragma unroll
        for (int n = 0; n < N; n++) ss[n] = x0[n] * x0[n] + x1[n] * x1[n];
#pragma unroll
        for (int n = 0; n < N; n++) {
            ss[n] += bfly_f<0>(ss[n], lane);
            ss[n] += bfly_f<1>(ss[n], lane);
            ss[n] += bfly_f<2>(ss[n], lane);
            ss[n] += bfly_f<3>(ss[n], lane);
            ss[n] += bfly_f<4>(ss[n], lane);
            if constexpr (HL == 64) ss[n] += bfly_f<5>(ss[n], lane);
            const float inv = rsqrt_any(ss[n] * (1.0f / HD) + a.eps);
            x0[n] = (x0[n] * inv) * w0;
            x1[n] = (x1[n] * inv) * w1;
        }
    }
    if (half) {
        float sn, cs;
        sincos_far(((float)pos * a.esc) * freq, sn, cs);
        if (l >= half) sn = 0.0f, cs = 1.0f;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const float r0 = x0[n] * cs - x1[n] * sn, r1 = x0[n] * sn + x1[n] * cs;
            x0[n] = l < half ? r0 : x0[n];
            x1[n] = l < half ? r1 : x1[n];
        }
        if (a.neox) {  // back to neighbouring channels
#pragma unroll
            for (int n = 0; n < N; n++) {
                float* row = row_s[wave][n] + (lane - l) * 2;
                row[i0] = x0[n];
                row[i1] = x1[n];
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int n = 0; n < N; n++) {
                const float2 x = *reinterpret_cast<const float2*>(row_s[wave][n] + lane * 2);
                x0[n] = x.x;
                x1[n] = x.y;
            }
        }
    }
    if (t >= T) return;
    const uint32_t c = 2 * l;
    if (isq) {
        const uint64_t out = a.qo + 4 * ((uint64_t)t0 * nx + h0) * HD;
#pragma unroll
        for (int n = 0; n < N; n++)
            if (h0 + n < nx) gstore<float2>(out + n * HD * 4 + (row0 + c) * 4, make_float2(x0[n], x1[n]));
        return;
    }
    uint32_t slot = pos0 + t;
    if (a.cap) slot %= a.cap;
    if (slot >= a.rows) return;
    const uint32_t kvd = a.nkv * HD, R = mx_slots(a.rows);
#pragma unroll
    for (int n = 0; n < N; n++) {
        const uint32_t h = h0 + n, ch = h * HD + c;
        if (h >= nx) break;
        if (a.fmt == 0) {
            gstore<float2>((isv ? a.vc : a.kc) + 4 * ((uint64_t)slot * kvd + ch), make_float2(x0[n], x1[n]));
        } else if (a.fmt == 1) {
            if (isv) {
                mptr<uint16_t>(a.vc)[vt_index(slot, kvd, ch)] = f2h(x0[n]);
                mptr<uint16_t>(a.vc)[vt_index(slot, kvd, ch + 1)] = f2h(x1[n]);
            } else {
                gstore<uint32_t>(a.kc + 2 * ((uint64_t)slot * kvd + ch), (uint32_t)f2h(x0[n]) | ((uint32_t)f2h(x1[n]) << 16));
            }
        } else {
            // the largest magnitude of 32 channels (16 lanes; a NaN's or an infinity's bits lie above all others)
            uint32_t m = max(__float_as_uint(x0[n]) & 0x7fffffffu, __float_as_uint(x1[n]) & 0x7fffffffu);
            m = max(m, bfly<0>(m, lane));
            m = max(m, bfly<1>(m, lane));
            m = max(m, bfly<2>(m, lane));
            m = max(m, bfly<3>(m, lane));
            const uint32_t x = mx_scale(__uint_as_float(m)), b0 = mx_byte(x0[n], x), b1 = mx_byte(x1[n], x);
            if (isv) {
                mptr<uint8_t>(a.vc)[mx_v_at(h, slot, c, R, HD)] = (uint8_t)b0;
                mptr<uint8_t>(a.vc)[mx_v_at(h, slot, c + 1, R, HD)] = (uint8_t)b1;
                if ((l & 15) == 0) mptr<uint8_t>(a.vc)[mx_vx_at(h, slot, l >> 4, R, HD, a.nkv)] = (uint8_t)x;
            } else {
                gstore<uint16_t>(a.kc + mx_k_at(h, slot, c, R, HD), (uint16_t)(b0 | (b1 << 8)));
                if ((l & 15) == 0) mptr<uint8_t>(a.kc)[mx_kx_at(h, slot, l >> 4, R, HD, a.nkv)] = (uint8_t)x;
            }
        }
    }
}
#define NORM_ROPE_KV(HD, N) \
    KERNEL __launch_bounds__(256) void qp_norm_rope_kv_h##HD##_##N(QpRopeKvArgs a) { norm_rope_kv_body<HD, N>(a); }
NORM_ROPE_KV(64, 1) NORM_ROPE_KV(64, 4) NORM_ROPE_KV(128, 1) NORM_ROPE_KV(128, 4)

// ====================================================================================== reading back
// Rows of positions p0 .. p0 + n - 1 as f32 or f16 [n][nkv hd]: a thread takes two channels of K and of V, of row blockIdx.y
// times the rows that a workgroup holds (grid (pairs of channels / 256, rows), the rows strided over past 65535 workgroups).
// Latency; with a division of 64 bits in each thread's index it was the instructions (512 rows of 16 heads of 64: 4.0 us,
// now 3.9; 2048 of 4 of 128: 5.3, now 5.1).
KERNEL __launch_bounds__(256) void qp_kv_read(QpKvReadArgs a) {
    const uint32_t kvd = a.nkv * a.hd, R = mx_slots(a.rows);
    const uint32_t pairs = kvd >> 1, wide = min(pairs, 256u), hold = 256 / wide, sh = a.hd == 128 ? 7 : 6;
    const uint32_t ch = 2 * (blockIdx.x * 256 + threadIdx.x % wide), h = ch >> sh, c = ch & (a.hd - 1);
    if (ch >= kvd || threadIdx.x >= hold * wide) return;
    for (uint64_t t64 = (uint64_t)blockIdx.y * hold + threadIdx.x / wide; t64 < a.n; t64 += (uint64_t)gridDim.y * hold) {
        const uint32_t t = (uint32_t)t64;
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
// grid (pieces / 256, 2 caches): cache 2 i is layer i's K, 2 i + 1 its V.  Latency: 6 rows in 32 layers of 8 f16 heads of 128
// 6.0 us, 4 rows in 2 layers of 16 8-bit heads of 64 4.2 us, of which a launch that does nothing is 2.
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

// Scores are S^T = K Q^T and outputs O^T += V^T P^T with v_mfma_f32_16x16x32_f16: a lane holds 8 scores of one row, which are its
// operand of the second product.  Queries and probabilities are f16 high and low parts (22 bits) below a power of two.  Keys and
// values are q 2^(x - E + 5) with an E of their own, exact and normal for x - E = -19 .. 0; a tile with blocks outside that
// range moves E (and the sums so far with it).  Where no E will do (blocks of one tile further apart than 2^19, values that would
// move E over more than 2^60, or not finite; eight inputs of a query that are all below 2^-16 of its largest, whose parts would
// lose bits, or not finite), the workgroup computes its rows with the f32 matrix instruction instead (attn_mx8_f32: one token
// behind 4100 keys of the 8B shape 81 us for 11, 32 behind 480 35 for 15, 2048 1220 for 108).  So no row loses bits to a key that
// it does not see.
//
// Probabilities are 2^(s - m) with a reference m of the row that lies MX_UP below its largest score, so that their f16 parts
// stay normal.  m follows the largest score only when a tile passes it by MX_LAG: until then probabilities of up to
// 2^(MX_UP + MX_LAG) are summed as they are, and no wavefront exchanges maxima or rescales its outputs.  (Where 2^20 is past, m
// is the largest score itself: less 10 it could be rounded to 16 or 32 below, and a probability to 2^16, past f16's range.)
constexpr float MX_LAG = 5.0f, MX_UP = 10.0f;
//
// Blocks of 128 rows (8B shape, 2048 tokens: 108 us, 0.64 PFLOP/s of issued products; a tree of 64 of 8 heads behind 32700 keys
// 88 us): matrix cores busy 35 % of the time and the vector unit 47 %, at a clock of 1.8 GHz; a SIMD's four wavefronts run the
// two after each other more than at once, although nothing orders them (one half of the wavefronts half a tile behind the other:
// 118 us).  Without the shared unpacking (blocks of 16 rows) the vector unit has it to itself, 156 us.  Blocks of 16 rows: one
// token behind 131000 keys 46 us (277 MB at 6.1 TB/s, some of it from the last-level cache), behind 4100 keys 9.4 us: the chain
// Paso, tile, scores, outputs, and the meeting of four wavefronts.

// What a wavefront works on.  WIDE: a workgroup takes 128 RG (query, head) rows of one KV head, 16 RG for each of its eight
// wavefronts, and all of them take all tiles of its share of the keys; else its four have the same 16 RG rows.
template <int HD, int RG, bool TREE, bool WIDE>
struct MxWork {
    static constexpr int CC = HD / 64, KS = HD / 32, DT = HD / 16, NB = HD / 32;
    struct Tile { uint32_t slot, lo, hi; int off; };  // 32 slots from slot on; lo .. hi of them hold keys slot + off
    uint32_t lane, wave, g, n16, T, pos0, G, kvh, nrow, R;
    uint32_t b0, b_lo, b_hi, r0, t_lo, t_hi;  // the workgroup's rows and their tokens, the wavefront's
    uint32_t kbeg, first, end_a, end_b, ta, i0, i1;
    uint64_t hk, hx;                          // the head's bytes and scales in a cache
    int lim[RG];                              // the lane's rows' positions: they see keys lim - swa < key <= lim,
    uint32_t word[RG];                        // TREE: those below pos0, and the drafted ones of their mask words
    const QpAttnArgs& a;

    QP_DEV MxWork(const QpAttnArgs& args) : a(args) {
        lane = threadIdx.x & 63, g = lane >> 4, n16 = lane & 15;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        G = a.group, kvh = blockIdx.x, R = mx_slots(a.rows);
        hk = (uint64_t)kvh * R * HD, hx = (uint64_t)a.nkv * R * HD + (uint64_t)kvh * R * NB;
        // long prompts: the blocks with the most keys first, then those with the fewest on (two workgroups share a CU)
        const uint32_t y = blockIdx.y, ny = gridDim.y, blk = TREE ? y : y < (ny + 1) / 2 ? ny - 1 - y : y - (ny + 1) / 2;
        b0 = blk * (WIDE ? 128 * RG : 16 * RG);
        r0 = b0 + (WIDE ? wave * 16 * RG : 0);
    }
    // What depends on the Paso; false where it has no rows for the workgroup.
    QP_DEV bool begin() {
        const uint2 paso = gload<uint2>(a.paso);
        T = min(__builtin_amdgcn_readfirstlane(paso.x), a.tcov), pos0 = __builtin_amdgcn_readfirstlane(paso.y), nrow = T * G;
        if (b0 >= nrow) return false;
        b_lo = token(b0), b_hi = token(min(b0 + (WIDE ? 128 * RG : 16 * RG), nrow) - 1);
        t_lo = token(min(r0, nrow - 1)), t_hi = token(min(r0 + 16 * RG, nrow) - 1);
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t t = token(row(r));
            uint32_t p = pos0 + t;
            if constexpr (TREE) {
                if (a.where) p = min(max(cptr<uint32_t>(a.where)[t], pos0), pos0 + T - 1);
                word[r] = t * a.mw;
            }
            lim[r] = (int)p;
        }
        // the key tiles: keys kbeg .. kend in slots first .. (ring: then 0 ..), whole tiles of 32 slots
        const uint32_t last = TREE ? T - 1 : b_hi, early = TREE ? 0 : b_lo;
        const uint32_t kend = a.cap ? pos0 + last + 1 : min(pos0 + last + 1, a.rows);
        kbeg = a.swa && pos0 + early + 1 > a.swa ? min(pos0 + early + 1 - a.swa, kend) : 0;
        first = a.cap ? kbeg % a.cap : kbeg;
        const uint32_t nkey = a.cap ? min(kend - kbeg, a.cap) : kend - kbeg;
        end_a = a.cap ? min(first + nkey, a.cap) : first + nkey, end_b = first + nkey - end_a;
        ta = nkey ? (end_a + 31) / 32 - first / 32 : 0;
        const uint32_t nt = ta + (end_b + 31) / 32, per = a.nsplit_inv ? __umulhi(nt + a.nsplit - 1, a.nsplit_inv) : nt;
        i0 = blockIdx.z * per, i1 = min(nt, i0 + per);
        return true;
    }
    // the token of (query, head) row x (below 2^23)
    QP_DEV uint32_t token(uint32_t x) const { return a.group_inv ? __umulhi(x, a.group_inv) : x; }
    // the lane's row of group r (past those that the dispatch covers: the last), and its query from the lane's inputs on
    QP_DEV uint32_t row(int r) const { return min(r0 + r * 16 + n16, a.tcov * G - 1); }
    QP_DEV uint64_t query(int r) const {
        const uint32_t rc = row(r), t = token(rc);
        return a.q + 4 * (((uint64_t)t * a.nh + kvh * G + rc - t * G) * HD + 16 * g);
    }
    QP_DEV Tile tile(uint32_t i) const {
        if (i < ta) return {(first / 32 + i) * 32, first, end_a, (int)(kbeg - first)};
        return {(i - ta) * 32, 0, end_b, (int)(kbeg + a.cap - first)};
    }
    // slot k of the tile holds a key; all do
    QP_DEV bool held(const Tile& t, uint32_t k) const { return t.slot + k >= t.lo && t.slot + k < t.hi; }
    QP_DEV bool full(const Tile& t) const { return t.slot >= t.lo && t.slot + 32 <= t.hi; }
    // TREE: bits of the lane's row's mask for the tile's 32 slots (drafted tokens only)
    QP_DEV uint32_t drafted(const Tile& t, int r) const {
        if constexpr (!TREE) return 0;
        const int j = (int)t.slot + t.off - (int)pos0, w = j >> 5, sh = j & 31;
        const uint32_t w0 = w >= 0 && w < (int)a.mw ? gload<uint32_t>(a.mask + 4ull * (word[r] + (uint32_t)w)) : 0;
        const uint32_t w1 = w + 1 >= 0 && w + 1 < (int)a.mw ? gload<uint32_t>(a.mask + 4ull * (word[r] + (uint32_t)(w + 1))) : 0;
        return (uint32_t)((((uint64_t)w1 << 32) | w0) >> sh);
    }
    // the lane's row sees the key in slot k of the tile
    QP_DEV bool sees(const Tile& t, int r, uint32_t k, uint32_t bits) const {
        const int key = (int)(t.slot + k) + t.off;
        const bool in = !a.swa || key > lim[r] - (int)a.swa;
        if constexpr (TREE) return held(t, k) & (key < (int)pos0 ? in : ((bits >> k) & 1) != 0);
        else return held(t, k) & (key <= lim[r]) & in;
    }
    // all slots hold keys that all rows of tokens lo .. hi see
    QP_DEV bool all_see(const Tile& t, uint32_t lo, uint32_t hi) const {
        const int k0 = (int)t.slot + t.off;
        return full(t) && k0 + 31 <= (int)pos0 + (TREE ? -1 : (int)lo) && (!a.swa || k0 > (int)(pos0 + (TREE ? T - 1 : hi)) - (int)a.swa);
    }
    // some row of the wavefront may see a key of the tile
    QP_DEV bool wanted(const Tile& t) const {
        const int k0 = (int)t.slot + t.off;
        return r0 < nrow && (TREE || (k0 <= (int)(pos0 + t_hi) && (!a.swa || k0 + 31 > (int)(pos0 + t_lo) - (int)a.swa)));
    }
    // Channels c .. c + 3 of (query, head) row `row`, over the keys of the state (m, l): the output, or this share's partial
    // state.  (States hold outputs that are divided by their l: o itself can be 2^15 times as large, past f32's range.)
    QP_DEV void put(uint32_t row, uint32_t c, float4 s, float m, float l) const {
        const uint32_t t = token(row);
        const uint64_t at = (uint64_t)t * a.nh + kvh * G + row - t * G;
        if (a.nsplit == 1) {
            gstore<float4>(a.o + 4 * (at * HD + c), s);
        } else {
            gstore<float4>(a.part_o + 4 * ((at * a.nsplit + blockIdx.z) * HD + c), s);
            if (c == 0) gstore<float2>(a.part_ml + 8 * (at * a.nsplit + blockIdx.z), make_float2(m, l));
        }
    }
};

// A wavefront's softmax state.  o: row n16 of group r, channels DT (4 g + x) + d in o[r][d][x].
template <int HD, int RG>
struct MxState {
    static constexpr int DT = HD / 16;
    f32x4 o[RG][DT];
    float m[RG], l[RG], p[RG][8];
    bool far;  // some row's m lies past 2^20

    QP_DEV void start() {
        far = false;
#pragma unroll
        for (int r = 0; r < RG; r++) {
            m[r] = -3.0e38f;
            l[r] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[r][d] = f32x4{0, 0, 0, 0};
        }
    }
    // Accumulators s of the lane's 8 keys of each row: those of keys that the row does not see become -inf.
    template <class W>
    QP_DEV void hide(const W& w, const typename W::Tile& t, f32x4 (&s)[RG][2]) const {
        if (w.all_see(t, w.t_lo, w.t_hi)) return;
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t bits = w.drafted(t, r);
#pragma unroll
            for (int j = 0; j < 8; j++)
                s[r][j >> 2][j & 3] = w.sees(t, r, (j >> 2) * 16 + 4 * w.g + (j & 3), bits) ? s[r][j >> 2][j & 3] : -__builtin_inff();
        }
    }
    // The same, and the row's reference m follows them (scores: s times unit, in units of log2).  c: what s is to be multiplied by
    // from now on.
    template <class W>
    QP_DEV void follow(const W& w, const typename W::Tile& t, f32x4 (&s)[RG][2], const float (&unit)[RG], float (&c)[RG]) {
#pragma unroll
        for (int r = 0; r < RG; r++) c[r] = unit[r];
        hide(w, t, s);
        float mx[RG];
        bool past = false;
#pragma unroll
        for (int r = 0; r < RG; r++) {
            mx[r] = s[r][0][0];
#pragma unroll
            for (int j = 1; j < 8; j++) mx[r] = fmaxf(mx[r], s[r][j >> 2][j & 3]);
            past = past | (fmaf(mx[r], c[r], -m[r]) > MX_UP + MX_LAG);  // (m + 15 may be rounded to the next 16)
        }
        if (__any(past)) {
            bool b = false;
#pragma unroll
            for (int r = 0; r < RG; r++) {
                mx[r] = fmaxf(mx[r], bfly_f<4>(mx[r], w.lane));
                mx[r] = fmaxf(mx[r], bfly_f<5>(mx[r], w.lane));
                const float top = mx[r] * c[r], mn = fmaxf(m[r], top - (fabsf(top) > 0x1p20f ? 0.0f : MX_UP));
                const float f = __builtin_amdgcn_exp2f(m[r] - mn);
                m[r] = mn;
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int x = 0; x < 4; x++) o[r][d][x] *= f;
                b = b | (fabsf(mn) > 0x1p20f && mn > -3.0e38f);
            }
            far = __any(b) != 0;
        }
        if (far) {  // (s c - m in one rounding could be as large as half of m's last place: s c first)
#pragma unroll
            for (int r = 0; r < RG; r++) {
#pragma unroll
                for (int j = 0; j < 8; j++) s[r][j >> 2][j & 3] *= c[r];
                c[r] = 1.0f;
            }
        }
    }
    // Their probabilities p: of keys j and j + 1 of row r.
    QP_DEV void weigh2(const f32x4 (&s)[RG][2], const float (&c)[RG], int r, int j) {
        p[r][j] = __builtin_amdgcn_exp2f(fmaf(s[r][j >> 2][j & 3], c[r], -m[r]));
        p[r][j + 1] = __builtin_amdgcn_exp2f(fmaf(s[r][j >> 2][(j & 3) + 1], c[r], -m[r]));
        l[r] += p[r][j];
        l[r] += p[r][j + 1];
    }
    QP_DEV void weigh(const f32x4 (&s)[RG][2], const float (&c)[RG]) {
#pragma unroll
        for (int r = 0; r < RG; r++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) weigh2(s, c, r, j);
    }
    // A value that is not finite reaches the rows that see its key, and no others: the lane's channels (which are of one
    // block) become NaN in the rows that see a key of the tile whose block is NaN.
    template <class W>
    QP_DEV void poison(const W& w, const typename W::Tile& t) {
        const uint64_t xs = w.a.vc + w.hx + (uint64_t)t.slot * W::NB + (DT * 4 * w.g / 32) * 32;
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t bits = w.drafted(t, r);
            bool nan = false;
#pragma unroll 1
            for (uint32_t i = 0; i < 32; i++) {  // byte i: lane group i / 8, value i % 8
                const uint32_t k = ((i >> 2) & 1) * 16 + 4 * (i >> 3) + (i & 3);
                nan |= w.sees(t, r, k, bits) && gload<uint8_t>(xs + i) == MX_NAN;
            }
            if (nan) {
#pragma unroll
                for (int d = 0; d < DT; d++) o[r][d] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
        }
    }
    QP_DEV void sum_l(uint32_t lane) {
#pragma unroll
        for (int r = 0; r < RG; r++) {
            l[r] += bfly_f<4>(l[r], lane);
            l[r] += bfly_f<5>(l[r], lane);
        }
    }
    // The same for a state that holds its outputs over their sums, with the largest scores themselves as references: o becomes
    // o (l 2^(m - m')) / l' and p 2^(s - m') / l', so that o stays within the values whatever they are.  l: the row's, not the
    // lane's.  (No key seen: l = 0, o = 0.)
    template <class W>
    QP_DEV void follow_over(const W& w, const typename W::Tile& t, f32x4 (&s)[RG][2], float c) {
        hide(w, t, s);
#pragma unroll
        for (int r = 0; r < RG; r++) {
            float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float v = s[r][j >> 2][j & 3] * c;
                asm("" : "+v"(v));  // (s c - m in one rounding could be as large as half of m's last place)
                s[r][j >> 2][j & 3] = v;
                top = fmaxf(top, v);
            }
            top = fmaxf(top, bfly_f<4>(top, w.lane));
            top = fmaxf(top, bfly_f<5>(top, w.lane));
            const float mn = fmaxf(m[r], top), was = l[r] * __builtin_amdgcn_exp2f(m[r] - mn);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[r][j] = __builtin_amdgcn_exp2f(s[r][j >> 2][j & 3] - mn);
                sum += p[r][j];
            }
            sum += bfly_f<4>(sum, w.lane);
            sum += bfly_f<5>(sum, w.lane);
            m[r] = mn;
            l[r] = was + sum;
            const float n = l[r] == 0.0f ? 0.0f : 1.0f / l[r], f = was * n;
#pragma unroll
            for (int j = 0; j < 8; j++) p[r][j] *= n;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[r][d][x] *= f;
        }
    }
    // channels DT (4 g + x) + d .. d + 3, times 2^back, over l (no key seen: l = 0, o = 0)
    QP_DEV float4 out4(int r, int x, int d, int back) const {
        const float f = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        return make_float4(__builtin_ldexpf(o[r][d][x] * f, back), __builtin_ldexpf(o[r][d + 1][x] * f, back),
                           __builtin_ldexpf(o[r][d + 2][x] * f, back), __builtin_ldexpf(o[r][d + 3][x] * f, back));
    }
    template <bool OVER, class W>
    QP_DEV void put_all(const W& w, int back) const {  // OVER: o is over l already
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t row = w.r0 + r * 16 + w.n16;
            if (row >= w.nrow) continue;
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int d = 0; d < DT; d += 4)
                    w.put(row, DT * (4 * w.g + x) + d,
                          OVER ? make_float4(o[r][d][x], o[r][d + 1][x], o[r][d + 2][x], o[r][d + 3][x]) : out4(r, x, d, back), m[r], l[r]);
        }
    }
};

// The workgroup's rows in f32, its share of the keys from the first tile on.  Not WIDE: by the first wavefront alone.  Values come
// as they are, up to f32's largest and beside small ones: no power of two below them all, so outputs are held over their sums.
template <int HD, int RG, bool TREE, bool WIDE>
__device__ __attribute__((noinline)) void attn_mx8_f32(const __attribute__((address_space(4))) QpAttnArgs* args) {
    const QpAttnArgs a = *args;
    using W = MxWork<HD, RG, TREE, WIDE>;
    W w(a);
    if (!w.begin() || (WIDE ? w.r0 >= w.nrow : w.wave != 0)) return;
    MxState<HD, RG> st;
    st.start();
    const float scale = a.scale * MX_LOG2E, sign = scale < 0.0f ? -1.0f : 1.0f;
    const uint64_t kb = a.kc + w.hk + w.lane * 16, vb = a.vc + w.hk + w.lane * 16, kx = a.kc + w.hx, vx = a.vc + w.hx;
    for (uint32_t i = w.i0; i < w.i1; i++) {
        const typename W::Tile t = w.tile(i);
        if (!w.wanted(t)) continue;
        f32x4 s[RG][2];
#pragma unroll
        for (int r = 0; r < RG; r++) s[r][0] = s[r][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll 1
            for (int cc = 0; cc < W::CC; cc++) {
                const u32x4 k = gload<u32x4>(kb + (uint64_t)t.slot * HD + (h * W::CC + cc) * 1024);
                const uint32_t x = gload<uint8_t>(kx + ((uint64_t)t.slot + h * 16 + w.n16) * W::NB + 2 * cc + (w.g >> 1));
#pragma unroll
                for (int b = 0; b < 16; b++)
#pragma unroll
                    for (int r = 0; r < RG; r++)
                        s[r][h] = mx_mfma(mx_value((k[b >> 2] >> (8 * (b & 3))) & 255, x), gload<float>(w.query(r) + cc * 256 + 4 * b) * sign, s[r][h]);
            }
        st.follow_over(w, t, s, fmaxf(fabsf(scale), 1.2e-38f));
        const bool whole = w.all_see(t, w.t_lo, w.t_hi);
        uint32_t x[8];
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = gload<uint8_t>(vx + (uint64_t)t.slot * W::NB + (w.n16 * W::DT / 32) * 32 + w.g * 8 + j);
            bad = bad | (x[j] == MX_NAN);
            if (!whole && (x[j] == MX_NAN || !w.held(t, (j >> 2) * 16 + 4 * w.g + (j & 3)))) x[j] = 0;
        }
        if (!whole && __any(bad)) st.poison(w, t);
#pragma unroll
        for (int d = 0; d < W::DT; d++) {
            const uint64_t at = vb + (uint64_t)t.slot * HD + (d >> 1) * 1024 + 8 * (d & 1);
            const uint2 v = gload<uint2>(at);
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int r = 0; r < RG; r++)
                    st.o[r][d] = mx_mfma(mx_value(((j < 4 ? v.x : v.y) >> (8 * (j & 3))) & 255, x[j]), st.p[r][j], st.o[r][d]);
        }
    }
    st.template put_all<true>(w, 0);
}

template <int HD, int RG, bool TREE, bool WIDE>
QP_DEV void attn_mx8_body(const QpAttnArgs& a) {
    using W = MxWork<HD, RG, TREE, WIDE>;
    using Tile = typename W::Tile;
    constexpr int CC = W::CC, KS = W::KS, DT = W::DT, NB = W::NB;
    extern __shared__ float4 mx_lds[];
    W w(a);
    // The queries' loads do not wait for the Paso, the first tiles' not for the queries (one token behind 4100 keys: 9.4 us,
    // 10.0 with each after the other), nor for the Paso where neither a window nor shares put them anywhere but at the start (one
    // token behind 100 keys: 7.0 us, 7.3).
    float4 qv[RG][KS][2];
#pragma unroll
    for (int r = 0; r < RG; r++) {
        const uint64_t at = w.query(r);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 2; i++) qv[r][s][i] = gload<float4>(at + (s >> 1) * 256 + (s & 1) * 32 + i * 16);
    }
    const uint32_t lane = w.lane, g = w.g, n16 = w.n16, wave = w.wave;
    const float scale = fabsf(a.scale) * MX_LOG2E;
    const __amdgpu_buffer_rsrc_t kr = kq_rsrc(a.kc + w.hk, (uint64_t)w.R * HD), vr = kq_rsrc(a.vc + w.hk, (uint64_t)w.R * HD);
    const __amdgpu_buffer_rsrc_t kxr = kq_rsrc(a.kc + w.hx, (uint64_t)w.R * NB), vxr = kq_rsrc(a.vc + w.hx, (uint64_t)w.R * NB);
    constexpr uint32_t NONE = 0xffffffffu;
    uint32_t kx[2], vx[2];  // the scales of the lane's key of each half, and of its 8 values' keys
    auto load_kx = [&](uint32_t slot) __attribute__((always_inline)) {  // (of a tile at `slot`; none: NONE)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t x = slot != NONE ? (slot + h * 16 + n16) * NB : QP_NOOFF;
            if constexpr (NB == 4) kx[h] = __builtin_amdgcn_raw_buffer_load_b32(kxr, x, 0, 0);
            else kx[h] = __builtin_amdgcn_raw_buffer_load_b16(kxr, x, 0, 0);
        }
    };
    auto load_vx = [&](uint32_t slot) __attribute__((always_inline)) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b64(vxr, slot != NONE ? slot * NB + (n16 * DT / 32) * 32 + g * 8 : QP_NOOFF, 0, 0);
        vx[0] = x[0];
        vx[1] = x[1];
    };
    u32x4 kw[2 * CC], vw[DT / 2];  // not WIDE: the wavefront's tile
    auto load_k = [&](uint32_t slot) __attribute__((always_inline)) {
        const uint32_t o = slot != NONE ? slot * HD + lane * 16 : QP_NOOFF;
        load_kx(slot);
#pragma unroll
        for (int c = 0; c < 2 * CC; c++) kw[c] = __builtin_amdgcn_raw_buffer_load_b128(kr, o, c * 1024, 0);
    };
    auto load_v = [&](uint32_t slot) __attribute__((always_inline)) {
        const uint32_t o = slot != NONE ? slot * HD + lane * 16 : QP_NOOFF;
        load_vx(slot);
#pragma unroll
        for (int c = 0; c < DT / 2; c++) vw[c] = __builtin_amdgcn_raw_buffer_load_b128(vr, o, c * 1024, 0);
    };
    const bool ahead = !WIDE && a.nsplit == 1 && !a.swa && wave * 32 < w.R;
    if (ahead) {
        load_k(wave * 32);
        load_v(wave * 32);
    }
    if (!w.begin()) return;
    const uint32_t i1 = w.i1;
    auto slot_of = [&](uint32_t i) __attribute__((always_inline)) { return i < i1 ? w.tile(i).slot : NONE; };
    if (!WIDE && !ahead) {
        load_k(slot_of(w.i0 + wave));
        load_v(slot_of(w.i0 + wave));
    }
    // ---- the rows' queries
    h8 qh[RG][KS], ql[RG][KS];
    int qe[RG];
    bool alike = true;  // the lane's fit the f16 parts
#pragma unroll
    for (int r = 0; r < RG; r++) {
        const bool covered = w.r0 + r * 16 + n16 < w.nrow;  // (rows of the call past Paso's: anything may stand there)
        float v[KS][8], mine = 0.0f, least = 3.4e38f;  // the largest element, the least of the largest of 8 (not 0)
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const float4 x = qv[r][s][0], z = qv[r][s][1];
            float f[8] = {x.x, x.y, x.z, x.w, z.x, z.y, z.z, z.w};
            float eight = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                f[i] = covered ? f[i] : 0.0f;
                const float u = fabsf(f[i]);
                v[s][i] = a.scale < 0.0f ? -f[i] : f[i];
                eight = fmaxf(eight, u);
                alike = alike & (u < __builtin_inff());  // (a NaN neither)
            }
            mine = fmaxf(mine, eight);
            least = fminf(least, eight == 0.0f ? 3.4e38f : eight);
        }
        float all = fmaxf(mine, bfly_f<4>(mine, lane));
        all = fmaxf(all, bfly_f<5>(all, lane));
        const int e = max((int)((__float_as_uint(all) >> 23) & 255) - 127, -110);
        alike = alike & (least >= all * 0x1p-16f);
        qe[r] = e;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x = __builtin_ldexpf(v[s][i], 14 - e);  // below 2^15
                qh[r][s][i] = (_Float16)x;
                ql[r][s][i] = (_Float16)(x - (float)qh[r][s][i]);
            }
    }
    MxState<HD, RG> st;
    st.start();
    int ek = 20, ev = 20;  // E of the keys and values (20 at least)
    int ev_span = -1;      // the lowest and (<< 8) the highest that ev has been since it was set; -1: it has not been
    int moved = 0;         // the sums are to be multiplied by 2^moved (ev has changed)
    float cs[RG];          // score = accumulator times cs, in units of log2, of keys unpacked with E = ek
    // (at most 2^88: accumulators are multiples of 2^-38 below 2^34, so that from there on two that differ are a weight of 0 apart,
    // and no score leaves f32's range)
    auto unit = [&](int e, float (&c)[RG]) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RG; r++) c[r] = __builtin_amdgcn_fmed3f(__builtin_ldexpf(scale, e + qe[r] - 152), 1.2e-38f, 0x1p88f);
    };
    auto wave_most = [&](int x) __attribute__((always_inline)) {  // of whole numbers below 2^24
        return (int)__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_max_v((float)x, lane))));
    };
    // E for the scales lo .. hi of the lanes (lo: of those that are not 0, 65536 where all are), e for those before: e where
    // it will do, else 4 above the largest or as far up as the smallest allows; 256 where no E will do.
    auto settle = [&](int lo, int hi, int e) __attribute__((always_inline)) {
        const int most = wave_most(hi), least = 65536 - wave_most(65536 - lo);
        if (most == 0) return e;
        if (most == (int)MX_NAN || least < most - 19) return 256;
        return most > e || least < e - 19 ? max(min(min(most + 4, least + 19), 254), 20) : e;
    };
    // The scales of a tile's slots without a key (which may hold anything) become 0.
    auto clear_k = [&](const Tile& t) __attribute__((always_inline)) {
        if (w.full(t)) return;
#pragma unroll
        for (int h = 0; h < 2; h++) kx[h] = w.held(t, h * 16 + n16) ? kx[h] : 0;
    };
    auto clear_v = [&](const Tile& t) __attribute__((always_inline)) {
        if (w.full(t)) return;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 4; j++) vx[h] &= w.held(t, h * 16 + 4 * g + j) ? 0xffffffffu : ~(255u << (8 * j));
    };
    // The least (of those that are not 0, 65536 where all are) and the largest scale that the lane looks at: lanes that hold the
    // same ones look at a part of them each, byte g of their keys' (hd = 64: g % 2), bytes n16 % 4 of their values'.
    struct Range { int lo, hi; };
    auto range = [&](const uint32_t (&x)[2], uint32_t byte) __attribute__((always_inline)) {
        const int a0 = (x[0] >> (8 * byte)) & 255, a1 = (x[1] >> (8 * byte)) & 255;
        return Range{min((a0 - 1) & 0xffff, (a1 - 1) & 0xffff) + 1, max(a0, a1)};
    };
    auto range_k = [&]() __attribute__((always_inline)) { return range(kx, g % NB); };
    auto range_v = [&]() __attribute__((always_inline)) { return range(vx, n16 & 3); };
    auto fits = [&](Range x, int e) __attribute__((always_inline)) { return (x.hi <= e) & (x.lo >= e - 19); };
    // E such that the tile's keys, its values fit; false where none will do.
    auto settle_k = [&]() __attribute__((always_inline)) {
        const Range x = range_k();
        ek = settle(x.lo, x.hi, ek);
        return ek < 256;
    };
    auto settle_v = [&](const Tile& t) __attribute__((always_inline)) {
        Range x = range_v();
        if (__any(x.hi == (int)MX_NAN) && !w.all_see(t, w.b_lo, w.b_hi)) {  // not every row sees every key: taken out
            st.poison(w, t);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (((vx[i] >> (8 * j)) & 255) == MX_NAN) vx[i] &= ~(255u << (8 * j));
            x = range_v();
        }
        const int e = settle(x.lo, x.hi, ev);
        const bool set = ev_span >= 0;
        const int lo = set ? min(ev_span & 255, e) : e, hi = set ? max(ev_span >> 8, e) : e;
        moved = set ? ev - e : 0;
        if (__any(x.hi != 0)) ev_span = lo | (hi << 8);
        ev = e;
        return e < 256 && hi - lo <= 60;  // (the sums, moved by all steps together, could leave f32's range)
    };
    auto move = [&]() __attribute__((always_inline)) {
        if (moved == 0) return;
#pragma unroll
        for (int r = 0; r < RG; r++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) st.o[r][d][x] = __builtin_ldexpf(st.o[r][d][x], moved);
        moved = 0;
    };
    auto pair = [&](uint32_t v, uint32_t i, uint32_t j) __attribute__((always_inline)) {  // bytes i and j of v
        return __builtin_bit_cast(us2, __builtin_amdgcn_perm(0u, v, 0x0c000c00u | i | (j << 16)));
    };
    // 2^(x - E + 5) of two blocks as f16 (0 below the normal ones)
    auto factor = [&](us2 x, int e) __attribute__((always_inline)) {
        const uint16_t lo = (uint16_t)(e - 20);  // (exponent 20: 2^5)
        return __builtin_bit_cast(h2, (us2)(__builtin_elementwise_sub_sat(x, us2{lo, lo}) << us2{10, 10}));
    };
    const h2 k1152 = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    auto key_factors = [&](uint32_t x, int c, h2 (&s)[4], h2 (&off)[4]) __attribute__((always_inline)) {
        const uint32_t at = 2 * c + (g >> 1);
        s[0] = factor(pair(x, at, at), ek);
        off[0] = s[0] * k1152;
#pragma unroll
        for (int i = 1; i < 4; i++) s[i] = s[0], off[i] = off[0];
    };
    auto value_factors = [&](const uint32_t (&x)[2], h2 (&s)[4], h2 (&off)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            s[c] = factor(pair(x[c >> 1], 2 * (c & 1), 2 * (c & 1) + 1), ev);
            off[c] = s[c] * k1152;
        }
    };
    unit(ek, cs);
    // eight bytes q + 128 as f16 times the factors s (of two bytes each), off = -1152 s
    auto unpack8 = [&](uint32_t w0, uint32_t w1, const h2 (&s)[4], const h2 (&off)[4]) __attribute__((always_inline)) {
        h8 v;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const h2 u = __builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(0x64646464u, c < 2 ? w0 : w1, c & 1 ? 0x04030402u : 0x04010400u)), s[c], off[c]);
            v[2 * c] = u[0];
            v[2 * c + 1] = u[1];
        }
        return v;
    };
    h8 ph[RG], pl[RG];
    float one = 1.0f;  // (not known to the compiler: p - high in one instruction that takes an f16 operand)
    asm("" : "+s"(one));
    auto split2 = [&](int r, int j) __attribute__((always_inline)) {
        // (rounded towards zero: the low part takes the rest, 21 bits together)
        const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(st.p[r][j], st.p[r][j + 1]));
        ph[r][j] = hi[0];
        ph[r][j + 1] = hi[1];
        pl[r][j] = (_Float16)fmaf(st.p[r][j], one, -(float)hi[0]);
        pl[r][j + 1] = (_Float16)fmaf(st.p[r][j + 1], one, -(float)hi[1]);
    };
    // Step c of the scores of both halves of the tile (their operands k0, k1), and the outputs d and d + 1 (v0, v1): no matrix
    // instruction adds to the sums of the one before it, which it would wait for.
    auto scores = [&](f32x4 (&s)[RG][2], int c, h8 k0, h8 k1) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RG; r++) {
            s[r][0] = mx_mfma(k0, qh[r][c], c ? s[r][0] : f32x4{0, 0, 0, 0});
            s[r][1] = mx_mfma(k1, qh[r][c], c ? s[r][1] : f32x4{0, 0, 0, 0});
        }
#pragma unroll
        for (int r = 0; r < RG; r++) {
            s[r][0] = mx_mfma(k0, ql[r][c], s[r][0]);
            s[r][1] = mx_mfma(k1, ql[r][c], s[r][1]);
        }
    };
    auto outputs = [&](int d, h8 v0, h8 v1) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RG; r++) {
            st.o[r][d] = mx_mfma(v0, ph[r], st.o[r][d]);
            st.o[r][d + 1] = mx_mfma(v1, ph[r], st.o[r][d + 1]);
        }
#pragma unroll
        for (int r = 0; r < RG; r++) {
            st.o[r][d] = mx_mfma(v0, pl[r], st.o[r][d]);
            st.o[r][d + 1] = mx_mfma(v1, pl[r], st.o[r][d + 1]);
        }
    };
    bool ok = __syncthreads_and(alike) != 0;
    if constexpr (!WIDE) {
        // the tiles are dealt to the wavefronts, each with a state of its own
        uint32_t i = w.i0 + wave;
        for (; ok && i < i1; i += 4) {
            const Tile t = w.tile(i);
            clear_k(t);
            clear_v(t);
            if (!__all(fits(range_k(), ek) & fits(range_v(), ev))) {
                ok = settle_k() && settle_v(t);
                if (!ok) break;
                unit(ek, cs);
                move();
            }
            f32x4 s[RG][2];
            h2 f[4], off[4], f1[4], off1[4];
#pragma unroll
            for (int c = 0; c < CC; c++) {
                key_factors(kx[0], c, f, off);
                key_factors(kx[1], c, f1, off1);
#pragma unroll
                for (int u = 0; u < 2; u++)
                    scores(s, 2 * c + u, unpack8(kw[c][2 * u], kw[c][2 * u + 1], f, off),
                           unpack8(kw[CC + c][2 * u], kw[CC + c][2 * u + 1], f1, off1));
            }
            load_k(slot_of(i + 4));
            float c[RG];
            st.follow(w, t, s, cs, c);
            st.weigh(s, c);
#pragma unroll
            for (int r = 0; r < RG; r++)
#pragma unroll
                for (int j = 0; j < 8; j += 2) split2(r, j);
            value_factors(vx, f, off);
#pragma unroll
            for (int d = 0; d < DT; d += 2)
                outputs(d, unpack8(vw[d >> 1][0], vw[d >> 1][1], f, off), unpack8(vw[d >> 1][2], vw[d >> 1][3], f, off));
            load_v(slot_of(i + 4));
        }
        ok = __syncthreads_and(ok) != 0;
    } else {
        // Every wavefront takes every tile, of which each unpacks a chunk of 1 KB to f16 in LDS (two buffers): chunk c (of K
        // below 2 CC, then of V) is wavefront c's.  It looks at that chunk's scales alone; where they do not fit E, it leaves a
        // word in LDS (one for each buffer), and all settle E anew and unpack the tile again.
        constexpr uint32_t NCH = 2 * CC + DT / 2;
        h8* lds = reinterpret_cast<h8*>(mx_lds);  // [buffer][chunk][half of the lane's bytes][lane]
        volatile uint32_t* misfit = reinterpret_cast<volatile uint32_t*>(lds + 2 * NCH * 128);
        const bool is_k = wave < 2 * CC, has = wave < NCH;
        const __amdgpu_buffer_rsrc_t mine = is_k ? kr : vr, mine_x = is_k ? kxr : vxr;
        const uint32_t at = (is_k ? wave : wave - 2 * CC) * 1024 + lane * 16;
        const uint32_t at_x = is_k ? ((wave / CC) * 16 + n16) * NB : (n16 * DT / 32) * 32 + g * 8;
        u32x4 raw;
        uint32_t x[2];  // the chunk's scales: K's of the lane's key, V's of its 8 keys
        auto load = [&](uint32_t j) __attribute__((always_inline)) {  // (past the last tile: the last)
            const uint32_t slot = w.tile(min(j, i1 - 1)).slot;
            if (is_k && NB == 2) {
                x[0] = __builtin_amdgcn_raw_buffer_load_b16(mine_x, at_x, slot * NB, 0);
            } else if (is_k) {
                x[0] = __builtin_amdgcn_raw_buffer_load_b32(mine_x, at_x, slot * NB, 0);
            } else if (has) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(mine_x, at_x, slot * NB, 0);
                x[0] = v[0];
                x[1] = v[1];
            }
            if (has) raw = __builtin_amdgcn_raw_buffer_load_b128(mine, at, slot * HD, 0);
        };
        auto stage = [&](uint32_t j) __attribute__((always_inline)) {
            if (!has) return;
            const Tile t = w.tile(j);
            h2 f[4], off[4];
            bool fit;
            if (is_k) {
                if (!w.full(t)) x[0] = w.held(t, (wave / CC) * 16 + n16) ? x[0] : 0;
                const int b = (x[0] >> (8 * (2 * (wave % CC) + (g >> 1)))) & 255;
                fit = (b <= ek) & ((b >= ek - 19) | (b == 0));
                key_factors(x[0], wave % CC, f, off);
            } else {
                if (!w.full(t)) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int j = 0; j < 4; j++) x[h] &= w.held(t, h * 16 + 4 * g + j) ? 0xffffffffu : ~(255u << (8 * j));
                }
                fit = fits(range(x, n16 & 3), ev);
                value_factors(x, f, off);
            }
            if (!__all(fit) && lane == 0) misfit[j & 1] = 1;
            h8* to = lds + ((j & 1) * NCH + wave) * 128 + lane;
            to[0] = unpack8(raw[0], raw[1], f, off);
            to[64] = unpack8(raw[2], raw[3], f, off);
        };
        uint32_t i = w.i0;
        if (ok && i < i1) {
            bool settle_now = true;  // (the first tile)
            if (threadIdx.x < 2) misfit[threadIdx.x] = 0;
            for (;;) {
                const Tile t = w.tile(i);
                if (settle_now) {
                    __syncthreads();
                    load(i);
                    load_kx(slot_of(i));
                    load_vx(slot_of(i));
                    clear_k(t);
                    clear_v(t);
                    ok = settle_k() && settle_v(t);  // (the same in all wavefronts: they see the same scales)
                    if (!ok) break;
                    unit(ek, cs);
                    move();
                    // (blocks that settle_v took out: unpacked as 0)
                    if (!is_k) x[0] = vx[0], x[1] = vx[1];
                    if (threadIdx.x == 0) misfit[i & 1] = 0;
                    stage(i);
                    load(i + 1);
                    __syncthreads();
                }
                if (w.wanted(t)) {
                    const h8* from = lds + (i & 1) * NCH * 128 + lane;
                    f32x4 s[RG][2];
#pragma unroll
                    for (int c = 0; c < KS; c++) scores(s, c, from[c * 64], from[(KS + c) * 64]);
                    float c[RG];
                    st.follow(w, t, s, cs, c);
                    st.weigh(s, c);
#pragma unroll
                    for (int r = 0; r < RG; r++)
#pragma unroll
                        for (int j = 0; j < 8; j += 2) split2(r, j);
#pragma unroll
                    for (int d = 0; d < DT; d += 2) outputs(d, from[(2 * KS + d) * 64], from[(2 * KS + d + 1) * 64]);
                }
                if (++i >= i1) break;
                stage(i);
                load(i + 1);
                __syncthreads();
                settle_now = __builtin_amdgcn_readfirstlane(misfit[i & 1]) != 0;
            }
        }
    }
    if (!ok) {
        attn_mx8_f32<HD, RG, TREE, WIDE>((const __attribute__((address_space(4))) QpAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr());
        return;
    }
    const int back = ev - 138;  // o times 2^back: the outputs
    st.sum_l(lane);
    if constexpr (WIDE) {
        st.template put_all<false>(w, back);
    } else {
        // ---- the four wavefronts' states meet: [wave][row][HD + 4], then [wave][row] (m, l)
        constexpr int LD = HD + 4;
        float* ol = reinterpret_cast<float*>(mx_lds);
        float* ml = ol + 4 * RG * 16 * LD;
#pragma unroll
        for (int r = 0; r < RG; r++) {
            const uint32_t at = wave * RG * 16 + r * 16 + n16;
            if (g == 0) {
                ml[2 * at] = st.m[r];
                ml[2 * at + 1] = st.l[r];
            }
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int d = 0; d < DT; d += 4) *reinterpret_cast<float4*>(ol + at * LD + DT * (4 * g + x) + d) = st.out4(r, x, d, back);
        }
        __syncthreads();
        for (uint32_t k = threadIdx.x; k < RG * 16 * (HD / 4); k += 256) {
            const uint32_t lr = k / (HD / 4), c = 4 * (k % (HD / 4)), row = w.r0 + lr;
            if (row >= w.nrow) continue;
            float M = -3.0e38f;
#pragma unroll
            for (int v = 0; v < 4; v++) M = fmaxf(M, ml[2 * (v * RG * 16 + lr)]);
            float f[4], L = 0.0f;  // the wavefronts' weights
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const float lw = ml[2 * (v * RG * 16 + lr) + 1];
                f[v] = lw != 0.0f ? lw * __builtin_amdgcn_exp2f(ml[2 * (v * RG * 16 + lr)] - M) : 0.0f;
                L += f[v];
            }
            const float n = L == 0.0f ? 0.0f : 1.0f / L;
            float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int v = 0; v < 4; v++) {
                if (ml[2 * (v * RG * 16 + lr) + 1] == 0.0f) continue;  // (it saw no key)
                const float4 x = *reinterpret_cast<const float4*>(ol + (v * RG * 16 + lr) * LD + c);
                const float g = f[v] * n;
                s = make_float4(s.x + x.x * g, s.y + x.y * g, s.z + x.z * g, s.w + x.w * g);
            }
            w.put(row, c, s, M, L);
        }
    }
}

#define ATTN_MX8(HD, NAME, TREE)                                                                                      \
    KERNEL __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void qp_attn_mx8_h##HD##_##NAME(            \
        QpAttnArgs a) { attn_mx8_body<HD, 1, TREE, false>(a); }                                                       \
    KERNEL __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4))) void qp_attn_mx8_h##HD##_##NAME##_wide(     \
        QpAttnArgs a) { attn_mx8_body<HD, 1, TREE, true>(a); }
ATTN_MX8(64, causal, false) ATTN_MX8(128, causal, false) ATTN_MX8(64, tree, true) ATTN_MX8(128, tree, true)

// The shares' partial states of each (query, head) row -> o, in a fixed order: grid rows, NY hd threads (at most 64 shares), the NY
// threads of one channel dealing the shares out.  A row that no share saw a key of is 0.  64 shares of 32 rows: 5.3 us (one
// thread for each channel: 7.7); 4 shares of 1024 rows: 3.9 (four threads: 4.4).  (Joined by the last workgroup of the
// attention's own launch instead, through counters: one token behind 4100 keys 13.2 us, 12.6 with this launch; 8 tokens 20.3 and
// 15.5, since that workgroup joins 16 rows; with fences that write back the L2 in place of stores through it 19.4 and 35.6.)
template <uint32_t NY>
QP_DEV void attn_mx8_comb(const QpAttnArgs& a) {
    __shared__ float wt[64], sum[NY][128];
    const uint32_t t = blockIdx.x / a.nh, d = NY == 1 ? threadIdx.x : threadIdx.x & (a.hd - 1);
    const uint32_t y = NY == 1 ? 0 : threadIdx.x / a.hd;
    const uint32_t ns = a.nsplit, T = paso_T(a.paso);
    const uint64_t row = blockIdx.x, po = a.part_o + 4 * (row * ns * a.hd + d);
    float v[8];
#pragma unroll
    for (uint32_t s = 0; s < 8; s++) v[s] = NY * s + y < ns ? gload<float>(po + 4ull * (NY * s + y) * a.hd) : 0.0f;
    const float2 mine = threadIdx.x < ns ? gload<float2>(a.part_ml + 8 * (row * ns + threadIdx.x)) : make_float2(-3.0e38f, 0.0f);
    if (t >= T) return;  // (the loads above are of the buffer all the same)
    if (threadIdx.x < 64) {
        const float M = wave_max_v(mine.x, d), f = mine.y != 0.0f ? mine.y * __builtin_amdgcn_exp2f(mine.x - M) : 0.0f;
        const float L = wave_sum_v(f, d);
        wt[d] = mine.y != 0.0f ? f / L : -1.0f;
    }
    __syncthreads();
    float o = 0.0f;
    for (uint32_t s0 = y; s0 < ns; s0 += 8 * NY) {
#pragma unroll
        for (uint32_t s = 0; s < 8; s++)
            if (s0 + NY * s < ns && wt[s0 + NY * s] != -1.0f) o += v[s] * wt[s0 + NY * s];
#pragma unroll
        for (uint32_t s = 0; s < 8; s++) v[s] = s0 + NY * (8 + s) < ns ? gload<float>(po + 4ull * (s0 + NY * (8 + s)) * a.hd) : 0.0f;
    }
    if constexpr (NY == 4) {
        sum[y][d] = o;
        __syncthreads();
        if (y) return;
        o = (o + sum[1][d]) + (sum[2][d] + sum[3][d]);
    }
    gstore<float>(a.o + 4 * (row * a.hd + d), o);
}
KERNEL __launch_bounds__(128) void qp_attn_mx8_comb(QpAttnArgs a) { attn_mx8_comb<1>(a); }
KERNEL __launch_bounds__(512) void qp_attn_mx8_comb4(QpAttnArgs a) { attn_mx8_comb<4>(a); }
