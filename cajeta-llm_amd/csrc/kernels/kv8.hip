// kv8.hip — K/V pages held in 8 bits: append with rotation, read, attention.
//
// A block is 16 consecutive positions of one kv head; K and V of a block have
// one scale each, a power of two 2^e (e from KV8_LOW to KV8_HIGH), and codes
// in −127..127. Powers of two, because blocks fill a token at a time: when a
// louder token raises e, the block's older codes are rescaled by a shift, and
// the half steps lost over all the rescalings stay under one step of the last
// scale (1/2 + 1/4 + ...), where a free scale that creeps up can lose half a
// step at each of 15 tokens. It costs up to one bit against amax / 127.
//
// A block whose values are not finite, or past 127·2^KV8_HIGH, is poisoned:
// its scale is NaN, so that every row which attends it comes out NaN.
#pragma once
#include "common.h"

#define KV8_PAGE 64
#define KV8_BLOCK 16
// 2^-48 is far below what fp16 planes hold, 127·2^63 far above; their spread
// keeps the attention's weights (scaled by 2^e against the largest) in f32's
// range, so no mixture of blocks underflows the softmax's sum.
#define KV8_LOW (-48)
#define KV8_HIGH 63

struct Kv8Seg {
    int slot, pos, row, rows;
};

// The segment s; false where it has no rows, or where its slot, rows or
// positions are out of range, which is reported.
DEV bool kv8_seg(const cj_kv8_args &a, int s, Kv8Seg &g) {
    const int4 v = ((const int4 *)a.segs)[s];
    g.slot = v.x; g.pos = v.y; g.row = v.z; g.rows = v.w;
    if (v.w == 0) return false;
    const bool ok = v.x >= 0 && v.x < a.n_slots && v.w > 0 && v.w <= a.max_rows && v.z >= 0 && v.z <= a.n_rows - v.w &&
                    v.y >= 0 && v.y <= a.limit - v.w;
    if (!ok && a.status && threadIdx.x == 0) *a.status = 1;
    return ok;
}

// The page of the slot's positions from 64·i on; −1 where the table has none.
DEV int kv8_page(const cj_kv8_args &a, int slot, int i) {
    const int p = a.pgtab[(int64_t)slot * a.slot_pages + i];
    return p >= 0 && p < a.n_pages ? p : -1;
}

// Another lane's double by DPP, and the two halves of the exchanges with lane
// ^ 16 and lane ^ 32. Pairs, quads, mirrored eights and mirrored rows: a sum
// over 8 or 16 lanes, a maximum over all.
template <int CTRL>
DEV double kv8_dpp(double v) {
    return __hiloint2double(dpp_i<CTRL>(__double2hiint(v)), dpp_i<CTRL>(__double2loint(v)));
}
#define KV8_MIRROR 0x140   // row_mirror
template <int LANES>
DEV double kv8_sum(double v) {
    v += kv8_dpp<DPP_XOR1>(v);
    v += kv8_dpp<DPP_XOR2>(v);
    v += kv8_dpp<DPP_HMIRROR>(v);
    return LANES == 8 ? v : v + kv8_dpp<KV8_MIRROR>(v);
}
DEV double kv8_max64(double v) {
    v = fmax(v, kv8_dpp<DPP_XOR1>(v));
    v = fmax(v, kv8_dpp<DPP_XOR2>(v));
    v = fmax(v, kv8_dpp<DPP_HMIRROR>(v));
    v = fmax(v, kv8_dpp<KV8_MIRROR>(v));
    int a, b, c, d;
    swap16(__double2hiint(v), a, b);
    swap16(__double2loint(v), c, d);
    v = fmax(__hiloint2double(a, c), __hiloint2double(b, d));
    swap32(__double2hiint(v), a, b);
    swap32(__double2loint(v), c, d);
    return fmax(__hiloint2double(a, c), __hiloint2double(b, d));
}
// 1 / sqrt(x) to the last bits of 64: the hardware's estimate and three
// steps of Newton's iteration.
DEV double kv8_rsqrt(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 3; i++) y = y * (1.5 - 0.5 * x * y * y);
    return y;
}

// The exponent of the scale for values up to `top`: the least e with
// top ≤ 127·2^e (127·2^(k−6) is 1.984·2^k).
DEV int kv8_exponent(double top) {
    const int k = ((__double2hiint(top) >> 20) & 0x7ff) - 1023;
    const int e = top <= ldexp(127.0, k - 6) ? k - 6 : k - 5;
    return e < KV8_LOW ? KV8_LOW : e;
}

// A stored scale's exponent, or KV8_HIGH + 1 where it is none.
DEV int kv8_exponent_of(float scale) {
    const uint32_t b = __float_as_uint(scale);
    const int e = (int)(b >> 23) - 127;
    return (b & 0x7fffffu) || (int)b < 0 || e < KV8_LOW || e > KV8_HIGH ? KV8_HIGH + 1 : e;
}

DEV float kv8_pow2(int e) { return e > KV8_HIGH ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(e + 127) << 23); }

// Four codes (bytes offset by 128) times 2^-shift, rounded half to even.
DEV uint32_t kv8_rescale4(uint32_t w, int shift) {
    uint32_t r = 0;
    const float f = __uint_as_float((uint32_t)(127 - min(shift, 120)) << 23);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float c = (float)((int)((w >> (8 * i)) & 255u) - 128);
        r |= (uint32_t)((int)rintf(c * f) + 128) << (8 * i);
    }
    return r;
}

// Rotation (and norm) of the pairs a[i], b[i] of one head's row, held by LANES
// lanes, lane j with pairs j·NP..; in 64 bits, so that the code of a value
// next to a rounding border is that of the exact one.
template <int NP, int LANES>
DEV void kv8_turn(double (&a)[NP], double (&b)[NP], const cj_kv8_args &g, const float *w, int pos, int j) {
    if (g.norm) {
        double ss = 0;
#pragma unroll
        for (int i = 0; i < NP; i++) ss += a[i] * a[i] + b[i] * b[i];
        const double s = kv8_rsqrt(kv8_sum<LANES>(ss) * (1.0 / (2 * LANES * NP)) + (double)g.eps), one = g.form ? 1.0 : 0.0;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            a[i] = a[i] * s * (one + (double)w[j * NP + i]);
            b[i] = b[i] * s * (one + (double)w[LANES * NP + j * NP + i]);
        }
    }
    const float *cs = g.rope_cs + (int64_t)pos * (2 * LANES * NP) + 2 * NP * j;
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const double c = (double)cs[2 * i], s = (double)cs[2 * i + 1], x = a[i], y = b[i];
        a[i] = x * c - y * s;
        b[i] = x * s + y * c;
    }
}

template <int NP>
DEV void kv8_load(const float *p, double (&a)[NP]) {
    float f[NP];
    if constexpr (NP == 4) *(f32x4 *)f = *(const f32x4 *)p;
    else {
        const float2 t = *(const float2 *)p;
        f[0] = t.x; f[1] = t.y;
    }
#pragma unroll
    for (int i = 0; i < NP; i++) a[i] = (double)f[i];
}

DEV void kv8_store4(float *p, const double (&a)[4]) { *(f32x4 *)p = f32x4{(float)a[0], (float)a[1], (float)a[2], (float)a[3]}; }

DEV double kv8_size(double x) { return fabs(x) <= 1.0e300 ? fabs(x) : __longlong_as_double(0x7ff0000000000000ll); }

DEV uint32_t kv8_code(double x, double inv) { return (uint32_t)((int)rint(x * inv) + 128); }

// Append: a workgroup a (segment, block, kv head), thread t position t / 16
// of the block and its rotation pairs (t % 16)·NP.., so a head's row is 16
// lanes; then workgroups of (row, query head) pairs, 16 bytes a lane (8 bytes
// a lane at head size 64: 37 → 33 us).
// Bound: HBM for many rows (3130 rows of 64 / 8 heads of 64 with the norm: 32
// us, 3.7 TB/s; without 29; q's rows alone 22), a launch for few. The 64-bit
// arithmetic costs the norm's 3 us and nothing else.
template <int HD>
DEV void kv8_append(const cj_kv8_args &a) {
    constexpr int NP = HD / 32;
    const int t = threadIdx.x, tt = t >> 4, j = t & 15;
    Kv8Seg g;
    if ((int)blockIdx.x >= a.kv_wgs) {
        // query rows: KV8_QS turns of 256 / LANES (row, head) pairs, all loaded first
        constexpr int LANES = HD / 8, PER = 256 / LANES;
        const int w = (int)blockIdx.x - a.kv_wgs, s = w / a.per_seg, it = t / LANES, d = t % LANES * 4;
        if (!kv8_seg(a, s, g)) return;
        double x[KV8_QS][4], y[KV8_QS][4];
        int r[KV8_QS], h[KV8_QS];
#pragma unroll
        for (int k = 0; k < KV8_QS; k++) {
            const int i = ((w - s * a.per_seg) * KV8_QS + k) * PER + it;
            r[k] = i / a.n_q;
            h[k] = i - r[k] * a.n_q;
            if (r[k] < g.rows) {
                const float *src = a.q + (int64_t)(g.row + r[k]) * a.q_stride + (int64_t)h[k] * HD + d;
                kv8_load<4>(src, x[k]);
                kv8_load<4>(src + HD / 2, y[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < KV8_QS; k++)
            if (r[k] < g.rows) {
                kv8_turn<4, LANES>(x[k], y[k], a, a.qw, g.pos + r[k], t % LANES);
                float *dst = a.q_out + (int64_t)(g.row + r[k]) * a.out_stride + (int64_t)h[k] * HD + d;
                kv8_store4(dst, x[k]);
                kv8_store4(dst + HD / 2, y[k]);
            }
        return;
    }
    __shared__ double tops[2][4];
    __shared__ __align__(16) uint8_t tv[HD * KV8_BLOCK];
    const int nb = (a.max_rows + KV8_BLOCK - 2) / KV8_BLOCK + 1;
    const int h = blockIdx.x % a.n_kv, w = blockIdx.x / a.n_kv, blk = w % nb, s = w / nb;
    if (!kv8_seg(a, s, g)) return;
    if (blk > (g.pos + g.rows - 1) / KV8_BLOCK - g.pos / KV8_BLOCK) return;
    const int b0 = (g.pos / KV8_BLOCK + blk) * KV8_BLOCK;
    // a slot has one segment in a call: two would write one block at once
    int twice = 0;
    for (int i = t; i < a.n_segs; i += 256) {
        const int4 o = ((const int4 *)a.segs)[i];
        twice |= i != s && o.x == g.slot && o.w > 0;
    }
    const int page = kv8_page(a, g.slot, b0 / KV8_PAGE);
    if (__syncthreads_or(twice) || page < 0) {
        if (a.status && t == 0) *a.status = 1;
        return;
    }
    const int p = b0 + tt, n_old = g.pos > b0 ? g.pos - b0 : 0;
    const bool fresh = tt >= n_old && p < g.pos + g.rows;
    const int64_t ph = (int64_t)page * a.n_kv + h, si = ph * 4 + (b0 % KV8_PAGE) / KV8_BLOCK;
    uint8_t *kb = a.kc + (ph * KV8_PAGE + b0 % KV8_PAGE) * HD;
    uint8_t *vb = a.vc + (ph * KV8_PAGE + b0 % KV8_PAGE) * HD;
    double kx[NP], ky[NP], vx[NP], vy[NP];
    double ktop = 0, vtop = 0;
    if (fresh) {
        const int64_t at = (int64_t)(g.row + (p - g.pos)) * a.kv_stride + (int64_t)h * HD + j * NP;
        kv8_load<NP>(a.k + at, kx);
        kv8_load<NP>(a.k + at + HD / 2, ky);
        kv8_load<NP>(a.v + at, vx);
        kv8_load<NP>(a.v + at + HD / 2, vy);
        kv8_turn<NP, 16>(kx, ky, a, a.kw, p, j);
#pragma unroll
        for (int i = 0; i < NP; i++) {
            ktop = fmax(ktop, fmax(kv8_size(kx[i]), kv8_size(ky[i])));
            vtop = fmax(vtop, fmax(kv8_size(vx[i]), kv8_size(vy[i])));
        }
    }
    ktop = kv8_max64(ktop);
    vtop = kv8_max64(vtop);
    if ((t & 63) == 0) {
        tops[0][t >> 6] = ktop;
        tops[1][t >> 6] = vtop;
    }
    __syncthreads();
    ktop = fmax(fmax(tops[0][0], tops[0][1]), fmax(tops[0][2], tops[0][3]));
    vtop = fmax(fmax(tops[1][0], tops[1][1]), fmax(tops[1][2], tops[1][3]));
    int ke = kv8_exponent(ktop), ve = kv8_exponent(vtop), ks = 0, vs = 0;   // exponents, and the older codes' shifts
    if (n_old) {
        const int ko = kv8_exponent_of(a.ks[si]), vo = kv8_exponent_of(a.vs[si]);
        ke = max(ke, ko);
        ve = max(ve, vo);
        ks = ke - ko;
        vs = ve - vo;
    }
    __syncthreads();   // every thread has read the old scales
    if (t == 0) {
        a.ks[si] = kv8_pow2(ke);
        a.vs[si] = kv8_pow2(ve);
        if (a.status && (ke > KV8_HIGH || ve > KV8_HIGH)) *a.status = 1;
    }
    const bool kgood = ke <= KV8_HIGH, vgood = ve <= KV8_HIGH;
    if (fresh) {
        const double ki = kgood ? ldexp(1.0, -ke) : 0.0, vi = vgood ? ldexp(1.0, -ve) : 0.0;
        uint32_t c0 = 0, c1 = 0;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            c0 |= (kgood ? kv8_code(kx[i], ki) : 128u) << (8 * i);
            c1 |= (kgood ? kv8_code(ky[i], ki) : 128u) << (8 * i);
            tv[(j * NP + i) * KV8_BLOCK + tt] = (uint8_t)(vgood ? kv8_code(vx[i], vi) : 128u);
            tv[(HD / 2 + j * NP + i) * KV8_BLOCK + tt] = (uint8_t)(vgood ? kv8_code(vy[i], vi) : 128u);
        }
        uint8_t *d = kb + tt * HD + j * NP;
        if constexpr (NP == 4) {
            *(uint32_t *)d = c0;
            *(uint32_t *)(d + HD / 2) = c1;
        } else {
            *(uint16_t *)d = (uint16_t)c0;
            *(uint16_t *)(d + HD / 2) = (uint16_t)c1;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            tv[(j * NP + i) * KV8_BLOCK + tt] = 128;
            tv[(HD / 2 + j * NP + i) * KV8_BLOCK + tt] = 128;
        }
        if (tt < n_old && ks > 0 && kgood) {
#pragma unroll
            for (int c = 0; c < 2 * NP; c += 4) {
                uint32_t *d = (uint32_t *)(kb + tt * HD + 2 * NP * j + c);
                *d = kv8_rescale4(*d, ks);
            }
        }
    }
    __syncthreads();
    if (t < HD) {
        // the channel's 16 positions: older codes from the plane, then the fresh ones
        u32x4 n = *(const u32x4 *)(tv + t * KV8_BLOCK);
        u32x4 *d = (u32x4 *)(vb + t * KV8_BLOCK);
        if (n_old) {
            const u32x4 o = *d;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = min(4, max(0, n_old - 4 * i));
                const uint32_t keep = k == 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
                const uint32_t x = vs > 0 && vgood ? kv8_rescale4(o[i], vs) : o[i];
                n[i] = (n[i] & ~keep) | (x & keep);
            }
        }
        *d = n;
    }
}

// Read: a workgroup a (segment, block, kv head); thread t the position t / 16
// and HD / 16 of its channels, V through LDS. Bound: HBM (3300 positions of 8
// heads of 64 in 6.5 us, 2.6 TB/s), a launch for few.
template <int HD>
DEV void kv8_read(const cj_kv8_args &a) {
    constexpr int W = HD / 16;
    __shared__ __align__(16) uint8_t tv[HD * KV8_BLOCK];
    const int t = threadIdx.x, tt = t >> 4, j = t & 15;
    const int nb = (a.max_rows + KV8_BLOCK - 2) / KV8_BLOCK + 1;
    const int h = blockIdx.x % a.n_kv, w = blockIdx.x / a.n_kv, blk = w % nb, s = w / nb;
    Kv8Seg g;
    if (!kv8_seg(a, s, g)) return;
    if (blk > (g.pos + g.rows - 1) / KV8_BLOCK - g.pos / KV8_BLOCK) return;
    const int b0 = (g.pos / KV8_BLOCK + blk) * KV8_BLOCK;
    int page = kv8_page(a, g.slot, b0 / KV8_PAGE);
    const bool bad = page < 0;
    if (bad) {
        page = 0;
        if (a.status && t == 0) *a.status = 1;
    }
    const int64_t ph = (int64_t)page * a.n_kv + h, si = ph * 4 + (b0 % KV8_PAGE) / KV8_BLOCK;
    const int64_t at = (ph * KV8_PAGE + b0 % KV8_PAGE) * HD;
    if (t < HD) *(u32x4 *)(tv + t * KV8_BLOCK) = *(const u32x4 *)(a.vc + at + t * KV8_BLOCK);
    __syncthreads();
    const int p = b0 + tt;
    if (p < g.pos || p >= g.pos + g.rows) return;
    const float none = __uint_as_float(0x7fc00000u), ks = bad ? none : a.ks[si], vs = bad ? none : a.vs[si];
    const int64_t o = (int64_t)(g.row + (p - g.pos)) * a.out_stride + (int64_t)h * HD + j * W;
    if (a.out)
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint32_t c = *(const uint32_t *)(a.kc + at + tt * HD + j * W + i);
            f32x4 f;
#pragma unroll
            for (int k = 0; k < 4; k++) f[k] = (float)((int)((c >> (8 * k)) & 255u) - 128) * ks;
            *(f32x4 *)(a.out + o + i) = f;
        }
    if (a.out2)
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            f32x4 f;
#pragma unroll
            for (int k = 0; k < 4; k++) f[k] = (float)((int)tv[(j * W + i + k) * KV8_BLOCK + tt] - 128) * vs;
            *(f32x4 *)(a.out2 + o + i) = f;
        }
}

// ------------------------------------------------------------- attention
//
// Softmax over the positions with running maxima, split over workgroups and
// joined by cj_kv8_join. The f16 matrix cores carry both products at f32's
// accuracy: codes are whole numbers up to 127, exact in f16, and q and the
// weights enter as two f16 halves each (hi + lo, 22 bits).
//
// The block's V scale 2^e rides on the weight: with s the score in base 2 the
// weight is w = 2^(s + e − M + 14), M the running maximum of ceil(s + e), so
// that the output is Σ w·code / Σ w·2^−e. A whole M makes every rescaling
// exact; 14 keeps the lo halves of all weights down to 2^-17 of the largest
// out of f16's subnormals.

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define KV8_LOG2E 1.44269504088896340736f
#define KV8_WEIGHT 14.0f

// Eight code bytes as f16: 0x64xx is 1024 + xx.
DEV h16x8 kv8_half8(uint32_t a, uint32_t b) {
    union { uint32_t u[4]; h16x8 h; } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    return r.h - (_Float16)1152.0f;
}

DEV uint32_t kv8_pack2(float x, float y) {
    const f32x2 v = {x, y};
    union { h16x2 h; uint32_t u; } r;
    r.h = __builtin_convertvector(v, h16x2);
    return r.u;
}

// w less its f16 half: v_fma_mix_f32 reads the half as it lies (the compiler
// widens it first).
DEV float kv8_less_lo(uint32_t h, float w) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(w));
    return r;
}
DEV float kv8_less_hi(uint32_t h, float w) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(w));
    return r;
}

// x as hi + lo halves.
DEV void kv8_halves(const float (&x)[8], h16x8 &hi, h16x8 &lo) {
    union { uint32_t u[4]; h16x8 h; } a, b;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a.u[i] = kv8_pack2(x[2 * i], x[2 * i + 1]);
        b.u[i] = kv8_pack2(kv8_less_lo(a.u[i], x[2 * i]), kv8_less_hi(a.u[i], x[2 * i + 1]));
    }
    hi = a.h;
    lo = b.h;
}

// The exponent of a block's scale as a float; NaN where the scale is.
DEV float kv8_exp_f(float s) { return (float)((int)((__float_as_uint(s) >> 23) & 255u) - 127) + s * 0.0f; }
DEV float kv8_recip(float s) { return __uint_as_float((254u << 23) - (__float_as_uint(s) & 0x7f800000u)); }

// A column's q, an exponent k apart from [1, 2)·2^14: the factor that the
// scores take back, scale·log2(e)·2^(k − 14).
DEV int kv8_q_exponent(float top) { return (int)(__float_as_uint(top) >> 23) - 127; }

// Keeps a branch that few pages take a branch: the compiler would carry out
// its comparisons and selects for every page.
DEV void kv8_branch() { asm volatile(""); }

DEV float kv8_max4(float v) {   // over the lanes l, l ^ 16, l ^ 32, l ^ 48
    int a, b;
    swap16(__float_as_int(v), a, b);
    v = fmaxf(__int_as_float(a), __int_as_float(b));
    swap32(__float_as_int(v), a, b);
    return fmaxf(__int_as_float(a), __int_as_float(b));
}
DEV float kv8_sum4(float v) {
    int a, b;
    swap16(__float_as_int(v), a, b);
    v = __int_as_float(a) + __int_as_float(b);
    swap32(__float_as_int(v), a, b);
    return __int_as_float(a) + __int_as_float(b);
}

// The pages [p0, p1) that split sp of the segment's rows r0 .. r1 covers, and
// how many splits these rows have.
DEV int kv8_split(const cj_kv8_args &a, const Kv8Seg &g, int r0, int r1, int sp, int &p0, int &p1) {
    const int lo = a.window > 0 && g.pos + r0 >= a.window ? (g.pos + r0 + 1 - a.window) / KV8_PAGE : 0;
    const int n = (g.pos + r1) / KV8_PAGE + 1 - lo;
    p0 = lo + min(n, sp * a.split_pages);
    p1 = lo + min(n, (sp + 1) * a.split_pages);
    return (n + a.split_pages - 1) / a.split_pages;
}

// A split's results: [segment][kv head][column tile][split] of the tile's
// columns (HD sums each), then their maxima and sums of weights.
#define KV8_FEW 16
template <int HD>
DEV float *kv8_part(const cj_kv8_args &a, int s, int h, int ct, int sp) {
    return a.part + ((((int64_t)s * a.n_kv + h) * a.col_tiles + ct) * a.splits + sp) * (a.tile_cols * (HD + 2));
}

// Page ids of a run of pages, 64 at a time, one a lane: read where a page is
// loaded, each would cost the wave a round trip to memory (8 sequences of
// 65500: 177 us, so 170).
struct Kv8Table {
    const cj_kv8_args &a;
    const int slot, from, end;   // pages from, from + 4, .. before end
    int ids;
    // the id of page from + 4k (k from 0 up, one after the other), −1 where there is none
    DEV int at(int k) {
        if ((k & 63) == 0) ids = kv8_page(a, slot, min(end - 1, from + 4 * (k + (int)(threadIdx.x & 63))));
        return __builtin_amdgcn_readlane(ids, k & 63);
    }
};

// A page's K codes go from memory straight into the wave's part of LDS, eight
// (HD 128) or four lanes a row, so that a copy touches whole lines. (A lane a
// row, 64 lines an instruction: 32 ragged sequences of up to 4096 positions
// 44.8 us, so 35.6; 64 rows behind 1033 24 and 19.6.)
// LDS row ρ holds key `key(ρ)` of the page; its 16-byte word c stands at c ^
// swizzle(ρ), so that 16 rows' reads of one word fall on all 64 banks once.
template <int HD>
DEV int kv8_swizzle(int row) { return HD == 128 ? row >> 1 & 7 : row >> 2 & 3; }
template <int HD, class Key>
DEV void kv8_copy_k(const uint8_t *page, uint8_t *lds, int l, Key &&key) {
    constexpr int W = HD / 16;   // words a row
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the page that stood there has been read
#pragma unroll
    for (int e = 0; e < W; e++) {
        const int row = e * (64 / W) + l / W, c = l % W ^ kv8_swizzle<HD>(row);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(page + key(row) * HD + c * 16),
                                         (__attribute__((address_space(3))) void *)(lds + e * 1024), 16, 0, 0);
    }
}
template <int HD>
DEV u32x4 kv8_read_k(const uint8_t *lds, int row, int c) {
    return *(const u32x4 *)(lds + row * HD + (c ^ kv8_swizzle<HD>(row)) * 16);
}
// The wave's copies and loads have landed.
DEV void kv8_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The columns' q as halves into LDS in the products' operand order: C columns
// of 256 / C threads, thread j of column c with its channels 4j + i·1024/C..;
// `at(d)` is the operand word and lane part of channel d. cs[c] takes back the
// column's exponent: scale·log2(e)·2^(k − 14), for the largest in [1, 2)·2^k.
template <int HD, int C>
struct Kv8Q {
    static constexpr int T = 256 / C, N = HD / (4 * T);
    f32x4 x[N];
    DEV void load(const float *src, int j) {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = *(const f32x4 *)(src + i * 4 * T + j * 4);
    }
    template <class At>
    DEV void store(uint8_t *qs, float *cs, int c, int j, float scale, At &&at) const {
        float top = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) top = fmaxf(top, fabsf(x[i][k]));
        top = fmaxf(top, dpp_f<DPP_XOR1>(top));
        top = fmaxf(top, dpp_f<DPP_XOR2>(top));
        top = fmaxf(top, dpp_f<DPP_HMIRROR>(top));
        if (T == 16) top = fmaxf(top, dpp_f<KV8_MIRROR>(top));
        const int e = kv8_q_exponent(top);
        const float sign = scale < 0 ? -1.0f : 1.0f;
        if (j == 0) cs[c] = ldexpf(scale * sign * KV8_LOG2E, e - 14);
#pragma unroll
        for (int i = 0; i < N; i++) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = ldexpf(x[i][k] * sign, 14 - e);
            const uint32_t h0 = kv8_pack2(y[0], y[1]), h1 = kv8_pack2(y[2], y[3]);
            const uint32_t l0 = kv8_pack2(kv8_less_lo(h0, y[0]), kv8_less_hi(h0, y[1]));
            const uint32_t l1 = kv8_pack2(kv8_less_lo(h1, y[2]), kv8_less_hi(h1, y[3]));
            uint8_t *d = qs + at(i * 4 * T + j * 4);
            *(uint2 *)d = make_uint2(h0, h1);
            *(uint2 *)(d + 1024) = make_uint2(l0, l1);
        }
    }
};

// Few columns (a column is a row and one query head of the kv head's group;
// up to 16): a workgroup a (segment, kv head, split), its four waves a page
// each in turn. The tiles' rows are placed so that the scores' accumulators
// are the next product's operand as they lie:
//  - scores: A rows are keys, row m of tile t is position (m/4)·16 + 4t + m%4
//    of the page, so lane group g = l/16 gets its 16 positions of block g in
//    order, and one K and one V scale a lane;
//  - output: B is the weights, A the V codes, 16 positions of a channel in 16
//    bytes, a page ahead in registers.
// Bound: HBM where there is enough to read (8 sequences of 65500 positions, 8
// kv heads of 128: 171 us, 6.27 TB/s; 32 ragged ones of up to 4096: 33 us,
// 5.05 TB/s with ramp and tail), else the chain of round trips (segment, page
// table, page, output: 6 us for one of 2049, and the join's 3).
template <int HD>
DEV void kv8_attend_c16(const cj_kv8_args &a) {
    constexpr int KS = HD / 32, DT = HD / 16;   // steps over the channels; channel tiles
    constexpr int KB = KV8_PAGE * HD, OB = 4 * KV8_FEW * (HD + 4) * 4;
    __shared__ __align__(16) uint8_t lds[4 * KB > OB ? 4 * KB : OB], qs[2 * KS * 1024];
    __shared__ float sc[KV8_FEW], sm[4][KV8_FEW], sl[4][KV8_FEW];
    const int t = threadIdx.x, l = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), n = l & 15, g4 = l >> 4;
    const uint32_t id = blockIdx.x;
    const int h = (int)(id % a.n_kv), sp = (int)(id / a.n_kv % a.splits), s = (int)(id / a.n_kv / a.splits);
    Kv8Seg g;
    if (!kv8_seg(a, s, g)) return;
    const int grp = a.n_q / a.n_kv, cols = g.rows * grp;
    int p0, p1;
    const int splits = kv8_split(a, g, 0, g.rows - 1, sp, p0, p1);
    if (sp >= splits) return;

    // q of column t / 16 (past the last: the first again)
    Kv8Q<HD, KV8_FEW> q;
    {
        const int c = t / 16 < cols ? t / 16 : 0;
        q.load(a.q + (int64_t)(g.row + c / grp) * a.q_stride + (int64_t)(h * grp + c % grp) * HD, t % 16);
    }
    uint8_t *kl = lds + wv * KB;
    u32x4 vr[DT], vn[DT];
    float ks, vs;
    int pi = p0 + wv;
    Kv8Table table{a, g.slot, pi, p1, 0};
    bool bad = false;
    int64_t ph = 0;
    auto page_at = [&](int i) {
        const int p = table.at((i - p0) >> 2);
        bad = p < 0;
        ph = (int64_t)(bad ? 0 : p) * a.n_kv + h;
    };
    auto copy_k = [&]() {
        kv8_copy_k<HD>(a.kc + ph * KB, kl, l, [](int row) { return (row >> 2 & 3) * 16 + (row >> 4) * 4 + (row & 3); });
    };
    auto load_v = [&]() {
        ks = a.ks[ph * 4 + g4];
        vs = a.vs[ph * 4 + g4];
        const uint8_t *b = a.vc + ph * KB + (g4 * HD + n) * 16;
#pragma unroll
        for (int j = 0; j < DT; j++) vn[j] = __builtin_nontemporal_load((const u32x4 *)(b + j * 256));
    };
    if (pi < p1) {
        page_at(pi);
        copy_k();
        load_v();
    }
    q.store(qs, sc, t / 16, t % 16, a.scale, [t](int d) {
        return (d % (HD / 4) / 8) * 2048 + (d / (HD / 4) * 16 + t / 16) * 16 + d % 8 * 2;
    });
    lds_barrier();
    const int c = n < cols ? n : 0, last = g.pos + c / grp, first = a.window > 0 ? last + 1 - a.window : 0;
    const float cs = sc[n];
    h16x8 qh[KS], ql[KS];
#pragma unroll
    for (int k = 0; k < KS; k++) {
        qh[k] = *(const h16x8 *)(qs + k * 2048 + l * 16);
        ql[k] = *(const h16x8 *)(qs + k * 2048 + 1024 + l * 16);
    }
    f32x4 o[DT] = {};
    float M = -INFINITY, L = 0;
    for (; pi < p1; pi += 4) {
        kv8_landed();
        if (bad && a.status && l == 0) *a.status = 1;
        float kf = (bad ? __uint_as_float(0x7fc00000u) : ks) * cs;
        const float ve = kv8_exp_f(vs), vi = kv8_recip(vs);
#pragma unroll
        for (int j = 0; j < DT; j++) vr[j] = vn[j];
        const bool more = pi + 4 < p1;
        if (more) {
            page_at(pi + 4);
            load_v();
        }
        f32x4 x[4] = {};
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
            u32x4 w[4];
            h16x8 f[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                w[q] = kv8_read_k<HD>(kl, q * 16 + n, g4 * (HD / 64) + k / 2);
                f[q] = kv8_half8(w[q][0], w[q][1]);
                x[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[q], qh[k], x[q], 0, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < 4; q++) x[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[q], ql[k], x[q], 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                f[q] = kv8_half8(w[q][2], w[q][3]);
                x[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[q], qh[k + 1], x[q], 0, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < 4; q++) x[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[q], ql[k + 1], x[q], 0, 0, 0);
        }
        if (more) copy_k();
        float top = -INFINITY;
        const int at = pi * KV8_PAGE + g4 * 16;
        if (pi * KV8_PAGE + KV8_PAGE - 1 > g.pos || (a.window > 0 && pi * KV8_PAGE < g.pos + g.rows - a.window)) {
            kv8_branch();
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    x[q][i] = (uint32_t)(at - first + 4 * q + i) <= (uint32_t)(last - first) ? __builtin_fmaf(x[q][i], kf, ve) : -INFINITY;
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[q][i] = __builtin_fmaf(x[q][i], kf, ve);
        }
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, x[q][i]);
        const float Mn = fmaxf(M, ceilf(kv8_max4(top)));
        const float base = (Mn == -INFINITY ? 0.0f : Mn) - KV8_WEIGHT;
        if (__any(Mn != M)) {
            const float r = exp2f(M - (base + KV8_WEIGHT));
#pragma unroll
            for (int j = 0; j < DT; j++) o[j] *= r;
            L *= r;
            M = Mn;
        }
        h16x8 wh[2], wl[2];
        float sum = 0;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = __builtin_amdgcn_exp2f(x[2 * u + i / 4][i % 4] - base);
                sum += w[i];
            }
            kv8_halves(w, wh[u], wl[u]);
        }
        L += sum == 0.0f ? 0.0f : sum * vi;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j0 = 0; j0 < DT; j0 += 4) {
                h16x8 f[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f[j] = kv8_half8(vr[j0 + j][2 * u], vr[j0 + j][2 * u + 1]);
                    o[j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[j], wh[u], o[j0 + j], 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) o[j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[j], wl[u], o[j0 + j], 0, 0, 0);
            }
    }

    // the four waves' results as one, where the K codes stood
    float (*so)[KV8_FEW][HD + 4] = (float (*)[KV8_FEW][HD + 4])lds;
    L = kv8_sum4(L);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < DT; j++) *(f32x4 *)&so[wv][n][j * 16 + g4 * 4] = o[j];
    if (g4 == 0) {
        sm[wv][n] = M;
        sl[wv][n] = L;
    }
    __syncthreads();
    float *part = splits > 1 ? kv8_part<HD>(a, s, h, 0, sp) : nullptr;
    for (int i = t; i < KV8_FEW * HD / 4; i += 256) {
        const int k = i / (HD / 4), d = i % (HD / 4) * 4;
        if (k >= cols) break;
        const float m = fmaxf(fmaxf(sm[0][k], sm[1][k]), fmaxf(sm[2][k], sm[3][k])), z = m == -INFINITY ? 0.0f : m;
        f32x4 y = {};
        float b = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = exp2f(sm[w][k] - z);
            y += *(const f32x4 *)&so[w][k][d] * f;
            b += sl[w][k] * f;
        }
        if (part) {
            *(f32x4 *)(part + k * HD + d) = y;
            if (d == 0) {
                part[KV8_FEW * HD + 2 * k] = m;
                part[KV8_FEW * HD + 2 * k + 1] = b;
            }
        } else {
            *(f32x4 *)(a.out + (int64_t)(g.row + k / grp) * a.out_stride + (int64_t)(h * grp + k % grp) * HD + d) = y / b;
        }
    }
}

// Scores of a page's two 32-row tiles (below): what the column at `last` does
// not see from `first` on, at position p and after, is −inf; a block of which
// it sees nothing may have no scale.
DEV void kv8_mask(f32x16 (&x)[2], f32x2 &ks, f32x2 &vs, int p, int first, int last) {
    kv8_branch();
    const uint32_t seen = (uint32_t)(last - first);
#pragma unroll
    for (int q = 0; q < 2; q++, p += 16) {
        const uint32_t at = (uint32_t)(p - first);   // (before first: past any `seen`)
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (at + i > seen) x[q][i] = -INFINITY;
        if (p > last || p + 15 < first) ks[q] = vs[q] = 1.0f;
    }
}

// The softmax step of those tiles: the running maximum M raised, the output
// and sum rescaled where it grew, then the weights of tile q as halves.
template <int DT>
struct Kv8Weights {
    float kf[2], off[2], back[2];
    DEV Kv8Weights(const f32x16 (&x)[2], f32x2 ks, f32x2 vs, float cs, float &M, float &L, f32x16 (&o)[DT]) {
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < 2; q++) {
            kf[q] = ks[q] * cs;
            kf[q] = kf[q] < 1e-37f ? 1e-37f : kf[q];   // (never zero: −inf stays −inf)
            off[q] = kv8_exp_f(vs[q]);
            back[q] = kv8_recip(vs[q]);
            float m = x[q][0];
#pragma unroll
            for (int i = 1; i < 16; i++) m = fmaxf(m, x[q][i]);
            top = fmaxf(top, __builtin_fmaf(m, kf[q], off[q]));
        }
        int u, v;
        swap32(__float_as_int(top), u, v);
        const float Mn = fmaxf(M, ceilf(fmaxf(__int_as_float(u), __int_as_float(v))));
        const float base = (Mn == -INFINITY ? 0.0f : Mn) - KV8_WEIGHT;
        if (__any(Mn != M)) {
            const float r = __builtin_amdgcn_exp2f(M - (base + KV8_WEIGHT));
#pragma unroll
            for (int j = 0; j < DT; j++) o[j] *= r;
            L *= r;
            M = Mn;
        }
        off[0] -= base;
        off[1] -= base;
    }
    DEV void halves(int q, const f32x16 &x, h16x8 (&wh)[2], h16x8 (&wl)[2], float &L) const {
        float sum = 0;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + i], kf[q], off[q]));
                sum += w[i];
            }
            kv8_halves(w, wh[u], wl[u]);
        }
        L += sum == 0.0f ? 0.0f : sum * back[q];
    }
};

// Some columns (17 and more, where 128 a workgroup would leave the chip
// empty): as for few, every wave its own pages, but 32 columns and the 32-row
// products. q's halves stay in LDS, being the same for all waves. Tile q's row
// r is position 32·(r/4 % 2) + 16q + 4·(r/8) + r%4, which gives lane half h =
// l/32 blocks 2h and 2h + 1 in order.
// Bound: the waves' own work, VALU (the codes' conversion, once a wave, and
// the softmax: 45% of the cycles) and matrix cores (28%) hardly overlapping
// (512 rows behind 1545 of 32 / 8 heads of 128: 41 us, 370 TFLOP/s; three rows
// of 16 sequences of 4097, 64 / 8 heads of 64: 18 us and the join's 5).
#define KV8_SOME 32
template <int HD>
DEV void kv8_attend_c32(const cj_kv8_args &a) {
    constexpr int KS = HD / 16, DT = HD / 32;   // steps over the channels; channel tiles
    constexpr int KB = KV8_PAGE * HD, OB = 2 * KV8_SOME * (HD + 4) * 4;
    __shared__ __align__(16) uint8_t lds[4 * KB > OB ? 4 * KB : OB], qs[2 * KS * 1024];
    __shared__ float sc[KV8_SOME], sm[4][KV8_SOME], sl[4][KV8_SOME];
    const int t = threadIdx.x, l = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), n = l & 31, hf = l >> 5;
    // workgroups eight apart share an L2: a segment's column tiles follow one another there
    const uint32_t id = blockIdx.x, per = id / 8 / a.col_tiles, rest = per * 8 + id % 8;
    const int ct = a.col_tiles - 1 - (int)(id / 8 % a.col_tiles);
    const int h = (int)(rest % a.n_kv), sp = (int)(rest / a.n_kv % a.splits), s = (int)(rest / a.n_kv / a.splits);
    Kv8Seg g;
    if (s >= a.n_segs || !kv8_seg(a, s, g)) return;
    const int grp = a.n_q / a.n_kv, cols = g.rows * grp, c0 = ct * KV8_SOME;
    if (c0 >= cols) return;
    const int r0 = c0 / grp, r1 = (min(c0 + KV8_SOME, cols) - 1) / grp;
    int p0, p1;
    const int splits = kv8_split(a, g, r0, r1, sp, p0, p1);
    if (sp >= splits) return;

    // q of column t / 8 (past the last: the tile's first again)
    Kv8Q<HD, KV8_SOME> q;
    {
        const int c = c0 + t / 8 < cols ? c0 + t / 8 : c0;
        q.load(a.q + (int64_t)(g.row + c / grp) * a.q_stride + (int64_t)(h * grp + c % grp) * HD, t % 8);
    }
    uint8_t *kl = lds + wv * KB;
    u32x4 vr[2][DT], vn[2][DT];
    f32x2 ks, vs;
    int pi = p0 + wv;
    Kv8Table table{a, g.slot, pi, p1, 0};
    bool bad = false;
    int64_t ph = 0;
    auto page_at = [&](int i) {
        const int p = table.at((i - p0) >> 2);
        bad = p < 0;
        ph = (int64_t)(bad ? 0 : p) * a.n_kv + h;
    };
    auto copy_k = [&]() {
        kv8_copy_k<HD>(a.kc + ph * KB, kl, l, [](int row) { return (row >> 2 & 1) * 32 + (row >> 5) * 16 + (row >> 3 & 3) * 4 + (row & 3); });
    };
    auto load_v = [&]() {
        ks = *(const f32x2 *)(a.ks + ph * 4 + 2 * hf);
        vs = *(const f32x2 *)(a.vs + ph * 4 + 2 * hf);
        const uint8_t *b = a.vc + ph * KB + (2 * hf * HD + n) * 16;
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int j = 0; j < DT; j++) vn[q][j] = *(const u32x4 *)(b + (q * HD + j * 32) * 16);
    };
    if (pi < p1) {
        page_at(pi);
        copy_k();
        load_v();
    }
    q.store(qs, sc, t / 8, t % 8, a.scale, [t](int d) {
        return (d % (HD / 2) / 8) * 2048 + (d / (HD / 2) * 32 + t / 8) * 16 + d % 8 * 2;
    });
    lds_barrier();
    const int c = c0 + n < cols ? c0 + n : c0, last = g.pos + c / grp, first = a.window > 0 ? last + 1 - a.window : 0;
    const float cs = sc[n];
    f32x16 o[DT] = {};
    float M = -INFINITY, L = 0;
    for (; pi < p1; pi += 4) {
        kv8_landed();
        if (bad && a.status && l == 0) *a.status = 1;
        f32x2 kb = ks, vb = vs;
        if (bad) kb[0] = kb[1] = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int j = 0; j < DT; j++) vr[q][j] = vn[q][j];
        const bool more = pi + 4 < p1;
        if (more) {
            page_at(pi + 4);
            load_v();
        }
        f32x16 x[2] = {};
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
            u32x4 w[2];
#pragma unroll
            for (int q = 0; q < 2; q++) w[q] = kv8_read_k<HD>(kl, q * 32 + n, hf * (HD / 32) + k / 2);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const h16x8 qh = *(const h16x8 *)(qs + (k + i) * 2048 + l * 16), ql = *(const h16x8 *)(qs + (k + i) * 2048 + 1024 + l * 16);
                h16x8 f[2];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    f[q] = kv8_half8(w[q][2 * i], w[q][2 * i + 1]);
                    x[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[q], qh, x[q], 0, 0, 0);
                }
#pragma unroll
                for (int q = 0; q < 2; q++) x[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[q], ql, x[q], 0, 0, 0);
            }
        }
        if (more) copy_k();
        if (pi * KV8_PAGE + KV8_PAGE - 1 > g.pos + r0 || (a.window > 0 && pi * KV8_PAGE < g.pos + r1 + 1 - a.window))
            kv8_mask(x, kb, vb, pi * KV8_PAGE + hf * 32, first, last);
        Kv8Weights<DT> w(x, kb, vb, cs, M, L, o);
#pragma unroll
        for (int q = 0; q < 2; q++) {
            h16x8 wh[2], wl[2];
            w.halves(q, x[q], wh, wl, L);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < DT; j++) {
                    const h16x8 f = kv8_half8(vr[q][j][2 * u], vr[q][j][2 * u + 1]);
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, wh[u], o[j], 0, 0, 0);
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, wl[u], o[j], 0, 0, 0);
                }
        }
    }

    // the four waves' results as one: rescaled to the largest maximum, then 2 and 3 onto 0 and 1, then the two
    int u, v;
    swap32(__float_as_int(L), u, v);
    if (hf == 0) {
        sm[wv][n] = M;
        sl[wv][n] = __int_as_float(u) + __int_as_float(v);
    }
    __syncthreads();   // (also: the K codes are not read any more)
    const float z = fmaxf(fmaxf(sm[0][n], sm[1][n]), fmaxf(sm[2][n], sm[3][n])), f = M == -INFINITY ? 0.0f : exp2f(M - z);
    float (*so)[KV8_SOME][HD + 4] = (float (*)[KV8_SOME][HD + 4])lds;
    if (wv >= 2)
#pragma unroll
        for (int j = 0; j < DT; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                f32x4 y;
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = o[j][4 * q + i] * f;
                *(f32x4 *)&so[wv - 2][n][j * 32 + q * 8 + hf * 4] = y;
            }
    __syncthreads();
    if (wv < 2)
#pragma unroll
        for (int j = 0; j < DT; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                f32x4 *y = (f32x4 *)&so[wv][n][j * 32 + q * 8 + hf * 4];
                f32x4 r = *y;
#pragma unroll
                for (int i = 0; i < 4; i++) r[i] += o[j][4 * q + i] * f;
                *y = r;
            }
    __syncthreads();
    float *part = splits > 1 ? kv8_part<HD>(a, s, h, ct, sp) : nullptr;
    for (int i = t; i < KV8_SOME * HD / 4; i += 256) {
        const int k = i / (HD / 4), d = i % (HD / 4) * 4, cc = c0 + k;
        if (cc >= cols) break;
        const float m = fmaxf(fmaxf(sm[0][k], sm[1][k]), fmaxf(sm[2][k], sm[3][k]));
        float b = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) b += sm[w][k] == -INFINITY ? 0.0f : sl[w][k] * exp2f(sm[w][k] - m);
        const f32x4 y = *(const f32x4 *)&so[0][k][d] + *(const f32x4 *)&so[1][k][d];
        if (part) {
            *(f32x4 *)(part + k * HD + d) = y;
            if (d == 0) {
                part[KV8_SOME * HD + 2 * k] = m;
                part[KV8_SOME * HD + 2 * k + 1] = b;
            }
        } else {
            *(f32x4 *)(a.out + (int64_t)(g.row + cc / grp) * a.out_stride + (int64_t)(h * grp + cc % grp) * HD + d) = y / b;
        }
    }
}

// Many columns (prefill chunks): a workgroup a (segment, kv head, 128
// columns), a wave 32 columns, every wave over the same pages. A page's codes
// become f16 once, on their way into LDS, and serve the four waves; the next
// page's codes are on their way to registers meanwhile, so a page costs one
// barrier. Rows as above.
//  - K in LDS: row 32t + r of 16-byte words, word c at c ^ (row & 15), so that
//    16 lanes' rows lie in different banks;
//  - V in LDS: [t][u][h][channel] words of the 8 positions 8u.. of block 2h + t.
// Bound: the matrix cores' power: four prompts of 4096 rows, 32 / 8 heads of
// 128, in 985 us are 1.12 PFLOP/s of f16 products (two for each one of the
// attention's, whose 560 TFLOP/s that makes) at 1.8 GHz, where an 8192^3 f16
// product of the library reaches 1.15. In a 128-position window (16 prompts of
// up to 300 rows, 64 / 8 heads of 64: 35 us) the softmax's VALU work.
#define KV8_MANY 128
template <int HD>
DEV void kv8_attend_c128(const cj_kv8_args &a) {
    constexpr int KS = HD / 16, DT = HD / 32, CH = HD / 64;   // steps, channel tiles, 16-byte words of codes a thread and plane
    constexpr int ROW = HD * 2, BUF = KV8_PAGE * ROW;
    __shared__ __align__(16) uint8_t sk[2][BUF], sv[2][BUF];
    const int t = threadIdx.x, l = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), n = l & 31, hf = l >> 5;
    const uint32_t id = blockIdx.x;
    const int h = (int)(id % a.n_kv), s = (int)(id / a.n_kv % a.n_segs);
    const int ct = a.col_tiles - 1 - (int)(id / a.n_kv / a.n_segs);   // the longest first
    Kv8Seg g;
    if (!kv8_seg(a, s, g)) return;
    const int grp = a.n_q / a.n_kv, cols = g.rows * grp, c0 = ct * KV8_MANY;
    if (c0 >= cols) return;
    int p0, p1;
    kv8_split(a, g, c0 / grp, (min(c0 + KV8_MANY, cols) - 1) / grp, 0, p0, p1);   // all of them

    // the wave's columns, this lane's, and its q as halves (columns past the last: the last again)
    const int w0 = min(c0 + wv * 32, cols - 1), w1 = min(c0 + wv * 32 + 31, cols - 1), c = min(c0 + wv * 32 + n, cols - 1), ri = c / grp;
    const int wfirst = g.pos + w0 / grp, wlast = g.pos + w1 / grp, last = g.pos + ri, first = a.window > 0 ? last + 1 - a.window : 0;
    const int wlow = a.window > 0 ? wfirst + 1 - a.window : 0;   // the first position that any column of the wave sees
    float qx[KS][8], top = 0, cs;   // (requested before the first page, whose way they then share)
    {
        const float *src = a.q + (int64_t)(g.row + ri) * a.q_stride + (int64_t)(h * grp + c % grp) * HD + hf * 8;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            *(f32x4 *)&qx[k][0] = *(const f32x4 *)(src + 16 * k);
            *(f32x4 *)&qx[k][4] = *(const f32x4 *)(src + 16 * k + 4);
        }
    }
    // staging: thread t moves words t, t + 256, .. of the page's K and V codes
    u32x4 kr[CH], vr[CH];
    f32x2 ksn, vsn;
    bool bad = false;
    auto load = [&](int i) {
        const int p = kv8_page(a, g.slot, i);
        bad = p < 0;
        const int64_t ph = (int64_t)(bad ? 0 : p) * a.n_kv + h;
        const u32x4 *kb = (const u32x4 *)(a.kc + ph * (KV8_PAGE * HD)), *vb = (const u32x4 *)(a.vc + ph * (KV8_PAGE * HD));
#pragma unroll
        for (int k = 0; k < CH; k++) {
            kr[k] = kb[t + 256 * k];
            vr[k] = vb[t + 256 * k];
        }
        ksn = *(const f32x2 *)(a.ks + ph * 4 + 2 * hf);
        vsn = *(const f32x2 *)(a.vs + ph * 4 + 2 * hf);
        if (bad && a.status && t == 0) *a.status = 1;
    };
    auto store = [&](int b) {
#pragma unroll
        for (int k = 0; k < CH; k++) {
            const int w = t + 256 * k;
            const int key = w / (HD / 16), c = w % (HD / 16) * 2;
            const int row = (key >> 4 & 1) * 32 + (key >> 2 & 3) * 8 + (key >> 5) * 4 + (key & 3);
            uint8_t *d = sk[b] + row * ROW;
            *(h16x8 *)(d + ((c ^ row) & (HD / 8 - 1)) * 16) = kv8_half8(kr[k][0], kr[k][1]);
            *(h16x8 *)(d + (((c + 1) ^ row) & (HD / 8 - 1)) * 16) = kv8_half8(kr[k][2], kr[k][3]);
            const int blk = w / HD, ch = w % HD;
            uint8_t *e = sv[b] + ((blk & 1) * 4 + (blk >> 1)) * (HD * 16) + ch * 16;
            *(h16x8 *)e = kv8_half8(vr[k][0], vr[k][1]);
            *(h16x8 *)(e + 2 * HD * 16) = kv8_half8(vr[k][2], vr[k][3]);
        }
    };
    load(p0);
    h16x8 qh[KS], ql[KS];
    {
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(qx[k][i]));
        int u, v;
        swap32(__float_as_int(top), u, v);
        const int e = kv8_q_exponent(fmaxf(__int_as_float(u), __int_as_float(v)));
        const float sign = a.scale < 0 ? -1.0f : 1.0f;
        cs = ldexpf(a.scale * sign * KV8_LOG2E, e - 14);
#pragma unroll
        for (int k = 0; k < KS; k++) {
#pragma unroll
            for (int i = 0; i < 8; i++) qx[k][i] = ldexpf(qx[k][i] * sign, 14 - e);
            kv8_halves(qx[k], qh[k], ql[k]);
        }
    }
    f32x16 o[DT] = {};
    float M = -INFINITY, L = 0;

    store(0);
    f32x2 ks = ksn, vs = vsn;
    if (bad) ks[0] = ks[1] = __uint_as_float(0x7fc00000u);
    for (int pi = p0, b = 0; pi < p1; pi++, b ^= 1) {
        __syncthreads();   // the page is in buffer b; buffer b ^ 1 is free
        const bool more = pi + 1 < p1;
        if (more) load(pi + 1);
        if (pi * KV8_PAGE <= wlast && pi * KV8_PAGE + KV8_PAGE > wlow) {
            f32x16 x[2] = {};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                h16x8 f[2];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    f[q] = *(const h16x8 *)(sk[b] + (32 * q + n) * ROW + (((2 * k + hf) ^ n) & (HD / 8 - 1)) * 16);
                    x[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[q], qh[k], x[q], 0, 0, 0);
                }
#pragma unroll
                for (int q = 0; q < 2; q++) x[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[q], ql[k], x[q], 0, 0, 0);
            }
            f32x2 kb = ks, vb = vs;
            if (pi * KV8_PAGE + KV8_PAGE - 1 > wfirst || (a.window > 0 && pi * KV8_PAGE < wlast + 1 - a.window))
                kv8_mask(x, kb, vb, pi * KV8_PAGE + hf * 32, first, last);
            Kv8Weights<DT> sm(x, kb, vb, cs, M, L, o);
#pragma unroll
            for (int q = 0; q < 2; q++) {
                h16x8 wh[2], wl[2];
                sm.halves(q, x[q], wh, wl, L);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < DT; j++) {
                        const h16x8 f = *(const h16x8 *)(sv[b] + ((q * 2 + u) * 2 + hf) * (HD * 16) + (j * 32 + n) * 16);
                        o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, wh[u], o[j], 0, 0, 0);
                        o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, wl[u], o[j], 0, 0, 0);
                    }
            }
        }
        if (more) {
            store(b ^ 1);
            ks = ksn;
            vs = vsn;
            if (bad) ks[0] = ks[1] = __uint_as_float(0x7fc00000u);
        }
    }
    int u, v;
    swap32(__float_as_int(L), u, v);
    L = __int_as_float(u) + __int_as_float(v);
    if (c0 + wv * 32 + n >= cols) return;
    L = 1.0f / L;
    float *d = a.out + (int64_t)(g.row + ri) * a.out_stride + (int64_t)(h * grp + c % grp) * HD;
#pragma unroll
    for (int j = 0; j < DT; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            f32x4 y;
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = o[j][4 * q + i] * L;
            *(f32x4 *)(d + j * 32 + q * 8 + hf * 4) = y;
        }
}

// The splits of the columns as one row each: HD / 4 threads a channel group,
// a.join_ways of them side by side over a column's splits, which are then
// joined in order; the other threads of the workgroup are other columns. kv
// head = id mod n_kv, as the parts were written, so that they are read through
// the L2 that holds them. Bound: a launch (3 to 5 us).
template <int HD>
DEV void kv8_join(const cj_kv8_args &a) {
    constexpr int C4 = HD / 4, W = 256 / C4;
    __shared__ __align__(16) float so[W][HD];
    __shared__ float sm[W], sl[W];
    const int t = threadIdx.x, d = t % C4 * 4, w = t / C4, ways = a.join_ways, per = W / ways, way = w % ways;
    const int grp = a.n_q / a.n_kv, most = a.max_rows * grp, tiles = (most + per - 1) / per;
    const uint32_t id = blockIdx.x;
    const int h = (int)(id % a.n_kv), s = (int)(id / a.n_kv / tiles), c = (int)(id / a.n_kv % tiles) * per + w / ways;
    Kv8Seg g;
    if (!kv8_seg(a, s, g)) return;
    const int cols = g.rows * grp, tc = a.tile_cols, ct = c / tc, k = c - ct * tc, c0 = ct * tc;
    int p0, p1, splits = 0;
    if (c < cols) splits = kv8_split(a, g, c0 / grp, (min(c0 + tc, cols) - 1) / grp, 0, p0, p1);
    float M = -INFINITY, L = 0;
    f32x4 y = {};
    if (splits > 1) {
        const float *part = kv8_part<HD>(a, s, h, ct, 0);
        const int64_t step = (int64_t)tc * (HD + 2);
#pragma unroll 4
        for (int sp = way; sp < splits; sp += ways) {
            const float *p = part + sp * step;
            const float m = p[tc * HD + 2 * k], b = p[tc * HD + 2 * k + 1];
            const f32x4 v = *(const f32x4 *)(p + k * HD + d);
            const float Mn = fmaxf(M, m), z = Mn == -INFINITY ? 0.0f : Mn, f0 = exp2f(M - z), f1 = exp2f(m - z);
            y = y * f0 + v * f1;
            L = L * f0 + b * f1;
            M = Mn;
        }
    }
    if (ways > 1) {
        *(f32x4 *)&so[w][d] = y;
        if (d == 0) {
            sm[w] = M;
            sl[w] = L;
        }
        __syncthreads();
        if (way) return;
        for (int i = 1; i < ways; i++) M = fmaxf(M, sm[w + i]);
        const float z = M == -INFINITY ? 0.0f : M;
        y = f32x4{};
        L = 0;
        for (int i = 0; i < ways; i++) {
            const float f = exp2f(sm[w + i] - z);
            y += *(const f32x4 *)&so[w + i][d] * f;
            L += sl[w + i] * f;
        }
    }
    if (splits > 1) *(f32x4 *)(a.out + (int64_t)(g.row + c / grp) * a.out_stride + (int64_t)(h * grp + c % grp) * HD + d) = y / L;
}

extern "C" __global__ void __launch_bounds__(256) cj_kv8_append_h64(cj_kv8_args a) { kv8_append<64>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_append_h128(cj_kv8_args a) { kv8_append<128>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_read_h64(cj_kv8_args a) { kv8_read<64>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_read_h128(cj_kv8_args a) { kv8_read<128>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) cj_kv8_attend_c16_h64(cj_kv8_args a) { kv8_attend_c16<64>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) cj_kv8_attend_c16_h128(cj_kv8_args a) { kv8_attend_c16<128>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_join_h64(cj_kv8_args a) { kv8_join<64>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_join_h128(cj_kv8_args a) { kv8_join<128>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) cj_kv8_attend_c32_h64(cj_kv8_args a) { kv8_attend_c32<64>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) cj_kv8_attend_c32_h128(cj_kv8_args a) { kv8_attend_c32<128>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) cj_kv8_attend_c128_h64(cj_kv8_args a) { kv8_attend_c128<64>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) cj_kv8_attend_c128_h128(cj_kv8_args a) { kv8_attend_c128<128>(a); }
