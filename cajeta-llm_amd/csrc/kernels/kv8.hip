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

// The segment s, and whether its slot, rows and positions are in range.
DEV bool kv8_seg(const cj_kv8_args &a, int s, Kv8Seg &g) {
    const int4 v = ((const int4 *)a.segs)[s];
    g.slot = v.x; g.pos = v.y; g.row = v.z; g.rows = v.w;
    const bool ok = v.x >= 0 && v.x < a.n_slots && v.w >= 0 && v.w <= a.max_rows && v.z >= 0 && v.z <= a.n_rows - v.w &&
                    v.y >= 0 && v.y <= a.limit - v.w;
    if (!ok && a.status && threadIdx.x == 0) *a.status = 1;
    return ok;
}

// The page of the slot's positions from 64·i on; −1 where the table has none.
DEV int kv8_page(const cj_kv8_args &a, int slot, int i) {
    const int p = a.pgtab[(int64_t)slot * a.slot_pages + i];
    return p >= 0 && p < a.n_pages ? p : -1;
}

DEV double kv8_shfl_xor(double v, int m) {
    return __hiloint2double(__shfl_xor(__double2hiint(v), m), __shfl_xor(__double2loint(v), m));
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

// Rotation (and norm) of the pairs a[i], b[i] of one head's row, held by 16
// lanes, lane j with pairs j·NP..; in 64 bits, so that the code of a value
// next to a rounding border is that of the exact one.
template <int NP>
DEV void kv8_turn(double (&a)[NP], double (&b)[NP], const cj_kv8_args &g, const float *w, int pos, int j) {
    if (g.norm) {
        double ss = 0;
#pragma unroll
        for (int i = 0; i < NP; i++) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
        for (int m = 1; m < 16; m *= 2) ss += kv8_shfl_xor(ss, m);
        const double s = 1.0 / sqrt(ss / (32 * NP) + (double)g.eps), one = g.form ? 1.0 : 0.0;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            a[i] = a[i] * s * (one + (double)w[j * NP + i]);
            b[i] = b[i] * s * (one + (double)w[16 * NP + j * NP + i]);
        }
    }
    const float *cs = g.rope_cs + (int64_t)pos * (32 * NP) + 2 * NP * j;
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

DEV double kv8_size(double x) { return fabs(x) <= 1.0e300 ? fabs(x) : __longlong_as_double(0x7ff0000000000000ll); }

DEV uint32_t kv8_code(double x, double inv) { return (uint32_t)((int)rint(x * inv) + 128); }

// Append: a workgroup a (segment, block, kv head), then workgroups of 16
// (row, query head) pairs. Thread t holds position (or pair) t / 16 and its
// rotation pairs (t % 16)·NP.., so a head's row is 16 lanes.
template <int HD>
DEV void kv8_append(const cj_kv8_args &a) {
    constexpr int NP = HD / 32;
    const int t = threadIdx.x, tt = t >> 4, j = t & 15;
    Kv8Seg g;
    if ((int)blockIdx.x >= a.kv_wgs) {
        // query rows
        const int w = (int)blockIdx.x - a.kv_wgs, s = w / a.per_seg;
        if (!kv8_seg(a, s, g)) return;
        const int i = (w - s * a.per_seg) * 16 + tt, r = i / a.n_q, h = i - r * a.n_q;
        if (r >= g.rows) return;
        double x[NP], y[NP];
        const float *src = a.q + (int64_t)(g.row + r) * a.q_stride + (int64_t)h * HD + j * NP;
        kv8_load<NP>(src, x);
        kv8_load<NP>(src + HD / 2, y);
        kv8_turn<NP>(x, y, a, a.qw, g.pos + r, j);
        float *dst = a.q_out + (int64_t)(g.row + r) * a.out_stride + (int64_t)h * HD + j * NP;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            dst[i] = (float)x[i];
            dst[HD / 2 + i] = (float)y[i];
        }
        return;
    }
    __shared__ double tops[2][4];
    __shared__ __align__(16) uint8_t tv[HD * KV8_BLOCK];
    const int nb = (a.max_rows + KV8_BLOCK - 2) / KV8_BLOCK + 1;
    const int h = blockIdx.x % a.n_kv, w = blockIdx.x / a.n_kv, blk = w % nb, s = w / nb;
    if (!kv8_seg(a, s, g)) return;
    const int b0 = (g.pos / KV8_BLOCK + blk) * KV8_BLOCK;
    if (g.rows == 0 || b0 >= g.pos + g.rows) return;
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
        const int64_t at = (int64_t)(g.row + p - g.pos) * a.kv_stride + (int64_t)h * HD + j * NP;
        kv8_load<NP>(a.k + at, kx);
        kv8_load<NP>(a.k + at + HD / 2, ky);
        kv8_load<NP>(a.v + at, vx);
        kv8_load<NP>(a.v + at + HD / 2, vy);
        kv8_turn<NP>(kx, ky, a, a.kw, p, j);
#pragma unroll
        for (int i = 0; i < NP; i++) {
            ktop = fmax(ktop, fmax(kv8_size(kx[i]), kv8_size(ky[i])));
            vtop = fmax(vtop, fmax(kv8_size(vx[i]), kv8_size(vy[i])));
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        ktop = fmax(ktop, kv8_shfl_xor(ktop, m));
        vtop = fmax(vtop, kv8_shfl_xor(vtop, m));
    }
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
// and HD / 16 of its channels.
template <int HD>
DEV void kv8_read(const cj_kv8_args &a) {
    constexpr int W = HD / 16;
    __shared__ __align__(16) uint8_t tv[HD * KV8_BLOCK];
    const int t = threadIdx.x, tt = t >> 4, j = t & 15;
    const int nb = (a.max_rows + KV8_BLOCK - 2) / KV8_BLOCK + 1;
    const int h = blockIdx.x % a.n_kv, w = blockIdx.x / a.n_kv, blk = w % nb, s = w / nb;
    Kv8Seg g;
    if (!kv8_seg(a, s, g)) return;
    const int b0 = (g.pos / KV8_BLOCK + blk) * KV8_BLOCK;
    if (b0 >= g.pos + g.rows) return;
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
    const int64_t o = (int64_t)(g.row + p - g.pos) * a.out_stride + (int64_t)h * HD + j * W;
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

// Attention, one wave a (row, query head): a page's 64 positions a pass, a
// lane a position for the scores, then lanes over the channels.
template <int HD>
DEV void kv8_attend_row(const cj_kv8_args &a) {
    __shared__ float sq[HD], sp[KV8_PAGE];
    const int t = threadIdx.x, h = blockIdx.x % a.n_q, w = blockIdx.x / a.n_q, i = w % a.max_rows, s = w / a.max_rows;
    Kv8Seg g;
    if (!kv8_seg(a, s, g) || i >= g.rows) return;
    const int kvh = h / (a.n_q / a.n_kv), last = g.pos + i;
    const int first = a.window > 0 && last >= a.window ? last + 1 - a.window : 0;
    for (int d = t; d < HD; d += 64) sq[d] = a.q[(int64_t)(g.row + i) * a.q_stride + (int64_t)h * HD + d] * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0, acc[HD / 64] = {};
    for (int pi = first / KV8_PAGE; pi <= last / KV8_PAGE; pi++) {
        int page = kv8_page(a, g.slot, pi);
        const bool bad = page < 0;
        if (bad) {
            page = 0;
            if (a.status && t == 0) *a.status = 1;
        }
        const int64_t ph = (int64_t)page * a.n_kv + kvh;
        const float none = __uint_as_float(0x7fc00000u);
        const int p = pi * KV8_PAGE + t;
        const bool seen = p >= first && p <= last;
        float x = 0;
        const uint32_t *kr = (const uint32_t *)(a.kc + (ph * KV8_PAGE + t) * HD);
        for (int c = 0; c < HD / 4; c++) {
            const uint32_t b = kr[c];
#pragma unroll
            for (int k = 0; k < 4; k++) x = fmaf(sq[4 * c + k], (float)((int)((b >> (8 * k)) & 255u) - 128), x);
        }
        x = seen ? x * (bad ? none : a.ks[ph * 4 + t / 16]) : -INFINITY;
        const float mt = fmaxf(m, xmax64(x));
        const float r = m == -INFINITY ? 0.0f : __expf(m - mt), e = seen ? __expf(x - mt) : 0.0f;
        float sum = e;
#pragma unroll
        for (int k = 1; k < 64; k *= 2) sum += __shfl_xor(sum, k);
        l = l * r + sum;
        m = mt;
        __syncthreads();
        sp[t] = seen ? e * a.vs[ph * 4 + t / 16] : 0.0f;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < HD / 64; c++) {
            float y = 0;
            for (int k = 0; k < KV8_PAGE; k++) {
                const uint8_t *v = a.vc + ph * KV8_PAGE * HD + (int64_t)(k / 16) * HD * 16 + (c * 64 + t) * 16 + k % 16;
                y = fmaf(sp[k], (float)((int)*v - 128), y);
            }
            acc[c] = acc[c] * r + y;
        }
    }
#pragma unroll
    for (int c = 0; c < HD / 64; c++)
        a.out[(int64_t)(g.row + i) * a.out_stride + (int64_t)h * HD + c * 64 + t] = acc[c] / l;
}

extern "C" __global__ void __launch_bounds__(256) cj_kv8_append_h64(cj_kv8_args a) { kv8_append<64>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_append_h128(cj_kv8_args a) { kv8_append<128>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_read_h64(cj_kv8_args a) { kv8_read<64>(a); }
extern "C" __global__ void __launch_bounds__(256) cj_kv8_read_h128(cj_kv8_args a) { kv8_read<128>(a); }
extern "C" __global__ void __launch_bounds__(64) cj_kv8_attend_row_h64(cj_kv8_args a) { kv8_attend_row<64>(a); }
extern "C" __global__ void __launch_bounds__(64) cj_kv8_attend_row_h128(cj_kv8_args a) { kv8_attend_row<128>(a); }
