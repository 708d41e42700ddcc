// qsa_rope.hip -- rotary positions: rows turned by their positions (with the
// RMSNorm before it), and the append of a token's K and V into the paged cache
// with that rotation on the way (qwfn_rope_rows, qwfn_kv_append_rope).
//
// Mathematics.  A head row x of hd values is normed, z_d = x_d w_d /
// sqrt(mean(x^2) + eps) (or z = x), and the pairs (a, b) of its first rd values
// turn by the angle 2 pi pos turns_i: (a c - b s, b c + a s), c and s times
// mscale.  Everything is evaluated in 64 bits and rounded once to fp32: a
// cached quant is decided by values next to a rounding border, and a far
// position needs the product pos * turns_i past 24 bits.  The vector pipes run an
// fp64 fma at the rate of an fp32 one.
//
// Two ways.  k_rope_rows8 and k_rope_append8 take rows of 64, 128 or 256 values in
// 16-byte pieces: a lane holds the two 8-value chunks of a head row whose values
// turn together, hd / 16 lanes a head row, computes its cos and sin once and goes
// over several heads with them.  k_rope_rows and k_rope_append take everything
// else, a wave a head row through LDS (8,192 x 16 rows 73 us).
//
// Measured (MI355X): 8,192 x 16 bfloat16 rows of 128, normed: 18.9 us by the kernel, 3.6 TB/s of the 5.2 that a
// large copy reaches; 1,628 vector instructions a wave of 8 rows x 4 heads are 60 % of the time, a
// fourth of them cos and sin.  8,000 rows of K and V into q8_0: 20.4 us (a wave's chain of loads, norm
// and division), their 16 query heads beside it 27.0 us for 98 MB.  64 single rows 5.8 us, one 5.0.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "qsa_append.h"
#include "qsa_io.h"

namespace qwfn_qsa {

namespace {

constexpr int kWaves = 4;                 // head rows a workgroup

__device__ __forceinline__ float row_value(const RowsArg &r, int64_t i) {
    if (r.dtype == QWFN_SRC_F32) return ((const float *)r.data)[i];
    const uint16_t h = ((const uint16_t *)r.data)[i];
    return r.dtype == QWFN_SRC_F16 ? h2f(h) : __uint_as_float((uint32_t)h << 16);
}
__device__ __forceinline__ void put_row_value(const RowsArg &r, int64_t i, float y) {
    if (r.dtype == QWFN_SRC_F32) ((float *)r.data)[i] = y;
    else if (r.dtype == QWFN_SRC_F16) ((uint16_t *)r.data)[i] = f2h(y);
    else ((__bf16 *)r.data)[i] = (__bf16)y;
}

// fp32 of a 64-bit result, a rounding of its own: without the barrier the compiler may join it
// with a following rounding to fp16 (floating-point contraction), which differs at ties.
__device__ __forceinline__ float round32(double y) {
    float f = (float)y;
    asm("" : "+v"(f));
    return f;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// cos and sin (times mscale, sin negated for the inverse) of pair i at pos.
__device__ __forceinline__ double2 rope_cs(const RopeArg &rp, int pos, int i) {
    const double f = rp.turns[i], p = (double)pos;
    double s, c;
    sincospi(2.0 * fma(p, f, -rint(p * f)), &s, &c);          // the product exact, less its whole turns
    return make_double2(c * rp.mscale, (rp.inverse ? -s : s) * rp.mscale);
}

// A wave turns one head row: x (LDS, its own hd doubles) holds the row, lane l
// has loaded values l, l + 64, ...; f(d, y) takes each result.  norm: fp32 [hd]
// weights or NULL.  Reached by every wave of the workgroup (it synchronises).
template <class Put>
__device__ __forceinline__ void turn_row(const RopeArg &rp, const float *norm, double *x, int hd, int pos, int lane,
                                         bool live, Put put) {
    double f = 1.0;
    if (live && norm) {
        double ss = 0.0;
        for (int d = lane; d < hd; d += 64) ss += x[d] * x[d];
        f = 1.0 / sqrt(wave_sum_f64(ss) / hd + rp.eps);
        for (int d = lane; d < hd; d += 64) x[d] *= f * (double)norm[d];
    }
    __syncthreads();
    if (!live) return;
    const int half = rp.rd / 2;
    for (int d = lane; d < hd; d += 64) {
        double y = x[d];
        if (d < rp.rd) {
            const int i = rp.interleaved ? d >> 1 : d < half ? d : d - half;
            const bool second = rp.interleaved ? d & 1 : d >= half;
            const int o = rp.interleaved ? d ^ 1 : second ? d - half : d + half;
            const double2 cs = rope_cs(rp, pos, i);
            y = second ? y * cs.x + x[o] * cs.y : y * cs.x - x[o] * cs.y;
        }
        put(d, round32(y));
    }
}

// ---- rows in 16-byte pieces ----

// cos and sin of 2 pi p f, p f exact: the whole turns off, the quarter turns aside,
// then the Taylor series at |y| <= pi / 4, to y^15 and y^16 (the next terms are below
// 2^-54).
__device__ __forceinline__ double2 turn(double p, double f) {
    const double r = fma(p, f, -rint(p * f)), q = rint(4.0 * r);
    const double y = fma(-0.25, q, r) * 6.283185307179586476925, z = y * y;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
    s = fma(s, z, 1.0 / 6227020800.0);
    c = fma(c, z, -1.0 / 87178291200.0);
    s = fma(s, z, -1.0 / 39916800.0);
    c = fma(c, z, 1.0 / 479001600.0);
    s = fma(s, z, 1.0 / 362880.0);
    c = fma(c, z, -1.0 / 3628800.0);
    s = fma(s, z, -1.0 / 5040.0);
    c = fma(c, z, 1.0 / 40320.0);
    s = fma(s, z, 1.0 / 120.0);
    c = fma(c, z, -1.0 / 720.0);
    s = fma(s, z, -1.0 / 6.0);
    c = fma(c, z, 1.0 / 24.0);
    s = fma(s * z, y, y);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int k = (int)q & 3;
    const double a = k & 1 ? s : c, b = k & 1 ? c : s;    // |cos|, |sin|
    return make_double2(k == 1 || k == 2 ? -a : a, k >= 2 ? -b : b);
}

// v of lane l ^ 1, 2, 4, 8 (by halves on the DPP network).
template <int CTRL>
__device__ __forceinline__ double dppd(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dppi<CTRL>((int)(uint32_t)u, (int)(uint32_t)u);
    const uint32_t hi = (uint32_t)dppi<CTRL>((int)(u >> 32), (int)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A lane's place in a head row of HD values: chunks a and b of 8 values.  HALF: while the
// rotation lasts, b is the chunk a turns with.  LH lanes a head row.
template <int HD, bool IL>
struct Place {
    static constexpr int LH = HD / 16;
    int e, a, b;
    bool ta, tb;                                          // the chunk turns
    __device__ __forceinline__ Place(int lane, int rd) {
        e = lane % LH;
        if (IL) {
            a = e;
            b = e + LH;
            ta = 8 * a < rd;
            tb = 8 * b < rd;
        } else {
            const int n = rd / 16;                        // lanes whose chunks turn
            ta = tb = e < n;
            a = ta ? e : 2 * n + (e - n);
            b = ta ? e + n : a + (LH - n);
        }
    }
};

// A lane's cos and sin: IL: of chunk a's four pairs and b's; HALF: of the eight pairs of a and b.
template <int HD, bool IL>
__device__ __forceinline__ void place_cs(const Place<HD, IL> &pl, const RopeArg &rp, int pos, const double (&f)[8],
                                         double2 (&cs)[8]) {
    double p = (double)pos;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        cs[k] = make_double2(0.0, 0.0);
        if (k < 4 || !IL ? pl.ta : pl.tb) {
            const double2 t = turn(p, f[k]);
            cs[k] = make_double2(t.x * rp.mscale, (rp.inverse ? -t.y : t.y) * rp.mscale);
        }
        // one pair after the other: eight chains at once would take the registers of a wave more a SIMD
        asm volatile("" : "+v"(p), "+v"(cs[k].x), "+v"(cs[k].y));
    }
}

// The lane's 16 values x (chunk a's, then b's) of a head row, normed (norm: with the weights w)
// and turned, rounded to fp32 in place.
template <int HD, bool IL>
__device__ __forceinline__ void turn16(const Place<HD, IL> &pl, float (&x)[16], bool norm, const float (&w)[16],
                                       const double2 (&cs)[8], double eps) {
    double f = 1.0;
    if (norm) {
        double ss = 0.0, st = 0.0;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
            ss = fma((double)x[k], (double)x[k], ss);
            st = fma((double)x[k + 1], (double)x[k + 1], st);
        }
        ss += st;
        ss += dppd<kDppQuadXor1>(ss);
        ss += dppd<kDppQuadXor2>(ss);
        if constexpr (HD >= 128) ss += dppd<kDppRowHalfMirror>(ss);
        if constexpr (HD >= 256) ss += dppd<kDppRowMirror>(ss);
        f = rsqrt(fma(ss, 1.0 / HD, eps));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int i = IL ? 2 * k : k, j = IL ? i + 1 : k + 8;
        const double p = (double)x[i] * ((double)w[i] * f), q = (double)x[j] * ((double)w[j] * f);
        const bool on = IL && k >= 4 ? pl.tb : pl.ta;     // (a product with 0 would spread a NaN to the other chunk)
        x[i] = round32(on ? fma(p, cs[k].x, -(q * cs[k].y)) : p);
        x[j] = round32(on ? fma(q, cs[k].x, p * cs[k].y) : q);
    }
}

}  // namespace

// One wave a head row: item = row * heads + head.
__global__ void __launch_bounds__(64 * kWaves)
k_rope_rows(RopeArg rp, RowsArg src, const float *norm, const int32_t *pos, int64_t n_items, int heads, int hd,
            RowsArg dst) {
    __shared__ double xs[kWaves][kRopeMaxDim];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t item = (int64_t)blockIdx.x * kWaves + w;
    const bool live = item < n_items;
    const int64_t r = live ? item / heads : 0;
    const int h = (int)(live ? item % heads : 0);
    if (live)
        for (int d = lane; d < hd; d += 64) xs[w][d] = row_value(src, r * src.row_stride + h * src.head_stride + d);
    turn_row(rp, norm, xs[w], hd, live ? pos[r] : 0, lane, live,
             [&](int d, float y) { put_row_value(dst, r * dst.row_stride + h * dst.head_stride + d, y); });
}

// One wave a head row of a token's Q (n_q heads, 0: none), K or V: item = row *
// (n_q + 2 Hkv) + head.
__global__ void __launch_bounds__(64 * kWaves)
k_rope_append(Geo g, qwfn_kv_view v, RopeArg rp, RowsArg q, RowsArg k, RowsArg vv, const float *q_norm,
              const float *k_norm, const int32_t *seq_ids, const int32_t *pos, int64_t n_items, int n_q, RowsArg q_out) {
    __shared__ double xs[kWaves][kRopeMaxDim];
    __shared__ float ys[kWaves][kRopeMaxDim];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, per = n_q + 2 * g.Hkv;
    const int64_t item = (int64_t)blockIdx.x * kWaves + w;
    const bool live = item < n_items;
    const int64_t r = live ? item / per : 0;
    int h = (int)(live ? item % per : 0);
    const int which = h < n_q ? 0 : h < n_q + g.Hkv ? 1 : 2;          // Q, K, V
    h -= which == 0 ? 0 : which == 1 ? n_q : n_q + g.Hkv;
    const RowsArg &src = which == 0 ? q : which == 1 ? k : vv;
    if (live)
        for (int d = lane; d < g.hd; d += 64) xs[w][d] = row_value(src, r * src.row_stride + h * src.head_stride + d);
    const int t = live ? pos[r] : 0;
    RopeArg rw = rp;
    if (which == 2) rw.rd = 0;                                        // V passes as it is
    turn_row(rw, which == 0 ? q_norm : which == 1 ? k_norm : nullptr, xs[w], g.hd, t, lane, live, [&](int d, float y) {
        if (which == 0) put_row_value(q_out, r * q_out.row_stride + h * q_out.head_stride + d, y);
        else ys[w][d] = y;
    });
    __syncthreads();
    if (!live || which == 0) return;
    const int seq = seq_ids ? seq_ids[r] : 0;
    const bool report = lane == 0 && h == 0 && which == 1;
    if (seq < 0 || seq >= g.n_seq_view) { if (report) set_status(v.status, QWFN_STATUS_SEQ_RANGE); return; }
    if (t < 0 || (int64_t)t >= (int64_t)g.pps * g.pt) { if (report) set_status(v.status, QWFN_STATUS_POS_RANGE); return; }
    const int32_t pp = phys_page(g, v.page_table, seq, t);
    if (pp < 0) { if (report) set_status(v.status, QWFN_STATUS_PAGE_RANGE); return; }
    uint8_t *page = (uint8_t *)(which == 2 ? v.v_pages : v.k_pages) + (int64_t)pp * g.page_bytes;
    const float *y = ys[w];
    for (int i = lane; i < g.hd / 4; i += 64)
        store_block_lane(g, page, which == 2, h, t % g.pt, i >> 3, i & 7,
                         [&](int d, float *x) { x[0] = y[d]; x[1] = y[d + 1]; },
                         [&](int d, float *x) { x[0] = y[d]; x[1] = y[d + 1]; x[2] = y[d + 2]; x[3] = y[d + 3]; });
}

// A lane's two chunks as they lie in memory (loaded a head ahead of their use).
template <int SZ>
struct Raw {
    u4v c[SZ];                                            // 2 chunks of 8 values of SZ bytes
    __device__ __forceinline__ void load(const RowsArg &r, int64_t at, int a, int b) {
        const uint8_t *p = (const uint8_t *)r.data + at * SZ;
#pragma unroll
        for (int k = 0; k < SZ / 2; ++k) {
            c[k] = *reinterpret_cast<const u4v *>(p + 8 * SZ * a + 16 * k);
            c[SZ / 2 + k] = *reinterpret_cast<const u4v *>(p + 8 * SZ * b + 16 * k);
        }
    }
    __device__ __forceinline__ void values(int dtype, float (&x)[16]) const {
#pragma unroll
        for (int k = 0; k < 4 * SZ; ++k) {
            const uint32_t w = c[k >> 2][k & 3];
            if constexpr (SZ == 4) {
                x[k] = __uint_as_float(w);
            } else {
                x[2 * k] = dtype == QWFN_SRC_F16 ? h2f((uint16_t)w) : bf16_f(w & 0xFFFFu);
                x[2 * k + 1] = dtype == QWFN_SRC_F16 ? h2f((uint16_t)(w >> 16)) : bf16_f(w >> 16);
            }
        }
    }
};

// What a lane reads before it knows more than its row: the first head's chunks, the norm's weights
// and the frequencies of its pairs, all in flight together (and before a page is looked up).
template <int HD, bool IL, int SZ>
struct Front {
    Raw<SZ> raw;
    float w[16];
    double f[8];
    __device__ __forceinline__ Front(const RopeArg &rp, const Place<HD, IL> &pl, const RowsArg &src, const float *norm,
                                     int64_t rr, int h0) {
        raw.load(src, rr * src.row_stride + h0 * src.head_stride, pl.a, pl.b);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool on = k < 4 || !IL ? pl.ta : pl.tb;
            f[k] = rp.turns[on ? IL ? 4 * (k < 4 ? pl.a : pl.b) + (k & 3) : 8 * pl.a + k : 0];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) w[k] = 1.0f;
        if (norm) {
            load8(norm, QWFN_SRC_F32, 8 * pl.a, w);
            load8(norm, QWFN_SRC_F32, 8 * pl.b, w + 8);
        }
    }
};

// Rows of HD values in 16-byte pieces: a wave 64 / LH rows at a time, heads h0 .. h1 - 1 with
// one cos and sin; put(h, x) takes the lane's 16 results of head h.
template <int HD, bool IL, int SZ, class Put>
__device__ __forceinline__ void heads8(const RopeArg &rp, const Place<HD, IL> &pl, const RowsArg &src, bool norm,
                                       Front<HD, IL, SZ> &in, int64_t rr, int pos, int h0, int h1, Put put) {
    const int64_t at = rr * src.row_stride;
    double2 cs[8];
    place_cs(pl, rp, pos, in.f, cs);
    for (int h = h0; h < h1; ++h) {
        float x[16];
        in.raw.values(src.dtype, x);
#pragma unroll
        for (int k = 0; k < 16; ++k) asm("" : "+v"(in.w[k]));         // (its 64-bit form is not held over the loop)
        if (h + 1 < h1) in.raw.load(src, at + (h + 1) * src.head_stride, pl.a, pl.b);
        turn16(pl, x, norm, in.w, cs, rp.eps);
        put(h, x);
    }
}

// grid (row blocks, groups of hg heads).
template <int HD, bool IL, int SZ>
__global__ void __launch_bounds__(256, SZ == 4 ? 3 : 4)
k_rope_rows8(RopeArg rp, RowsArg src, const float *norm, const int32_t *pos, int64_t n_rows, int heads, int hg, RowsArg dst) {
    constexpr int kRowsWave = 64 * 16 / HD;
    const int lane = threadIdx.x & 63, h0 = blockIdx.y * hg;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kRowsWave;
    if (row0 >= n_rows) return;
    const Place<HD, IL> pl(lane, rp.rd);
    const int64_t r = row0 + lane / pl.LH, rr = min(r, n_rows - 1), to = rr * dst.row_stride;
    Front<HD, IL, SZ> in(rp, pl, src, norm, rr, h0);
    heads8<HD, IL, SZ>(rp, pl, src, norm != nullptr, in, rr, pos[rr], h0, min(h0 + hg, heads), [&](int h, const float *x) {
        if (r >= n_rows) return;
        store8(dst.data, dst.dtype, to + h * dst.head_stride + 8 * pl.a, x);
        store8(dst.data, dst.dtype, to + h * dst.head_stride + 8 * pl.b, x + 8);
    });
}

// Where row r's K and V go: its page and row in it; false (and reported once, with `report`) for a
// bad sequence, position or page.
struct Dest { int32_t page, row; };
__device__ __forceinline__ bool dest_of(const Geo &g, const qwfn_kv_view &v, int seq, int t, bool report, Dest &d) {
    int32_t bad = 0;
    if (seq < 0 || seq >= g.n_seq_view) bad = QWFN_STATUS_SEQ_RANGE;
    else if (t < 0 || (int64_t)t >= (int64_t)g.pps * g.pt) bad = QWFN_STATUS_POS_RANGE;
    else if ((d.page = phys_page(g, v.page_table, seq, t)) < 0) bad = QWFN_STATUS_PAGE_RANGE;
    if (bad && report) set_status(v.status, bad);
    d.row = bad ? 0 : t % g.pt;
    return !bad;
}

// q8_0 of a 32-value block held by a quad of lanes, 8 values each, as quant4 computes it.
__device__ __forceinline__ uint2 quad_q8(const float *x, int variant, uint16_t *dh) {
#pragma clang fp contract(off)
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float ax = fabsf(x[k]);
        a = ax > a ? ax : a;
    }
    a = fmaxf(a, dppf<kDppQuadXor1>(a, a));
    a = fmaxf(a, dppf<kDppQuadXor2>(a, a));
    const float d = a / 127.0f;
    *dh = f2h(d);
    const float id = variant == QWFN_Q8_X86_RNE ? (a != 0.0f ? 127.0f / a : 0.0f) : (d != 0.0f ? 1.0f / d : 0.0f);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float y = x[k] * id;
        w[k / 4] |= (uint32_t)(uint8_t)to_i8(variant == QWFN_Q8_X86_RNE ? __builtin_rintf(y) : roundf(y)) << (8 * (k & 3));
    }
    return make_uint2(w[0], w[1]);
}

// q4_0 of a quad's block, as quant_q4 computes it (the first value of the largest magnitude
// sets the scale): the quants of the lane's 8 values, a byte each; lane e of the quad.
__device__ __forceinline__ uint2 quad_q4(const float *x, int e, uint16_t *dh) {
#pragma clang fp contract(off)
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) a = fmaxf(a, fabsf(x[k]));
    a = fmaxf(a, dppf<kDppQuadXor1>(a, a));
    a = fmaxf(a, dppf<kDppQuadXor2>(a, a));
    int bi = 32;
    float bv = 0.0f;
#pragma unroll
    for (int k = 7; k >= 0; --k)
        if (a > 0.0f && fabsf(x[k]) == a) { bi = 8 * e + k; bv = x[k]; }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
        const int oi = step ? dppi<kDppQuadXor2>(bi, bi) : dppi<kDppQuadXor1>(bi, bi);
        const float ov = step ? dppf<kDppQuadXor2>(bv, bv) : dppf<kDppQuadXor1>(bv, bv);
        if (oi < bi) { bi = oi; bv = ov; }
    }
    const float d = bv / -8.0f;
    *dh = f2h(d);
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float y = x[k] * id + 8.5f;
        const int t = y != y ? 0 : (int)y;
        w[k / 4] |= (uint32_t)(t < 15 ? t : 15) << (8 * (k & 3));
    }
    return make_uint2(w[0], w[1]);
}

// Chunk c (8 values, four lanes of a quad holding chunks 4 j .. 4 j + 3) of a head row into a
// K-layout page.  The quad is together; `live` is the same in it.
template <int KT>
__device__ __forceinline__ void store_chunk(const Geo &g, uint8_t *page, int gh, int row, int c, const float *x, bool live) {
    if constexpr (KT == QWFN_KV_F16) {
        if (live) store8(page + chunk_off(g, gh, row, c), QWFN_SRC_F16, 0, x);
    } else {
        uint16_t dh;
        if constexpr (KT == QWFN_KV_Q4_0) {
            const uint2 w = quad_q4(x, c & 3, &dh);
            // dims 0 .. 15 of the block in the low nibbles, 16 .. 31 in the high ones
            const uint32_t hx = (uint32_t)dppi<kDppQuadXor2>((int)w.x, (int)w.x), hy = (uint32_t)dppi<kDppQuadXor2>((int)w.y, (int)w.y);
            if (live && (c & 3) < 2)
                *reinterpret_cast<uint2 *>(page + chunk_off(g, gh, row, c / 4) + 8 * (c & 1)) = make_uint2(w.x | hx << 4, w.y | hy << 4);
        } else {
            const uint2 w = quad_q8(x, g.variant, &dh);
            if (live) *reinterpret_cast<uint2 *>(page + quant_off(g, gh, row, 8 * c)) = w;
        }
        if (live && (c & 3) == 0) *reinterpret_cast<uint16_t *>(page + scale_off(g, gh, row, c / 4)) = dh;
    }
}

// The V rows of a q8_0 page that is dimension-major in its 64-token tiles: a workgroup's up to
// 64 rows of 64 dimensions (chunks c0 .. c0 + 7) of one head are quantized by rows, eight lanes
// a row, and turned in LDS.  Rows at positions that follow each other (a prompt's) leave it as
// whole words, others byte by byte.
constexpr int kTurnRow = 68;                              // 64 bytes of a dimension, displaced by up to 3
__device__ __forceinline__ void values_turned(const Geo &g, const qwfn_kv_view &v, const RowsArg &vv, const int32_t *seq_ids,
                                              const int32_t *pos, int64_t row0, int64_t end, int h, int c0, uint8_t *lds) {
    const int lane = threadIdx.x & 63, tid = threadIdx.x, c = c0 + lane % 8, o0 = tid / 8;
    const int m = (int)(end - row0);
    float x[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k)
        load8(vv.data, vv.dtype, (row0 + min(o0 + 32 * k, m - 1)) * vv.row_stride + h * vv.head_stride + 8 * c, x[k]);
    const int t0 = pos[row0], s0 = seq_ids ? seq_ids[row0] : 0;
    bool run = t0 >= 0 && (int64_t)t0 + m <= (int64_t)g.pps * g.pt && s0 >= 0 && s0 < g.n_seq_view;
    if (tid < m) run = run && (int64_t)pos[row0 + tid] == (int64_t)t0 + tid && (!seq_ids || seq_ids[row0 + tid] == s0);
    run = __syncthreads_and(run);
    const int a = run ? t0 & 3 : 0;
    // a run's rows lie in one page or two: looked up once, not a row (tb: the second's first cell)
    int tb = 0;
    int32_t pa = -1, pb = -1;
    if (run) {
        tb = (t0 / g.pt + 1) * g.pt;
        pa = phys_page(g, v.page_table, s0, t0);
        if (t0 + m > tb) pb = phys_page(g, v.page_table, s0, tb);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int o = o0 + 32 * k, t = t0 + o;
        const int64_t rr = row0 + min(o, m - 1);
        Dest d{t < tb ? pa : pb, t < tb ? t - tb + g.pt : t - tb};
        bool live = o < m;
        if (run) live = live && d.page >= 0;
        else live = dest_of(g, v, seq_ids ? seq_ids[rr] : 0, pos[rr], false, d) && live;
        uint8_t *page = (uint8_t *)v.v_pages + (live ? (int64_t)d.page * g.page_bytes : 0);
        uint16_t dh;
        const uint2 w = quad_q8(x[k], g.variant, &dh);
        if (live && (c & 3) == 0) *reinterpret_cast<uint16_t *>(page + scale_off(g, h, d.row, c / 4)) = dh;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t b = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
            if (run) {
                if (o < m) lds[(8 * (c - c0) + j) * kTurnRow + a + o] = b;
            } else if (live) {
                page[vquant_off(g, h, d.row, 8 * c + j)] = b;
            }
        }
    }
    if (!run) return;
    __syncthreads();
    // word k of a dimension: cells t0 - a + 4 k .. + 3, which lie in one tile
    uint8_t *va = (uint8_t *)v.v_pages + (int64_t)pa * g.page_bytes, *vb = (uint8_t *)v.v_pages + (int64_t)pb * g.page_bytes;
    for (int i = tid; i < 64 * 17; i += 256) {
        const int dim = i / 17, k = i % 17, o = 4 * k - a, t = t0 + o;
        if (o >= m || (t < tb ? pa : pb) < 0) continue;
        uint8_t *to = t < tb ? va + vquant_off(g, h, t - tb + g.pt, 8 * c0 + dim) : vb + vquant_off(g, h, t - tb, 8 * c0 + dim);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(lds + dim * kTurnRow + 4 * k);
        if (o >= 0 && o + 4 <= m) {
            *reinterpret_cast<uint32_t *>(to) = w;
        } else {
            for (int j = 0; j < 4; ++j)
                if (o + j >= 0 && o + j < m) to[j] = (uint8_t)(w >> (8 * j));
        }
    }
}

// Q, K and V: grid (row blocks, a pass of the four waves each; groups of hq query heads, then of
// hk key heads, then one a value head, or a 64-dimension part of one that is turned).  SZ: bytes of
// a source value.
template <int HD, int KT, bool IL, int SZ>
__global__ void __launch_bounds__(256, 3)
k_rope_append8(Geo g, qwfn_kv_view v, RopeArg rp, RowsArg q, RowsArg k, RowsArg vv, const float *q_norm,
               const float *k_norm, const int32_t *seq_ids, const int32_t *pos, int64_t n_rows, int n_q, int hq, int hk,
               RowsArg q_out) {
    constexpr int kRowsWave = 64 * 16 / HD;
    __shared__ __attribute__((aligned(16))) uint8_t lds[KT == QWFN_KV_Q8_0 ? 64 * kTurnRow : 16];
    const int qg = (n_q + hq - 1) / hq, kg = (g.Hkv + hk - 1) / hk;
    const int64_t b0 = (int64_t)blockIdx.x * (4 * kRowsWave);
    const int role = blockIdx.y, which = role < qg ? 0 : role < qg + kg ? 1 : 2;         // Q, K, V
    if (KT == QWFN_KV_Q8_0 && which == 2 && g.vdim) {
        const int i = role - qg - kg;                                                    // (64 rows, 64 dimensions)
        if (b0 % 64 == 0)
            values_turned(g, v, vv, seq_ids, pos, b0, min(b0 + 64, n_rows), i / (HD / 64), i % (HD / 64) * 8, lds);
        return;
    }
    const RowsArg src = which == 0 ? q : which == 1 ? k : vv;
    const float *norm = which == 0 ? q_norm : which == 1 ? k_norm : nullptr;
    const int h0 = which == 0 ? role * hq : which == 1 ? (role - qg) * hk : role - qg - kg;
    const int h1 = which == 0 ? min(h0 + hq, n_q) : which == 1 ? min(h0 + hk, g.Hkv) : h0 + 1;
    const int lane = threadIdx.x & 63;
    const Place<HD, IL> pl(lane, which == 2 ? 0 : rp.rd);                                // (V does not turn)
    const int64_t row0 = b0 + (threadIdx.x >> 6) * kRowsWave;
    if (row0 >= n_rows) return;
    const int64_t r = row0 + lane / pl.LH, rr = min(r, n_rows - 1);
    const int t = pos[rr], seq = seq_ids ? seq_ids[rr] : 0;
    Front<HD, IL, SZ> in(rp, pl, src, norm, rr, h0);
    Dest d{0, 0};
    bool live = r < n_rows;
    if (which) {
        const bool report = live && which == 1 && h0 == 0 && pl.e == 0;
        live = dest_of(g, v, seq, t, report, d) && live;
    }
    uint8_t *page = (uint8_t *)(which == 1 ? v.k_pages : v.v_pages) + (live ? (int64_t)d.page * g.page_bytes : 0);
    heads8<HD, IL, SZ>(rp, pl, src, norm != nullptr, in, rr, t, h0, h1, [&](int h, const float *x) {
        if (which) {
            store_chunk<KT>(g, page, h, d.row, pl.a, x, live);
            store_chunk<KT>(g, page, h, d.row, pl.b, x + 8, live);
        } else if (live) {
            const int64_t to = rr * q_out.row_stride + h * q_out.head_stride;
            store8(q_out.data, q_out.dtype, to + 8 * pl.a, x);
            store8(q_out.data, q_out.dtype, to + 8 * pl.b, x + 8);
        }
    });
}

// Rows that begin, every one, at a 16-byte boundary.
static bool pieces(const RowsArg &r) {
    const int64_t n = r.dtype == QWFN_SRC_F32 ? 4 : 8;
    return (uintptr_t)r.data % 16 == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
}
// A rotation whose pairs lie in a chunk, or in two whole chunks.
static bool pieces_fit(const RopeArg &rp, int hd) {
    return (hd == 64 || hd == 128 || hd == 256) && rp.rd % (rp.interleaved ? 8 : 16) == 0;
}

// Heads a wave takes with one cos and sin: the fewest of 1, 2 and 4 that leave the grid within
// the 1,024 workgroups resident at once, else 4 (cos and sin are a fourth of a wave's
// instructions at 4 heads and more than half at 1; fewer heads a wave fill the device with few
// rows: 64 rows of 20 heads 5.7 us with 1, 14 with 4).
static int heads_a_wave(int blocks, int heads) {
    for (int n = 1; n < 4; n *= 2)
        if ((int64_t)blocks * ((heads + n - 1) / n) <= 1024) return n;
    return 4;
}
// Rows up to which the append takes the queries in its own launch.  Past them the launch is a few
// per cent and the queries' kernel alone holds a wave more a SIMD.
constexpr int kFewRows = 256;

template <class F>
static hipError_t by_shape(int hd, int dtype, F of) {
    const auto sz = [&](auto hdc) {
        return dtype == QWFN_SRC_F32 ? of(hdc, std::integral_constant<int, 4>()) : of(hdc, std::integral_constant<int, 2>());
    };
    return hd == 64 ? sz(std::integral_constant<int, 64>()) : hd == 128 ? sz(std::integral_constant<int, 128>())
                                                                       : sz(std::integral_constant<int, 256>());
}

hipError_t launch_rope_rows(const RopeArg &rp, const RowsArg &src, const float *norm, const int32_t *pos,
                            int32_t n_rows, int32_t heads, int32_t hd, const RowsArg &dst, hipStream_t st) {
    const int64_t rows = 4 * 64 * 16 / hd > 0 ? 4 * 64 * 16 / hd : 1;
    const int blocks = (int)((n_rows + rows - 1) / rows), hg = heads_a_wave(blocks, heads);
    if (pieces_fit(rp, hd) && pieces(src) && pieces(dst) && (!norm || (uintptr_t)norm % 16 == 0) &&
        (heads + hg - 1) / hg <= 65535) {
        const auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)blocks, (unsigned)((heads + hg - 1) / hg)), dim3(256), 0, st, rp, src,
                               norm, pos, n_rows, heads, hg, dst);
            return hipGetLastError();
        };
        const auto of = [&](auto hdc, auto szc) {
            constexpr int HD = decltype(hdc)::value, SZ = decltype(szc)::value;
            return rp.interleaved ? go(k_rope_rows8<HD, true, SZ>) : go(k_rope_rows8<HD, false, SZ>);
        };
        return by_shape(hd, src.dtype, of);
    }
    const int64_t items = (int64_t)n_rows * heads;
    hipLaunchKernelGGL(k_rope_rows, dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(64 * kWaves), 0, st, rp, src,
                       norm, pos, items, heads, hd, dst);
    return hipGetLastError();
}

hipError_t launch_rope_append(const Geo &g, const qwfn_kv_view &v, const RopeArg &rp, const RowsArg &q,
                              const RowsArg &k, const RowsArg &vv, const float *q_norm, const float *k_norm,
                              const int32_t *seq_ids, const int32_t *pos, int32_t n_rows, const RowsArg &q_out,
                              hipStream_t st) {
    const int n_q = q.data ? g.H : 0;
    // quantized blocks of 32 are a quad of lanes' chunks: whole, when half the rotated values are
    const bool quads = g.kt == QWFN_KV_F16 || rp.interleaved || rp.rd % 64 == 0;
    const auto whole = [](const float *w) { return (uintptr_t)w % 16 == 0; };
    const auto size = [](const RowsArg &r) { return r.dtype == QWFN_SRC_F32 ? 4 : 2; };
    if (quads && pieces_fit(rp, g.hd) && pieces(k) && pieces(vv) && (!n_q || (pieces(q) && pieces(q_out) && size(q) == size(k))) && size(k) == size(vv) && whole(q_norm) &&
        whole(k_norm)) {
        if (n_q && n_rows > kFewRows) {                   // the queries in a launch of their own
            const hipError_t e = launch_rope_rows(rp, q, q_norm, pos, n_rows, n_q, g.hd, q_out, st);
            return e != hipSuccess ? e : launch_rope_append(g, v, rp, RowsArg{}, k, vv, nullptr, k_norm, seq_ids, pos, n_rows,
                                                            RowsArg{}, st);
        }
        const int rows = 4 * 64 * 16 / g.hd, blocks = (n_rows + rows - 1) / rows;
        const int hq = heads_a_wave(blocks, std::max(n_q, 1)), hk = std::min(heads_a_wave(blocks, g.Hkv), 2);
        const unsigned roles = (n_q + hq - 1) / hq + (g.Hkv + hk - 1) / hk + g.Hkv * (g.vdim ? g.hd / 64 : 1);
        const auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)blocks, roles), dim3(256), 0, st, g, v, rp, q, k, vv, q_norm, k_norm,
                               seq_ids, pos, n_rows, n_q, hq, hk, q_out);
            return hipGetLastError();
        };
        const auto of = [&](auto hdc, auto szc) {
            constexpr int HD = decltype(hdc)::value, SZ = decltype(szc)::value;
            if (g.kt == QWFN_KV_Q4_0)
                return rp.interleaved ? go(k_rope_append8<HD, QWFN_KV_Q4_0, true, SZ>) : go(k_rope_append8<HD, QWFN_KV_Q4_0, false, SZ>);
            if (g.kt == QWFN_KV_F16)
                return rp.interleaved ? go(k_rope_append8<HD, QWFN_KV_F16, true, SZ>) : go(k_rope_append8<HD, QWFN_KV_F16, false, SZ>);
            return rp.interleaved ? go(k_rope_append8<HD, QWFN_KV_Q8_0, true, SZ>) : go(k_rope_append8<HD, QWFN_KV_Q8_0, false, SZ>);
        };
        return by_shape(g.hd, k.dtype, of);
    }
    const int64_t items = (int64_t)n_rows * (n_q + 2 * g.Hkv);
    hipLaunchKernelGGL(k_rope_append, dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(64 * kWaves), 0, st, g, v,
                       rp, q, k, vv, q_norm, k_norm, seq_ids, pos, items, n_q, q_out);
    return hipGetLastError();
}

}  // namespace qwfn_qsa
