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
#include <hip/hip_runtime.h>

#include "qsa_append.h"

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
        put(d, (float)y);
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

hipError_t launch_rope_rows(const RopeArg &rp, const RowsArg &src, const float *norm, const int32_t *pos,
                            int32_t n_rows, int32_t heads, int32_t hd, const RowsArg &dst, hipStream_t st) {
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
    const int64_t items = (int64_t)n_rows * (n_q + 2 * g.Hkv);
    hipLaunchKernelGGL(k_rope_append, dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(64 * kWaves), 0, st, g, v,
                       rp, q, k, vv, q_norm, k_norm, seq_ids, pos, items, n_q, q_out);
    return hipGetLastError();
}

}  // namespace qwfn_qsa
