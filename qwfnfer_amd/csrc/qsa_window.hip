// qsa_window.hip -- attention with a sliding window and a few first tokens that
// stay visible, over the paged cache (qwfn_window_attn_decode,
// qwfn_window_attn_prefill).
//
// Mathematics.  The query at position p of a sequence sees the cells t <= p with
// t > p - window or t < sinks; o = sum_t e^(q.k_t / sqrt(hd) - m) v_t / sum_t
// e^(q.k_t / sqrt(hd) - m), m the largest visible logit.
#include <hip/hip_runtime.h>

#include "qsa_append.h"
#include "qsa_window.h"

namespace qwfn_qsa {

namespace {

__device__ __forceinline__ float io_value(const void *p, int dtype, int64_t i) {
    if (dtype == QWFN_SRC_F32) return ((const float *)p)[i];
    const uint16_t h = ((const uint16_t *)p)[i];
    return dtype == QWFN_SRC_F16 ? h2f(h) : __uint_as_float((uint32_t)h << 16);
}
__device__ __forceinline__ void put_io_value(void *p, int dtype, int64_t i, float y) {
    if (dtype == QWFN_SRC_F32) ((float *)p)[i] = y;
    else if (dtype == QWFN_SRC_F16) ((uint16_t *)p)[i] = f2h(y);
    else ((__bf16 *)p)[i] = (__bf16)y;
}

}  // namespace

// One workgroup a (row, query head): tiles of 64 cells, the running maximum and
// sum over them, thread d the output's dimension d.
__global__ void __launch_bounds__(256)
k_window(Geo g, qwfn_kv_view v, WinArg wa) {
    __shared__ float part[4][64], p[64], qs[256];
    const int row = blockIdx.x, h = blockIdx.y, gh = h / g.G, tid = threadIdx.x;
    int s = row, len, first = 0, n_q = 1;
    if (wa.q_start) {                       // the last sequence that starts at or before the row
        int lo = 0, hi = wa.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (wa.q_start[mid] <= row) lo = mid; else hi = mid - 1;
        }
        s = lo;
        first = wa.q_start[s];
        n_q = wa.q_start[s + 1] - first;
        if (row < first || row >= first + n_q) return;          // behind the last sequence
    } else {
        first = row;
    }
    len = wa.seq_len[s];
    const int64_t o = ((int64_t)row * g.H + h) * g.hd;
    const bool bad = len < 0 || len > wa.max_seq_len || n_q > len + (wa.q_start ? 0 : 1) || n_q > wa.max_q;
    if (bad || len == 0) {
        for (int d = tid; d < g.hd; d += 256) put_io_value(wa.out, wa.dtype, o + d, 0.0f);
        if (bad && tid == 0 && h == 0) set_status(v.status, QWFN_STATUS_LEN_RANGE);
        return;
    }
    const int pos = len - n_q + row - first;
    for (int d = tid; d < g.hd; d += 256) qs[d] = io_value(wa.q, wa.dtype, o + d) * g.scale_log2;
    const int lo = pos - wa.window + 1 > 0 ? pos - wa.window + 1 : 0;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int t0 = 0; t0 <= pos; t0 += 64) {
        if (t0 >= wa.sinks && t0 + 64 <= lo) { t0 = lo / 64 * 64 - 64; continue; }
        __syncthreads();
        const int32_t pp = phys_page(g, v.page_table, s, t0);
        if (pp < 0) { if (tid == 0) set_status(v.status, QWFN_STATUS_PAGE_RANGE); continue; }
        const uint8_t *kp = (const uint8_t *)v.k_pages + (int64_t)pp * g.page_bytes;
        const uint8_t *vp = (const uint8_t *)v.v_pages + (int64_t)pp * g.page_bytes;
        const int c = tid & 63, w = tid >> 6, n = g.hd / 4;
        float x = 0.0f;
        for (int d = w * n; d < (w + 1) * n; ++d) x += qs[d] * member_k(g, kp, gh, (t0 + c) % g.pt, d);
        part[w][c] = x;
        __syncthreads();
        const int t = t0 + c;
        const bool seen = t <= pos && (t >= lo || t < wa.sinks);
        x = seen ? (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]) : -INFINITY;
        const float mt = fmaxf(m, wave_max(x));
        const float f = m == -INFINITY ? 0.0f : exp2f(m - mt), e = seen ? exp2f(x - mt) : 0.0f;
        l = l * f + wave_sum(e);
        m = mt;
        if (w == 0) p[c] = e;
        __syncthreads();
        acc *= f;
        if (tid < g.hd)
            for (int i = 0; i < 64; ++i) {
                const int ti = t0 + i;
                if (ti <= pos && (ti >= lo || ti < wa.sinks)) acc += p[i] * member_k(g, vp, gh, ti % g.pt, tid, true);
            }
    }
    if (tid < g.hd) put_io_value(wa.out, wa.dtype, o + tid, l != 0.0f ? acc / l : 0.0f);
}

size_t window_ws_bytes(const Geo &g, const WinPlan &p) { return p.prefill ? 256 : win_dec_ws_bytes(g, p); }

hipError_t launch_window(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, const WinPlan &p, void *ws,
                         hipStream_t st) {
    if (!p.prefill) return launch_win_dec(g, v, wa, p, ws, st);
    hipLaunchKernelGGL(k_window, dim3((unsigned)p.n_rows, (unsigned)g.H), dim3(256), 0, st, g, v, wa);
    return hipGetLastError();
}

}  // namespace qwfn_qsa
