// qsa_window.hip -- attention with a sliding window and a few first tokens that
// stay visible, over the paged cache (qwfn_window_attn_prefill; the single-token
// kernels are in qsa_window_dec.hip).
//
// Mathematics.  The query at position p of a sequence sees the cells t <= p with
// t > p - window or t < sinks; o = sum_t 2^(s_t - r) v_t / sum_t 2^(s_t - r), s = q.k
// log2(e) / sqrt(hd), r a running reference near the largest visible s, one pass
// over the cells.
//
// k_win_stage brings the cells that a call's queries see into matrix-core operands
// once: each would otherwise be unpacked by every block of queries that sees it (a
// block of 16 queries a time at 8 heads a KV head, so 256 times for a window of
// 4,096).  k_win_rows walks a block of rows (query x head of one KV head) over its
// tiles:
//   S^T = K Q^T on v_mfma_f32_32x32x16_f16, A = 32 cells, columns = 32 rows;
//   O^T = V^T P^T, the accumulator layout of S^T being (with V's cells staged in its
//     order) the operand layout of P^T, so weights never leave their lane.
//
// Measured (MI355X): 8,192 bfloat16 queries over windows of 4,096 and 64 first tokens (279 GFLOP):
// k_win_rows 293-325 us, 870-950 TFLOP/s of the 1,215 that a large fp16 product reaches here (the
// clock falls to 1.9 GHz under either), MFMA busy 52 %, VALU 47 %; k_win_stage 10 us.  3,001 float32
// queries from nothing (three products for each): 88 us, the CUs that hold two workgroups.  Computing
// the next step's logits under a step's exponentials (two K tiles ahead, scheduled by groups) took 60
// registers more and measured the same; steps of 32 cells at three workgroups a CU 360 us, as 1,024
// workgroups are then one round and a third.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "qsa_append.h"
#include "qsa_window.h"

namespace qwfn_qsa {

typedef float f16v __attribute__((ext_vector_type(16)));

namespace {

// A staged tile of 64 cells of one KV head, NP planes (fp16, or fp16 hi and lo):
//   K [plane][hd / 8][64 cells][8 dims]
//   V [plane][64 / 16][2][hd][8 cells]: cells 16 ks + 4 half + {0 .. 3, 8 .. 11}
template <int HD, int NP> constexpr int staged_half() { return NP * 64 * HD * 2; }     // bytes of K, or of V
// What the rows' kernel needs to know of a tile: values are staged times 2^ke, 2^ve.
struct TileInfo {
    int32_t ke, ve;
    int32_t there;          // the tile's page is in the pool
    int32_t odd;            // V holds values that are not finite: staged as 0, their bits in OddBits
};
// Where an odd tile's V is not finite: bit d % 32 of word [cell][d / 32].
template <int HD> constexpr int odd_words() { return 64 * HD / 32; }

// A plan's staging area: tiles [n_seq][Hkv][cap], their TileInfo, then the parts.
struct PfLayout {
    int cap, parts, blocks;
    size_t info, odd, part_o, part_rl, total;
};

constexpr int kEighths = 1024;   // workgroups from which neighbouring blocks share an XCD (340 against 351 us at 1,024)
constexpr int kExact = 2;   // planes of float32 and float16 rows

// The sequence's queries and length, and whether they can be served.
struct PfSeq { int start, n_q, len; bool ok; };
__device__ __forceinline__ PfSeq pf_seq(const WinArg &wa, int s) {
    PfSeq q;
    q.start = wa.q_start[s];
    q.n_q = wa.q_start[s + 1] - q.start;
    q.len = wa.seq_len[s];
    if (q.start < 0 || q.n_q < 0 || q.n_q > wa.n_rows - q.start) { q.n_q = 0; q.ok = false; return q; }
    q.ok = q.len >= 0 && q.len <= wa.max_seq_len && q.n_q <= q.len && q.n_q <= wa.max_q;
    return q;
}

// Whether the query at pos sees cell t0 + c: c against three numbers, so that a lane holds no
// cell indices.
struct Seen {
    int last, before, sinks;
    __device__ __forceinline__ Seen(int pos, int window, int sink_tokens, int t0)
        : last(pos - t0), before(pos - window - t0), sinks(sink_tokens - t0) {}
    __device__ __forceinline__ bool operator()(int c) const { return c <= last && (c > before || c < sinks); }
};

// The order of a run of N products whose operand (NP planes) comes from LDS: reads kAhead
// products ahead.  Left to itself the compiler reads each operand where it is used, and its LDS
// latency (some 130 cycles) shows between the products.
template <int NP, int N>
__device__ __forceinline__ void lds_ahead() {
    constexpr int kAhead = N < 4 ? N : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead * NP, 0);                    // LDS reads
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, NP == 2 ? 3 : 1, 0);            // MFMA
        if (i + kAhead < N) __builtin_amdgcn_sched_group_barrier(0x100, NP, 0);
    }
}

// e with |x| 2^e < 2^15 for |x| <= m, in steps, so that neighbouring tiles mostly share it
// (a change costs the rows' kernel a pass over its sums).  fp16's absolute half step 2^-25 is
// then small against the tile's largest value: one plane, 0 while m is in [2^-4, 2^15), so
// 2^-21 of m; two planes, multiples of 8, which leave m >= 2^7, so 2^-32.
template <int NP>
__device__ __forceinline__ int stage_exp(float m) {
    const int e = m == 0.0f ? 0 : pow2_to(m, 14);
    return NP == 2 ? e & ~7 : m >= 0.0625f && m < 32768.0f ? 0 : e;
}

}  // namespace

// grid (tile slots, Hkv, n_seq): slot i of a sequence's list of tiles into its place.  Bound by its
// chain of loads (the sequence, the page, the tile): 8 to 10 us from 100 tiles to 400.
template <int HD, int KT, bool VD, int NP>
__global__ void __launch_bounds__(256)
k_win_stage(Geo g, qwfn_kv_view v, WinArg wa, int cap, uint8_t *staged, TileInfo *info,
            uint32_t *odd_bits) {
    constexpr int NB = HD / 32, C8 = HD / 8, kRow = HD + 8;
    __shared__ float dk[64][NB + 1], dv[64][NB + 1];
    __shared__ float red[2][4];
    __shared__ __attribute__((aligned(16))) uint16_t vt[VD ? 1 : 64][VD ? 8 : kRow];
    const int slot = blockIdx.x, gh = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const PfSeq q = pf_seq(wa, s);
    if (!q.ok) {
        if (slot == 0 && gh == 0 && tid == 0) set_status(v.status, QWFN_STATUS_LEN_RANGE);
        return;
    }
    if (q.n_q == 0) return;
    const WinTiles tl = win_tiles(q.len, q.n_q, wa.window, wa.sinks);
    if (slot >= tl.n || slot >= cap) return;
    const int t0 = tl.cell(slot);
    const int64_t at = ((int64_t)s * g.Hkv + gh) * cap + slot;
    const int32_t pp = phys_page(g, v.page_table, s, t0);
    if (pp < 0) {
        if (tid == 0) {
            info[at] = TileInfo{0, 0, 0, 0};
            set_status(v.status, QWFN_STATUS_PAGE_RANGE);
        }
        return;
    }
    const int64_t tile = (int64_t)pp * g.page_bytes + (int64_t)(gh * (g.pt / 64) + t0 % g.pt / 64) * g.chunks * 1024;
    const uint8_t *kq = (const uint8_t *)v.k_pages + tile, *vq = (const uint8_t *)v.v_pages + tile;
    const int live = q.len - t0;                          // cells of the tile that are written
    // ---- every piece the thread converts, in flight before the scales are waited for ----
    // item i of K (and of V in a K layout): dims 8 (i / 64) .. of cell i % 64; of a dimension-major V: cells
    // c0 .. c0 + 3 and c0 + 8 .. c0 + 11 of dim i % HD
    constexpr int N = HD / 32;                            // items a thread: tid + 256 n
    using Piece = std::conditional_t<KT == QWFN_KV_F16, u4v, uint2>;
    Piece kr[N], vr[N];
    auto piece = [&](const uint8_t *tq, int i) {
        const int c8 = i >> 6, cell = i & 63;
        if constexpr (KT == QWFN_KV_F16) return *reinterpret_cast<const u4v *>(tq + c8 * 1024 + cell * 16);
        else if constexpr (KT == QWFN_KV_Q4_0) return *reinterpret_cast<const uint2 *>(tq + (c8 / 4) * 1024 + cell * 16 + (c8 & 1) * 8);
        else return *reinterpret_cast<const uint2 *>(tq + (c8 / 2) * 1024 + cell * 16 + (c8 & 1) * 8);
    };
    auto cell0 = [](int i) { return i / HD / 2 * 16 + (i / HD & 1) * 4; };
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = tid + 256 * n;
        kr[n] = piece(kq, i);
        if constexpr (VD) {
            const uint8_t *p = vq + i % HD * 64 + cell0(i);
            vr[n] = make_uint2(*reinterpret_cast<const uint32_t *>(p), *reinterpret_cast<const uint32_t *>(p + 8));
        } else {
            vr[n] = piece(vq, i);
        }
    }
    // ---- the scales, and the exponents they ask for ----
    int ke = 0, ve = 0;
    if constexpr (KT != QWFN_KV_F16) {
        const int64_t so = (int64_t)pp * g.page_bytes + g.qbytes + (int64_t)(gh * g.pt + t0 % g.pt) * (NB * 2);
        const uint16_t *ks = reinterpret_cast<const uint16_t *>((const uint8_t *)v.k_pages + so);
        const uint16_t *vs = reinterpret_cast<const uint16_t *>((const uint8_t *)v.v_pages + so);
        float mk = 0.0f, mv = 0.0f;
        for (int i = tid; i < 64 * NB; i += 256) {
            const float a = i / NB < live ? h2f(ks[i]) : 0.0f, b = i / NB < live ? h2f(vs[i]) : 0.0f;
            dk[i / NB][i % NB] = a;
            dv[i / NB][i % NB] = b;
            mk = fabsf(a) < INFINITY ? fmaxf(mk, fabsf(a)) : mk;
            mv = fabsf(b) < INFINITY ? fmaxf(mv, fabsf(b)) : mv;
        }
        mk = wave_max(mk);
        mv = wave_max(mv);
        if ((tid & 63) == 0) { red[0][tid >> 6] = mk; red[1][tid >> 6] = mv; }
        __syncthreads();
        constexpr float kTop = KT == QWFN_KV_Q4_0 ? 8.0f : 128.0f;
        ke = stage_exp<NP>(kTop * fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])));
        ve = stage_exp<NP>(kTop * fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3])));
    }
    const float fk = ldexpf(1.0f, ke), fv = ldexpf(1.0f, ve);
    uint8_t *out = staged + at * (2 * staged_half<HD, NP>());
    // the eight values of a K-layout piece, times the exponent's power of two
    auto eight = [&](Piece w, const float (*d)[NB + 1], int i, float f, float *x) {
        const int c8 = i >> 6, cell = i & 63;
        if constexpr (KT == QWFN_KV_F16) {
#pragma unroll
            for (int k = 0; k < 4; ++k) { x[2 * k] = h2f((uint16_t)w[k]); x[2 * k + 1] = h2f((uint16_t)(w[k] >> 16)); }
            if (cell >= live)
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = 0.0f;
        } else {
            const float dd = d[cell][c8 / 4] * f;
            const int sh = c8 & 2 ? 4 : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t u = (k < 4 ? w.x : w.y) >> (8 * (k & 3));
                x[k] = dd * (KT == QWFN_KV_Q4_0 ? (float)((int)(u >> sh & 15) - 8) : (float)(int8_t)u);
            }
        }
    };
    // plane p of a value: its fp16, or what the fp16 leaves
    auto plane = [&](float x, int p) {
        const _Float16 h = (_Float16)x;
        return p == 0 ? h : (_Float16)(x - (float)h);
    };
    int odd = 0;
    // a V value, 0 in place of one that is not finite: a row that does not see it multiplies it by 0
    auto finite = [&](float x) {
        const bool fin = fabsf(x) < INFINITY;
        odd |= !fin;
        return fin ? x : 0.0f;
    };
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = tid + 256 * n;
        float x[8];
        eight(kr[n], dk, i, fk, x);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            h8v y;
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = plane(x[k], p);
            *reinterpret_cast<h8v *>(out + (p * C8 * 64 + i) * 16) = y;
        }
    }
    out += staged_half<HD, NP>();
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        if constexpr (!VD) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int i = tid + 256 * n;
                float x[8];
                eight(vr[n], dv, i, fv, x);
                h8v y;
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = plane(finite(x[k]), p);
                *reinterpret_cast<h8v *>(&vt[i & 63][(i >> 6) * 8]) = y;
            }
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = tid + 256 * n, dim = i % HD, c0 = cell0(i);           // i = (ks * 2 + half) * HD + dim
            h8v y;
            if constexpr (VD) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int cell = c0 + (k < 4 ? k : k + 4);
                    y[k] = plane(finite(dv[cell][dim / 32] * fv * (float)(int8_t)((k < 4 ? vr[n].x : vr[n].y) >> (8 * (k & 3)))), p);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = __builtin_bit_cast(_Float16, vt[c0 + (k < 4 ? k : k + 4)][dim]);
            }
            *reinterpret_cast<h8v *>(out + (p * HD * 8 + i) * 16) = y;
        }
    }
    odd = __syncthreads_or(odd);
    if (odd)
        for (int i = tid; i < odd_words<HD>(); i += 256) {
            uint32_t bits = 0;
            for (int d = 0; d < 32; ++d)
                bits |= (uint32_t)(i / NB < live && !(fabsf(member_k(g, (const uint8_t *)v.v_pages + (int64_t)pp * g.page_bytes, gh,
                                                                     t0 % g.pt + i / NB, i % NB * 32 + d, true)) < INFINITY)) << d;
            odd_bits[at * odd_words<HD>() + i] = bits;
        }
    if (tid == 0) info[at] = TileInfo{ke, ve, 1, odd};
}

// Four waves of 32 rows each; row = query * G + head of the KV head's group.  TC cells a
// step, double-buffered in LDS.  One-dimensional grid over blocks * parts * Hkv: a workgroup's
// XCD is its index modulo 8, and each XCD takes a run of neighbouring blocks of one KV head,
// whose windows overlap and fit its L2 (4 MB).
template <int HD, int NP, int TC>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2)
k_win_rows(Geo g, qwfn_kv_view v, WinArg wa, int cap, int blocks, int parts, const uint8_t *staged, const TileInfo *info,
           const uint32_t *odd_bits, float *part_o, float2 *part_rl) {
    constexpr int KS = HD / 16, DT = HD / 32, CT = TC / 32, kRows = 128;
    constexpr int kHalf = NP * TC * HD * 2, kStep = 2 * kHalf;            // bytes of K (or V), of both
    constexpr float kOff = NP == 2 ? 13.0f : 6.0f, kSlack = NP == 2 ? 2.0f : 8.0f;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, half = lane >> 5;
    // one more block a sequence than whole ones.  More than the device holds at once: each XCD an
    // eighth of them, by heads and rows.  Fewer: the last rows of all heads first, as the first
    // ones see less (a compute unit's second workgroup is then a short one: 102 -> 90 us at 3,001
    // float32 queries from nothing)
    int id = (int)blockIdx.x, gh, part, blk;
    if (blocks * parts * g.Hkv >= kEighths) {
        const int full = blocks - wa.n_seq, n_full = full * parts * g.Hkv, tail = id >= n_full;
        if (tail) id -= n_full;
        else if (id < n_full / 8 * 8) id = id % 8 * (n_full / 8) + id / 8;
        const int per = tail ? wa.n_seq : full;
        gh = id / (per * parts), part = id % parts, blk = id / parts % per + (tail ? full : 0);
    } else {
        gh = id % g.Hkv, part = id / g.Hkv % parts, blk = blocks - 1 - id / (g.Hkv * parts);
    }
    // the block's sequence: blocks of sequence s start at q_start[s] * G / kRows + s
    int s = 0;
    for (int hi = wa.n_seq - 1; s < hi;) {
        const int mid = (s + hi + 1) / 2;
        if ((int64_t)wa.q_start[mid] * g.G / kRows + mid <= blk) s = mid; else hi = mid - 1;
    }
    const PfSeq q = pf_seq(wa, s);
    const int64_t r0 = (blk - ((int64_t)q.start * g.G / kRows + s)) * kRows;
    const int64_t total = (int64_t)q.n_q * g.G;
    if (r0 < 0 || r0 >= total) return;
    const int base = q.len - q.n_q;                       // position of the sequence's first query

    // ---- the rows' queries ----
    h8v qf[NP][KS];
    const int64_t rr = r0 + w * 32 + n;
    const bool row = rr < total;
    const int qi = (int)(rr / g.G), pos = base + (row ? qi : q.n_q - 1);
    const int64_t io = (((int64_t)q.start + qi) * g.H + gh * g.G + (int)(rr % g.G)) * HD;     // the row's first value
    float c0;
    {
        float x[KS][8], m = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if (row) {
                load8(wa.q, wa.dtype, io + 16 * k + 8 * half, x[k]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[k][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[k][j]));
        }
        const int e = pow2_to(swap32_op(m, [](float a, float c) { return fmaxf(a, c); }), 13);
        const float f = ldexpf(1.0f, e);
        c0 = ldexpf(g.scale_log2, -e);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[k][j] * f;
                qf[0][k][j] = (_Float16)y;
                if constexpr (NP == 2) qf[NP - 1][k][j] = (_Float16)(y - (float)(_Float16)y);
            }
    }

    // ---- its tiles: first tokens' tiles before the window, then the window's ----
    const WinTiles tl = win_tiles(q.ok ? q.len : 0, q.n_q, wa.window, wa.sinks);
    const int p_lo = base + (int)(r0 / g.G), p_hi = base + (int)((min(r0 + kRows, total) - 1) / g.G);
    const int wt = max(0, p_lo - wa.window + 1) / 64;
    const int n1 = min(min(wa.sinks, p_hi + 1) / 64 + (min(wa.sinks, p_hi + 1) % 64 ? 1 : 0), wt);
    const int nt = q.ok ? (n1 + p_hi / 64 + 1 - wt) * (64 / TC) : 0;
    const int k0 = (int)((int64_t)nt * part / parts), k1 = (int)((int64_t)nt * (part + 1) / parts);
    const int64_t first = ((int64_t)s * g.Hkv + gh) * cap;
    auto cell_of = [&](int k) { const int t = k / (64 / TC); return (t < n1 ? t : wt + t - n1) * 64 + k % (64 / TC) * TC; };
    auto slot_of = [&](int cell) { const int t = cell / 64; return t < tl.ns ? t : tl.ns + t - tl.w0; };
    // one step's K and V, 16 bytes a lane, into buffer k & 1.  The wave's transfers of 1 KiB differ
    // by uniform offsets alone, so each costs no vector register: K [plane][chunk][TC][8] is runs of
    // TC cells of the tile's 64, V [plane][TC / 16][2][HD][8] is one run a plane.
    const uint32_t lane_k = lane / TC * 1024 + lane % TC * 16, lane_v = lane * 16;
    auto fetch = [&](int k) {
        const int cell = cell_of(k), sub = cell % 64;
        const uint8_t *src = staged + (first + slot_of(cell)) * (int64_t)(2 * staged_half<HD, NP>());
        const uint32_t dst = (uint32_t)(uintptr_t)lds + (k & 1) * kStep;
#pragma unroll
        for (int i = 0; i < kHalf / 4096; ++i) {
            const int at = (i * 4 + w) * 1024;            // LDS bytes of the wave's transfer
            lds_dma16_sv(src + at / (TC * 16) * 1024 + sub * 16, lane_k, dst + at);
        }
#pragma unroll
        for (int i = 0; i < kHalf / 4096; ++i) {
            const int at = (i * 4 + w) * 1024, pl = at / (TC * HD * 2);
            lds_dma16_sv(src + staged_half<HD, NP>() + pl * (64 - TC) * HD * 2 + sub * HD * 2 + at, lane_v, dst + kHalf + at);
        }
    };
    // (through the scalar cache: a vector load would wait for the transfers issued before it)
    auto info_of = [&](int k) {
        typedef const __attribute__((address_space(4))) int32_t *Const;
        const Const p = (Const)(uintptr_t)(info + first + slot_of(cell_of(k)));
        return TileInfo{p[0], p[1], p[2], p[3]};
    };

    f16v o[DT];
    float r = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    int ve = 0, any_odd = 0;
    // the wave's own range of positions, for the masks
    const int64_t rw = min(r0 + w * 32, total - 1);
    const int pw_lo = base + (int)(rw / g.G), pw_hi = base + (int)(min(r0 + w * 32 + 31, total - 1) / g.G);

    TileInfo next{0, 0, 0, 0};
    if (k0 < k1) {
        fetch(k0);
        next = info_of(k0);
    }
    for (int k = k0; k < k1; ++k) {
        wait_vmem_all();
        __syncthreads();
        if (k + 1 < k1) fetch(k + 1);
        const int t0 = cell_of(k);
        const TileInfo ti = next;
        if (k + 1 < k1) next = info_of(k + 1);
        if (!ti.there) continue;
        any_odd |= ti.odd;
        const uint8_t *kb = lds + (k & 1) * kStep, *vb = kb + kHalf;
        if (ti.ve != ve) {                                // V in other units from here on
            const float f = ldexpf(1.0f, ti.ve - ve);
            ve = ti.ve;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
        // ---- S^T; the matrix halves go before the other wave's vector half (340 -> 322 us) ----
        __builtin_amdgcn_s_setprio(1);
        f16v x[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[c][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                h8v a[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    a[p] = *reinterpret_cast<const h8v *>(kb + p * (TC * HD * 2) + ((2 * ks + half) * TC + c * 32 + n) * 16);
                if constexpr (NP == 2) {
                    x[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], qf[0][ks], x[c], 0, 0, 0);
                    x[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], qf[1][ks], x[c], 0, 0, 0);
                }
                x[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], qf[0][ks], x[c], 0, 0, 0);
            }
        }
        lds_ahead<NP, CT * KS>();
        __builtin_amdgcn_s_setprio(0);
        // ---- masks, the running reference, the weights ----
        const bool whole = t0 + TC - 1 <= pw_lo && (t0 > pw_hi - wa.window || t0 + TC <= wa.sinks);
        if (!whole) {
            const Seen see(pos, wa.window, wa.sinks, t0 + 4 * half);
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    x[c][i] = see(c * 32 + 8 * (i >> 2) + (i & 3)) ? x[c][i] : -INFINITY;
        }
        float mx = x[0][0];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[c][i]);
        mx = swap32_op(mx, [](float p, float q2) { return fmaxf(p, q2); });
        const float cs = ldexpf(c0, -ti.ke), want = mx * cs - kOff;
        if (__any(want > r + kSlack)) {
            const float rn = fmaxf(r, want), f = __builtin_amdgcn_exp2f(r - (rn == -INFINITY ? 0.0f : rn));
            r = rn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
        const float ref = r == -INFINITY ? 0.0f : r;
        h8v pf[NP][CT * 2];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(x[c][i], cs, -ref));
                l += e;
                pf[0][2 * c + (i >> 3)][i & 7] = (_Float16)e;
                if constexpr (NP == 2) pf[NP - 1][2 * c + (i >> 3)][i & 7] = (_Float16)(e - (float)(_Float16)e);
            }
        // ---- O^T ----
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int ks = 0; ks < TC / 16; ++ks) {
                h8v a[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    a[p] = *reinterpret_cast<const h8v *>(vb + p * (TC * HD * 2) + ((2 * ks + half) * HD + 32 * d + n) * 16);
                if constexpr (NP == 2) {
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], pf[0][ks], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], pf[1][ks], o[d], 0, 0, 0);
                }
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], pf[0][ks], o[d], 0, 0, 0);
            }
        lds_ahead<NP, DT * TC / 16>();
        __builtin_amdgcn_s_setprio(0);
    }
    // ---- values that are not finite: a row that sees one gets a NaN there ----
    for (int k = k0; any_odd && k < k1; ++k) {
        const TileInfo ti = info_of(k);
        if (!ti.there || !ti.odd) continue;
        const int t0 = cell_of(k);
        const uint32_t *bits = odd_bits + (first + slot_of(t0)) * odd_words<HD>() + t0 % 64 * DT;
#pragma unroll 1
        for (int c = 0; c < TC; ++c)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint32_t m = bits[c * DT + d] >> (4 * half);
                if (m == 0) continue;
                const bool see = Seen(pos, wa.window, wa.sinks, t0)(c);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = see && (m >> (8 * (i >> 2) + (i & 3)) & 1) ? NAN : o[d][i];
            }
    }

    // ---- out ----
    const float ls = swap32_op(l, [](float p, float q2) { return p + q2; });
    if (!row) return;
    const float f = ldexpf(1.0f, -ve) * (parts == 1 ? (ls != 0.0f ? 1.0f / ls : 0.0f) : 1.0f);
    const int64_t pr = ((((int64_t)q.start + qi) * g.Hkv + gh) * parts + part) * g.G + rr % g.G;
    if (parts > 1 && half == 0) part_rl[pr] = make_float2(r, ls);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f4v y = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            y *= f;
            const int at = 32 * d + 8 * i + 4 * half;
            if (parts > 1) *reinterpret_cast<f4v *>(part_o + pr * HD + at) = y;
            else store4(wa.out, wa.dtype, io + at, y);
        }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

static int planes(const WinPlan &p) { return p.dtype == QWFN_SRC_BF16 ? 1 : kExact; }
static constexpr int rows_a_block() { return 128; }

static PfLayout pf_layout(const Geo &g, const WinPlan &p) {
    PfLayout l;
    const int rows = rows_a_block();
    l.cap = win_most_tiles(p);
    const int64_t blocks = (int64_t)p.n_rows * g.G / rows + p.n_seq;
    l.blocks = (int)blocks;
    // few blocks: their tiles over several workgroups, at least two tiles each
    const int64_t wgs = blocks * g.Hkv;
    l.parts = (int)std::max<int64_t>(1, std::min<int64_t>({l.cap / 2, 512 / wgs, kWinMostParts}));
    size_t off = win_align((size_t)p.n_seq * g.Hkv * l.cap * (size_t)(planes(p) * 64 * g.hd * 2) * 2);
    auto take = [&](size_t bytes) { const size_t o = off; off = win_align(off + bytes); return o; };
    l.info = take((size_t)p.n_seq * g.Hkv * l.cap * sizeof(TileInfo));
    l.odd = take((size_t)p.n_seq * g.Hkv * l.cap * (64 * g.hd / 32) * sizeof(uint32_t));
    const size_t pr = l.parts > 1 ? (size_t)p.n_rows * g.Hkv * l.parts * g.G : 0;
    l.part_o = take(pr * g.hd * sizeof(float));
    l.part_rl = take(pr * sizeof(float2));
    l.total = off;
    return l;
}

template <int HD, int KT, bool VD, int NP>
static void stage_t(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, const PfLayout &l, uint8_t *ws, hipStream_t st) {
    hipLaunchKernelGGL((k_win_stage<HD, KT, VD, NP>), dim3((unsigned)l.cap, (unsigned)g.Hkv, (unsigned)wa.n_seq), dim3(256),
                       0, st, g, v, wa, l.cap, ws, (TileInfo *)(ws + l.info), (uint32_t *)(ws + l.odd));
}

template <int HD, int NP, int TC>
static hipError_t prefill_t(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, const PfLayout &l, uint8_t *ws, hipStream_t st) {
    if (g.kt == QWFN_KV_Q4_0) stage_t<HD, QWFN_KV_Q4_0, false, NP>(g, v, wa, l, ws, st);
    else if (g.kt == QWFN_KV_F16) stage_t<HD, QWFN_KV_F16, false, NP>(g, v, wa, l, ws, st);
    else if (g.vdim) stage_t<HD, QWFN_KV_Q8_0, true, NP>(g, v, wa, l, ws, st);
    else stage_t<HD, QWFN_KV_Q8_0, false, NP>(g, v, wa, l, ws, st);
    constexpr int kLds = 2 * 2 * NP * TC * HD * 2;
    const hipError_t e = hipFuncSetAttribute((const void *)k_win_rows<HD, NP, TC>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_win_rows<HD, NP, TC>), dim3((unsigned)(l.blocks * l.parts * g.Hkv)), dim3(256), kLds, st, g, v, wa, l.cap, l.blocks, l.parts, ws, (const TileInfo *)(ws + l.info), (const uint32_t *)(ws + l.odd), (float *)(ws + l.part_o),
                       (float2 *)(ws + l.part_rl));
    if (l.parts > 1) launch_win_merge(g, wa, l.parts, (const float *)(ws + l.part_o), (const float2 *)(ws + l.part_rl), st);
    return hipGetLastError();
}

// A query a sequence at most: the single-token kernels serve it.
static bool single(const WinPlan &p) { return !p.prefill || p.max_q == 1; }

size_t window_ws_bytes(const Geo &g, const WinPlan &p) { return single(p) ? win_dec_ws_bytes(g, p) : pf_layout(g, p).total; }

hipError_t launch_window(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, const WinPlan &p, void *ws,
                         hipStream_t st) {
    if (single(p)) return launch_win_dec(g, v, wa, p, ws, st);
    const PfLayout l = pf_layout(g, p);
    uint8_t *b = (uint8_t *)ws;
    const bool exact = planes(p) == kExact;
    switch (g.hd) {
    case 64: return exact ? prefill_t<64, 2, 64>(g, v, wa, l, b, st) : prefill_t<64, 1, 64>(g, v, wa, l, b, st);
    case 128: return exact ? prefill_t<128, 2, 32>(g, v, wa, l, b, st) : prefill_t<128, 1, 64>(g, v, wa, l, b, st);
    case 256: return exact ? prefill_t<256, 2, 32>(g, v, wa, l, b, st) : prefill_t<256, 1, 32>(g, v, wa, l, b, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace qwfn_qsa
