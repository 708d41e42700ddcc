// qsa_window_dec.hip -- sliding-window attention of one query a sequence
// (qwfn_window_attn_decode): k_win_dec, and k_win_merge, which joins the parts
// of a sequence's tiles.
//
// A wave walks 64-cell tiles of one (sequence, KV head); the group's query heads
// are the columns of v_mfma_f32_16x16x32_f16.  Lane l = 16 lg + hn.
//   QK: A = cells x 32 dims of one quantization block (quants exact in fp16), B =
//     the queries, each row scaled by a power of two and split into fp16 hi + lo;
//     the key's scale multiplies the block's product in fp32.  Row 4 lg + i of
//     cell group cg is the tile's cell 16 lg + 4 cg + i, so a lane ends with the
//     logits of the 16 cells 16 lg .. 16 lg + 15 for its column, which are both
//     its k-elements of the PV operand and 16 contiguous bytes of a V row.
//   PV: A = 16 dims x 32 cells of V, B = weight x V scale, as fp16 hi + lo.
// LOC (groups of up to 8 heads): the low halves are columns 8 .. 15 of the same
// product, and the two halves of a column are added by one DPP step, so hi + lo
// cost no second MFMA.
// Weights are e^(s - r) with r at least max(s) + log2(V scale bound) - 14: the fp16
// products stay below 2^14 and keep 22 bits down to 2^-38 of the largest.
//
// Measured (MI355X): 64 sequences of up to 4,160 cells, q8_0, 2 x 128 KV heads: 39.7 us for 135 MB,
// 3.4 TB/s of the 5.2 that a large copy reaches.  The waves' tiles come in whole rounds (up to 5 for
// 3.8 on average) and a round waits for its loads: VALU active 34 %, 1,045 instructions a tile.
// Workgroups for two a CU: three, four and six a CU measured 46, 47 and 50 us.  One sequence over
// 1,024 cells: 8.5 us, a chain of dependent loads (length, page, tile), one tile a wave, then the
// merge's 3.2 us.  A tile held ahead in registers needs heads of at most 128 values.
#include <hip/hip_runtime.h>

#include "qsa_append.h"
#include "qsa_window.h"

namespace qwfn_qsa {

namespace {

// One tile's registers.  K: 8-byte (q8_0, q4_0: 8 dims, or 8 bytes of nibbles) or
// 16-byte (F16: 8 dims) pieces of cell 16 (hn / 4) + 4 cg + hn % 4.
template <int KT> struct KPiece { using T = uint2; };
template <> struct KPiece<QWFN_KV_F16> { using T = u4v; };

template <int HD, int KT>
struct KTile {
    typename KPiece<KT>::T k[4][HD / 32];
    u4v sc[KT == QWFN_KV_F16 ? 1 : HD / 16];            // the scales of cells 16 lg .. 16 lg + 15
};
// V: dim-major (VD), dims 16 dt + hn's cells 16 lg ..; else the chunks of cells 2 p, 2 p + 1
// (p = lane % 32), those of the lane's parity.
template <int HD, int KT, bool VD> constexpr int v_chunks() {
    return VD ? HD / 16 : (KT == QWFN_KV_F16 ? HD / 8 : KT == QWFN_KV_Q4_0 ? HD / 32 : HD / 16) / 2 * 2;
}
template <int HD, int KT, bool VD>
struct VTile {
    u4v v[v_chunks<HD, KT, VD>()];
    u4v sc[KT == QWFN_KV_F16 ? 1 : HD / 16];
};

template <int HD, int KT>
__device__ __forceinline__ void load_k(KTile<HD, KT> &t, const uint8_t *q, const uint8_t *sc, int hn, int lg) {
#pragma unroll
    for (int cg = 0; cg < 4; ++cg) {
        const int cell = 16 * (hn >> 2) + 4 * cg + (hn & 3);
#pragma unroll
        for (int b = 0; b < HD / 32; ++b) {
            if constexpr (KT == QWFN_KV_F16)
                t.k[cg][b] = *reinterpret_cast<const u4v *>(q + (4 * b + lg) * 1024 + cell * 16);
            else if constexpr (KT == QWFN_KV_Q4_0)
                t.k[cg][b] = *reinterpret_cast<const uint2 *>(q + b * 1024 + cell * 16 + (lg & 1) * 8);
            else
                t.k[cg][b] = *reinterpret_cast<const uint2 *>(q + (2 * b + (lg >> 1)) * 1024 + cell * 16 + (lg & 1) * 8);
        }
    }
    if constexpr (KT != QWFN_KV_F16)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) t.sc[i] = *reinterpret_cast<const u4v *>(sc + lg * HD + i * 16);
}

template <int HD, int KT, bool VD>
__device__ __forceinline__ void load_v(VTile<HD, KT, VD> &t, const uint8_t *q, const uint8_t *sc, int lane) {
    constexpr int N = v_chunks<HD, KT, VD>();
    if constexpr (VD) {
#pragma unroll
        for (int dt = 0; dt < N; ++dt)
            t.v[dt] = *reinterpret_cast<const u4v *>(q + (16 * dt + (lane & 15)) * 64 + (lane >> 4) * 16);
    } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                t.v[2 * k + c] = *reinterpret_cast<const u4v *>(q + (2 * k + (lane >> 5)) * 1024 + (2 * (lane & 31) + c) * 16);
    }
    if constexpr (KT != QWFN_KV_F16)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) t.sc[i] = *reinterpret_cast<const u4v *>(sc + (lane >> 4) * HD + i * 16);
}

// Nibbles n of the low or high halves of 8 bytes -> n - 8 as exact fp16.
__device__ __forceinline__ h8v q4x8_to_h8(uint2 w, int shift) {
    const half2v bias = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    h8v r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t u = ((i ? w.y : w.x) >> shift) & 0x0F0F0F0Fu;
        const half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
        const half2v b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
        r[4 * i] = a[0]; r[4 * i + 1] = a[1]; r[4 * i + 2] = b[0]; r[4 * i + 3] = b[1];
    }
    return r;
}

template <int KT>
__device__ __forceinline__ h8v k_operand(typename KPiece<KT>::T w, int lg) {
    if constexpr (KT == QWFN_KV_F16) return __builtin_bit_cast(h8v, w);
    else if constexpr (KT == QWFN_KV_Q4_0) return q4x8_to_h8(w, lg >= 2 ? 4 : 0);
    else return q8x8_to_h8(w);
}

__device__ __forceinline__ uint32_t word(const u4v *a, int i) { return a[i >> 2][i & 3]; }

// The V tile of a K layout into LDS transposed: vt[dim][cell], rows of 72 halves.  A word
// holds cells 2 p and 2 p + 1 of one dim.
constexpr int kVtRow = 72;
template <int HD, int KT>
__device__ __forceinline__ void stage_v(const VTile<HD, KT, false> &t, uint32_t *vt, int lane, uint32_t keep) {
    const int p = lane & 31, h = lane >> 5;
    constexpr int N = v_chunks<HD, KT, false>() / 2;
    const half2v b8 = {(_Float16)-1152.0f, (_Float16)-1152.0f}, b4 = {(_Float16)-1032.0f, (_Float16)-1032.0f};
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const u4v x = t.v[2 * k], y = t.v[2 * k + 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (KT == QWFN_KV_F16) {
                const int d = (2 * k + h) * 8 + 2 * j;
                vt[d * (kVtRow / 2) + p] = __builtin_amdgcn_perm(y[j], x[j], 0x05040100u) & keep;
                vt[(d + 1) * (kVtRow / 2) + p] = __builtin_amdgcn_perm(y[j], x[j], 0x07060302u) & keep;
            } else if constexpr (KT == QWFN_KV_Q4_0) {
                const int d = (2 * k + h) * 32 + 4 * j;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = __builtin_amdgcn_perm(y[j], x[j], 0x0c040c00u + 0x00010001u * e);
                    vt[(d + e) * (kVtRow / 2) + p] =
                        __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (w & 0x000F000Fu) | 0x64006400u) + b4);
                    vt[(d + e + 16) * (kVtRow / 2) + p] =
                        __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (w >> 4 & 0x000F000Fu) | 0x64006400u) + b4);
                }
            } else {
                const int d = (2 * k + h) * 16 + 4 * j;
                const uint32_t xu = x[j] ^ 0x80808080u, yu = y[j] ^ 0x80808080u;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = __builtin_amdgcn_perm(yu, xu, 0x0c040c00u + 0x00010001u * e) | 0x64006400u;
                    vt[(d + e) * (kVtRow / 2) + p] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, w) + b8);
                }
            }
        }
    }
}

// hi and lo words of two weights (no V scales).
__device__ __forceinline__ void split2(float p0, float p1, uint32_t &hi, uint32_t &lo) {
    const half2v h = {(_Float16)p0, (_Float16)p1};
    const half2v l = {(_Float16)(p0 - (float)h[0]), (_Float16)(p1 - (float)h[1])};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ float ror8_add(float x) { return x + dppf<kDppRowRor8>(x, x); }

}  // namespace

// grid (parts, Hkv, n_seq), four waves; tile i of the sequence's list belongs to wave
// i % (4 parts) of them.  One part: the normalised output; else the part's (r, l) and
// unnormalised O.
template <int HD, int KT, bool VD, bool LOC>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2)
k_win_dec(Geo g, qwfn_kv_view v, WinArg wa, int parts, float *part_o, float2 *part_rl) {
    constexpr int NB = HD / 32, DT = HD / 16;
    constexpr int kVtBytes = VD ? 0 : HD * kVtRow * 2;
    constexpr int kOutBytes = (LOC ? 8 : 16) * HD * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4][kVtBytes > kOutBytes ? kVtBytes : kOutBytes];
    __shared__ float2 rl[4][16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hn = lane & 15, lg = lane >> 4, part = blockIdx.x, gh = blockIdx.y, s = blockIdx.z;
    const int head = LOC ? hn & 7 : hn;
    const bool low = LOC && hn >= 8;
    int row = s, rows = 1;
    const int len = wa.seq_len[s];
    bool bad = len < 0 || len > wa.max_seq_len;
    if (wa.q_start) {                                   // a row a sequence at most, anywhere
        row = wa.q_start[s];
        rows = wa.q_start[s + 1] - row;
        if (row < 0 || rows < 0 || rows > wa.n_rows - row) rows = 0, bad = true;
        bad = bad || rows > 1 || rows > len;
    }
    const WinTiles tl = win_tiles(bad ? 0 : len, 1, wa.window, wa.sinks);
    if (bad && part == 0 && gh == 0 && threadIdx.x == 0) set_status(v.status, QWFN_STATUS_LEN_RANGE);
    if (rows != 1) {                                    // none, or too many, which get zeros
        for (int64_t i = threadIdx.x; i < (int64_t)rows * g.G; i += 256) {
            const int64_t at = row + i / g.G;
            const int64_t pr = ((at * g.Hkv + gh) * parts + part) * g.G + i % g.G;
            if (parts > 1) part_rl[pr] = make_float2(-INFINITY, 0.0f);
            for (int d = 0; d < HD; d += 4) {
                if (parts > 1) *reinterpret_cast<f4v *>(part_o + pr * HD + d) = f4v{0, 0, 0, 0};
                else store4(wa.out, wa.dtype, (at * g.H + gh * g.G + i % g.G) * HD + d, f4v{0, 0, 0, 0});
            }
        }
        return;
    }

    // the column's query: a power of two brings its largest value to [2^13, 2^14), then hi (+ lo)
    h8v qh[NB], ql[LOC ? 1 : NB];
    float qscale;
    {
        float x[NB][8];
        const int64_t o = ((int64_t)row * g.H + gh * g.G + head) * HD;
        float m = 0.0f;
        if (head < g.G) {
#pragma unroll
            for (int b = 0; b < NB; ++b) load8(wa.q, wa.dtype, o + 32 * b + 8 * lg, x[b]);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[b][j] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[b][j]));
        const int e = pow2_to(col_max4(m), 13);
        const float f = ldexpf(1.0f, e);
        qscale = ldexpf(g.scale_log2, -e);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[b][j] * f;
                const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
                qh[b][j] = low ? lo : hi;
                if constexpr (!LOC) ql[b][j] = lo;
            }
    }

    const int step = 4 * parts;
    const int64_t tile_bytes = (int64_t)g.chunks * 1024;
    const int32_t *pt = v.page_table + (int64_t)s * g.pps;
    // tile i's page, or -1 past the list or for a page that is not there
    auto page_of = [&](int i) -> int32_t {
        if (i >= tl.n) return -1;
        const int t0 = tl.cell(i);
        const int32_t p = pt[t0 / g.pt];
        if (p >= 0 && p < g.n_phys) return p;
        if (lane == 0) set_status(v.status, QWFN_STATUS_PAGE_RANGE);
        return -1;
    };
    auto quants = [&](const void *pages, int32_t p, int t0) {
        return (const uint8_t *)pages + (int64_t)p * g.page_bytes + (gh * (g.pt / 64) + t0 % g.pt / 64) * tile_bytes;
    };
    auto scales = [&](const void *pages, int32_t p, int t0) {
        return (const uint8_t *)pages + (int64_t)p * g.page_bytes + g.qbytes + (int64_t)(gh * g.pt + t0 % g.pt) * (NB * 2);
    };
    // the next tile of the wave that is there
    auto next = [&](int i, int32_t &p) {
        p = -1;
        while (i < tl.n && (p = page_of(i)) < 0) i += step;
        return i;
    };

    f4v o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f4v{0, 0, 0, 0};
    float r = -INFINITY, l = 0.0f;
    KTile<HD, KT> kt;
    VTile<HD, KT, VD> vt;
    int32_t p;
    int i = next(part * 4 + w, p);
    // heads of 256 values: a tile's K, and after it its V, take the registers that the next tile
    // would be held in
    constexpr bool kAhead = HD < 256;
    if (kAhead && i < tl.n) {
        const int t0 = tl.cell(i);
        load_k<HD, KT>(kt, quants(v.k_pages, p, t0), scales(v.k_pages, p, t0), hn, lg);
        load_v<HD, KT, VD>(vt, quants(v.v_pages, p, t0), scales(v.v_pages, p, t0), lane);
    }
    while (i < tl.n) {
        const int t0 = tl.cell(i);
        int32_t pn;
        const int in = next(i + step, pn);
        const bool more = in < tl.n;
        const int tn = more ? tl.cell(in) : 0;
        // ---- QK ----
        if (!kAhead) load_k<HD, KT>(kt, quants(v.k_pages, p, t0), scales(v.k_pages, p, t0), hn, lg);
        float x[4][4];
#pragma unroll
        for (int cg = 0; cg < 4; ++cg) {
            f4v a = {0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const h8v ka = k_operand<KT>(kt.k[cg][b], lg);
                if constexpr (KT == QWFN_KV_F16) {
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[b], a, 0, 0, 0);
                    if constexpr (!LOC) a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[b], a, 0, 0, 0);
                } else {
                    f4v c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[b], f4v{0, 0, 0, 0}, 0, 0, 0);
                    if constexpr (!LOC) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[b], c, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int at = (4 * cg + j) * NB + b;
                        const uint32_t sw = word(kt.sc, at >> 1);
                        a[j] += c[j] * h2f((uint16_t)(at & 1 ? sw >> 16 : sw));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) x[cg][j] = (LOC ? ror8_add(a[j]) : a[j]) * qscale;
        }
        if (!kAhead) load_v<HD, KT, VD>(vt, quants(v.v_pages, p, t0), scales(v.v_pages, p, t0), lane);
        if (kAhead && more) load_k<HD, KT>(kt, quants(v.k_pages, pn, tn), scales(v.k_pages, pn, tn), hn, lg);
        // ---- the tile's edges ----
        uint32_t keep = 0xFFFFFFFFu;                    // F16 V: cells 2 p, 2 p + 1 of the staging lane
        if (!tl.whole(i, len)) {
            auto seen = [&](int c) { return tl.seen(t0 + c, len); };
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const bool on = seen(16 * lg + c);
                x[c >> 2][c & 3] = on ? x[c >> 2][c & 3] : -INFINITY;
                if constexpr (KT != QWFN_KV_F16)
#pragma unroll
                    for (int k = 0; k < NB / 2; ++k) {
                        const int at = c * (NB / 2) + k;
                        vt.sc[at >> 2][at & 3] = on ? vt.sc[at >> 2][at & 3] : 0u;
                    }
            }
            if constexpr (!VD && KT == QWFN_KV_F16)
                keep = (seen(2 * (lane & 31)) ? 0xFFFFu : 0u) | (seen(2 * (lane & 31) + 1) ? 0xFFFF0000u : 0u);
        }
        // ---- the running reference and the weights ----
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 16; ++c) mx = fmaxf(mx, x[c >> 2][c & 3]);
        int bound = 14;                                 // log2 of 2^14 over a bound on the lane's V scales
        if constexpr (KT != QWFN_KV_F16) {
            uint32_t any = 0;                           // its exponent is at least every scale's
#pragma unroll
            for (int k = 0; k < 8 * NB; ++k) any |= word(vt.sc, k);
            any |= any >> 16;
            bound = 28 - min((int)(any >> 10 & 31), 30);
        }
        const float want = col_max4(mx - (float)bound);
        if (__any(want > r + 1.0f)) {
            const float rn = fmaxf(r, want), f = __builtin_amdgcn_exp2f(r - (rn == -INFINITY ? 0.0f : rn));
            r = rn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
        const float ref = r == -INFINITY ? 0.0f : r;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            x[c >> 2][c & 3] = __builtin_amdgcn_exp2f(x[c >> 2][c & 3] - ref);
            l += x[c >> 2][c & 3];
        }
        // ---- PV ----
        uint32_t *vl = reinterpret_cast<uint32_t *>(lds[w]);
        if constexpr (!VD) {
            stage_v<HD, KT>(vt, vl, lane, keep);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            u4v ph[2], plo[2];                          // cells 16 lg + 8 m .. + 7
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int c = 8 * m + 2 * k;
                    const float p0 = x[c >> 2][c & 3], p1 = x[(c + 1) >> 2][(c + 1) & 3];
                    uint32_t hi, lo;
                    if constexpr (KT == QWFN_KV_F16) {
                        split2(p0, p1, hi, lo);
                    } else {
                        const uint32_t d0 = word(vt.sc, (c * NB + b) >> 1), d1 = word(vt.sc, ((c + 1) * NB + b) >> 1);
                        if (b & 1) p_split2<1>(p0, d0, p1, d1, hi, lo);
                        else p_split2<0>(p0, d0, p1, d1, hi, lo);
                    }
                    ph[m][k] = low ? lo : hi;
                    if constexpr (!LOC) plo[m][k] = lo;
                }
#pragma unroll
            for (int d = 2 * b; d < 2 * b + 2; ++d)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    h8v va;
                    if constexpr (VD)
                        va = q8x8_to_h8(m ? make_uint2(vt.v[d][2], vt.v[d][3]) : make_uint2(vt.v[d][0], vt.v[d][1]));
                    else
                        va = *reinterpret_cast<const h8v *>(vl + (16 * d + hn) * (kVtRow / 2) + 8 * lg + 4 * m);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, __builtin_bit_cast(h8v, ph[m]), o[d], 0, 0, 0);
                    if constexpr (!LOC)
                        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, __builtin_bit_cast(h8v, plo[m]), o[d], 0, 0, 0);
                }
        }
        if constexpr (!VD) {
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (kAhead && more) load_v<HD, KT, VD>(vt, quants(v.v_pages, pn, tn), scales(v.v_pages, pn, tn), lane);
        i = in;
        p = pn;
    }

    // ---- the four waves' states into one ----
    l = col_sum4(l);
    __syncthreads();                                    // (lds: the waves' V tiles before)
    float *ow = reinterpret_cast<float *>(lds[w]);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        f4v y = o[d];
        if constexpr (LOC)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = ror8_add(y[j]);
        if (!low) *reinterpret_cast<f4v *>(ow + head * HD + 16 * d + 4 * lg) = y;
    }
    if (lg == 0 && !low) rl[w][head] = make_float2(r, l);
    __syncthreads();
    for (int at = threadIdx.x * 4; at < g.G * HD; at += 1024) {
        const int h = at / HD;
        float rm = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) rm = fmaxf(rm, rl[k][h].x);
        const float ref = rm == -INFINITY ? 0.0f : rm;
        f4v y = {0, 0, 0, 0};
        float ls = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // (weights of 0 are multiplied all the same: a seen value that is not finite shows)
            const float f = rl[k][h].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rl[k][h].x - ref);
            y += f * *reinterpret_cast<const f4v *>(reinterpret_cast<const float *>(lds[k]) + at);
            ls += f * rl[k][h].y;
        }
        if (parts == 1) {
            store4(wa.out, wa.dtype, ((int64_t)row * g.H + gh * g.G) * HD + at, y * (ls != 0.0f ? 1.0f / ls : 0.0f));
        } else {
            const int64_t pr = (((int64_t)row * g.Hkv + gh) * parts + part) * g.G;
            *reinterpret_cast<f4v *>(part_o + pr * HD + at) = y;
            if (at % HD == 0) part_rl[pr + h] = make_float2(rm, ls);
        }
    }
}

// The parts of one row and query head, grid (rows, Hkv * G): every wave finds the weights (lane k
// takes part k, k + 64, ...), thread (j, d) sums parts j, j + 1024 / HD, ... of values 4 d ..
// + 3, the loads of four parts in flight, and LDS joins the j.
template <int HD>
__global__ void __launch_bounds__(256)
k_win_merge(Geo g, WinArg wa, int parts, const float *part_o, const float2 *part_rl) {
    constexpr int D = HD / 4, J = 256 / D;
    __shared__ f4v sum[256];
    __shared__ float ws[4 * 64];                          // weights of up to kWinMostParts parts
    const int h = blockIdx.y, gh = h / g.G, row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, d = tid % D, j = tid / D;
    if (wa.q_start && (row < wa.q_start[0] || row >= wa.q_start[wa.n_seq])) return;
    const int64_t first = ((int64_t)row * g.Hkv + gh) * parts * g.G + h % g.G;
    float2 rl[kWinMostParts / 64];
    float rm = -INFINITY;
#pragma unroll
    for (int k = 0; k < kWinMostParts / 64; ++k) {
        const int p = 64 * k + lane;
        rl[k] = p < parts ? part_rl[first + (int64_t)p * g.G] : make_float2(-INFINITY, 0.0f);
        rm = fmaxf(rm, rl[k].x);
    }
    rm = wave_max(rm);
    const float ref = rm == -INFINITY ? 0.0f : rm;
    float ls = 0.0f;
#pragma unroll
    for (int k = 0; k < kWinMostParts / 64; ++k) {
        const float f = rl[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rl[k].x - ref);
        ls += f * rl[k].y;
        if (tid < 64) ws[64 * k + lane] = f;
    }
    ls = wave_sum(ls);
    __syncthreads();
    f4v y = {0, 0, 0, 0};
    for (int p = j; p < parts; p += 4 * J) {
        f4v o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = min(p + k * J, parts - 1);
            o[k] = *reinterpret_cast<const f4v *>(part_o + (first + (int64_t)at * g.G) * HD + 4 * d);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (p + k * J < parts) y += ws[p + k * J] * o[k];
    }
    sum[tid] = y;
    __syncthreads();
    if (j) return;
#pragma unroll
    for (int k = 1; k < J; ++k) y += sum[k * D + d];
    store4(wa.out, wa.dtype, ((int64_t)row * g.H + h) * HD + 4 * d, y * (ls != 0.0f ? 1.0f / ls : 0.0f));
}

// The same for up to kFewParts parts: a thread four values of a row and head, no exchange, the
// rows of several workgroups' worth in one (many rows of few parts: 700 x 16 heads x 5 parts
// 17 us by k_win_merge).
constexpr int kFewParts = 8;
template <int HD>
__global__ void __launch_bounds__(256)
k_win_merge_few(Geo g, WinArg wa, int parts, const float *part_o, const float2 *part_rl) {
    const int64_t i = (int64_t)blockIdx.x * (1024 / HD) + threadIdx.x / (HD / 4);           // row * H + head
    const int64_t row = i / g.H;
    const int h = (int)(i % g.H), d = threadIdx.x % (HD / 4) * 4;
    if (row >= wa.n_rows) return;
    if (wa.q_start && (row < wa.q_start[0] || row >= wa.q_start[wa.n_seq])) return;
    const int64_t first = (row * g.Hkv + h / g.G) * parts * g.G + h % g.G;
    float2 rl[kFewParts];
    f4v o[kFewParts];
    float rm = -INFINITY;
#pragma unroll
    for (int k = 0; k < kFewParts; ++k) {
        const int64_t at = first + (int64_t)min(k, parts - 1) * g.G;
        rl[k] = part_rl[at];
        o[k] = *reinterpret_cast<const f4v *>(part_o + at * HD + d);
    }
#pragma unroll
    for (int k = 0; k < kFewParts; ++k) {
        if (k >= parts) rl[k].x = -INFINITY;
        rm = fmaxf(rm, rl[k].x);
    }
    const float ref = rm == -INFINITY ? 0.0f : rm;
    f4v y = {0, 0, 0, 0};
    float ls = 0.0f;
#pragma unroll
    for (int k = 0; k < kFewParts; ++k) {
        if (k >= parts) break;
        const float f = rl[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rl[k].x - ref);
        ls += f * rl[k].y;
        y += f * o[k];
    }
    store4(wa.out, wa.dtype, (row * g.H + h) * HD + d, y * (ls != 0.0f ? 1.0f / ls : 0.0f));
}

template <int HD>
static void merge_t(const Geo &g, const WinArg &wa, int parts, const float *part_o, const float2 *part_rl, hipStream_t st) {
    if (parts <= kFewParts) {
        const int64_t rows = (int64_t)wa.n_rows * g.H, a_wg = 1024 / HD;
        hipLaunchKernelGGL(k_win_merge_few<HD>, dim3((unsigned)((rows + a_wg - 1) / a_wg)), dim3(256), 0, st, g, wa, parts,
                           part_o, part_rl);
    } else {
        hipLaunchKernelGGL(k_win_merge<HD>, dim3((unsigned)wa.n_rows, (unsigned)g.H), dim3(256), 0, st, g, wa, parts, part_o,
                           part_rl);
    }
}

void launch_win_merge(const Geo &g, const WinArg &wa, int parts, const float *part_o, const float2 *part_rl, hipStream_t st) {
    if (g.hd == 64) merge_t<64>(g, wa, parts, part_o, part_rl, st);
    else if (g.hd == 128) merge_t<128>(g, wa, parts, part_o, part_rl, st);
    else merge_t<256>(g, wa, parts, part_o, part_rl, st);
}

// Parts of a sequence's tiles: enough workgroups for two a CU, at most a tile a wave.
int win_dec_parts(const Geo &g, const WinPlan &p) {
    const int tiles = win_most_tiles(p);
    const int pairs = p.n_seq * g.Hkv;
    return std::max(1, std::min({(tiles + 3) / 4, (512 + pairs - 1) / pairs, kWinMostParts}));
}

size_t win_dec_ws_bytes(const Geo &g, const WinPlan &p) {
    const int parts = win_dec_parts(g, p);
    if (parts == 1) return 256;
    const size_t rows = (size_t)p.n_rows * g.Hkv * parts * g.G;
    return win_align(rows * g.hd * sizeof(float)) + win_align(rows * sizeof(float2));
}

template <int HD, int KT, bool VD, bool LOC>
static void launch_t(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, int parts, float *po, float2 *rl, hipStream_t st) {
    hipLaunchKernelGGL((k_win_dec<HD, KT, VD, LOC>), dim3((unsigned)parts, (unsigned)g.Hkv, (unsigned)wa.n_seq), dim3(256),
                       0, st, g, v, wa, parts, po, rl);
}

template <int HD, bool LOC>
static void launch_kt(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, int parts, float *po, float2 *rl, hipStream_t st) {
    if (g.kt == QWFN_KV_Q4_0) launch_t<HD, QWFN_KV_Q4_0, false, LOC>(g, v, wa, parts, po, rl, st);
    else if (g.kt == QWFN_KV_F16) launch_t<HD, QWFN_KV_F16, false, LOC>(g, v, wa, parts, po, rl, st);
    else if (g.vdim) launch_t<HD, QWFN_KV_Q8_0, true, LOC>(g, v, wa, parts, po, rl, st);
    else launch_t<HD, QWFN_KV_Q8_0, false, LOC>(g, v, wa, parts, po, rl, st);
}

bool win_shape(int32_t hd, int32_t G) { return G <= 8 ? hd == 64 || hd == 128 || hd == 256 : hd == 256 && G <= 16; }

hipError_t launch_win_dec(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, const WinPlan &p, void *ws, hipStream_t st) {
    const int parts = win_dec_parts(g, p);
    float *po = (float *)ws;
    float2 *rl = (float2 *)((uint8_t *)ws + win_align((size_t)p.n_rows * g.Hkv * parts * g.G * g.hd * sizeof(float)));
    switch (g.hd) {
    case 64: launch_kt<64, true>(g, v, wa, parts, po, rl, st); break;
    case 128: launch_kt<128, true>(g, v, wa, parts, po, rl, st); break;
    case 256: g.G <= 8 ? launch_kt<256, true>(g, v, wa, parts, po, rl, st) : launch_kt<256, false>(g, v, wa, parts, po, rl, st); break;
    default: return hipErrorInvalidValue;
    }
    if (parts > 1) launch_win_merge(g, wa, parts, po, rl, st);
    return hipGetLastError();
}

}  // namespace qwfn_qsa
