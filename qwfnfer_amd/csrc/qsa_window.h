// qsa_window.h -- what the sliding-window kernels share: a sequence's list of
// 64-cell tiles, a row's power of two, the parts' merge.
#pragma once

#include <algorithm>

#include "qsa_io.h"

namespace qwfn_qsa {

constexpr int kWinMostParts = 256;       // parts a row's tiles are split into

inline size_t win_align(size_t x) { return (x + 255) & ~(size_t)255; }

// The 64-cell tiles that the last n_q queries of a sequence of length len see: the
// first tokens' tiles 0 .. ns - 1, then the window's from tile w0 (no tile twice).
struct WinTiles {
    int n, ns, w0, window, sinks;
    __host__ __device__ __forceinline__ int cell(int i) const { return (i < ns ? i : w0 + i - ns) * 64; }
    // the cells the query at position len - 1 sees
    __device__ __forceinline__ bool seen(int t, int len) const { return t < len && (t >= len - window || t < sinks); }
    __device__ __forceinline__ bool whole(int i, int len) const {
        const int t = cell(i);
        return t + 64 <= len && (t >= len - window || t + 64 <= sinks);
    }
};
__host__ __device__ __forceinline__ WinTiles win_tiles(int len, int n_q, int window, int sinks) {
    WinTiles t;
    t.window = window;
    t.sinks = sinks;
    t.n = t.ns = t.w0 = 0;
    if (len <= 0) return t;
    const int64_t lo = (int64_t)len - n_q - window + 1;
    const int first = lo > 0 ? (int)lo : 0;
    const int s = sinks < first ? sinks : first;        // first tokens before the window
    t.ns = (s + 63) / 64;
    t.w0 = first / 64 > t.ns ? first / 64 : t.ns;
    t.n = t.ns + (len + 63) / 64 - t.w0;
    return t;
}
// The most tiles such a list has within a plan's bounds.
inline int win_most_tiles(const WinPlan &p) {
    const int64_t all = ((int64_t)p.max_seq_len + 63) / 64;
    const int64_t win = ((int64_t)p.window + p.max_q - 1 + 126) / 64, sink = ((int64_t)p.sinks + 63) / 64;
    return (int)std::min<int64_t>(all, win + sink);
}

// The exponent e that brings a row's largest magnitude m to [2^k, 2^(k + 1)): x 2^e.  A
// zero row and one that is not finite stay as they are.  Bounded so that 2^e and 2^-e
// are normal numbers.
__device__ __forceinline__ int pow2_to(float m, int k) {
    const int b = (int)(__float_as_uint(m) >> 23);      // m >= 0
    return b == 0 || b == 255 ? 0 : min(max(k + 127 - b, -100), 100);
}

// Decode (qsa_window_dec.hip)
int win_dec_parts(const Geo &g, const WinPlan &p);
size_t win_dec_ws_bytes(const Geo &g, const WinPlan &p);
hipError_t launch_win_dec(const Geo &g, const qwfn_kv_view &v, const WinArg &wa, const WinPlan &p, void *ws, hipStream_t st);

// The parts of every row of the call (part_o, part_rl: [row][Hkv][parts][G]) into out; rows
// outside every sequence are left as they were.
void launch_win_merge(const Geo &g, const WinArg &wa, int parts, const float *part_o, const float2 *part_rl, hipStream_t st);

}  // namespace qwfn_qsa
