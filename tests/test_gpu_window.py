"""Sliding-window attention over the paged cache, on the GPU, against the same attention in
64 bits over the cache's own values (read back by the dequantizing gather)."""
import itertools
import math

import numpy as np
import pytest
import torch

from qwfnfer_amd import qsa

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = {                              # n_head, n_head_kv, head_dim, block_tokens
    "base": (16, 2, 128, 64), "ckpt": (24, 2, 256, 4), "small": (16, 2, 64, 64), "wide": (16, 8, 128, 64),
    "mid": (8, 2, 128, 64), "big": (16, 2, 256, 64), "four": (16, 2, 128, 4),
}


def config(shape, kv):
    h, hkv, hd, bt = SHAPES[shape]
    return qsa.QsaConfig(n_head=h, n_head_kv=hkv, head_dim=hd, block_tokens=bt, kv_type=kv)


class Setup:
    """A filled cache of sequences of the given lengths, in permuted pages, and its values in 64 bits."""

    def __init__(self, cfg, lens, seed=0, rows=None):
        self.cfg, self.lens = cfg, list(lens)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        n_seq = len(self.lens)
        pages = max(1, -(-max(self.lens) // cfg.page_tokens))
        perm = torch.randperm(n_seq * pages, device="cuda", generator=gen).to(torch.int32).view(n_seq, pages)
        self.cache = qsa.KvCache.allocate(cfg, n_seq, pages, page_table=perm)
        self.max_len = pages * cfg.page_tokens
        hkv, hd = cfg.n_head_kv, cfg.head_dim
        for s, n in enumerate(self.lens):
            if n == 0:
                continue
            k, v = (torch.randn(n, hkv, hd, device="cuda", generator=gen) for _ in range(2))
            scale = torch.empty(n, hkv, hd // 32, 1, device="cuda")
            k, v = ((x.view(n, hkv, -1, 32) * scale.uniform_(math.log(0.25), math.log(2), generator=gen).exp_()).reshape(n, hkv, hd).contiguous()
                    for x in (k, v))
            if rows:
                k, v = rows(s, k, v)
            pos = torch.arange(n, dtype=torch.int32, device="cuda")
            qsa.append_q8_0(self.cache, k, v, pos, torch.full_like(pos, s))
        self.gen = gen
        self.read()

    def read(self):
        lens = torch.tensor([max(n, 1) for n in self.lens], dtype=torch.int32, device="cuda")
        k, v, _ = qsa.gather_dequant(self.cache, lens, None, None, -(-self.max_len // self.cfg.block_tokens))
        self.k, self.v = k.double(), v.double()              # [seq, KV head, cell, dim]
        qsa.read_status(self.cache)

    def queries(self, n, dtype, scale=1.0):
        return (torch.randn(n, self.cfg.n_head, self.cfg.head_dim, device="cuda", generator=self.gen) * scale).to(dtype)

    def expected(self, q, seq, first, window, sinks):
        """(result, sum p|v|, sum p A (|v| + |o|), most cells, sum |v|, largest |v|, D) of queries q of sequence seq
        at positions first ..: A is a logit's sum of magnitudes, D the logits' change where every key value is off
        by the largest of them."""
        cfg, n = self.cfg, len(q)
        g = cfg.n_head // cfg.n_head_kv
        p = torch.arange(first, first + n, device="cuda")[:, None]
        t = torch.arange(int(p.max()) + 1, device="cuda")
        seen = (t <= p) & ((t > p - window) | (t < sinks))
        k, v = self.k[seq, :, :len(t)], self.v[seq, :, :len(t)]
        qd = q.double().view(n, cfg.n_head_kv, g, cfg.head_dim).permute(1, 2, 0, 3)     # [Hkv, G, n, hd]
        kt = k[:, None].transpose(-1, -2)
        hidden = ~seen
        x = (qd.float().double() @ torch.nan_to_num(kt, nan=0.0, posinf=0.0, neginf=0.0)) / math.sqrt(cfg.head_dim)
        a = (qd.abs() @ torch.nan_to_num(kt.abs(), nan=0.0, posinf=0.0)) / math.sqrt(cfg.head_dim)
        w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
        vv = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)[:, None]
        o = w @ vv
        b0 = w @ vv.abs()
        b1 = (w * a) @ vv.abs() + (w * a).sum(-1, keepdim=True) * o.abs()
        sv = (~hidden).double() @ vv.abs()
        top = vv.abs().amax()
        d = (qd.abs().sum(-1, keepdim=True) * torch.nan_to_num(k.abs(), nan=0.0, posinf=0.0).amax() / math.sqrt(cfg.head_dim)).expand_as(o)
        back = lambda y: y.permute(2, 0, 1, 3).reshape(n, cfg.n_head, cfg.head_dim)  # noqa: E731
        return back(o), back(b0), back(b1), int(seen.sum(1).max()), back(sv.expand_as(o)), top, back(d)


def bound_of(want, dtype, hd):
    """Tolerance: a logit is off by at most eps_s of its sum of magnitudes A, which moves the output by at most
    sum p (eps_s A)(|v| + |o|) to first order (the factor 2 covers the rest); weights and values are off by
    eps_v, sums of n terms by n 2^-24 of their magnitudes.
    F32 and F16: operands held to 2^-21 (a sum of two fp16 numbers), fp32 sums: eps_s = (hd + 16) 2^-24 + 2^-19.
    BF16: keys, values and weights rounded to fp16: eps = 2^-11 each.
    fp16's step is absolute below 2^-14, half of it 2^-25.  The largest weight is at least 2^13 (BF16: 2^6) of the
    units the weights are in, so a weight is off by up to 2^-38 (2^-31) of the largest besides, the output by that
    times sum |v|.  Keys and values are scaled so that a tile's largest is at least 2^7 (BF16: 2^-4): they are off
    by up to 2^-32 (2^-21) of it besides.  Then one rounding to the output's type."""
    o, b0, b1, n, sv, top, d = want
    if dtype == torch.bfloat16:
        eps_s, eps_v, abs_w, abs_v = 2.0 ** -11 + (hd + 16) * 2.0 ** -24, 2 * 2.0 ** -11, 2.0 ** -31, 2.0 ** -21
    else:
        eps_s, eps_v, abs_w, abs_v = (hd + 16) * 2.0 ** -24 + 2.0 ** -19, 2.0 ** -19, 2.0 ** -38, 2.0 ** -32
    return (2 * eps_s * b1 + (eps_v + (n + 16) * 2.0 ** -24) * (b0 + o.abs()) + abs_w * sv + abs_v * (top + 2 * d * (b0 + o.abs()))
            + torch.finfo(dtype).eps / 2 * o.abs() * 1.01)


def check(got, want, dtype, hd):
    """bound_of(), and the absolute half step of a float16 output."""
    assert got.dtype == dtype
    o = want[0]
    err, bound = (got.double() - o).abs(), bound_of(want, dtype, hd) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    bad = ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), float(err.max()), float((err / bound).max()))


def decode(st, dtype, window, sinks, lens=None, q=None, ws=None, **kw):
    lens = st.lens if lens is None else lens
    q = st.queries(len(lens), dtype) if q is None else q
    ws = ws or qsa.Workspace.for_window(st.cfg, len(lens), st.max_len, window, sinks, dtype=dtype)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return q, qsa.window_attn_decode(st.cache, q, sl, st.max_len, window, ws, sink_tokens=sinks, **kw)


def check_decode(st, q, out, dtype, window, sinks, lens=None):
    for s, n in enumerate(st.lens if lens is None else lens):
        if n <= 0:
            assert not out[s].any()
        else:
            check(out[s:s + 1], st.expected(q[s:s + 1], s, n - 1, window, sinks), dtype, st.cfg.head_dim)


def prefill(st, n_q, dtype, window, sinks, lens=None, q=None, gap=0, ws=None):
    lens = st.lens if lens is None else lens
    rows = sum(n_q) + gap
    q = st.queries(rows, dtype) if q is None else q
    start = torch.tensor([0, *np.cumsum(n_q).tolist()], dtype=torch.int32, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = ws or qsa.Workspace.for_window(st.cfg, len(lens), st.max_len, window, sinks, n_rows=rows, max_q=max(n_q), dtype=dtype)
    out = torch.full((rows, st.cfg.n_head, st.cfg.head_dim), 7.0, dtype=dtype, device="cuda")
    qsa.window_attn_prefill(st.cache, q, start, sl, max(n_q), st.max_len, window, ws, sink_tokens=sinks, out=out)
    return q, out


def check_prefill(st, q, out, n_q, dtype, window, sinks, lens=None):
    at = 0
    for s, (n, m) in enumerate(zip(st.lens if lens is None else lens, n_q)):
        if m:
            check(out[at:at + m], st.expected(q[at:at + m], s, n - m, window, sinks), dtype, st.cfg.head_dim)
        at += m
    assert (out[at:] == 7.0).all()                       # rows behind the last sequence are left as they were


KV_IO = [(kv, io) for kv in (0, 1, 2) for io in TYPES]


# ---- single tokens --------------------------------------------------------------

@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("kv,io", KV_IO)
def test_decode_shapes_and_types(shape, kv, io):
    st = Setup(config(shape, kv), [1, 63, 64, 65, 300, 517])
    q, out = decode(st, TYPES[io], 130, 5)
    check_decode(st, q, out, TYPES[io], 130, 5)
    assert qsa.read_status(st.cache) == 0


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 128, 200, 1000, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 64, 70, 300, 2 ** 31 - 1])
def test_decode_windows(window, sinks):
    st = Setup(config("base", 0), [1, 2, 64, 129, 700, 1024], seed=window % 97)
    for io in ("f32", "bf16"):
        q, out = decode(st, TYPES[io], window, sinks)
        check_decode(st, q, out, TYPES[io], window, sinks)


@pytest.mark.parametrize("kv", [0, 1, 2])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("lens,window", [([9000], 4096), ([20000, 3, 12000], 9001), ([5000] * 40, 700)])
def test_decode_long(kv, io, lens, window):
    st = Setup(config("base", kv), lens)
    q, out = decode(st, TYPES[io], window, 33)
    check_decode(st, q, out, TYPES[io], window, 33)


def test_decode_empty_and_bad_rows():
    """Length 0 is a padded row, zeros without a report; a bad length is reported and gives zeros."""
    st = Setup(config("base", 0), [100, 0, 300])
    ws = qsa.Workspace.for_window(st.cfg, 3, st.max_len, 64, 4)
    q, out = decode(st, torch.float32, 64, 4, ws=ws)
    check_decode(st, q, out, torch.float32, 64, 4)
    assert qsa.read_status(st.cache) == 0
    for bad in (-1, st.max_len + 1, -2 ** 31, 2 ** 31 - 1):
        lens = [100, bad, 300]
        q, out = decode(st, torch.float32, 64, 4, lens=lens, ws=ws)
        assert not out[1].any()
        check_decode(st, q[:1], out[:1], torch.float32, 64, 4, lens=lens[:1])
        assert qsa.read_status(st.cache) == qsa._lib.STATUS_LEN_RANGE


@pytest.mark.parametrize("kv", [0, 2])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_pages_out_of_sight_are_not_read(kv, io):
    """Entries of pages that no visible cell is in hold -1, a far number, or a page of NaN."""
    dtype = TYPES[io]
    st = Setup(config("base", kv), [2000, 1500], seed=4)
    window, sinks = 300, 7
    n_q = [40, 3]
    q = st.queries(2, dtype)
    st.cache.page_table[0, 1:6] = torch.tensor([-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1, -1], dtype=torch.int32)
    st.cache.page_table[1, 1:4] = -1
    _, out = decode(st, dtype, window, sinks, q=q)
    check_decode(st, q, out, dtype, window, sinks)
    q, out = prefill(st, n_q, dtype, window, sinks)
    check_prefill(st, q, out, n_q, dtype, window, sinks)
    assert qsa.read_status(st.cache) == 0
    # a visible page that is gone: reported, its cells not attended
    st.cache.page_table[0, 7] = -1                      # cells 1792 .. 1999: all of the rest is 1700 .. 1791 and the sinks
    st.k[0, :, 1792:] = 0
    q, out = decode(st, dtype, window, sinks)
    assert qsa.read_status(st.cache) == qsa._lib.STATUS_PAGE_RANGE
    seen = torch.cat([st.k[0, :, :7], st.k[0, :, 1700:1792]], 1), torch.cat([st.v[0, :, :7], st.v[0, :, 1700:1792]], 1)
    g = st.cfg.n_head // st.cfg.n_head_kv
    x = (q[0].double().view(st.cfg.n_head_kv, g, -1) @ seen[0].transpose(1, 2)) / math.sqrt(st.cfg.head_dim)
    o = (torch.softmax(x, -1) @ seen[1]).reshape(st.cfg.n_head, -1)
    assert (out[0].double() - o).abs().max() < 0.02      # a page more or less moves values by 0.1 and more
    check(out[1:], st.expected(q[1:], 1, 1499, window, sinks), dtype, 128)
    q, out = prefill(st, n_q, dtype, window, sinks)
    assert qsa.read_status(st.cache) == qsa._lib.STATUS_PAGE_RANGE
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("kv,io", [(2, "f32"), (2, "bf16"), (0, "bf16"), (0, "f32")])
def test_non_finite_cells_out_of_sight(kv, io):
    """Infinities and NaN in cells that a query does not see, in the same tile as cells that it sees."""
    dtype = TYPES[io]
    bad = [3, 40, 130, 131, 200, 511]

    def rows(s, k, v):
        for i, t in enumerate(bad):
            k[t, :, i * 20 % 128] = math.nan if i % 2 else math.inf
            v[t, :, i * 30 % 128] = math.inf if i % 2 else math.nan
        return k, v

    st = Setup(config("base", kv), [600], rows=rows)
    for n, window, sinks in ((510, 300, 3), (350, 149, 3), (139, 7, 0), (600, 80, 2), (204, 3, 0)):
        q, out = decode(st, dtype, window, sinks, lens=[n])
        check_decode(st, q, out, dtype, window, sinks, lens=[n])
    # prefill: some queries of a tile's group see a bad cell, others do not
    n_q, window = [390], 50
    q, out = prefill(st, n_q, dtype, window, 2)
    o = st.expected(q, 0, 210, window, 2)
    sees = torch.zeros(390, dtype=torch.bool, device="cuda")
    for t in bad:
        p = torch.arange(210, 600, device="cuda")
        sees |= (t <= p) & (t > p - window)
    assert sees.any() and not sees.all()
    check(out[~sees], (o[0][~sees], o[1][~sees], o[2][~sees], o[3], o[4][~sees], o[5], o[6][~sees]), dtype, 128)
    # queries that see one: their keys give NaN weights
    assert torch.isnan(out[sees].float()).any(-1).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", [0, 1, 2])
def test_seen_non_finite_values_show(io, kv):
    """A NaN or infinity in a visible V value makes that dimension of the output not finite, no other one."""
    dtype = TYPES[io]

    def rows(s, k, v):
        v[100, 1, 5] = math.inf
        v[101, 1, 70] = math.nan
        return k, v

    st = Setup(config("base", kv), [300], rows=rows)
    # the quantized types hold a scale that is not finite, or quants of 0: what the cache holds decides
    held = ~torch.isfinite(st.v[0, 1, 100:102]).all(0)
    for got in (decode(st, dtype, 250, 0)[1][0], prefill(st, [3], dtype, 250, 0)[1][2]):
        finite = torch.isfinite(got.float()).view(2, 8, 128)
        assert finite[0].all()
        assert (finite[1] == ~held).all()


@pytest.mark.parametrize("io", list(TYPES))
@pytest.mark.parametrize("kscale,vscale,qscale", [(1e3, 1e4, 1e-3), (1e-4, 1e-5, 1e3), (30.0, 3e4, 1.0), (1.0, 1e-6, 1.0)])
@pytest.mark.parametrize("kv", [0, 2])
def test_magnitudes(io, kscale, vscale, qscale, kv):
    """Large and small keys, values and queries: logits of a few units, or of hundreds (a weight of 1)."""
    dtype = TYPES[io]
    if kv == 2 or io == "f16":
        vscale = min(max(vscale, 1e-5), 5e3)             # what fp16 cells and outputs hold
    st = Setup(config("base", kv), [333, 150], rows=lambda s, k, v: (k * kscale, v * vscale))
    for got, want in _both(st, dtype, qscale):
        check(got, want, dtype, 128)


def _both(st, dtype, qscale):
    q = st.queries(2, dtype, qscale)
    _, out = decode(st, dtype, 140, 4, q=q)
    for s, n in enumerate(st.lens):
        yield out[s:s + 1], st.expected(q[s:s + 1], s, n - 1, 140, 4)
    q = st.queries(60, dtype, qscale)
    _, out = prefill(st, [50, 10], dtype, 140, 4, q=q)
    yield out[:50], st.expected(q[:50], 0, 283, 140, 4)
    yield out[50:], st.expected(q[50:], 1, 140, 140, 4)


# ---- several queries a sequence --------------------------------------------------

@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("kv,io", KV_IO)
def test_prefill_shapes_and_types(shape, kv, io):
    st = Setup(config(shape, kv), [333, 64, 1, 200])
    n_q = [100, 64, 1, 7]
    q, out = prefill(st, n_q, TYPES[io], 90, 5, gap=3)
    check_prefill(st, q, out, n_q, TYPES[io], 90, 5)
    assert qsa.read_status(st.cache) == 0


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 70, 300, 2 ** 31 - 1])
def test_prefill_windows(window, sinks):
    st = Setup(config("base", 0), [700, 130], seed=window % 89)
    for io in ("f32", "bf16"):
        q, out = prefill(st, [450, 130], TYPES[io], window, sinks)
        check_prefill(st, q, out, [450, 130], TYPES[io], window, sinks)


@pytest.mark.parametrize("n_q", [[1], [2], [15], [16], [17], [33], [128], [129], [1, 1, 1, 1, 1], [0, 5, 0, 0, 300, 0],
                                 [31, 32, 33, 1, 0, 64]])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_prefill_row_counts(n_q, io):
    st = Setup(config("base", 0), [max(5 * m, 77) for m in n_q], seed=len(n_q))
    q, out = prefill(st, n_q, TYPES[io], 120, 9, gap=20)
    check_prefill(st, q, out, n_q, TYPES[io], 120, 9)
    assert qsa.read_status(st.cache) == 0


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("lens,n_q,window,sinks", [
    ([6000], [3], 4500, 64), ([6000], [700], 2048, 64), ([3001], [3001], 1000, 4), ([9000, 50], [17, 50], 8000, 0),
])
def test_prefill_long(io, lens, n_q, window, sinks):
    st = Setup(config("base", 0), lens)
    q, out = prefill(st, n_q, TYPES[io], window, sinks)
    check_prefill(st, q, out, n_q, TYPES[io], window, sinks)


def test_prefill_bad_sequences():
    """More queries than tokens, a bad length, more than max_q: reported, zero rows; the others unharmed."""
    st = Setup(config("base", 0), [200, 100, 150, 90])
    n_q = [30, 10, 20, 40]
    for lens, bad in (([200, 9, 150, 90], 1), ([200, -7, 150, 90], 1), ([200, 100, st.max_len + 1, 90], 2), ([0, 100, 150, 90], 0)):
        q, out = prefill(st, n_q, torch.bfloat16, 64, 3, lens=lens)
        assert qsa.read_status(st.cache) == qsa._lib.STATUS_LEN_RANGE
        at = 0
        for s, (n, m) in enumerate(zip(lens, n_q)):
            if s == bad:
                assert not out[at:at + m].any()
            else:
                check(out[at:at + m], st.expected(q[at:at + m], s, n - m, 64, 3), torch.bfloat16, 128)
            at += m
    q = st.queries(100, torch.float32)
    start = torch.tensor([0, 30, 40, 60, 100], dtype=torch.int32, device="cuda")
    ws = qsa.Workspace.for_window(st.cfg, 4, st.max_len, 64, 3, n_rows=100, max_q=35)
    out = qsa.window_attn_prefill(st.cache, q, start, torch.tensor(st.lens, dtype=torch.int32, device="cuda"), 35,
                                  st.max_len, 64, ws, sink_tokens=3)
    assert qsa.read_status(st.cache) == qsa._lib.STATUS_LEN_RANGE
    assert not out[60:].any()
    check(out[:30], st.expected(q[:30], 0, 170, 64, 3), torch.float32, 128)


def test_prefill_of_single_rows():
    """max_q = 1: sequences of a row or none, rows behind the last, and a sequence of two, which is refused."""
    for lens, window in (([400, 90, 1000, 70], 200), ([9000, 5], 8000)):
        st = Setup(config("base", 0), lens)
        n_q = [1, 0, 1, 1] if len(lens) == 4 else [1, 1]
        for io in ("f32", "bf16"):
            q, out = prefill(st, n_q, TYPES[io], window, 10, gap=2)
            check_prefill(st, q, out, n_q, TYPES[io], window, 10)
            assert qsa.read_status(st.cache) == 0
        m = len(lens) + 1
        q = st.queries(m, torch.bfloat16)
        start = torch.tensor([0, 2, *range(3, m + 1)], dtype=torch.int32, device="cuda")
        ws = qsa.Workspace.for_window(st.cfg, len(lens), st.max_len, window, 10, n_rows=m, max_q=1, dtype=torch.bfloat16)
        out = qsa.window_attn_prefill(st.cache, q, start, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1,
                                      st.max_len, window, ws, sink_tokens=10)
        assert qsa.read_status(st.cache) == qsa._lib.STATUS_LEN_RANGE
        assert not out[:2].any()
        check(out[2:3], st.expected(q[2:3], 1, lens[1] - 1, window, 10), torch.bfloat16, 128)


def test_decode_is_the_prefill_of_one_query():
    st = Setup(config("base", 0), [400, 90, 1000])
    q, out = decode(st, torch.float32, 200, 10)
    _, rows = prefill(st, [1, 1, 1], torch.float32, 200, 10, q=q)
    for s, n in enumerate(st.lens):
        want = st.expected(q[s:s + 1], s, n - 1, 200, 10)
        check(out[s:s + 1], want, torch.float32, 128)
        check(rows[s:s + 1], want, torch.float32, 128)


def test_runs_are_bit_equal():
    """No atomics decide a sum's order."""
    st = Setup(config("base", 0), [5000, 300, 2500])
    for io in TYPES:
        q = st.queries(3, TYPES[io])
        a, b = (decode(st, TYPES[io], 3000, 10, q=q)[1] for _ in range(2))
        assert torch.equal(a, b)
        q = st.queries(200, TYPES[io])
        a, b = (prefill(st, [100, 60, 40], TYPES[io], 1500, 10, q=q)[1] for _ in range(2))
        assert torch.equal(a, b)


def test_captured_and_replayed_with_new_lengths():
    """One graph of a token's step (the append with its rotation, then the attention), replayed as the sequences
    grow, with eager steps of another cache between the replays; and two graphs that share one workspace."""
    cfg = config("base", 0)
    st, other = Setup(cfg, [250, 1, 511], seed=1), Setup(cfg, [250, 1, 511], seed=1)
    for s in (st, other):
        s.cache.page_table.copy_(torch.arange(s.cache.page_table.numel(), dtype=torch.int32).view_as(s.cache.page_table))
    other.cache.k_pages.copy_(st.cache.k_pages)
    other.cache.v_pages.copy_(st.cache.v_pages)
    rope = qsa.Rope(qsa.RopeConfig(rope_dim=128))
    x = torch.randn(3, 20, 128, device="cuda").bfloat16()
    pos, lens = torch.tensor([249, 0, 500], dtype=torch.int32, device="cuda"), torch.tensor([250, 1, 501], dtype=torch.int32, device="cuda")
    seq = torch.arange(3, dtype=torch.int32, device="cuda")
    ws = qsa.Workspace.for_window(cfg, 3, st.max_len, 100, 4, dtype=torch.bfloat16)
    qo, out, out2 = (torch.zeros(3, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in range(3))

    def step(cache, q_out, o):
        qsa.append_rope(cache, rope, x[:, 16:18], x[:, 18:], pos, seq, q=x[:, :16], q_out=q_out)
        return qsa.window_attn_decode(cache, q_out, lens, st.max_len, 100, ws, sink_tokens=4, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(st.cache, qo, out)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, o in zip(graphs, (out, out2)):
        with torch.cuda.graph(g):
            step(st.cache, qo, o)
    for i in range(5):
        x.copy_(torch.randn(3, 20, 128, device="cuda"))
        pos.copy_(torch.tensor([249 + i, i, 500 + i], dtype=torch.int32))
        lens.copy_(pos + 1)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step(other.cache, torch.empty_like(qo), torch.empty_like(out))
        assert torch.equal(out, want) and torch.equal(out2, want)


def test_prefill_captured_and_replayed():
    cfg = config("base", 0)
    st = Setup(cfg, [600, 300])
    q = st.queries(120, torch.bfloat16)
    start, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, 80, 120], [600, 300]))
    ws = qsa.Workspace.for_window(cfg, 2, st.max_len, 100, 4, n_rows=120, max_q=100, dtype=torch.bfloat16)
    out = torch.zeros_like(q)
    run = lambda o: qsa.window_attn_prefill(st.cache, q, start, lens, 100, st.max_len, 100, ws, sink_tokens=4, out=o)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out)
    for i, (a, b) in enumerate(itertools.product([[0, 80, 120], [0, 20, 120], [5, 100, 110]], [[600, 300], [431, 260]])):
        start.copy_(torch.tensor(a, dtype=torch.int32))
        lens.copy_(torch.tensor(b, dtype=torch.int32))
        q.copy_(st.queries(120, torch.bfloat16))
        out.fill_(float(i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(torch.full_like(q, float(i))))
        check(out[a[0]:a[1]], st.expected(q[a[0]:a[1]], 0, b[0] - (a[1] - a[0]), 100, 4), torch.bfloat16, 128)
        assert (out[a[2]:] == i).all() and (out[:a[0]] == i).all()


def test_on_another_stream():
    st = Setup(config("base", 0), [3000, 200])
    q = st.queries(2, torch.bfloat16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ws = qsa.Workspace.for_window(st.cfg, 2, st.max_len, 1000, 0, dtype=torch.bfloat16)
    _, want = decode(st, torch.bfloat16, 1000, 0, q=q)
    torch.cuda.synchronize()
    lens, out = torch.tensor(st.lens, dtype=torch.int32, device="cuda"), torch.zeros_like(q)
    torch.cuda.synchronize()
    qsa.window_attn_decode(st.cache, q, lens, st.max_len, 1000, ws, out=out, stream=side)
    side.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("kv", [0, 2])
def test_pages_past_32_bits(kv):
    """Pages more than 4 GiB into their pool: the bytes and results of the same rows in a small one."""
    cfg = config("base", kv)
    far = 2 ** 32 // cfg.page_bytes() + 2
    rope = qsa.Rope(qsa.RopeConfig(rope_dim=128))
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(700, 20, 128, device="cuda", generator=gen).bfloat16()
    pos = torch.arange(700, dtype=torch.int32, device="cuda")
    start, lens = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, 100], [700]))
    got = []
    for table, phys in ([[0, 1, 2]], 3), ([[far, far + 2, far + 1]], far + 3):
        c = qsa.KvCache.allocate(cfg, 1, 3, page_table=torch.tensor(table, dtype=torch.int32), n_phys_pages=phys)
        q = qsa.append_rope(c, rope, x[:, 16:18], x[:, 18:], pos, q=x[:, :16])
        ws = qsa.Workspace.for_window(cfg, 1, 768, 300, 4, n_rows=100, max_q=100)
        got.append((qsa.window_attn_decode(c, q[-1:].contiguous(), lens, 768, 300, ws, sink_tokens=4),
                    qsa.window_attn_prefill(c, q[600:].contiguous(), start, lens, 100, 768, 300, ws, sink_tokens=4)))
        assert qsa.read_status(c) == 0 and got[-1][0].any()
        del c
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ---- a run of them, as a program makes it ------------------------------------------

@pytest.mark.parametrize("kv", [0, 1, 2])
def test_prompt_then_tokens(kv):
    """A prompt read in chunks, then single tokens, pages given back as the window leaves them, against one
    64-bit attention over all rows: the cache's own values, turned as they went in."""
    cfg = config("base", kv)
    cache = qsa.KvCache.allocate(cfg, 1, 4)
    rope = qsa.Rope(qsa.RopeConfig(rope_dim=128, base=1e6))
    window, sinks, total = 200, 4, 900
    gen = torch.Generator(device="cuda").manual_seed(kv)
    x = torch.randn(total, 20, 128, device="cuda", generator=gen)
    norm = torch.rand(128, device="cuda", generator=gen) + 0.5
    pos = torch.arange(total, dtype=torch.int32, device="cuda")
    outs, qs, at = [], [], 0
    table = cache.page_table.clone()
    for n in (300, 1, 257, 64, *[1] * 20, 250, 8):
        rows = slice(at, at + n)
        q = qsa.append_rope(cache, rope, x[rows, 16:18], x[rows, 18:], pos[rows], k_norm=norm, q=x[rows, :16], q_norm=norm)
        at += n
        lens = torch.tensor([at], dtype=torch.int32, device="cuda")
        gone = max(0, at - n - window + 1) // 256        # whole pages before the window, but the sinks'
        cache.page_table[0, 1:gone] = -1
        if n == 1:
            ws = qsa.Workspace.for_window(cfg, 1, 1024, window, sinks)
            outs.append(qsa.window_attn_decode(cache, q, lens, 1024, window, ws, sink_tokens=sinks))
        else:
            ws = qsa.Workspace.for_window(cfg, 1, 1024, window, sinks, n_rows=n, max_q=n)
            start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            outs.append(qsa.window_attn_prefill(cache, q, start, lens, n, 1024, window, ws, sink_tokens=sinks))
        qs.append(q)
    assert at == total and (cache.page_table == -1).any() and qsa.read_status(cache) == 0
    cache.page_table.copy_(table)
    st = Setup.__new__(Setup)
    st.cfg, st.cache, st.lens, st.max_len = cfg, cache, [total], 1024
    st.read()
    check(torch.cat(outs), st.expected(torch.cat(qs), 0, 0, window, sinks), torch.float32, 128)
    # the rows went in turned: the values differ from the turned rows by the cache type's rounding alone
    k = qsa.rope_rows(rope, x[:, 16:18].contiguous(), pos, norm=norm)
    step = {0: 1 / 127, 1: 1 / 8, 2: 2.0 ** -10}[kv]
    amax = k.view(total, 2, 4, 32).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(total, 2, 128)
    assert ((st.k[0, :, :total].transpose(0, 1) - k).abs() <= step * amax).all()
