"""Rotary rows and the append with the rotation on the way, on the GPU: against the same
steps in 64-bit numpy, and the cache's bytes against the CPU oracle's append of the rows
so computed."""
import math

import numpy as np
import pytest
import torch

from oracle import oracle as O
from qwfnfer_amd import qsa
from tests._gpu import make_pair, np_of

pytestmark = pytest.mark.gpu

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rope_of(rd, layout="half", **kw):
    return qsa.Rope(qsa.RopeConfig(rope_dim=rd, base=1e6, layout=layout, norm_eps=EPS, **kw))


def part_turns(pos, turns):
    """pos * turns less its whole turns, float64 [n, pairs], the product exact (in integers)."""
    got = np.empty((len(pos), len(turns)))
    for i, t in enumerate(turns):
        num, den = float(t).as_integer_ratio()
        for j, p in enumerate(pos):
            r = int(p) * num % den
            got[j, i] = (r if 2 * r <= den else r - den) / den
    return got


def turned(rope, x, pos, norm=None, inverse=False):
    """float64 [n, heads, hd]: normed and turned, from the definition."""
    x = x.detach().cpu().double().numpy()
    if norm is not None:
        eps = float(np.float32(EPS))
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.cpu().double().numpy()
    rd, half = rope.cfg.rope_dim, rope.cfg.rope_dim // 2
    a = 2 * math.pi * part_turns(pos, rope.turns.cpu().tolist()) * (-1 if inverse else 1)
    m = float(np.float32(rope.cfg.scale()))
    c, s = np.cos(a)[:, None] * m, np.sin(a)[:, None] * m
    i = np.arange(half)
    p, q = (i, i + half) if rope.cfg.layout == "half" else (2 * i, 2 * i + 1)
    y = x.copy()
    y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., q] * c + x[..., p] * s
    return y


def check_rows(got, want, dtype):
    """One rounding to fp32 and one to the row's type, each at most half a step; the 64-bit evaluation
    itself is off by a few 2^-52 of the pair's size (1e-14 covers both sides' steps).  Below a type's
    normal range a step is absolute: half of the smallest subnormal."""
    got = got.detach().cpu().double().numpy()
    step = 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    size = np.abs(want).max(axis=-1, keepdims=True)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > step * np.abs(want) * (1 + 2.0 ** -20) + 1e-14 * size + tiny
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want).max()))


def positions(n, far, seed=0):
    return torch.from_numpy((np.random.default_rng(seed).integers(0, 1000, n) + far).astype(np.int32)).cuda()


@pytest.mark.parametrize("hd,rd", [(128, 128), (128, 64), (64, 64), (256, 256), (256, 64), (128, 32), (128, 2), (128, 126),
                                   (96, 40), (80, 80), (3, 2), (512, 512), (127, 64)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
def test_rows_shapes(hd, rd, layout, norm):
    gen = torch.Generator(device="cuda").manual_seed(hd + rd)
    rope = rope_of(rd, layout)
    x = torch.randn(37, 3, hd, device="cuda", generator=gen)
    w = torch.rand(hd, device="cuda", generator=gen) + 0.5 if norm else None
    pos = positions(37, 5000)
    check_rows(qsa.rope_rows(rope, x, pos, norm=w), turned(rope, x, np_of(pos), w), torch.float32)


@pytest.mark.parametrize("src", list(TYPES))
@pytest.mark.parametrize("dst", list(TYPES))
@pytest.mark.parametrize("rd,layout", [(128, "half"), (64, "interleaved"), (36, "half")])
def test_rows_types(src, dst, rd, layout):
    gen = torch.Generator(device="cuda").manual_seed(5)
    rope = rope_of(rd, layout, scaling="yarn", factor=8.0)
    x = torch.randn(70, 4, 128, device="cuda", generator=gen).to(TYPES[src])
    pos = positions(70, 100000)
    out = torch.empty(70, 4, 128, dtype=TYPES[dst], device="cuda")
    assert qsa.rope_rows(rope, x, pos, out=out) is out
    check_rows(out, turned(rope, x, np_of(pos)), TYPES[dst])


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 64, 65, 1000])
@pytest.mark.parametrize("heads", [1, 16])
def test_rows_counts(n, heads):
    gen = torch.Generator(device="cuda").manual_seed(n)
    rope = rope_of(128)
    x = torch.randn(n, heads, 128, device="cuda", generator=gen).bfloat16()
    pos = positions(n, 3)
    check_rows(qsa.rope_rows(rope, x, pos), turned(rope, x, np_of(pos)), torch.bfloat16)


def test_rows_of_many_heads():
    """More groups of heads than a grid's second dimension holds."""
    rope = rope_of(64)
    x = torch.randn(2, 300000, 64, device="cuda").half()
    pos = torch.tensor([7, 70000], dtype=torch.int32, device="cuda")
    check_rows(qsa.rope_rows(rope, x, pos), turned(rope, x, np_of(pos)), torch.float16)


def test_rows_extreme_positions():
    rope = rope_of(128)
    x = torch.randn(6, 2, 128, device="cuda")
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1], dtype=torch.int32, device="cuda")
    got = qsa.rope_rows(rope, x, pos)
    check_rows(got, turned(rope, x, np_of(pos)), torch.float32)
    assert torch.equal(got[0], x[0])                     # position 0 turns nothing


@pytest.mark.parametrize("off", [0, 1, 3])
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_rows_strides_and_alignment(off, src):
    """Rows of a fused projection, heads first, and rows that begin at an odd element."""
    gen = torch.Generator(device="cuda").manual_seed(off)
    rope, pos = rope_of(128), positions(33, 77)
    buf = torch.randn(33 * 20 * 128 + 8, device="cuda", generator=gen).to(TYPES[src])
    x = buf[off:off + 33 * 20 * 128].view(33, 20, 128)[:, 2:18]
    want = turned(rope, x, np_of(pos))
    check_rows(qsa.rope_rows(rope, x, pos), want, TYPES[src])
    heads_first = torch.zeros(16, 33 + 1, 132, device="cuda", dtype=TYPES[src]).transpose(0, 1)[:33, :, off:off + 128]
    qsa.rope_rows(rope, x, pos, out=heads_first)
    check_rows(heads_first, want, TYPES[src])
    same = x.clone(memory_format=torch.preserve_format)
    check_rows(qsa.rope_rows(rope, heads_first, pos * 0), np_of(heads_first.double()), TYPES[src])
    keep = buf.clone()
    qsa.rope_rows(rope, x, pos, out=x)                   # in place; the columns beside it stay
    check_rows(x, want, TYPES[src])
    keep[off:off + 33 * 20 * 128].view(33, 20, 128)[:, 2:18] = x
    assert torch.equal(keep, buf) and not torch.equal(same, x)


def test_rows_inverse_undoes_and_is_the_gradient():
    rope, pos = rope_of(64, "interleaved"), positions(50, 12345)
    x = torch.randn(50, 4, 128, device="cuda")
    y = qsa.rope_rows(rope, x, pos)
    back = qsa.rope_rows(rope, y, pos, inverse=True)
    # each way rounds once: 2^-24 of a value, turned into its pair partner by the second
    assert (back - x).abs().max() <= 3 * 2.0 ** -24 * x.abs().max()
    # <g, R x> = <R^T g, x> for every g: the inverse is the gradient of rows that are not normed
    g = torch.randn_like(x)
    gx = qsa.rope_rows(rope, g, pos, inverse=True)
    check_rows(gx, turned(rope, g, np_of(pos), inverse=True), torch.float32)
    lhs, rhs = (g.double() * y.double()).sum(-1), (gx.double() * x.double()).sum(-1)
    # y and gx are rounded once; a turned value is at most sqrt(2) of its row's largest
    bound = 3 * 2.0 ** -24 * (g.double().abs() @ torch.ones(128, dtype=torch.float64, device="cuda")) * x.abs().max()
    assert ((lhs - rhs).abs() <= bound).all()
    # and by differences, in the direction e: R is linear, so (R(x + e) - R(x)) . g is e . gx to rounding
    e = torch.randn_like(x)
    diff = (qsa.rope_rows(rope, x + e, pos).double() - y.double()) * g.double()
    dots = ((x + e).double() - x.double()) * gx.double()
    size = ((x + e).abs().max() + x.abs().max() + e.abs().max()).double()
    assert ((diff.sum(-1) - dots.sum(-1)).abs() <= 4 * 2.0 ** -24 * size * g.double().abs().sum(-1)).all()


def test_rows_nan_stays_in_its_pair():
    rope, pos = rope_of(64), positions(5, 9)
    x = torch.randn(5, 2, 128, device="cuda")
    x[1, 0, 3] = math.nan
    x[2, 1, 100] = math.inf
    got = np_of(qsa.rope_rows(rope, x, pos))
    bad = ~np.isfinite(got)
    want = np.zeros_like(bad)
    want[1, 0, [3, 35]] = True
    want[2, 1, 100] = True
    assert (bad == want).all()


def test_rows_refuse_partial_overlap():
    rope, pos = rope_of(128), positions(8, 0)
    buf = torch.randn(8 * 256 + 128, device="cuda")
    x, y = buf[:2048].view(8, 2, 128), buf[128:].view(8, 2, 128)
    with pytest.raises(qsa._lib.QsaError):
        qsa.rope_rows(rope, x, pos, out=y)
    with pytest.raises(qsa._lib.QsaError):
        qsa.rope_rows(rope, x, pos, out=x.view(8, 2, 128)[:, :1].expand(8, 2, 128))


# ---- the append ---------------------------------------------------------------

CONFIGS = {
    "base": dict(), "ckpt": dict(n_head=24, n_head_kv=2, head_dim=256, block_tokens=4),
    "small": dict(n_head=16, n_head_kv=2, head_dim=64), "wide": dict(n_head=16, n_head_kv=8),
    "ref": dict(quant_variant=O.Q8_REF_ROUNDF),
}


def rows(gen, n, heads, hd, dtype):
    """N(0, 1) by a log-uniform [0.1, 10] scale a 32-value block."""
    x = torch.randn(n, heads, hd // 32, 32, device="cuda", generator=gen)
    s = torch.empty(n, heads, hd // 32, 1, device="cuda").uniform_(math.log(0.1), math.log(10), generator=gen).exp_()
    return (x * s).reshape(n, heads, hd).to(dtype)


def run_append(cfg_kw, kv, n, io, rd, layout="half", norm=True, with_q=True, pos=None, seqs=None, n_seq=1, pps=4, fused=False):
    cfg = qsa.QsaConfig(**cfg_kw, kv_type=kv)
    H, Hkv, hd = cfg.n_head, cfg.n_head_kv, cfg.head_dim
    gen = torch.Generator(device="cuda").manual_seed(n + rd)
    rope = rope_of(rd, layout)
    if fused:
        x = rows(gen, n, H + 2 * Hkv, hd, TYPES[io])
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    else:
        q, k, v = (rows(gen, n, m, hd, TYPES[io]) for m in (H, Hkv, Hkv))
    kw = torch.rand(hd, device="cuda", generator=gen) + 0.5 if norm else None
    qw = torch.rand(hd, device="cuda", generator=gen) + 0.5 if norm else None
    pos = np.arange(n) if pos is None else np.asarray(pos)
    seqs = np.zeros(n) if seqs is None else np.asarray(seqs)
    dev, host = make_pair(cfg, n_seq, pps, seed=3)
    fill = np.random.default_rng(1).integers(0, 256, host.k_pages.size, dtype=np.uint8)
    host.k_pages[:], host.v_pages[:] = fill, fill[::-1]          # what no row writes must stay
    dev.k_pages.copy_(torch.from_numpy(host.k_pages))
    dev.v_pages.copy_(torch.from_numpy(host.v_pages))
    tp, ts = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (pos, seqs))
    q_out = qsa.append_rope(dev, rope, k, v, tp, ts, k_norm=kw, q=q if with_q else None, q_norm=qw if with_q else None)
    status = qsa.read_status(dev)
    want_k = turned(rope, k, pos, kw).astype(np.float32)
    assert host.append(want_k, np_of(v.float()), pos.astype(np.int32), seqs.astype(np.int32)) == status
    assert (np_of(dev.k_pages) == host.k_pages).all()
    assert (np_of(dev.v_pages) == host.v_pages).all()
    if with_q:
        assert q_out.dtype == torch.float32
        check_rows(q_out, turned(rope, q, pos, qw), torch.float32)
    else:
        assert q_out is None
    return status


@pytest.mark.parametrize("kv", [0, 1, 2])
@pytest.mark.parametrize("cfg", list(CONFIGS))
@pytest.mark.parametrize("io", list(TYPES))
def test_append_bytes(kv, cfg, io):
    hd = CONFIGS[cfg].get("head_dim", 128)
    assert run_append(CONFIGS[cfg], kv, 150, io, hd, fused=io == "bf16") == 0


@pytest.mark.parametrize("kv", [0, 1, 2])
@pytest.mark.parametrize("rd,layout", [(128, "interleaved"), (64, "half"), (64, "interleaved"), (32, "half"), (16, "half"),
                                       (2, "half"), (90, "half"), (90, "interleaved"), (96, "half"), (8, "interleaved")])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rotations(kv, rd, layout, norm):
    assert run_append({}, kv, 70, "f16", rd, layout, norm) == 0


@pytest.mark.parametrize("kv", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 2, 5, 31, 64, 65, 129, 700])
@pytest.mark.parametrize("with_q", [False, True])
def test_append_counts(kv, n, with_q):
    assert run_append({}, kv, n, "bf16", 128, with_q=with_q, fused=True) == 0


@pytest.mark.parametrize("kv", [0, 1, 2])
@pytest.mark.parametrize("start", [1, 3, 61, 255, 300])
def test_append_runs_that_start_inside_a_tile(kv, start):
    """A chunk continues where the last one ended: tiles and pages begin and end inside it."""
    assert run_append({}, kv, 200, "f32", 128, pos=np.arange(200) + start) == 0


@pytest.mark.parametrize("kv", [0, 1, 2])
def test_append_scattered(kv):
    """Rows of several sequences in any order, positions out of order, a permuted page table."""
    rng = np.random.default_rng(kv)
    seqs = rng.integers(0, 3, 180)
    pos = rng.permutation(1024)[:180]
    assert run_append({}, kv, 180, "bf16", 128, pos=pos, seqs=seqs, n_seq=3) == 0
    # one run but for two rows that have changed places
    pos = np.arange(180) + 7
    pos[[20, 90]] = pos[[90, 20]]
    assert run_append({}, kv, 180, "bf16", 128, pos=pos) == 0


@pytest.mark.parametrize("kv", [0, 1, 2])
def test_append_skips_bad_rows(kv):
    """Bad positions and sequences inside a run: their rows are skipped and reported, the others written."""
    pos, seqs = np.arange(150) + 3, np.zeros(150)
    pos[17], pos[40] = -1, 1024
    seqs[60], seqs[101] = 1, -5
    got = run_append({}, kv, 150, "f32", 128, pos=pos, seqs=seqs)
    assert got == qsa._lib.STATUS_POS_RANGE | qsa._lib.STATUS_SEQ_RANGE


@pytest.mark.parametrize("kv", [0, 2])
def test_append_page_given_back(kv):
    cfg = qsa.QsaConfig(kv_type=kv)
    table = torch.tensor([[2, -1, 0, 7]], dtype=torch.int32)
    c = qsa.KvCache.allocate(cfg, 1, 4, page_table=table, n_phys_pages=4)
    rope = rope_of(128)
    k = torch.randn(600, 2, 128, device="cuda")
    qsa.append_rope(c, rope, k, k, torch.arange(200, 800, dtype=torch.int32, device="cuda"))
    assert qsa.read_status(c) == qsa._lib.STATUS_PAGE_RANGE
    pages = c.k_pages.view(4, -1)
    assert pages[2].any() and pages[0].any() and not pages[1].any() and not pages[3].any()


@pytest.mark.parametrize("kv", [0, 1, 2])
def test_append_non_finite_rows(kv):
    """What the plain append stores for a row, from the same 32-bit values."""
    cfg = qsa.QsaConfig(kv_type=kv)
    a, b = (qsa.KvCache.allocate(cfg, 1, 1) for _ in range(2))
    rope = rope_of(128)
    k = torch.randn(80, 2, 128, device="cuda")
    k[5, 0, 7], k[6, 1, 70], k[70, 0, 0] = math.nan, math.inf, -math.inf
    k[30] = 0
    pos = torch.arange(80, dtype=torch.int32, device="cuda")
    qsa.append_rope(a, rope, k, k, pos)
    qsa.append_q8_0(b, qsa.rope_rows(rope, k, pos), k, pos)
    if kv == 2:                                          # a NaN's payload bits are its own
        for x, y in ((a.k_pages, b.k_pages), (a.v_pages, b.v_pages)):
            assert torch.equal(torch.nan_to_num(x.view(torch.float16), nan=7.0), torch.nan_to_num(y.view(torch.float16), nan=7.0))
    else:
        assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)


@pytest.mark.parametrize("kv", [0, 1, 2])
@pytest.mark.parametrize("types,off", [(("f32", "bf16", "bf16"), 0), (("bf16", "f16", "f32"), 0), (("bf16", "bf16", "bf16"), 3),
                                       (("f16", "f32", "f32"), 1)])
def test_append_mixed_types_and_alignment(kv, types, off):
    """Sources of several types, rows that begin at an odd element, a float16 q_out with gaps between heads."""
    cfg = qsa.QsaConfig(kv_type=kv)
    rope = rope_of(128)
    gen = torch.Generator(device="cuda").manual_seed(off)
    n = 90

    def source(heads, t):
        buf = torch.empty(n * heads * 160 + 8, device="cuda", dtype=TYPES[t])
        x = buf[off:off + n * heads * 160].view(n, heads, 160)[:, :, :128]
        x.copy_(rows(gen, n, heads, 128, TYPES[t]))
        return x

    q, k, v = (source(h, t) for h, t in zip((16, 2, 2), types))
    pos = torch.arange(5, 5 + n, dtype=torch.int32, device="cuda")
    a, b = (qsa.KvCache.allocate(cfg, 1, 1) for _ in range(2))
    q_out = torch.zeros(n, 16, 192, dtype=torch.float16, device="cuda")[:, :, 32:160]
    assert qsa.append_rope(a, rope, k, v, pos, q=q, q_out=q_out) is q_out
    check_rows(q_out, turned(rope, q, np_of(pos)), torch.float16)
    turned_k = torch.from_numpy(turned(rope, k, np_of(pos)).astype(np.float32)).cuda()
    qsa.append_q8_0(b, turned_k, v.float().contiguous(), pos)
    assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)


def test_append_captured_and_replayed():
    """One graph, replayed with new rows and positions between eager work, each replay against eager calls."""
    cfg = qsa.QsaConfig()
    rope = rope_of(128)
    c, e = (qsa.KvCache.allocate(cfg, 4, 4) for _ in range(2))
    x = torch.randn(4, 20, 128, device="cuda").bfloat16()
    pos, seq = torch.tensor([0, 10, 200, 999], dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    q_out = torch.zeros(4, 16, 128, device="cuda")
    args = dict(q=x[:, :16], q_out=q_out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qsa.append_rope(c, rope, x[:, 16:18], x[:, 18:], pos, seq, **args)
    torch.cuda.current_stream().wait_stream(side)
    qsa.append_rope(e, rope, x[:, 16:18], x[:, 18:], pos, seq)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qsa.append_rope(c, rope, x[:, 16:18], x[:, 18:], pos, seq, **args)
    for step in range(4):
        x.copy_(torch.randn(4, 20, 128, device="cuda"))
        pos.copy_(torch.tensor([step, 11 + step, 255 + step, 1000 + step], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = qsa.append_rope(e, rope, x[:, 16:18], x[:, 18:], pos, seq, q=x[:, :16])
        assert torch.equal(q_out, want)
        assert torch.equal(c.k_pages, e.k_pages) and torch.equal(c.v_pages, e.v_pages)
