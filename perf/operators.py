"""Rotary positions, their append into the paged cache, and sliding-window attention over
it, as cases that can be timed and checked.

A case is one call of ``qwfnfer_amd.qsa``: ``rope_rows`` (path "rope"), ``append_rope``
("append"), ``window_attn_decode`` ("decode") or ``window_attn_prefill`` ("prefill").
Where ``own`` is false, :func:`run` computes the same from elementary torch operations.

A cache is two pools of pages as ``include/qwfn_qsa.h`` lays them out.  Sequences keep the
pages of their window and of their first tokens only; the others' entries of the page
table hold -1, as where a server has given those pages back.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

Q8_0, Q4_0, F16 = 0, 1, 2
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAGE = 256
EPS = 1e-6

# query heads, KV heads, head dimension, tokens of an indexer block (with whole 64-token
# blocks q8_0 keeps V dimension-major)
SHAPES = {"base": (16, 2, 128, 64), "ckpt": (24, 2, 256, 4), "small": (16, 2, 64, 64), "wide": (16, 8, 128, 64),
          "mid": (8, 2, 128, 64), "big": (16, 2, 256, 64)}


# ---- the cases -------------------------------------------------------------

def _named(name, **case):
    return dict(case, name=name) if name else case


def _rope(name=None, n=1, heads=16, hd=128, rd=128, layout="half", scaling="none", io="f32", out="f32", norm=False,
          inverse=False, far=0, fused=False):
    return _named(name, path="rope", n=n, heads=heads, hd=hd, rd=rd, layout=layout, scaling=scaling, io=io, out=out,
                  norm=norm, inverse=inverse, far=far, fused=fused)


def _append(name=None, n=1, prompt=False, far=0, spread=0, shape="base", kv=F16, rd=128, layout="half",
            scaling="none", io="f32", norm=True, fused=False):
    return _named(name, path="append", n=n, prompt=prompt, far=far, spread=spread, shape=shape, kv=kv, rd=rd,
                  layout=layout, scaling=scaling, io=io, norm=norm, fused=fused)


def _decode(name=None, longest=4096, shortest=None, n_seq=1, window=1024, sinks=0, shape="base", kv=Q8_0, io="f32",
            spread=0):
    return _named(name, path="decode", longest=longest, shortest=shortest or longest, n_seq=n_seq, window=window,
                  sinks=sinks, shape=shape, kv=kv, io=io, spread=spread)


def _prefill(name=None, past=0, n_q=1024, n_seq=1, window=1024, sinks=0, shape="base", kv=Q8_0, io="bf16", spread=0):
    return _named(name, path="prefill", past=past, n_q=n_q, n_seq=n_seq, window=window, sinks=sinks, shape=shape,
                  kv=kv, io=io, spread=spread)


def listed():
    return [
        # the queries of one token of a chat, all latency
        _rope("rope_token"),
        # a long document's chunk, far into it: queries as they leave a bfloat16 projection of Q, K and V
        # in one matrix, their norm and the scaled rotation of half the head
        _rope("rope_chunk", n=8192, rd=64, scaling="yarn", io="bf16", out="bf16", norm=True, far=131072, fused=True),
        # one token of a chat: its query turned, its K and V into the cache
        _append("append_token", far=4096),
        # a server's step: 64 sequences, one token each, at far and ragged positions
        _append("append_batch64", n=64, far=100000, spread=3, io="bf16", fused=True),
        # a prompt's chunk into the default cache type, read back as values
        _append("append_chunk", n=8000, prompt=True, kv=Q8_0, io="bf16", fused=True),
        # one token of a chat over a short window
        _decode("decode_token", longest=4096, window=1024),
        # the benchmark's batch of eight, short to very long, with four first tokens kept
        _decode("decode_batch8", longest=262144, shortest=1000, n_seq=8, window=4096, sinks=4, io="bf16", spread=5),
        # a server's batch over the default cache type
        _decode("decode_batch64", longest=100000, shortest=2000, n_seq=64, window=4096, sinks=64, io="bf16", spread=7),
        # the same over an fp16 cache of narrow heads, windows of no round length
        _decode("decode_f16_batch24", longest=40000, shortest=500, n_seq=24, window=2001, sinks=5, shape="small",
                kv=F16, io="f16", spread=9),
        # a prompt from nothing, of no round length, in the engine's own float32
        _prefill("prefill_prompt", n_q=3001, window=1000, sinks=4, io="f32"),
        # several users' turns in one call: a few hundred new tokens each over long chats
        _prefill("prefill_turns", past=30000, n_q=300, n_seq=6, window=2048, sinks=64, spread=2),
        # a chunk of a very long document
        _prefill("prefill_chunk", past=98304, n_q=8192, window=4096, sinks=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["rope", "append", "append", "decode", "decode", "decode", "prefill", "prefill", "prefill"])
    spread, io = rng.randrange(1000), rng.choice(["f32", "f16", "bf16", "bf16"])
    scaling, layout = rng.choice(["none", "linear", "yarn"]), rng.choice(["half", "half", "interleaved"])
    far, sinks = rng.choice([0, _log(rng, 100, 200000)]), rng.choice([0, 4, _log(rng, 1, 256)])
    shape = rng.choice(["base", "base", "base", "ckpt", "small", "wide", "mid", "big"])
    kv = rng.choice([Q8_0, Q8_0, Q4_0, F16])
    if path == "rope":
        hd = rng.choice([64, 128, 128, 256])
        return _rope(n=_log(rng, 1, 8192 * 128 // hd), heads=rng.choice([1, 2, 4, 16]), hd=hd,
                     rd=rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)]), layout=layout,
                     scaling=scaling, io=io, out=rng.choice([io, "f32"]), norm=rng.random() < 0.5,
                     inverse=rng.random() < 0.25, far=far, fused=rng.random() < 0.5)
    if path == "append":
        prompt = rng.random() < 0.6
        hd = SHAPES[shape][2]
        return _append(n=_log(rng, 2, 8000 * 128 // (hd * SHAPES[shape][1] // 2)) if prompt else _log(rng, 1, 64),
                       prompt=prompt, far=0 if prompt else far, spread=spread, shape=shape, kv=kv,
                       rd=rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)]), layout=layout,
                       scaling=scaling, io=io, norm=rng.random() < 0.5, fused=rng.random() < 0.5)
    if path == "decode":
        longest, (_, hkv, hd, _) = _log(rng, 100, 200000), SHAPES[shape]
        most = max(2, 64 * 256 // (hkv * hd) // (2 if kv == F16 else 1))
        return _decode(longest=longest, shortest=max(1, longest // rng.choice([1, 8, 64])),
                       n_seq=rng.choice([1, 1, _log(rng, 2, most)]), window=_log(rng, 1, 4096), sinks=sinks, shape=shape,
                       kv=kv, io=io, spread=spread)
    n_seq, (h, _, hd, _) = rng.choice([1, 1, rng.randint(2, 8)]), SHAPES[shape]
    return _prefill(past=rng.choice([0, _log(rng, 10, 100000)]), n_q=_log(rng, 2, (4000 if n_seq == 1 else 500) * 2048 // (h * hd)),
                    n_seq=n_seq, window=_log(rng, 1, 4096), sinks=sinks, shape=shape, kv=kv, io=io, spread=spread)


# ---- geometry of a case ----------------------------------------------------

def _up(x, m):
    return -(-x // m) * m


def _between(case, lo, hi, n, salt=0):
    """n numbers spread over [lo, hi] by their logarithm, the first of them hi."""
    r = random.Random(case["spread"] + salt)
    got = [int(round(math.exp(r.uniform(math.log(max(lo, 1)), math.log(max(hi, 1)))))) for _ in range(n)]
    got[0] = hi
    return got


def _lengths(case):
    """(tokens of each sequence with the new ones, new tokens of each)."""
    if case["path"] == "decode":
        got = _between(case, case["shortest"], case["longest"], case["n_seq"])
        return got, [1] * len(got)
    n_q = _between(case, 1, case["n_q"], case["n_seq"], 17)
    past = _between(case, case["past"] // 8, case["past"], case["n_seq"]) if case["past"] else [0] * case["n_seq"]
    return [p + n for p, n in zip(past, n_q)], n_q


def _row_bytes(kv, hd):
    return {Q8_0: hd, Q4_0: hd // 2, F16: 2 * hd}[kv]


def _vdim(case):
    """Whether V lies dimension-major in its 64-token tiles."""
    return case["kv"] == Q8_0 and SHAPES[case["shape"]][3] % 64 == 0


def _page_bytes(case):
    _, hkv, hd, _ = SHAPES[case["shape"]]
    quants = hkv * PAGE * _row_bytes(case["kv"], hd)
    return quants, quants + (0 if case["kv"] == F16 else hkv * PAGE * (hd // 32) * 2)


def _seen(case):
    """Cells that some new query of each sequence sees."""
    w, s = case["window"], case["sinks"]
    return [min(n, w + q - 1) + min(s, max(0, n - w - q + 1)) for n, q in zip(*_lengths(case))]


def _pairs(case):
    """(query, cell) pairs of a call, for each query head."""
    w, s, total = case["window"], case["sinks"], 0
    for n, q in zip(*_lengths(case)):
        p = np.arange(n - q, n, dtype=np.int64)
        total += int((np.minimum(p + 1, w) + np.minimum(s, np.maximum(0, p + 1 - w))).sum())
    return total


# ---- inputs ----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _freqs(case):
    """The rotation's angle a position of each pair, in radians, and the factor on cos and sin."""
    rd, base, factor, trained = case["rd"], 1e6, 8.0, 32768
    i = np.arange(rd // 2, dtype=np.float64)
    f = base ** (-2.0 * i / rd)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "none":
        return f, 1.0
    # YaRN: pairs that turn often in the trained length stay, those that turn less than once
    # are stretched by the factor, a ramp between them
    dim = [rd * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), rd - 1)
    ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
    return f / factor * ramp + f * (1.0 - ramp), 0.1 * math.log(factor) + 1.0


def _randn(gen, *size):
    return torch.randn(size, device="cuda", generator=gen)


def _rotation(case, gen, hd, state):
    f, mscale = _freqs(case)
    state["turns"] = torch.from_numpy(f / (2 * math.pi)).cuda()
    state["mscale"] = float(np.float32(mscale))
    if case["norm"]:
        state["norm"] = torch.rand(hd, device="cuda", generator=gen) + 0.5


def _handle(case):
    from qwfnfer_amd import qsa
    scaled = {} if case["scaling"] == "none" else {"scaling": case["scaling"], "factor": 8.0, "trained_tokens": 32768}
    return qsa.Rope(qsa.RopeConfig(rope_dim=case["rd"], base=1e6, layout=case["layout"], norm_eps=EPS, **scaled))


def _cache(case, state):
    """The framework's handle of the pages."""
    from qwfnfer_amd import qsa
    h, hkv, hd, bt = SHAPES[case["shape"]]
    cfg = qsa.QsaConfig(n_head=h, n_head_kv=hkv, head_dim=hd, block_tokens=bt, page_tokens=PAGE, kv_type=case["kv"])
    pooled = torch.zeros(16, device="cuda")          # no call here reads or writes pooled keys
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    return qsa.KvCache(cfg, state["k_pages"], state["v_pages"], pooled, state["table"], status)


def _prepare_rope(case, seed):
    gen, n, heads, hd = _gen(seed), case["n"], case["heads"], case["hd"]
    state = {"case": case}
    # the queries of a fused projection lie beside two heads of K and two of V
    x = _randn(gen, n, heads + 4 if case["fused"] else heads, hd).to(DTYPES[case["io"]])
    state["x"] = x[:, :heads]
    state["pos"] = torch.arange(case["far"], case["far"] + n, dtype=torch.int32, device="cuda")
    _rotation(case, gen, hd, state)
    state["out"] = torch.zeros((n, heads, hd), dtype=DTYPES[case["out"]], device="cuda")
    if own:
        state["rope"] = _handle(case)
    return state


def _prepare_append(case, seed):
    gen, n = _gen(seed), case["n"]
    h, hkv, hd, _ = SHAPES[case["shape"]]
    state = {"case": case}
    io = DTYPES[case["io"]]
    if case["fused"]:
        x = _randn(gen, n, h + 2 * hkv, hd).to(io)
        state["q"], state["k"], state["v"] = x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]
    else:
        state["q"], state["k"], state["v"] = (_randn(gen, n, m, hd).to(io) for m in (h, hkv, hkv))
    state["q_out"] = torch.zeros((n, h, hd), dtype=torch.float32, device="cuda")
    _rotation(case, gen, hd, state)
    if case["prompt"]:
        n_seq, pos = 1, list(range(n))
        pages = _up(n, PAGE) // PAGE
        table = torch.arange(pages, dtype=torch.int32).view(1, pages)
        state["seq_ids"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    else:
        n_seq, pos = n, _between(case, 1, max(1, case["far"]), n)
        pages = max(pos) // PAGE + 1
        table = torch.full((n_seq, pages), -1, dtype=torch.int32)
        perm = torch.randperm(n_seq, device="cuda", generator=gen).to(device="cpu", dtype=torch.int32)
        table[torch.arange(n_seq), torch.tensor(pos) // PAGE] = perm      # the page being written is there
        state["seq_ids"] = torch.arange(n, dtype=torch.int32, device="cuda")
    state["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
    state["table"] = table.cuda()
    phys = pages if case["prompt"] else n_seq
    state["k_pages"], state["v_pages"] = (torch.zeros(phys * _page_bytes(case)[1], dtype=torch.uint8, device="cuda")
                                          for _ in range(2))
    if own:
        state["rope"], state["cache"] = _handle(case), _cache(case, state)
        state["seq_len"] = torch.tensor([n], dtype=torch.int32, device="cuda") if case["prompt"] else state["pos"] + 1
        if not case["prompt"]:                        # the block that each token is in, to be read back after the call
            bt = SHAPES[case["shape"]][3]
            state["sel"] = (state["pos"] // bt).view(n, 1, 1).expand(n, hkv, 1).contiguous()
            state["n_sel"] = torch.ones((n, hkv), dtype=torch.int32, device="cuda")
            state["at"] = (state["pos"] % bt).long()
    return state


def _random_pages(case, gen, phys):
    """Pages of random rows: N(0, 1) by a log-uniform [0.25, 2] scale a 32-value block."""
    _, hkv, hd, _ = SHAPES[case["shape"]]
    quants, total = _page_bytes(case)
    scale = lambda *size: torch.empty(size, device="cuda").uniform_(math.log(0.25), math.log(2.0), generator=gen).exp_()  # noqa: E731
    if case["kv"] == F16:
        return (_randn(gen, phys, quants // 2) * scale(phys, quants // 64, 1).expand(-1, -1, 32).reshape(phys, -1)).half().view(torch.uint8).reshape(-1)
    pages = torch.empty((phys, total), dtype=torch.uint8, device="cuda")
    if case["kv"] == Q8_0:
        pages[:, :quants] = (_randn(gen, phys, quants) * 42).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        step = 42.0
    else:
        pages[:, :quants] = torch.randint(0, 256, (phys, quants), device="cuda", generator=gen, dtype=torch.int32).to(torch.uint8)
        step = 4.6
    pages[:, quants:] = (scale(phys, (total - quants) // 2) / step).half().view(torch.uint8)
    return pages.reshape(-1)


def _prepare_attn(case, seed):
    gen = _gen(seed)
    h, hkv, hd, _ = SHAPES[case["shape"]]
    lens, n_q = _lengths(case)
    state, n_seq, w = {"case": case}, len(lens), case["window"]
    pages = _up(max(lens), PAGE) // PAGE
    kept = []
    for s, (n, q) in enumerate(zip(lens, n_q)):
        p = set(range(max(0, n - q - w + 1) // PAGE, (n - 1) // PAGE + 1))
        kept += [(s, x) for x in sorted(p | set(range(_up(min(case["sinks"], n), PAGE) // PAGE)))]
    table = torch.full((n_seq, pages), -1, dtype=torch.int32)
    at = torch.tensor(kept)
    table[at[:, 0], at[:, 1]] = torch.randperm(len(kept), device="cuda", generator=gen).to(device="cpu", dtype=torch.int32)
    state["table"] = table.cuda()
    state["k_pages"], state["v_pages"] = (_random_pages(case, gen, len(kept)) for _ in range(2))
    state["seq_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state["max_len"] = pages * PAGE
    rows = sum(n_q)
    state["q"] = _randn(gen, rows, h, hd).to(DTYPES[case["io"]])
    state["out"] = torch.zeros_like(state["q"])
    if case["path"] == "prefill":
        state["q_start"] = torch.tensor([0, *np.cumsum(n_q).tolist()], dtype=torch.int32, device="cuda")
        state["max_q"] = max(n_q)
    if own:
        from qwfnfer_amd import qsa
        state["cache"] = _cache(case, state)
        state["ws"] = qsa.Workspace.for_window(state["cache"].cfg, n_seq, state["max_len"], w, case["sinks"],
                                               n_rows=rows, max_q=max(n_q), dtype=state["q"].dtype)
    return state


def prepare(case, seed):
    return {"rope": _prepare_rope, "append": _prepare_append}.get(case["path"], _prepare_attn)(case, seed)


# ---- one pass --------------------------------------------------------------

def _run_own(s):
    from qwfnfer_amd import qsa
    case = s["case"]
    if case["path"] == "rope":
        return qsa.rope_rows(s["rope"], s["x"], s["pos"], norm=s.get("norm"), out=s["out"], inverse=case["inverse"])
    if case["path"] == "append":
        qsa.append_rope(s["cache"], s["rope"], s["k"], s["v"], s["pos"], s["seq_ids"], k_norm=s.get("norm"),
                        q=s["q"], q_norm=s.get("norm"), q_out=s["q_out"])
        if case["kv"] == F16:
            return {"q": s["q_out"], "k": s["k_pages"].view(torch.float16), "v": s["v_pages"].view(torch.float16)}
        n, bt = case["n"], SHAPES[case["shape"]][3]
        if case["prompt"]:                            # the cache read back as values
            k, v, _ = qsa.gather_dequant(s["cache"], s["seq_len"], None, None, _up(n, bt) // bt)
            return {"q": s["q_out"], "k": k[0, :, :n].transpose(0, 1), "v": v[0, :, :n].transpose(0, 1)}
        k, v, _ = qsa.gather_dequant(s["cache"], s["seq_len"], s["sel"], s["n_sel"], 1)
        i = torch.arange(n, device="cuda")
        return {"q": s["q_out"], "k": k[i, :, s["at"]], "v": v[i, :, s["at"]]}
    if case["path"] == "decode":
        return qsa.window_attn_decode(s["cache"], s["q"], s["seq_len"], s["max_len"], case["window"], s["ws"],
                                      sink_tokens=case["sinks"], out=s["out"])
    return qsa.window_attn_prefill(s["cache"], s["q"], s["q_start"], s["seq_len"], s["max_q"], s["max_len"],
                                   case["window"], s["ws"], sink_tokens=case["sinks"], out=s["out"])


def run(s):
    if own:
        return _run_own(s)
    path = s["case"]["path"]
    if path == "rope":
        return _rotated(s["x"], s["case"], s).to(DTYPES[s["case"]["out"]])
    if path == "append":
        return _plain_append(s)
    return _plain_attn(s)


def _rotated(x, case, s):
    """The norm and the rotation in 64 bits (a value next to a rounding border decides a cached quant, and
    far positions need the angle), rounded once to 32."""
    x = x.double()
    if case["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["norm"].double()
    turns = s["pos"].double()[:, None] * s["turns"]
    angle = (turns - turns.round())[:, None] * (2 * math.pi)
    c, sn = torch.cos(angle) * s["mscale"], torch.sin(angle) * s["mscale"]
    if case.get("inverse"):
        sn = -sn
    rd = case["rd"]
    r = x[..., :rd]
    a, b = (r[..., :rd // 2], r[..., rd // 2:]) if case["layout"] == "half" else (r[..., 0::2], r[..., 1::2])
    ya, yb = a * c - b * sn, b * c + a * sn
    y = torch.cat([ya, yb], -1) if case["layout"] == "half" else torch.stack([ya, yb], -1).flatten(-2)
    return torch.cat([y, x[..., rd:]], -1).float()


def _as_cached(x, kv):
    """The 32-bit rows as the values the cache holds for them."""
    if kv == F16:
        return x.half()
    b = x.unflatten(-1, (-1, 32))
    if kv == Q8_0:
        amax = b.abs().amax(-1, keepdim=True)
        most = torch.full_like(amax, 127.0)           # by a tensor: a division by a number is a product with its inverse
        d = (amax / most).half().float()
        return (torch.round(b * torch.where(amax != 0, most / amax, 0.0)).clamp(-128, 127) * d).flatten(-2)
    big = torch.gather(b, -1, b.abs().argmax(-1, keepdim=True))
    d = big / -8.0
    q = (b * torch.where(d != 0, 1.0 / d, 0.0) + 8.5).trunc().clamp(max=15.0)
    return ((q - 8.0) * d.half().float()).flatten(-2)


def _plain_append(s):
    case = s["case"]
    q, k, v = _rotated(s["q"], case, s), _as_cached(_rotated(s["k"], case, s), case["kv"]), _as_cached(s["v"].float(), case["kv"])
    if case["kv"] != F16:
        return {"q": q, "k": k, "v": v}
    _, hkv, hd, _ = SHAPES[case["shape"]]
    page, row = s["table"][s["seq_ids"].long(), s["pos"].long() // PAGE].long(), s["pos"].long() % PAGE
    got = {"q": q}
    for name, x in (("k", k), ("v", v)):
        pages = s[name + "_pages"].view(torch.float16)
        tiles = pages.view(-1, hkv, PAGE // 64, hd // 8, 64, 8)
        tiles[page, :, row // 64, :, row % 64] = x.unflatten(-1, (hd // 8, 8))
        got[name] = pages
    return got


def _cells(case, pages, is_v, page, row):
    """Cached rows at (page, row) as 32-bit values: [..., KV heads, head dimension]."""
    _, hkv, hd, _ = SHAPES[case["shape"]]
    quants, total = _page_bytes(case)
    pages = pages.view(-1, total)
    raw, t, r = pages[:, :quants], row // 64, row % 64
    if case["kv"] == F16:
        return raw.view(torch.float16).view(-1, hkv, PAGE // 64, hd // 8, 64, 8)[page, :, t, :, r].flatten(-2).float()
    d = pages[:, quants:].view(torch.float16).view(-1, hkv, PAGE, hd // 32)[page, :, row].float()
    if case["kv"] == Q4_0:
        b = raw.view(-1, hkv, PAGE // 64, hd // 32, 64, 16)[page, :, t, :, r]
        x = torch.cat([b & 15, b >> 4], -1).float() - 8.0
    elif is_v and _vdim(case):
        x = raw.view(torch.int8).view(-1, hkv, PAGE // 64, hd, 64)[page, :, t, :, r].float().unflatten(-1, (-1, 32))
    else:
        x = raw.view(torch.int8).view(-1, hkv, PAGE // 64, hd // 16, 64, 16)[page, :, t, :, r].flatten(-2).float().unflatten(-1, (-1, 32))
    return (x * d[..., None]).flatten(-2)


def _plain_attn(s):
    case = s["case"]
    h, hkv, hd, _ = SHAPES[case["shape"]]
    lens = s["seq_len"].long()
    n_seq, g, w = len(lens), h // hkv, min(case["window"], s["max_len"])
    if case["path"] == "decode":
        n_q, start, max_q = torch.ones_like(lens), torch.arange(n_seq, device="cuda"), 1
    else:
        n_q, start, max_q = s["q_start"].diff().long(), s["q_start"][:-1].long(), s["max_q"]
    # the cells that a sequence's queries see: its first tokens, then the run that ends with its last
    i = torch.arange(max_q, device="cuda")
    first = (lens - n_q - w + 1).clamp(min=0)[:, None]
    sinks = torch.arange(case["sinks"], device="cuda").expand(n_seq, -1)
    run_ = first + torch.arange(min(w + max_q - 1, s["max_len"]), device="cuda")
    t = torch.cat([sinks, run_], 1)
    there = torch.cat([sinks < first, run_ < lens[:, None]], 1)
    at = s["table"].gather(1, (t // PAGE).clamp(max=s["table"].shape[1] - 1)).long().clamp(min=0)
    k, v = (_cells(case, s[m + "_pages"], m == "v", at, t % PAGE) for m in ("k", "v"))       # [seq, cell, KV head, dim]
    row = (start[:, None] + i).clamp(max=len(s["q"]) - 1)
    q = s["q"][row].float().unflatten(2, (hkv, g))                                          # [seq, query, KV head, group, dim]
    p = (lens - n_q)[:, None] + i
    seen = there[:, None] & (t[:, None] <= p[..., None]) & ((t[:, None] > p[..., None] - w) | (t[:, None] < case["sinks"]))
    logits = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(hd)
    logits = logits.unflatten(2, (g, max_q)).masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    o = torch.matmul(e.flatten(2, 3), v.transpose(1, 2).contiguous()).unflatten(2, (g, max_q)) / e.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                               # [seq, query, head, dim]
    return o[i < n_q[:, None]].to(s["q"].dtype)


# ---- from the definition, in 64 bits ---------------------------------------

def _exact_rotated(x, case, s):
    x = x.cpu().double().numpy()
    if case["norm"]:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * s["norm"].cpu().double().numpy()
    f, _ = _freqs(case)
    turn = np.exp(1j * np.outer(s["pos"].cpu().numpy().astype(np.float64), f) * (-1 if case.get("inverse") else 1)) * s["mscale"]
    y, half = x.copy(), case["rd"] // 2
    i = np.arange(half)
    a, b = (i, i + half) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    z = (x[..., a] + 1j * x[..., b]) * turn[:, None]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_cached(x, kv):
    x = x.astype(np.float32)
    if kv == F16:
        return x.astype(np.float16)
    b = x.reshape(-1, 32)
    if kv == Q8_0:
        amax = np.abs(b).max(1, keepdims=True)
        with np.errstate(divide="ignore"):
            inv = np.where(amax > 0, np.float32(127) / amax, np.float32(0))
        y = np.rint(b * inv).astype(np.float64) * (amax / np.float32(127)).astype(np.float16)
    else:
        big = b[np.arange(len(b)), np.abs(b).argmax(1)][:, None]
        d = big / np.float32(-8)
        with np.errstate(divide="ignore"):
            inv = np.where(d != 0, np.float32(1) / d, np.float32(0))
        y = (np.minimum(15, np.floor(b * inv + np.float32(8.5))).astype(np.float64) - 8) * d.astype(np.float16)
    return y.reshape(x.shape)


def _exact_append(case, s):
    k, v = _exact_cached(_exact_rotated(s["k"], case, s), case["kv"]), _exact_cached(s["v"].cpu().float().numpy(), case["kv"])
    q = _exact_rotated(s["q"], case, s)
    if case["kv"] != F16:
        return {"q": q, "k": k, "v": v}
    _, hkv, hd, _ = SHAPES[case["shape"]]
    table, pos, got = s["table"].cpu().numpy(), s["pos"].cpu().numpy(), {"q": q}
    page = table[s["seq_ids"].cpu().numpy(), pos // PAGE].astype(np.int64)[:, None, None]
    head, d, row = np.arange(hkv)[:, None], np.arange(hd), (pos % PAGE)[:, None, None]
    at = (((page * hkv + head) * (PAGE // 64) + row // 64) * (hd // 8) + d // 8) * 512 + row % 64 * 8 + d % 8
    for name, x in (("k", k), ("v", v)):
        pages = np.zeros(s[name + "_pages"].numel() // 2)
        pages[at.reshape(-1)] = x.reshape(-1)
        got[name] = pages.astype(np.float16)
    return got


def _exact_rows(case, pages, is_v, table_row, t, head):
    """Cells t of one KV head as 64-bit values, each byte by its place in the page."""
    _, hkv, hd, _ = SHAPES[case["shape"]]
    quants, total = _page_bytes(case)
    base, row, d = table_row[t // PAGE].long()[:, None] * total, (t % PAGE)[:, None], torch.arange(hd, device="cuda")
    tile = head * (PAGE // 64) + row // 64
    if case["kv"] == F16:
        at = base + ((tile * (hd // 8) + d // 8) * 64 + row % 64) * 16 + d % 8 * 2
        return pages.view(torch.float16)[at // 2].double()
    scale = pages.view(torch.float16)[(base + quants) // 2 + (head * PAGE + row) * (hd // 32) + d // 32].double()
    if case["kv"] == Q4_0:
        byte = pages[base + ((tile * (hd // 32) + d // 32) * 64 + row % 64) * 16 + d % 16].long()
        return scale * (torch.where(d % 32 < 16, byte % 16, byte // 16) - 8)
    if is_v and _vdim(case):
        at = base + (tile * hd + d) * 64 + row % 64
    else:
        at = base + ((tile * (hd // 16) + d // 16) * 64 + row % 64) * 16 + d % 16
    return scale * pages.view(torch.int8)[at]


def _exact_attn(case, s):
    h, hkv, hd, _ = SHAPES[case["shape"]]
    g, w = h // hkv, case["window"]
    lens, n_q = _lengths(case)
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for seq, (n, m) in enumerate(zip(lens, n_q)):
        for i in range(0, m, 512):                     # queries at a time
            p = torch.arange(n - m + i, n - m + min(m, i + 512), device="cuda")
            lo = max(0, int(p[0]) - w + 1)
            t = torch.cat([torch.arange(min(case["sinks"], lo), device="cuda"), torch.arange(lo, int(p[-1]) + 1, device="cuda")])
            hidden = (t > p[:, None]) | ((t <= p[:, None] - w) & (t >= case["sinks"]))
            rows = slice(at + i, at + i + len(p))
            for head in range(hkv):
                k, v = (_exact_rows(case, s[x + "_pages"], x == "v", s["table"][seq], t, head) for x in ("k", "v"))
                q = s["q"][rows, head * g:(head + 1) * g].double()
                logits = torch.tensordot(q, k, ([2], [1])) / math.sqrt(hd)
                weights = torch.softmax(logits.masked_fill(hidden[:, None], -math.inf), -1)
                out[rows, head * g:(head + 1) * g] = torch.tensordot(weights, v, ([2], [0]))
        at += m
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "rope":
        return _exact_rotated(s["x"], case, s)
    return _exact_append(case, s) if case["path"] == "append" else _exact_attn(case, s)


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["path"] == "rope":
        values = case["n"] * case["heads"] * case["hd"]
        return {"bytes": values * (size[case["io"]] + size[case["out"]]) + case["n"] * 4, "flops": 3 * values}
    h, hkv, hd, _ = SHAPES[case["shape"]]
    cell = hkv * (_row_bytes(case["kv"], hd) + (0 if case["kv"] == F16 else hd // 16))       # of K, or of V
    if case["path"] == "append":
        n = case["n"]
        back = 0 if case["kv"] == F16 else n * hkv * hd * 8                                  # read back as values
        return {"bytes": n * (h + 2 * hkv) * hd * size[case["io"]] + n * h * hd * 4 + 2 * n * cell + back,
                "flops": 3 * n * (h + hkv) * hd}
    rows = sum(_lengths(case)[1])
    return {"bytes": 2 * cell * sum(_seen(case)) + 2 * rows * h * hd * size[case["io"]], "flops": 4 * h * hd * _pairs(case)}
