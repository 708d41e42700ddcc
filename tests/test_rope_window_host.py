"""The rotary and sliding-window calls on the host: frequency tables, sizes, and what is
refused before any launch (no GPU call is reached)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from qwfnfer_amd import _lib, qsa

EINVAL, ERANGE, ENOTSUP = _lib.QWFN_EINVAL, _lib.QWFN_ERANGE, _lib.QWFN_ENOTSUP


def _code(name, *args):
    rc = getattr(_lib.load(), name)(*args)
    if rc < 0:
        assert _lib.load().qwfn_qsa_last_error()
    return rc


# ---- frequencies ------------------------------------------------------------

def test_frequencies_unscaled_and_linear():
    f = qsa.RopeConfig(rope_dim=64, base=1e4).frequencies()
    want = 1e4 ** (-np.arange(32) * 2.0 / 64)
    np.testing.assert_allclose(f, want, rtol=4e-15)
    g = qsa.RopeConfig(rope_dim=64, base=1e4, scaling="linear", factor=4.0)
    np.testing.assert_allclose(g.frequencies(), want / 4, rtol=4e-15)
    assert g.scale() == 1.0


def test_frequencies_yarn():
    c = qsa.RopeConfig(rope_dim=128, base=1e4, scaling="yarn", factor=16.0, trained_tokens=4096)
    f, plain = np.array(c.frequencies()), 1e4 ** (-np.arange(64) / 64.0)
    turns = 4096 * plain / (2 * math.pi)                 # over the trained length
    assert np.allclose(f[turns > 40], plain[turns > 40], rtol=1e-14)           # fast pairs stay
    assert np.allclose(f[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-14)    # slow pairs are stretched
    ratio = f / plain
    # two evaluations of a power, each within a unit in the last place (2^-52 of it): quotients within 2^-50
    assert (np.diff(ratio) <= 2 ** -50).all() and ratio.max() <= 1 + 2 ** -50 and ratio.min() >= (1 - 2 ** -50) / 16
    assert c.scale() == pytest.approx(0.1 * math.log(16) + 1)
    assert qsa.RopeConfig(scaling="yarn", factor=16.0, mscale=1.25).scale() == 1.25


def test_rope_config_refusals():
    for bad in (dict(rope_dim=0), dict(rope_dim=63), dict(layout="neox"), dict(scaling="ntk"), dict(base=1.0),
                dict(factor=0.0), dict(trained_tokens=0)):
        with pytest.raises(ValueError):
            qsa.RopeConfig(**bad)
    with pytest.raises(ValueError):
        qsa.Rope(qsa.RopeConfig(rope_dim=64), device="cpu", turns=torch.zeros(31))


# ---- the C entry points -----------------------------------------------------

def _rope(**kw):
    a = dict(rope_dim=128, layout=0, turns=4096, mscale=1.0, norm_eps=1e-6, **{})
    a.update(kw)
    return _lib.RopeStruct(a["rope_dim"], a["layout"], a["turns"], a["mscale"], a["norm_eps"])


def _rows(data=1 << 20, dtype=0, rs=2048, hs=128):
    return _lib.RowsStruct(data, dtype, rs, hs)


def _rope_rows(rope=None, src=None, pos=4096, n=4, heads=16, hd=128, dst=None, norm=None):
    return _code("qwfn_rope_rows", C.byref(rope or _rope()), C.byref(src or _rows()), norm, pos, n, heads, hd, 0,
                 C.byref(dst or _rows(data=1 << 24)), None)


@pytest.mark.parametrize("kw", [
    dict(rope=_rope(rope_dim=0)), dict(rope=_rope(rope_dim=63)), dict(rope=_rope(rope_dim=130)),
    dict(rope=_rope(layout=2)), dict(rope=_rope(turns=0)), dict(rope=_rope(turns=4100)),
    dict(rope=_rope(mscale=math.inf)), dict(rope=_rope(mscale=math.nan)), dict(rope=_rope(norm_eps=-1.0)),
    dict(src=_rows(data=0)), dict(src=_rows(dtype=3)), dict(src=_rows(dtype=-1)), dict(src=_rows(data=(1 << 20) + 2)),
    dict(src=_rows(rs=-1)), dict(src=_rows(hs=-128)), dict(src=_rows(rs=1 << 62)), dict(dst=_rows(data=0)),
    dict(pos=None), dict(pos=4098), dict(norm=4098), dict(n=0), dict(heads=0), dict(hd=0), dict(hd=513),
    dict(dst=_rows(data=1 << 24, rs=0)), dict(dst=_rows(data=1 << 24, hs=127)), dict(dst=_rows(data=1 << 24, rs=2047)),
    dict(dst=_rows(data=(1 << 20) + 4)),                        # overlaps src by all but a value
    dict(dst=_rows(dtype=1)),                                   # src's place with another type
    dict(dst=_rows(rs=2052)),                                   # src's place with another stride
])
def test_rope_rows_refusals(kw):
    assert _rope_rows(**kw) == EINVAL


def test_rope_rows_too_many():
    assert _rope_rows(n=1 << 30, heads=4, src=_rows(rs=512), dst=_rows(data=1 << 60, rs=512)) == ERANGE
    assert _rope_rows(n=1 << 24, heads=4, src=_rows(rs=512), dst=_rows(data=1 << 60, rs=512)) == ERANGE
    assert _append(n=1 << 22) == ERANGE


def _view(pps=4, n_seq=1, nphys=4, k=4096):
    return _lib.KvView(k, 8192, 16384, 4096, None, n_seq, pps, nphys)


def _append(cfg=qsa.QsaConfig(), view=None, rope=None, k=None, v=None, q=None, q_out=None, pos=4096, n=4, k_norm=None,
            q_norm=None):
    s = cfg.shape()
    ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
    return _code("qwfn_kv_append_rope", C.byref(s), C.byref(view or _view()), C.byref(rope or _rope()),
                 C.byref(k or _rows(rs=256)), C.byref(v or _rows(data=1 << 22, rs=256)), k_norm, None, pos, n, ref(q),
                 q_norm, ref(q_out), None)


@pytest.mark.parametrize("kw", [
    dict(view=_view(k=0)), dict(rope=_rope(rope_dim=256)), dict(k=_rows(data=0)), dict(v=_rows(dtype=7)), dict(pos=None),
    dict(n=0), dict(n=-3), dict(q=_rows()), dict(q_out=_rows()), dict(q_norm=4096), dict(k_norm=4097),
    dict(q=_rows(data=1 << 24), q_out=_rows(data=1 << 24)),                    # q_out is q
    dict(q=_rows(data=1 << 24), q_out=_rows(data=1 << 22)),                    # q_out is v
    dict(q=_rows(data=1 << 24), q_out=_rows(data=1 << 26, rs=100)),
    dict(cfg=qsa.QsaConfig(head_dim=100)),
])
def test_append_rope_refusals(kw):
    assert _append(**kw) == EINVAL


def _attn(decode=True, cfg=qsa.QsaConfig(), view=None, q=1 << 20, dtype=0, q_start=4096, seq_len=4096, n_seq=1, n_rows=8,
          max_q=8, max_len=1024, window=100, sinks=0, out=1 << 24, ws=1 << 28, nbytes=1 << 30):
    s, v = cfg.shape(), view or _view(n_seq=2)
    if decode:
        return _code("qwfn_window_attn_decode", C.byref(s), C.byref(v), q, dtype, seq_len, n_seq, max_len, window, sinks,
                     out, ws, nbytes, None)
    return _code("qwfn_window_attn_prefill", C.byref(s), C.byref(v), q, dtype, q_start, seq_len, n_seq, n_rows, max_q,
                 max_len, window, sinks, out, ws, nbytes, None)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("kw,code", [
    (dict(view=_view(k=0)), EINVAL), (dict(q=None), EINVAL), (dict(q=(1 << 20) + 4), EINVAL), (dict(dtype=3), EINVAL),
    (dict(seq_len=None), EINVAL), (dict(n_seq=0), EINVAL), (dict(n_seq=3), EINVAL), (dict(max_len=0), EINVAL),
    (dict(max_len=1025), ERANGE), (dict(window=0), EINVAL), (dict(window=-1), EINVAL), (dict(sinks=-1), EINVAL),
    (dict(out=None), EINVAL), (dict(out=(1 << 24) + 8), EINVAL), (dict(out=1 << 20), EINVAL),
    (dict(out=(1 << 20) + 4096), EINVAL), (dict(ws=None), EINVAL), (dict(ws=(1 << 28) + 16), EINVAL),
    (dict(nbytes=16), ERANGE), (dict(view=_view(n_seq=5000), n_seq=2049), ERANGE),
])
def test_window_refusals(decode, kw, code):
    assert _attn(decode, **kw) == code


def test_window_prefill_refusals():
    assert _attn(False, q_start=None) == EINVAL
    assert _attn(False, n_rows=0) == EINVAL
    assert _attn(False, max_q=0) == EINVAL
    assert _attn(False, n_rows=1 << 28) == ERANGE
    assert _attn(False, n_rows=1 << 22) == ERANGE


def test_window_workspace_sizes():
    cfg = qsa.QsaConfig()
    one = cfg.window_workspace_bytes(1, 1, 1, 4096, 1024)
    assert 0 < one <= cfg.window_workspace_bytes(64, 64, 1, 4096, 1024)
    # a workspace for a prefill also serves the decode of its sequences
    assert cfg.window_workspace_bytes(8, 8, 1, 4096, 1024) <= cfg.window_workspace_bytes(8, 800, 100, 4096, 1024)
    for bad in (dict(n_seq=0), dict(n_rows=0), dict(max_q=0), dict(max_seq_len=0), dict(window=0), dict(sink_tokens=-1)):
        a = dict(n_seq=1, n_rows=1, max_q=1, max_seq_len=64, window=8, sink_tokens=0)
        with pytest.raises(_lib.QsaError):
            cfg.window_workspace_bytes(**{**a, **bad})
    with pytest.raises(TypeError):
        cfg.window_workspace_bytes(1, 1, 1, 64, 8, dtype=torch.float64)


# ---- the Python calls -------------------------------------------------------

def _cpu_cache(cfg=qsa.QsaConfig()):
    z = torch.zeros(4 * cfg.page_bytes(), dtype=torch.uint8)
    return qsa.KvCache(cfg, z, z.clone(), torch.zeros(16), torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_python_calls_refuse_host_tensors_and_shapes():
    rope = qsa.Rope(qsa.RopeConfig(rope_dim=64), device="cpu")
    pos = torch.zeros(3, dtype=torch.int32)
    x = torch.zeros(3, 4, 128)
    for call in (lambda: qsa.rope_rows(rope, x, pos), lambda: qsa.rope_rows(rope, x[0], pos),
                 lambda: qsa.append_rope(_cpu_cache(), rope, x[:, :2], x[:, :2], pos),
                 lambda: qsa.append_rope(_cpu_cache(), rope, x[:, :2], x[:, :2], pos, q_norm=torch.ones(128)),
                 lambda: qsa.append_rope(_cpu_cache(), rope, x[:, :2], x[:, :2], pos, q_out=torch.zeros(3, 16, 128))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        qsa.rope_rows(rope, x.double(), pos)
    with pytest.raises(ValueError):
        qsa.window_attn_decode(_cpu_cache(), torch.zeros(1, 16, 128), torch.ones(1, dtype=torch.int32), 64, 8, None)


def test_no_rows_is_no_call():
    rope = qsa.Rope(qsa.RopeConfig(rope_dim=64), device="cpu")
    none = torch.zeros(0, dtype=torch.int32)
    assert qsa.rope_rows(rope, torch.zeros(0, 4, 128), none).shape == (0, 4, 128)
    assert qsa.append_rope(_cpu_cache(), rope, torch.zeros(0, 2, 128), torch.zeros(0, 2, 128), none) is None
