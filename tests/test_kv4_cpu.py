"""Refusals of the 4-bit cache operators, and their host-side arithmetic: no GPU needed, nothing is launched."""
import importlib
from fractions import Fraction

import numpy as np
import pytest
import torch

from conftest import load_pkg

FAKE = 1 << 20  # never dereferenced: validation fails first
ARG, UNSUPPORTED, WORKSPACE = -1, -2, -4


def _lib():
    return load_pkg().lib


def _store(**kw):
    a = dict(k=FAKE, v=FAKE, dtype=1, B=2, T=4, NH=2, D=64, k_sb=1536, k_st=384, k_sh=64, v_sb=1536, v_st=384, v_sh=64,
             codes=FAKE, params=FAKE, c_si=64, c_sb=32, c_sh=16, cap=16, starts=None, start=0, counts=None, weights=None,
             positions=None, w_sb=0, w_sh=0, seen=None, seen0=0, stream=None)
    a.update(kw)
    return _lib().attn_kv4_store(*a.values())


def _load(**kw):
    a = dict(codes=FAKE, params=FAKE, c_si=64, c_sb=32, c_sh=16, cap=16, B=2, T=4, NH=2, D=64, starts=None, start=0,
             counts=None, k=FAKE, v=FAKE, dtype=0, o_sb=512, o_st=128, o_sh=64, stream=None)
    a.update(kw)
    return _lib().attn_kv4_load(*a.values())


def _decode(**kw):
    a = dict(q=FAKE, codes=FAKE, params=FAKE, o=FAKE, lse=None, B=2, NH=4, NKV=2, L=9, D=64, q_sb=256, q_sh=64, o_sb=256,
             o_sh=64, c_si=64, c_sb=32, c_sh=16, cap=16, lengths=None, w_in=None, w_out=None, w_sb=0, w_sh=0, scale=0.125,
             dtype=1, ws=FAKE, ws_bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib().attn_kv4_decode(*a.values())


def _weights(**kw):
    a = dict(q=FAKE, k=FAKE, lse=FAKE, w_in=None, w_out=FAKE, B=1, NH=4, NKV=2, T=8, D=64, q_sb=2048, q_st=256, q_sh=64,
             k_sb=1024, k_st=128, k_sh=64, w_sb=16, w_sh=8, first=0, lengths=None, scale=0.125, dtype=0, ws=FAKE, ws_bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib().attn_key_weights(*a.values())


def _evict(**kw):
    a = dict(codes=FAKE, params=FAKE, weights=FAKE, positions=FAKE, c_si=64, c_sb=32, c_sh=16, cap=16, w_sb=32, w_sh=16,
             dc=None, dp=None, dw=None, dpos=None, d_si=0, d_sb=0, d_sh=0, dcap=0, dw_sb=0, dw_sh=0, B=2, NH=2, L=9, D=64,
             keep=4, recent=1, lengths=None, seen=None, seen0=9, slots=FAKE, ws=FAKE, ws_bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib().attn_kv4_evict(*a.values())


# one head over many rows: more splits than a cluster holds
LONG = dict(B=1, NH=1, NKV=1, L=32768, cap=32768, c_sh=32768, c_sb=32768, c_si=32768)

CACHE = [
    (dict(codes=None), ARG, "null"), (dict(params=None), ARG, "null"), (dict(D=48), UNSUPPORTED, "head_dim"),
    (dict(D=8), UNSUPPORTED, "head_dim"), (dict(D=256), UNSUPPORTED, "head_dim"), (dict(cap=17), ARG, "multiples of 16"),
    (dict(c_sh=24), ARG, "multiples of 16"), (dict(c_sb=33), ARG, "multiples of 16"), (dict(c_si=65), ARG, "multiples of 16"),
    (dict(cap=32), ARG, "stride"), (dict(codes=FAKE + 8), ARG, "aligned"), (dict(params=FAKE + 4), ARG, "aligned"),
    (dict(B=0), ARG, "positive"), (dict(B=-1), ARG, "positive"),
    (dict(cap=(1 << 30) + 16, c_sh=1 << 31, c_sb=1 << 32, c_si=1 << 33), ARG, "2^30"),
]


@pytest.mark.parametrize("call", [_store, _load, _decode, _evict])
@pytest.mark.parametrize("bad,code,text", CACHE)
def test_bad_caches_are_refused(call, bad, code, text):
    L = _lib()
    before = load_pkg().launch_count()
    assert call(**bad) == code
    assert text in L.attn_last_error_string().decode()
    assert load_pkg().launch_count() == before


@pytest.mark.parametrize("call,bad,code,text", [
    (_store, dict(k=None), ARG, "null"), (_store, dict(v=None), ARG, "null"), (_store, dict(dtype=2), ARG, "dtype"),
    (_store, dict(T=0), ARG, "positive"), (_store, dict(k_st=-1), ARG, "negative"), (_store, dict(start=13), ARG, "capacity"),
    (_store, dict(start=-1), ARG, "capacity"), (_store, dict(T=17), ARG, "capacity"), (_store, dict(c_sb=0), ARG, "overlap"),
    (_store, dict(c_si=0), ARG, "overlap"), (_store, dict(B=1 << 16, T=1 << 14, NH=4), ARG, "2^31"),
    (_store, dict(k=FAKE + 1), ARG, "misaligned"), (_store, dict(weights=FAKE, w_sb=-1), ARG, "strides"),
    (_load, dict(k=None), ARG, "null"), (_load, dict(dtype=2), ARG, "dtype"), (_load, dict(start=13), ARG, "capacity"),
    (_load, dict(o_st=-1), ARG, "negative"), (_load, dict(T=0), ARG, "positive"),
    (_decode, dict(q=None), ARG, "null"), (_decode, dict(o=None), ARG, "null"), (_decode, dict(dtype=2), ARG, "dtype"),
    (_decode, dict(NH=3), ARG, "multiple"), (_decode, dict(NKV=0), ARG, "multiple"), (_decode, dict(L=0), ARG, "length"),
    (_decode, dict(L=17), ARG, "length"), (_decode, dict(q_sb=-1), ARG, "negative"), (_decode, dict(w_in=FAKE), ARG, "weights_out"),
    (_decode, dict(ws=None, **LONG), WORKSPACE, "workspace"), (_decode, dict(ws_bytes=16, **LONG), WORKSPACE, "workspace"),
    (_decode, dict(ws=FAKE + 4), ARG, "aligned"),
    (_decode, dict(w_out=FAKE), ARG, "overlap"), (_decode, dict(w_out=FAKE, w_sb=32, w_sh=8), ARG, "overlap"),
    (_decode, dict(o_sh=0), ARG, "overlap"), (_weights, dict(w_sh=0), ARG, "overlap"), (_evict, dict(w_sb=0), ARG, "overlap"),
    (_store, dict(weights=FAKE, w_sb=32, w_sh=8), ARG, "overlap"), (_store, dict(positions=FAKE), ARG, "overlap"),
    (_weights, dict(q=None), ARG, "null"), (_weights, dict(w_out=None), ARG, "null"), (_weights, dict(dtype=5), ARG, "dtype"),
    (_weights, dict(T=(1 << 30) + 1, w_sh=1 << 31, w_sb=1 << 32), ARG, "2^30"),
    (_weights, dict(NH=3), ARG, "multiple"), (_weights, dict(first=-1), ARG, "first_query"), (_weights, dict(T=0), ARG, "positive"),
    (_weights, dict(D=160), UNSUPPORTED, "head_dim"), (_weights, dict(T=4096, w_sh=4096, ws_bytes=4), WORKSPACE, "workspace"), (_weights, dict(k_st=-1), ARG, "negative"),
    (_evict, dict(weights=None), ARG, "null"), (_evict, dict(slots=None), ARG, "null"), (_evict, dict(L=17), ARG, "length"),
    (_evict, dict(L=0), ARG, "length"), (_evict, dict(keep=0), ARG, "keep"), (_evict, dict(keep=17), ARG, "keep"),
    (_evict, dict(recent=5), ARG, "recent"), (_evict, dict(recent=-1), ARG, "recent"), (_evict, dict(L=20000, cap=20000, c_sh=20000, c_sb=40000, c_si=80000, ws=None), WORKSPACE, "workspace"),
    (_evict, dict(L=20000, cap=20000, c_sh=20000, c_sb=40000, c_si=80000, ws_bytes=4), WORKSPACE, "workspace"), (_evict, dict(c_sb=0), ARG, "overlap"),
    (_evict, dict(dc=FAKE, dp=2 * FAKE, dw=2 * FAKE, d_si=64, d_sb=32, d_sh=16, dcap=16), ARG, "another cache"),
    (_evict, dict(dc=2 * FAKE, dp=2 * FAKE, dw=None, d_si=64, d_sb=32, d_sh=16, dcap=16), ARG, "null"),
    (_evict, dict(dc=2 * FAKE, dp=2 * FAKE, dw=2 * FAKE, d_si=64, d_sb=32, d_sh=16, dcap=8), ARG, "multiples of 16"),
])
def test_bad_arguments_are_refused(call, bad, code, text):
    L = _lib()
    before = load_pkg().launch_count()
    assert call(**bad) == code
    assert text in L.attn_last_error_string().decode()
    assert load_pkg().launch_count() == before


def test_workspace_sizes_of_nothing():
    L = _lib()
    assert L.attn_kv4_decode_workspace_size(0, 8, 8, 10, 64, 1, 1) == 0
    assert L.attn_kv4_decode_workspace_size(1, 8, 3, 10, 64, 1, 1) == 0
    assert L.attn_kv4_evict_workspace_size(1, 8, 10, 0) == 0


def test_wrappers_refuse_host_tensors_and_wrong_types():
    ops = load_pkg().mha_ops
    codes = torch.zeros((2, 1, 1, 16, 32), dtype=torch.uint8)
    params = torch.zeros((2, 1, 1, 16, 1, 2), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_decode(torch.zeros((1, 1, 64)), codes, params, 4)
    with pytest.raises(TypeError, match="uint8"):
        ops.kv4_decode(torch.zeros((1, 1, 64)), codes.int(), params, 4)
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv4_empty(1, 1, 16, 48)
    c, p = ops.kv4_empty(2, 3, 17, 128, device="cpu")
    assert c.shape == (2, 2, 3, 32, 64) and p.shape == (2, 2, 3, 32, 2, 2)


def test_cache_class_refuses_bad_sizes():
    KV4Cache = load_pkg().KV4Cache
    for bad in (dict(B=0), dict(max_len=0), dict(NH=0), dict(prompt_window=0), dict(D=24)):
        a = dict(B=1, max_len=8, NH=2, D=64)
        a.update(bad)
        with pytest.raises(ValueError):
            KV4Cache(**a)


def _code(x, s, m):
    """kv4_code_exact's float32 steps (csrc/kv4.cuh), in NumPy."""
    f = np.float32
    d = f(x - m)
    bb = f(d - x)
    e = f(f(x - f(d - bb)) - f(m + bb))
    n = f(min(max(np.rint(f(d * f(f(1) / s))), f(0)), f(15)))
    hi, lo = f(f(n + f(0.5)) * s), f(f(n - f(0.5)) * s)
    odd = int(n) & 1
    if d > hi or (d == hi and (e > 0 or (e == 0 and odd))):
        n += 1
    elif d < lo or (d == lo and (e < 0 or (e == 0 and odd))):
        n -= 1
    return int(min(max(n, 0), 15))


def test_code_steps_decide_exactly():
    """The float32 steps of the code against exact rational arithmetic: values at, and one float32 step
    to either side of, every border of two codes, for scales and minima over float16's range."""
    rng = np.random.default_rng(11)
    checked = 0
    for _ in range(300):
        s = np.float32(np.float16(2.0 ** rng.uniform(-20, 8)))
        m = np.float32(np.float16(rng.normal() * 2.0 ** rng.uniform(-8, 8)))
        for n in range(15):
            border = np.float32(m + np.float32(np.float32(n + 0.5) * s))
            for x in (np.nextafter(border, np.float32(-np.inf)), border, np.nextafter(border, np.float32(np.inf))):
                t = (Fraction(float(x)) - Fraction(float(m))) / Fraction(float(s))
                want = min(max(round(t), 0), 15)  # Fraction's round: half to even
                assert _code(x, s, m) == want, (x, s, m, n)
                checked += 1
                # the quick way round is only taken where it decides alike
                f = np.float32
                q = f(min(max(f(f(x - m) * f(f(f(1) / s) * f(1 / 15))), f(0)), f(1))) * f(15)
                if abs(f(q - np.rint(q))) <= f(0.49999):
                    assert int(np.rint(q)) == want, (x, s, m, n)
    assert checked == 300 * 45
