"""Memory that a call of the 4-bit cache operators would write twice, or write while it reads it: refused on the
host.  Nothing is launched (every call that these checks let pass is stopped by a later one).  And torch without
the private names that the wrappers prefer."""
import random
import subprocess
import sys

import pytest

from conftest import ROOT, load_pkg
from test_kv4_cpu import ARG, FAKE, LONG, WORKSPACE, _decode, _evict, _load, _store, _weights

F = FAKE


def outcome(call, **kw):
    before = load_pkg().launch_count()
    code = call(**kw)
    assert load_pkg().launch_count() == before
    return code, load_pkg().lib.attn_last_error_string().decode()


@pytest.mark.parametrize("call,bad", [
    # two axes of one stride: head 1 of sequence 0 is head 0 of sequence 1
    (_store, dict(c_sb=16)), (_store, dict(c_si=32)), (_store, dict(c_si=16)), (_store, dict(c_si=48, c_sh=32, c_sb=16)),
    (_store, dict(weights=F, w_sb=16, w_sh=16)), (_store, dict(positions=F, w_sb=24, w_sh=16)),
    (_store, dict(weights=F, w_sb=16, w_sh=31)), (_store, dict(c_si=1 << 56)),
    (_load, dict(o_st=64)), (_load, dict(o_sb=256)), (_load, dict(o_sh=0)), (_load, dict(o_sb=0)), (_load, dict(o_st=0)),
    (_load, dict(k=F, v=F)), (_load, dict(k=F, v=F + 64 * 4)),
    (_decode, dict(o_sb=64)), (_decode, dict(o_sb=128, o_sh=64)), (_decode, dict(w_out=F, w_sb=9, w_sh=9)),
    (_decode, dict(w_out=F, w_in=F + 4, w_sb=32, w_sh=16)), (_decode, dict(w_out=F, w_in=F - 32, w_sb=32, w_sh=16)),
    (_decode, dict(w_out=F, w_in=F + 64 * 3, w_sb=128, w_sh=48)),
    (_weights, dict(B=2, w_sb=8, w_sh=8)), (_weights, dict(w_in=F + 4, w_out=F)), (_weights, dict(w_in=F, w_out=F + 32)),
    (_evict, dict(c_sb=16)), (_evict, dict(c_si=32)), (_evict, dict(w_sb=16, w_sh=16)),
    (_evict, dict(dc=4 * F, dp=5 * F, dw=6 * F, d_si=64, d_sb=16, d_sh=16, dcap=16, dw_sb=32, dw_sh=16)),
    (_evict, dict(dc=4 * F, dp=5 * F, dw=6 * F, d_si=64, d_sb=32, d_sh=16, dcap=16, dw_sb=4, dw_sh=4)),
])
def test_rows_that_overlap_are_refused(call, bad):
    code, text = outcome(call, **bad)
    assert code == ARG and "overlap" in text, text


# a destination of its own: codes, params, weights and positions
THERE = dict(dc=4 * F, dp=5 * F, dw=6 * F, dpos=7 * F, d_si=64, d_sb=32, d_sh=16, dcap=16, dw_sb=32, dw_sh=16,
             codes=F, params=2 * F, weights=3 * F, positions=8 * F)


@pytest.mark.parametrize("bad", [
    dict(dc=F), dict(dc=F + 32 * 16 * 7), dict(dc=F - 32 * 16 * 7), dict(dp=2 * F + 64), dict(dp=2 * F - 64), dict(dw=3 * F + 4), dict(dw=3 * F),
    dict(dpos=8 * F), dict(dpos=8 * F + 64), dict(dc=F + 32 * 64, d_si=192, d_sb=96, d_sh=48)])
def test_an_eviction_into_its_own_source_is_refused(bad):
    code, text = outcome(_evict, **{**THERE, **bad})
    assert code == ARG and "another cache" in text, text


def test_apart_but_interleaved_memory_is_accepted():
    """(As far as a later refusal.)"""
    # sums of one array of pairs; heads outside sequences; both halves of one cache
    assert outcome(_decode, **LONG, w_out=F, w_in=F + 4 * 32768, w_sb=65536, w_sh=65536, ws=None)[0] == WORKSPACE
    assert outcome(_weights, B=2, NKV=2, T=4096, w_sh=8192, w_sb=4096, w_in=F, w_out=F, ws_bytes=4)[0] == WORKSPACE
    far = dict(THERE, L=20000, cap=20000, c_sh=20000, c_sb=80000, c_si=160000, dc=F + 32 * 40000, d_sh=20000, d_sb=80000, d_si=160000,
               dp=2 * F * 64, dw=3 * F * 64, dpos=8 * F * 64, ws=None)
    assert outcome(_evict, **far)[0] == WORKSPACE
    assert "capacity" in outcome(_store, c_sb=16, c_sh=32, start=13)[1]
    assert "2^31" in outcome(_load, k=F, v=1 << 50, B=12288, T=129, NH=1024, D=16, c_sh=16, c_sb=16 * 1024, c_si=1 << 30, cap=16,
                             starts=F, o_sh=16, o_st=16 * 1024, o_sb=129 * 16 * 1024)[1]


def test_shared_memory_is_found_exactly():
    """Source and destination rows of an eviction at random strides and distances, against all pairs of rows."""
    rng = random.Random(5)
    L, keep, seen = 16400, 16, [0, 0]
    base = 1 << 40
    for _ in range(400):
        B, NH = rng.choice([1, 2, 3]), rng.choice([1, 2, 3])
        c_sh = L + 16 * rng.choice([0, 1, 5, 700, 3000])
        c_sb = c_sh * NH + 16 * rng.choice([0, 3, 900])
        c_si = c_sb * B + 16 * rng.choice([0, 2, 4000])
        if rng.random() < 0.5:
            d_sh, d_sb, d_si = c_sh, c_sb, c_si
        else:
            d_sh = 16 * rng.choice([1, 2, 100])
            d_sb = d_sh * NH + 16 * rng.choice([0, 3])
            d_si = d_sb * B + 16 * rng.choice([0, 2, 4000])
        off = 16 * rng.choice([rng.randrange(-3000, 3000), rng.randrange(-20, 12000), L // 16, c_sh // 16 - 1, c_sb // 16 - 1])
        rows = lambda start, si, sb, sh, n: [(start + i * si + b * sb + h * sh, n) for i in range(2) for b in range(B) for h in range(NH)]  # noqa: E731
        src, dst = rows(0, c_si, c_sb, c_sh, L), rows(off, d_si, d_sb, d_sh, keep)
        shared = any(x < y + m and y < x + n for x, n in src for y, m in dst)
        code, text = outcome(_evict, B=B, NH=NH, D=16, L=L, keep=keep, recent=0, codes=base, params=base << 2, weights=base << 3, positions=None,
                             cap=L, c_sh=c_sh, c_sb=c_sb, c_si=c_si, w_sb=NH * L, w_sh=L, dc=base + off * 8, dp=base << 4, dw=base << 5,
                             d_sh=d_sh, d_sb=d_sb, d_si=d_si, dcap=16, dw_sb=NH * 16, dw_sh=16, ws=None)
        assert (code == ARG and "another cache" in text) if shared else code == WORKSPACE, text
        seen[shared] += 1
    assert min(seen) > 80, seen


def test_package_imports_without_torchs_private_names():
    code = ("import importlib, torch\n"
            "for name in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "ops = importlib.import_module('llm-gpu-5_b200').mha_ops\n"
            "assert ops._current_device is torch.cuda.current_device and ops._raw_stream is ops._public_raw_stream\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
