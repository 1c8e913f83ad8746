"""The 4-bit key/value cache operators against plain 64-bit forms: store and load, decode with
accumulated weights, prompt weights, eviction, and all of them together through the modules.

Tolerances are bounds from the arithmetic, u = 2^-24 being float32's half step:
* a score is sums of at most D products (and D additions of the minimum's part) in float32, whose partial
  sums are at most A = scale * sum_d |q_d| (15 s + |m|); the query may be held as two float16 parts of
  its row (2^-22 of the row's largest value): delta = u ((D + 16) A + 4 scale D max|q| 15 s);
* p = exp(z - lse) has relative error rho = 2 delta + (L / 32 + 64) u (the exponent's own rounding, its
  argument's, and the row sum, at most L / 32 + 64 additions deep);
* an output adds p's rounding to float16 before the value product, once for bfloat16 outputs (2^-11)
  and in two parts for float32 ones (2^-22), on terms of at most 15 s, the value sums' own
  (L / 32 + 64) u, and half a step of the output's type.
"""
import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ops(pkg, cuda_dev):
    return pkg.mha_ops


# ------------------------------------------------------------------------------------ plain forms
def quantise(x):
    """(codes as integers [..., D], s, m [..., groups]) of float rows, on the CPU in exact steps."""
    x = x.detach().float().cpu()
    D = x.shape[-1]
    g = min(D, 64)
    x = x.reshape(*x.shape[:-1], D // g, g)
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) * torch.tensor(1.0 / 15, dtype=torch.float32)).clamp(max=65504.0).half()
    m = lo.clamp(-65504.0, 65504.0).half()
    bad = ~torch.isfinite(x).all(-1)
    s = torch.where(bad, torch.tensor(float("nan"), dtype=torch.float16), s)
    m = torch.where(bad, torch.tensor(float("nan"), dtype=torch.float16), m)
    n = ((x.double() - m.double()[..., None]) / s.double()[..., None]).round().clamp(0, 15)
    n = torch.where(s.double()[..., None] > 0, n, torch.zeros_like(n))
    return n.to(torch.uint8).flatten(-2), s, m


def unpack(codes):
    codes = codes.cpu()
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def values(codes, params):
    """The 64-bit numbers a cache holds: [2, B, NH, cap, D]."""
    n = unpack(codes).double()
    p = params.cpu().double()
    D = n.shape[-1]
    p = p.repeat_interleave(min(D, 64), dim=-2)
    return n * p[..., 0] + p[..., 1]


def make_cache(ops, B, NH, L, D, seed, extra=0):
    """A cache of L random rows per head; whatever lies behind them reads as NaN."""
    gen = torch.Generator().manual_seed(seed)
    codes, params = ops.kv4_empty(B, NH, L + extra, D)
    codes.fill_(255)
    params.fill_(float("nan"))
    x = torch.randn((2, B, L, NH, D), generator=gen) + 0.7 * torch.randn((2, 1, 1, NH, D), generator=gen)
    if L:
        ops.kv4_store(x[0].cuda(), x[1].cuda(), codes, params, 0)
    return codes, params


def decode_plain(q, codes, params, lens, scale, dtype):
    """(o, lse, w, and bounds on their errors) in 64 bits."""
    kv = values(codes, params)
    B, NH, D = q.shape
    NKV, cap = kv.shape[2], kv.shape[3]
    G = NH // NKV
    q = q.cpu().double()
    o, lse = torch.zeros((B, NH, D), dtype=torch.float64), torch.full((B, NH), -math.inf, dtype=torch.float64)
    w = torch.zeros((B, NKV, cap), dtype=torch.float64)
    eo, el, ew = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(w)
    rep = min(D, 64)
    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        for h in range(NH):
            c = h // G
            k, v = kv[0, b, c, :n], kv[1, b, c, :n]
            ks = params[0, b, c, :n].cpu().double().repeat_interleave(rep, dim=1)
            vs = params[1, b, c, :n].cpu().double().repeat_interleave(rep, dim=1)
            z = (k @ q[b, h]) * scale
            A = scale * ((15 * ks[..., 0] + ks[..., 1].abs()) @ q[b, h].abs())
            delta = float((U * ((D + 16) * A + 4 * scale * q[b, h].abs().max() * 15 * ks[..., 0].sum(1))).max())
            lse[b, h] = torch.logsumexp(z, 0)
            p = torch.exp(z - lse[b, h])
            depth = (n / 32 + 64) * U
            rho = 2 * delta + depth + U * float(A.max()) * 2
            o[b, h] = p @ v
            w[b, c, :n] += p
            ew[b, c, :n] += rho * p
            el[b, h] = delta + depth + 2 * U * (1 + lse[b, h].abs())
            part = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
            mag = p @ (15 * vs[..., 0] + vs[..., 1].abs())
            eo[b, h] = rho * mag + part * (p @ (15 * vs[..., 0])) + depth * mag + HALF_STEP[dtype] * o[b, h].abs() * 1.01
    return o, lse, w, eo, el, ew


def within(got, want, bound, what):
    got = got.detach().cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), what
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max())} over its bound"


# ------------------------------------------------------------------------------------ store and load
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,NH,D,pos,layout", [
    (1, 1, 1, 64, 0, "fused"), (2, 5, 3, 16, 11, "fused"), (3, 33, 2, 32, 0, "heads"), (2, 130, 4, 64, 7, "fused"),
    (1, 19, 2, 128, 1, "odd"), (2, 64, 5, 64, 100, "heads")])
def test_store_and_load_are_exact(ops, dtype, B, T, NH, D, pos, layout):
    gen = torch.Generator().manual_seed(B * 1000 + T)
    x = torch.randn((2, B, T, NH, D), generator=gen) * 2.0 ** torch.randint(-6, 7, (2, B, T, NH, 1), generator=gen)
    x += torch.randn((2, 1, 1, NH, D), generator=gen)
    x = x.to(dtype)
    if layout == "fused":
        buf = torch.zeros((B, T, 3 * NH, D), dtype=dtype, device="cuda")
        k, v = buf[:, :, NH:2 * NH], buf[:, :, 2 * NH:]
    elif layout == "heads":
        buf = torch.zeros((2, B, NH, T, D), dtype=dtype, device="cuda")
        k, v = buf[0].transpose(1, 2), buf[1].transpose(1, 2)
    else:  # rows that start at any element
        buf = torch.zeros((2, B, T, NH, D + 3), dtype=dtype, device="cuda")
        k, v = buf[0, ..., 1:D + 1], buf[1, ..., 2:D + 2]
    k.copy_(x[0])
    v.copy_(x[1])
    codes, params = ops.kv4_empty(B, NH, pos + T, D)
    codes.fill_(0xA5)
    params.fill_(-7.0)
    ops.kv4_store(k, v, codes, params, pos)
    n, s, m = quantise(x.transpose(2, 3))
    assert torch.equal(unpack(codes)[:, :, :, pos:pos + T], n)
    got = params.cpu()[:, :, :, pos:pos + T]
    assert torch.equal(got[..., 0], s) and torch.equal(got[..., 1], m)
    # nothing else was touched
    assert bool((codes[:, :, :, :pos] == 0xA5).all()) and bool((codes[:, :, :, pos + T:] == 0xA5).all())
    assert bool((params[:, :, :, :pos] == -7.0).all()) and bool((params[:, :, :, pos + T:] == -7.0).all())
    want = values(codes, params)[:, :, :, pos:pos + T].transpose(2, 3)
    for out in (torch.float32, torch.bfloat16):
        lk, lv = ops.kv4_load(codes, params, pos, T, dtype=out)
        for i, y in enumerate((lk, lv)):
            assert torch.equal(y.cpu(), want[i].float().to(out))


def test_store_ragged_starts_counts_marks(ops):
    """Per-sequence starts and counts on the device: rows behind a sequence's last, and rows that fall
    outside the cache, are left as they were; weights and positions are written beside the rows."""
    B, T, NH, D, cap = 5, 9, 3, 32, 48
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((2, B, T, NH, D), generator=gen).cuda()
    starts, counts, seen = [0, 17, 44, -3, 60], [9, 0, 9, 9, 4], [0, 100, 7, 50, 1]
    codes, params = ops.kv4_empty(B, NH, cap, D)
    codes.zero_()
    params.zero_()
    weights = torch.full((B, NH, cap), 3.0, device="cuda")
    positions = torch.full((B, NH, cap), -1, dtype=torch.int32, device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.kv4_store(x[0], x[1], codes, params, i32(starts), counts=i32(counts), weights=weights, positions=positions,
                  seen=i32(seen))
    n, s, _ = quantise(x.transpose(2, 3))
    want_n, want_s = torch.zeros((2, B, NH, cap, D), dtype=torch.uint8), torch.zeros((2, B, NH, cap, 1), dtype=torch.float16)
    want_w, want_p = torch.full((B, NH, cap), 3.0), torch.full((B, NH, cap), -1, dtype=torch.int32)
    for b in range(B):
        for t in range(counts[b]):
            slot = starts[b] + t
            if 0 <= slot < cap:
                want_n[:, b, :, slot], want_s[:, b, :, slot] = n[:, b, :, t], s[:, b, :, t]
                want_w[b, :, slot], want_p[b, :, slot] = 0.0, seen[b] + t
    assert torch.equal(unpack(codes), want_n) and torch.equal(params.cpu()[..., 0], want_s)
    assert torch.equal(weights.cpu(), want_w) and torch.equal(positions.cpu(), want_p)
    held = values(codes, params)
    lk, _ = ops.kv4_load(codes, params, i32(starts), T, counts=i32(counts))
    for b in range(B):
        for t in range(T):
            slot = starts[b] + t
            want = held[0, b, :, slot].float() if t < counts[b] and 0 <= slot < cap else torch.zeros((NH, D))
            assert torch.equal(lk[b, t].cpu(), want)


def test_store_of_special_groups(ops):
    """Constant rows, ranges around float16's smallest and largest scales, values on the border of two
    codes, infinities and NaN."""
    D = 64
    rows = torch.zeros((15, D))
    rows[1] = 3.25
    rows[2] = torch.arange(D) * 1e-9              # the scale vanishes
    rows[3] = torch.arange(D) * 2e-8              # a subnormal scale
    rows[4] = torch.linspace(-3e38, 3e38, D)      # torch's own steps overflow: not finite
    rows[5] = torch.linspace(-1e6, 5e5, D)
    rows[6] = torch.arange(D) % 31 * 0.5          # s = 1: every odd value is a tie
    rows[7] = torch.arange(D) % 31 * 0.5 - 7.0
    rows[8] = torch.linspace(100.0, 100.5, D)     # a small range far from zero
    rows[9, 5] = float("inf")
    rows[10, 63] = float("nan")
    rows[11, 0] = float("-inf")
    rows[12] = -0.0
    rows[13] = torch.linspace(70000.0, 80000.0, D)
    rows[14] = torch.where(torch.arange(D) % 3 == 0, 3e38, -3e38)  # max - min overflows: saturates
    x = rows.view(1, 15, 1, D).cuda()
    codes, params = ops.kv4_empty(1, 1, 15, D)
    ops.kv4_store(x, x, codes, params, 0)
    n, s, m = quantise(rows)
    assert torch.equal(unpack(codes)[0, 0, 0, :15], n) and torch.equal(unpack(codes)[1, 0, 0, :15], n)
    p = params.cpu()[0, 0, 0, :15]
    assert torch.equal(p[..., 0].nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))
    assert torch.equal(p[..., 1].nan_to_num(nan=-1.0), m.nan_to_num(nan=-1.0))
    k, _ = ops.kv4_load(codes, params, 0, 15)
    bad = torch.isnan(k[0, :, 0]).all(-1).cpu()
    assert torch.equal(bad, ~torch.isfinite(rows).all(-1)) and bad.sum() == 4


# ------------------------------------------------------------------------------------ decode
DECODES = [
    # B, NH, NKV, D, L, lengths
    (1, 1, 1, 64, 1, None), (2, 3, 3, 16, 2, None), (1, 12, 12, 64, 129, None), (3, 8, 8, 32, 257, [257, 0, 1]),
    (2, 8, 2, 64, 63, None), (2, 7, 1, 128, 65, [64, 65]), (1, 9, 1, 64, 300, None), (2, 24, 2, 32, 31, None),
    (4, 4, 4, 128, 1000, [0, 999, 16, 255]), (2, 5, 5, 64, 4100, [4097, 4100]), (1, 2, 1, 16, 2049, None),
    (2, 40, 2, 64, 640, [640, 3]), (3, 2, 2, 32, 17, [0, 0, 0]),
    (40, 8, 8, 32, 600, [(37 * b) % 601 for b in range(40)]),  # more CTAs than the GPU holds, two splits each
    (1, 33, 1, 16, 5000, None),                                # 33 query heads to a cached one
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,NH,NKV,D,L,lengths", DECODES)
def test_decode_matches_plain(ops, dtype, B, NH, NKV, D, L, lengths):
    codes, params = make_cache(ops, B, NKV, L, D, seed=L * 7 + D, extra=5)
    for b in range(B if lengths else 0):  # rows behind the sequence's last are never looked at
        params[:, b, :, lengths[b]:] = float("nan")
    gen = torch.Generator().manual_seed(D + L)
    q = (torch.randn((B, NH, D), generator=gen) * 1.5).to(dtype).cuda()
    lse = torch.empty((B, NH), device="cuda")
    w = torch.rand((B, NKV, codes.shape[3]), generator=gen).cuda()
    w0 = w.clone()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths else None
    out = ops.kv4_decode(q, codes, params, L, lengths=lens, lse=lse, weights=w)
    o, l, wp, eo, el, ew = decode_plain(q, codes, params, lengths or [L] * B, 1 / math.sqrt(D), dtype)
    within(out, o, eo, "o")
    within(lse, l, el, "lse")
    within(w, wp + w0.cpu().double(), ew + U * (wp + w0.cpu().double()) * 2, "weights")
    assert torch.equal(w[:, :, L:], w0[:, :, L:])
    # weights set, not added, into another array; and the same output without any
    w2 = torch.full_like(w, 9.0)
    out2 = ops.kv4_decode(q, codes, params, L, lengths=lens, weights_out=w2)
    within(w2[:, :, :L], wp[:, :, :L], ew[:, :, :L] + U * wp[:, :, :L], "weights set")
    assert bool((w2[:, :, L:] == 9.0).all())
    out3 = ops.kv4_decode(q, codes, params, L, lengths=lens)
    assert torch.equal(out, out2) and torch.equal(out, out3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_strides_scale_and_large_scores(ops, dtype):
    """A slice of a larger cache and batch, queries and outputs with strides of their own, scores far
    apart (one key takes everything) and a query of very small and very large elements."""
    B, NKV, D, L = 4, 6, 64, 200
    codes, params = make_cache(ops, B, NKV, L, D, seed=3)
    cs, ps = codes[:, 1:3, 2:5], params[:, 1:3, 2:5]
    gen = torch.Generator().manual_seed(8)
    big = torch.zeros((2, 6, 5, D), dtype=dtype, device="cuda")
    q = big[:, :, 2]
    x = torch.randn((2, 6, D), generator=gen)
    x[0, 1] *= 40.0
    x[0, 2] *= 1e-6
    x[0, 3, ::2] *= 1e-5
    x[1, 0] = 0.0
    q.copy_(x)
    out = torch.full((2, 6, 3, D), 5.0, dtype=dtype, device="cuda")
    lse = torch.empty((2, 6), device="cuda")
    w = torch.zeros((2, 4, 208), device="cuda")[:, :3]
    ops.kv4_decode(q, cs, ps, L, scale=0.7, out=out[:, :, 1], lse=lse, weights=w)
    o, l, wp, eo, el, ew = decode_plain(q, cs, ps, [L] * 2, 0.7, dtype)
    within(out[:, :, 1], o, eo, "o")
    within(lse, l, el, "lse")
    within(w, wp, ew + U * wp, "weights")
    assert bool((out[:, :, 0] == 5.0).all()) and bool((out[:, :, 2] == 5.0).all())


def test_decode_poisoned_rows_poison_only_their_sequence(ops):
    """A NaN held in one sequence's rows makes that head's output NaN and leaves the others alone."""
    codes, params = make_cache(ops, 3, 2, 100, 64, seed=1)
    q = torch.randn((3, 2, 64), generator=torch.Generator().manual_seed(2)).cuda()
    clean = ops.kv4_decode(q, codes, params, 100)
    params[0, 1, 0, 40] = float("nan")
    got = ops.kv4_decode(q, codes, params, 100)
    assert bool(torch.isnan(got[1, 0]).all())
    keep = torch.ones((3, 2), dtype=torch.bool)
    keep[1, 0] = False
    assert torch.equal(got.cpu()[keep], clean.cpu()[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_not_finite_query_stays_in_its_head(ops, dtype):
    """A NaN or an infinity in one query head of a shared group leaves the other heads' outputs alone."""
    codes, params = make_cache(ops, 2, 1, 70, 64, seed=1)
    q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    clean = ops.kv4_decode(q, codes, params, 70)
    q[0, 1, 3] = float("nan")
    q[1, 2, 5] = float("inf")
    got = ops.kv4_decode(q, codes, params, 70)
    bad = torch.zeros((2, 4), dtype=torch.bool)
    bad[0, 1] = bad[1, 2] = True
    assert bool(torch.isnan(got.cpu()[bad].float()).all())
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])


def test_decode_is_repeatable_and_order_free(ops):
    """Bit-equal from call to call; a permutation of the rows gives the same numbers to rounding."""
    codes, params = make_cache(ops, 2, 4, 3000, 64, seed=6)
    q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(4)).cuda()
    a = ops.kv4_decode(q, codes, params, 3000)
    for _ in range(3):
        assert torch.equal(a, ops.kv4_decode(q, codes, params, 3000))
    perm = torch.randperm(3000, generator=torch.Generator().manual_seed(1)).cuda()
    codes2, params2 = codes.clone(), params.clone()
    codes2[:, :, :, :3000], params2[:, :, :, :3000] = codes[:, :, :, perm], params[:, :, :, perm]
    o, _, _, eo, _, _ = decode_plain(q, codes, params, [3000] * 2, 0.125, torch.float32)
    within(ops.kv4_decode(q, codes2, params2, 3000), o, eo, "permuted")


def test_decode_on_a_side_stream_and_two_at_once(ops):
    """Calls on two streams at once, each with workspaces of its own."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    caches = [make_cache(ops, 2, 3, 2000, 64, seed=20 + i) for i in range(2)]
    qs = [torch.randn((2, 3, 64), generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    want = [ops.kv4_decode(qs[i], *caches[i], 2000) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(sides):
            with torch.cuda.stream(st):
                got[i].append(ops.kv4_decode(qs[i], *caches[i], 2000))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_captured_decode_loop_grows_with_device_lengths(pkg, ops):
    """Store, decode and the length's increment captured once and replayed: every replay appends at,
    and attends over, the length as it then is.  Two captured graphs, replayed in turn, do not disturb
    one another."""
    B, NH, D, cap = 3, 2, 64, 64
    gen = torch.Generator().manual_seed(77)
    steps = 6
    xs = torch.randn((2, steps, 3, B, 1, NH, D), generator=gen).cuda()
    start = [5, 0, 17]

    class Loop:
        def __init__(self, i):
            self.codes, self.params = make_cache(ops, B, NH, 20, D, seed=40 + i, extra=cap - 20)
            self.lens = torch.tensor(start, dtype=torch.int32, device="cuda")
            self.x = torch.empty((3, B, 1, NH, D), device="cuda")
            self.w = torch.zeros((B, NH, cap), device="cuda")
            self.pos = torch.zeros((B, NH, cap), dtype=torch.int32, device="cuda")

        def step(self):
            ops.kv4_store(self.x[1], self.x[2], self.codes, self.params, self.lens, weights=self.w, positions=self.pos)
            self.lens += 1
            return ops.kv4_decode(self.x[0, :, 0], self.codes, self.params, cap, lengths=self.lens, weights=self.w)

    eager = [Loop(0), Loop(1)]
    want = [[], []]
    for t in range(steps):
        for i in range(2):
            eager[i].x.copy_(xs[i, t])
            want[i].append(eager[i].step().clone())
    loops = [Loop(0), Loop(1)]
    graphs = []
    for i in range(2):
        loops[i].x.copy_(xs[i, 0])
        torch.cuda.synchronize()
        graphs.append(pkg.graphs.CapturedStep(loops[i].step))
    for t in range(steps):
        for i in range(2):
            loops[i].x.copy_(xs[i, t])
        outs = [graphs[i].replay() for i in range(2)]
        for i in range(2):
            assert torch.equal(outs[i], want[i][t]), (t, i)
    for i in range(2):
        assert torch.equal(loops[i].codes, eager[i].codes) and torch.equal(loops[i].w, eager[i].w)
        assert torch.equal(loops[i].pos, eager[i].pos) and loops[i].lens.tolist() == [s + steps for s in start]


@pytest.mark.parametrize("B,NH,L", [(1, 3, 2000), (1, 1, 9000), (70, 8, 600)])
def test_captured_calls_of_every_plan(pkg, ops, B, NH, L):
    """Decode as a cluster, and through the combine kernel, prompt weights in parts and an eviction, captured
    and replayed on new queries: the same numbers as eager calls."""
    D = 64
    codes, params = make_cache(ops, B, NH, L, D, seed=L)
    cap = codes.shape[3]
    gen = torch.Generator().manual_seed(L)
    q = torch.randn((B, NH, D), generator=gen).cuda()
    w = torch.rand((B, NH, cap), generator=gen).cuda()
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(B, NH, cap).contiguous()
    T = 700 if B > 1 else 2100
    qk = torch.randn((2, 1, T, 1, D), generator=gen).bfloat16().cuda()
    lse = torch.full((1, 1, T), 5.0, device="cuda")

    def step():
        w2 = torch.empty_like(w)
        o = ops.kv4_decode(q, codes, params, L, weights=w, weights_out=w2)
        out = ops.kv4_empty(B, NH, 512, D) + (torch.zeros((B, NH, 512), device="cuda"), torch.zeros((B, NH, 512), dtype=torch.int32, device="cuda"))
        slots = ops.kv4_evict(codes, params, w2, pos, L, 500, recent=7, out=out)
        return (o, w2, ops.key_weights(qk[0], qk[1], lse), slots, out[2], out[3], out[0][:, :, :, :500].clone())

    step()
    graph = pkg.graphs.CapturedStep(step)
    for i in range(3):
        q.copy_(torch.randn((B, NH, D), generator=gen))
        want = [t.clone() for t in step()]
        for a, b in zip(graph.replay(), want):
            assert torch.equal(a[..., :L], b[..., :L])


def test_decode_of_many_sequence_heads(ops):
    """More sequences x heads than a grid's second axis holds."""
    B, NH, D, L = 8200, 8, 16, 3
    codes, params = make_cache(ops, B, NH, L, D, seed=9)
    q = torch.randn((B, NH, D), generator=torch.Generator().manual_seed(3)).cuda()
    out = ops.kv4_decode(q, codes, params, L)
    pick = [0, 1, 4095, 8191, 8199]
    o, _, _, eo, _, _ = decode_plain(q[pick], codes[:, pick], params[:, pick], [L] * len(pick), 0.25, torch.float32)
    within(out[pick], o, eo, "o")


# ------------------------------------------------------------------------------------ prompt weights
PROMPTS = [
    # B, NH, NKV, T, D, first, lengths
    (1, 1, 1, 1, 16, 0, None), (2, 4, 4, 17, 32, 0, None), (2, 2, 2, 128, 64, 0, None), (1, 3, 3, 129, 64, 40, None),
    (3, 4, 2, 200, 64, 0, [200, 0, 77]), (2, 6, 2, 300, 32, 150, [160, 300]), (1, 2, 1, 513, 16, 500, None),
    (2, 2, 2, 64, 48, 63, None), (1, 2, 2, 257, 64, 257, None), (1, 5, 5, 385, 8, 130, None),
    (1, 1, 1, 2100, 64, 0, None), (1, 2, 1, 1300, 32, 100, [1290]), (1, 1, 1, 1100, 128, 0, None),  # queries in parts
]


def prompt_plain(q, k, lse, scale, first, lengths, tf32):
    """(w, bound on its error); the score's sums reach A = scale sum |q||k|, the lse is an input."""
    if tf32:
        q, k = ((x.contiguous().view(torch.int32) & ~0x1fff).view(torch.float32) for x in (q, k))
    q, k, lse = q.cpu().double(), k.cpu().double(), lse.cpu().double()
    B, T, NH, D = q.shape
    NKV = k.shape[2]
    w = torch.zeros((B, NKV, T), dtype=torch.float64)
    e = torch.zeros_like(w)
    for b in range(B):
        n = T if lengths is None else lengths[b]
        if n <= first:
            continue
        for h in range(NH):
            c = h // (NH // NKV)
            z = q[b, first:n, h] @ k[b, :n, c].T * scale - lse[b, h, first:n, None]
            a = q[b, first:n, h].abs() @ k[b, :n, c].abs().T * scale + lse[b, h, first:n, None].abs()
            p = torch.tril(torch.exp(z), diagonal=first)
            w[b, c, :n] += p.sum(0)
            e[b, c, :n] += (p * (U * ((D + 8) * a + 16))).sum(0)
    return w, e + (T / 16 + 64) * U * w


@pytest.mark.parametrize("kind", ["fp32", "tf32", "bf16"])
@pytest.mark.parametrize("B,NH,NKV,T,D,first,lengths", PROMPTS)
def test_prompt_weights_match_plain(ops, kind, B, NH, NKV, T, D, first, lengths):
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    gen = torch.Generator().manual_seed(T * 3 + D)
    qkv = torch.randn((B, T, NH + NKV + 1, D), generator=gen).to(dtype).cuda()
    q, k = qkv[:, :, :NH], qkv[:, :, NH:NH + NKV]
    scale = 1 / math.sqrt(D)
    kk = k.repeat_interleave(NH // NKV, dim=2)
    z = torch.einsum("bihd,bjhd->bhij", q.double(), kk.double()) * scale
    lse = z.masked_fill(torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1), -math.inf).logsumexp(-1).float().contiguous()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths else None
    w, e = prompt_plain(q, k, lse, scale, first, lengths, kind == "tf32")
    got = ops.key_weights(q, k, lse, first_query=first, lengths=lens, dtype="tf32" if kind == "tf32" else None)
    within(got, w, e, "weights")
    assert torch.equal(got, ops.key_weights(q, k, lse, first_query=first, lengths=lens, dtype="tf32" if kind == "tf32" else None))
    # added onto sums that are there, in place, in a wider array
    have = torch.rand((B, NKV, T + 9), generator=gen).cuda()
    before = have.cpu().double()
    ops.key_weights(q, k, lse, first_query=first, lengths=lens, weights=have[:, :, :T], dtype="tf32" if kind == "tf32" else None)
    within(have[:, :, :T], before[:, :, :T] + w, e + U * (before[:, :, :T] + w) * 2, "added")
    assert torch.equal(have.cpu().double()[:, :, T:], before[:, :, T:])


@pytest.mark.parametrize("kind", ["fp32", "tf32", "bf16"])
@pytest.mark.parametrize("T,D,pad,shift", [(150, 5, 0, 0), (70, 128, 1, 0), (200, 20, 0, 1), (65, 127, 0, 0), (300, 12, 4, 0)])
def test_prompt_weights_of_unaligned_rows(ops, kind, T, D, pad, shift):
    """Odd head_dim, rows whose stride is no multiple of four elements, and tensors that start off an alignment."""
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    B, NH, scale = 2, 2, 1 / math.sqrt(D)
    gen = torch.Generator().manual_seed(T + D)
    x = torch.randn((2 * B * T * NH * (D + pad) + shift,), generator=gen).to(dtype).cuda()[shift:].view(2, B, T, NH, D + pad)[..., :D]
    z = torch.einsum("bihd,bjhd->bhij", x[0].double(), x[1].double()) * scale
    lse = z.masked_fill(torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1), -math.inf).logsumexp(-1).float().contiguous()
    w, e = prompt_plain(x[0], x[1], lse, scale, 3, None, kind == "tf32")
    within(ops.key_weights(x[0], x[1], lse, first_query=3, dtype="tf32" if kind == "tf32" else None), w, e, "weights")


@pytest.mark.parametrize("kind", ["fp32", "tf32", "bf16"])
def test_prompt_weights_ignore_the_padding(ops, kind):
    """Whatever lies behind a sequence's last token (queries, keys, lse: NaN and infinities here) reaches
    no weight, and the weights there are 0."""
    B, T, NH, D = 3, 300, 2, 32
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    how = dict(lengths=torch.tensor([300, 129, 5], dtype=torch.int32, device="cuda"), dtype="tf32" if kind == "tf32" else None)
    gen = torch.Generator().manual_seed(4)
    q, k = (torch.randn((B, T, NH, D), generator=gen).to(dtype).cuda() for _ in range(2))
    lse = torch.full((B, NH, T), 4.0, device="cuda")
    clean = ops.key_weights(q, k, lse, **how)
    for b, n in enumerate((300, 129, 5)):
        q[b, n:], k[b, n:], lse[b, :, n:] = float("nan"), float("inf"), float("-inf")
    got = ops.key_weights(q, k, lse, **how)
    assert torch.equal(got, clean)
    assert not bool(got[1, :, 129:].any()) and not bool(got[2, :, 5:].any()) and bool(got[2, :, :5].all())


@pytest.mark.parametrize("kind", ["fp32", "tf32", "bf16"])
def test_prompt_weights_of_the_forward_sum_to_one_per_query(pkg, ops, kind):
    """With the lse of attn_fwd itself, the weights of all keys add up to one per query: each head's
    total is T, within the rounding of p against that lse (bfloat16 and tf32 forwards: their scores
    are the same products; 2e-5 of the total covers the forward's approximate exponentials)."""
    B, T, NH, D = 2, 321, 3, 32
    dt = torch.bfloat16 if kind == "bf16" else torch.float32
    mm = "tf32" if kind == "tf32" else dt
    gen = torch.Generator().manual_seed(6)
    qkv = torch.randn((B, T, 3, NH, D), generator=gen).to(dt).cuda()
    ctx = torch.empty((B, T, NH * D), dtype=dt, device="cuda")
    lse = torch.empty((B, NH, T), device="cuda")
    es = qkv.element_size()
    hv = [pkg.mha_ops.HeadView.tokens(qkv.data_ptr() + i * NH * D * es, T, 3 * NH * D, D) for i in range(3)]
    ops.attention_forward(*hv, pkg.mha_ops.HeadView.tokens(ctx.data_ptr(), T, NH * D, D), lse, B, NH, T, D, D ** -0.5, mm)
    w = ops.key_weights(qkv[:, :, 0], qkv[:, :, 1], lse, dtype=mm)
    total = w.double().sum(-1).cpu()
    assert float((total - T).abs().max()) <= 2e-5 * T
    probs = ops.attention_probs(hv[0], hv[1], lse, B, NH, T, D, D ** -0.5, mm)
    if kind != "tf32":  # the debug matrix recomputes float32 scores; its column sums are these weights
        assert float((probs.double().sum(2) - w.double()).abs().max()) <= 2e-5 * T


# ------------------------------------------------------------------------------------ eviction
def evict_plain(w, pos, n, keep, protect):
    """slots of one head, by sorting."""
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)

    def rank(j):
        x = float(w[j])
        first = 2 if pos[j] >= protect else 0 if math.isnan(x) else 1
        return (-first, -x if first == 1 else 0.0, j)
    kept = set(sorted(range(n), key=rank)[:keep])
    spare = iter(j for j in range(keep, n) if j in kept)
    return [i if i in kept else next(spare) for i in range(keep)]


EVICTIONS = [
    # B, NH, D, L, keep, recent, lengths
    (1, 1, 64, 2, 1, 0, None), (2, 3, 64, 129, 128, 16, None), (1, 2, 32, 500, 17, 17, None), (3, 2, 16, 200, 64, 5, [200, 64, 0]),
    (2, 2, 128, 1500, 700, 100, [1500, 701]), (1, 1, 64, 5000, 4999, 0, None), (2, 1, 64, 64, 64, 8, None),
    (1, 3, 32, 40000, 20000, 64, None), (1, 2, 16, 33, 40, 2, None), (1, 2, 32, 3000, 1000, 30, None),
    (1, 1, 64, 12000, 7000, 100, None), (2, 1, 16, 9000, 8999, 8999, [9000, 8999]),
    (1, 2, 32, 32768, 16384, 64, None), (2, 1, 16, 20001, 9999, 7, [20001, 9000]), (1, 1, 64, 32769, 30000, 0, None),
]


def evict_state(ops, B, NH, D, L, seed, cap=None):
    gen = torch.Generator().manual_seed(seed)
    cap = (max(cap or L, L) + 15) // 16 * 16
    codes = torch.randint(0, 256, (2, B, NH, cap, D // 2), dtype=torch.uint8, generator=gen).cuda()
    params = torch.randn((2, B, NH, cap, D // min(D, 64), 2), generator=gen).half().cuda()
    w = torch.rand((B, NH, cap), generator=gen).pow(4)
    w[w < 0.01] = 0.0        # many equal weights
    w[w > 0.9] = 0.9
    w[..., ::7] *= -0.0      # -0 counts as 0
    w[..., 3::50] = float("nan")
    w[..., 5::61] = float("inf")
    w[..., 6::71] = -1.0
    pos = torch.stack([torch.randperm(2 * cap, generator=gen)[:cap] for _ in range(B * NH)]).view(B, NH, cap).int()
    return codes, params, w.cuda(), pos.cuda()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,NH,D,L,keep,recent,lengths", EVICTIONS)
def test_evict_matches_plain(ops, B, NH, D, L, keep, recent, lengths, in_place):
    codes, params, w, pos = evict_state(ops, B, NH, D, L, seed=L + keep, cap=max(L, keep))
    seen = 2 * codes.shape[3]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths else None
    before = [t.clone() for t in (codes, params, w, pos)]
    ocap = (keep + 15) // 16 * 16
    if in_place:
        slots = ops.kv4_evict(codes, params, w, pos, L, keep, recent=recent, seen=seen, lengths=lens)
        after = (codes, params, w, pos)
    else:
        after = tuple(t.new_full(s, 77) for t, s in (
            (codes, (2, B, NH, ocap, D // 2)), (params, (2, B, NH, ocap, D // min(D, 64), 2)), (w, (B, NH, ocap)), (pos, (B, NH, ocap))))
        slots = ops.kv4_evict(codes, params, w, pos, L, keep, recent=recent, seen=seen, lengths=lens, out=after)
        for a, b in zip((codes, params, w, pos), before):  # the source is as it was, bit for bit
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    want = torch.tensor([[evict_plain(before[2][b, h].tolist(), before[3][b, h].tolist(), lengths[b] if lengths else L, keep, seen - recent)
                          for h in range(NH)] for b in range(B)], dtype=torch.int32)
    assert torch.equal(slots.cpu(), want)
    src = [t.cpu() for t in before]
    for b in range(B):
        n = min(lengths[b] if lengths else L, keep)
        for h in range(NH):
            at = want[b, h, :n].long()
            assert torch.equal(after[0].cpu()[:, b, h, :n], src[0][:, b, h, at])
            assert torch.equal(after[1].cpu()[:, b, h, :n], src[1][:, b, h, at])
            assert torch.equal(after[2].cpu()[b, h, :n].view(torch.int32), src[2][b, h, at].view(torch.int32))
            assert torch.equal(after[3].cpu()[b, h, :n], src[3][b, h, at])
            if not in_place:  # slots behind the kept rows were left alone
                assert bool((after[0][:, b, h, n:] == 77).all()) and bool((after[2][b, h, n:] == 77).all())
            else:
                assert torch.equal(after[0].cpu()[:, b, h, keep:], src[0][:, b, h, keep:])


def test_evict_without_positions_and_ragged_seen(ops):
    """positions None: a slot is its position; ``seen`` per sequence by default from the lengths."""
    B, NH, D, L, keep, recent = 3, 2, 64, 100, 30, 12
    codes, params, w, _ = evict_state(ops, B, NH, D, L, seed=2)
    lens = [100, 50, 31]
    out = tuple(t.new_zeros(s) for t, s in ((codes, (2, B, NH, 32, 32)), (params, (2, B, NH, 32, 1, 2)), (w, (B, NH, 32)))) \
        + (torch.zeros((B, NH, 32), dtype=torch.int32, device="cuda"),)
    slots = ops.kv4_evict(codes, params, w, None, L, keep, recent=recent, out=out,
                          lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    want = torch.tensor([[evict_plain(w[b, h].tolist(), list(range(L)), lens[b], keep, lens[b] - recent) for h in range(NH)]
                         for b in range(B)], dtype=torch.int32)
    assert torch.equal(slots.cpu(), want)
    assert torch.equal(out[3].cpu()[:, :, :keep], want)


@pytest.mark.parametrize("NH,L,out_of", [(2, 2050, 2), (2, 4100, 1), (1, 16500, 100), (3, 2049, 1)])
def test_evict_a_few_rows_of_a_long_cache(ops, NH, L, out_of):
    """In place, on both sides of the number of slots that one CTA looks through by itself."""
    codes, params, w, pos = evict_state(ops, 1, NH, 32, L, seed=L)
    keep, seen = L - out_of, 2 * codes.shape[3]
    src = [t.cpu() for t in (codes, params, w, pos)]
    slots = ops.kv4_evict(codes, params, w, pos, L, keep, recent=8, seen=seen)
    want = torch.tensor([[evict_plain(src[2][0, h].tolist(), src[3][0, h].tolist(), L, keep, seen - 8) for h in range(NH)]],
                        dtype=torch.int32)
    assert torch.equal(slots.cpu(), want)
    for h in range(NH):
        at = want[0, h].long()
        assert torch.equal(codes.cpu()[:, 0, h, :keep], src[0][:, 0, h, at])
        assert torch.equal(params.cpu()[:, 0, h, :keep], src[1][:, 0, h, at])
        assert torch.equal(w.cpu()[0, h, :keep].view(torch.int32), src[2][0, h, at].view(torch.int32))
        assert torch.equal(pos.cpu()[0, h, :keep], src[3][0, h, at])


# ------------------------------------------------------------------------------------ refusals on a device
def test_wrapper_refusals(ops):
    codes, params = make_cache(ops, 2, 2, 20, 64, seed=1)
    q = torch.zeros((2, 4, 64), device="cuda")
    w = torch.zeros((2, 2, 32), device="cuda")
    with pytest.raises(ValueError):
        ops.kv4_decode(q[:1], codes, params, 4)
    with pytest.raises(ValueError):
        ops.kv4_decode(q, codes, params[:, :, :, :16], 4)
    with pytest.raises(ValueError):
        ops.kv4_decode(q, codes[..., ::2], params, 4)
    with pytest.raises(ValueError):
        ops.kv4_decode(q, codes, params, 20, weights=w[:, :, :16])
    with pytest.raises(TypeError):
        ops.kv4_decode(q, codes, params, 20, lengths=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.kv4_decode(q, codes, params, 20, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.kv4_decode(q.half(), codes, params, 20)
    with pytest.raises(RuntimeError, match="length"):
        ops.kv4_decode(q, codes, params, 33)
    with pytest.raises(RuntimeError, match="multiple"):
        ops.kv4_decode(q[:, :3], codes, params, 20)
    with pytest.raises(ValueError):
        ops.kv4_store(q[:, None], q[:, None], codes, params, 0)
    with pytest.raises(RuntimeError, match="capacity"):
        ops.kv4_store(torch.zeros((2, 40, 2, 64), device="cuda"), torch.zeros((2, 40, 2, 64), device="cuda"), codes, params, 0)
    with pytest.raises(RuntimeError, match="recent"):
        ops.kv4_evict(codes, params, w, None, 20, 4, recent=5)
    with pytest.raises(RuntimeError, match="keep"):
        ops.kv4_evict(codes, params, w, None, 20, 0)
    with pytest.raises(ValueError):
        ops.key_weights(q[:, None], q[:, None, :3], torch.zeros((2, 4, 2), device="cuda"))


def test_empty_calls_do_nothing(ops):
    codes, params = ops.kv4_empty(2, 2, 16, 64)
    codes.zero_()
    params.zero_()
    none = torch.zeros((2, 0, 2, 64), device="cuda")
    ops.kv4_store(none, none, codes, params, 0)
    k, v = ops.kv4_load(codes, params, 0, 0)
    assert k.shape == (2, 0, 2, 64) and not bool(codes.any())


# ------------------------------------------------------------------------------------ through the module
@pytest.mark.parametrize("prec,tol", [("fp32", 1e-5), ("tf32", 2e-2), ("bf16", 2e-2)])
def test_module_generates_from_a_4bit_cache(pkg, ops, prec, tol):
    """Prompt, decode, evict, decode through MultiHeadAttention.  Each decode output is the output
    projection of attention over what the cache holds (read back with kv4_load, in 64 bits; module
    tolerances of the precision), and the tracked weights are the sums of the attention weights."""
    B, T, NH, D = 2, 70, 4, 16 if prec == "tf32" else 32
    C = NH * D
    np.random.seed(5)
    attn = pkg.MultiHeadAttention(pkg.GPTConfig(vocab_size=50, embedding_dim=C, num_heads=NH, attention_precision=prec))
    attn.c_attn_w.weights.mul_(8.0)
    attn.training = False
    cache = attn.new_kv_cache(B, 96, bits=4, track_weights=True)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((B, T, C), generator=gen).cuda()
    plain = attn.new_kv_cache(B, 96)
    y4, y = attn.forward(x.view(-1), B, T, kv_cache=cache), attn.forward(x.view(-1), B, T, kv_cache=plain)
    assert torch.equal(y4.tensor, y.tensor)  # the prompt's own attention is not quantised
    assert cache.length == T and cache.seen == T
    n, s, m = quantise(torch.stack((plain.k[:, :T], plain.v[:, :T])).transpose(2, 3))
    assert torch.equal(unpack(cache.codes)[:, :, :, :T], n)
    total = cache.weights[:, :, :T].double().sum(-1)
    assert float((total - T).abs().max()) <= 1e-3 * T  # every query's weights add up to one
    assert torch.equal(cache.positions[:, :, :T], torch.arange(T, device="cuda", dtype=torch.int32).expand(B, NH, T))
    wo, bo = attn.c_proj_w.weights.double(), attn.c_proj_b.weights.double()
    wq, bq = attn.c_attn_w.weights.double()[:, :C], attn.c_attn_b.weights.double()[:C]
    for step in range(6):
        if step == 3:
            before = cache.weights[:, :, :cache.length].clone(), cache.positions[:, :, :cache.length].clone()
            slots = cache.evict(40, recent=8)
            assert cache.length == 40 and slots.shape == (B, NH, 40) and cache.seen == T + 3
            for b in range(B):
                for h in range(NH):
                    assert slots[b, h].tolist() == evict_plain(before[0][b, h].tolist(), before[1][b, h].tolist(), T + 3, 40, T + 3 - 8)
            assert torch.equal(cache.positions[:, :, :40], before[1].gather(-1, slots.long()))
            assert cache.evict(40) is None
        xt = torch.randn((B, C), generator=gen).cuda()
        w0 = cache.weights[:, :, :cache.length].clone()
        out = attn.forward_decode(xt, B, cache)
        L = cache.length
        assert bool((cache.positions[:, :, L - 1] == T + step).all())
        k, v = (t.transpose(1, 2).double() for t in ops.kv4_load(cache.codes, cache.params, 0, L))
        q = (xt.double() @ wq + bq).view(B, NH, 1, D)
        p = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(D), -1)
        want = (p @ v).transpose(1, 2).reshape(B, C) @ wo + bo
        assert float((out.tensor.double() - want).abs().max() / want.abs().max()) <= tol
        gained = cache.weights[:, :, :L].double()
        gained[:, :, :L - 1] -= w0.double()
        assert float((gained - p[:, :, 0]).abs().max()) <= tol * 5
    with pytest.raises(RuntimeError):
        attn.new_kv_cache(B, 8, bits=4).evict(4)
    with pytest.raises(ValueError):
        attn.new_kv_cache(B, 8, bits=8)


def test_module_prompt_window_and_restart(pkg, ops):
    """prompt_window counts the last queries only; a prompt at position 0 replaces what was held."""
    B, T, NH, C = 1, 50, 2, 64
    np.random.seed(2)
    attn = pkg.MultiHeadAttention(pkg.GPTConfig(vocab_size=50, embedding_dim=C, num_heads=NH, attention_precision="fp32"))
    cache = attn.new_kv_cache(B, 64, bits=4, track_weights=True, prompt_window=10)
    x = torch.randn((B, T, C), generator=torch.Generator().manual_seed(3)).cuda()
    for _ in range(2):
        attn.forward(x.view(-1), B, T, kv_cache=cache)
        assert cache.length == T
        assert float((cache.weights[:, :, :T].double().sum(-1) - 10).abs().max()) <= 1e-4
    probs = torch.from_numpy(attn.cache_attn_weights).double()
    assert float((cache.weights[:, :, :T].cpu().double() - probs[:, :, 40:].sum(2)).abs().max()) <= 1e-5
    with pytest.raises(RuntimeError, match="position"):
        cache.store(torch.zeros((1, 1, 3 * C), device="cuda"), 7)
    with pytest.raises(RuntimeError, match="max_len"):
        cache.store(torch.zeros((1, 20, 3 * C), device="cuda"), T)
