"""The 4-bit cache operators where they went wrong once: numbers that are not finite in places a mask
leaves out, scales of zero and below, value scales far apart, the tf32 module's prompt weights, arguments
that the C boundary would cut short, batches of none.

Bounds on errors are those derived in test_gpu_kv4.py (u = 2^-24), or stand beside the test."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv4 import U, decode_plain, make_cache, prompt_plain, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg, cuda_dev):
    return pkg.mha_ops


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------ prompt weights
KINDS = ["fp32", "tf32", "bf16"]


def prompt(kind, B, T, NH, NKV, D, scale, seed):
    """q, k, and the lse of a causal softmax of these scores, whatever the scale."""
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    gen = torch.Generator().manual_seed(seed)
    qk = torch.randn((B, T, NH + NKV, D), generator=gen).to(dtype).cuda()
    q, k = qk[:, :, :NH], qk[:, :, NH:]
    z = torch.einsum("bihd,bjhd->bhij", q.double(), k.repeat_interleave(NH // NKV, dim=2).double()) * scale
    z = z.masked_fill_(torch.ones((T, T), dtype=torch.bool, device="cuda").triu_(1), -math.inf)
    return q, k, z.logsumexp(-1).float().contiguous()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
def test_prompt_weights_at_any_scale(ops, kind, scale):
    B, T, NH, NKV, D = 2, 300, 4, 2, 32
    q, k, lse = prompt(kind, B, T, NH, NKV, D, scale, 11)
    mode = "tf32" if kind == "tf32" else None
    for first, lengths in ((0, None), (77, None), (0, [300, 131])):
        w, _ = prompt_plain(q, k, lse, scale, first, lengths, kind == "tf32")
        # every score's sums of magnitudes are below a
        a = (q.float().abs().amax() * k.float().abs().amax()).item() * D * abs(scale) + float(lse.abs().max())
        bound = U * ((D + 8) * a + 16) * w + (T / 16 + 64) * U * w
        got = ops.key_weights(q, k, lse, scale=scale, first_query=first, lengths=i32(lengths) if lengths else None, dtype=mode)
        within(got, w, bound, (scale, first, lengths))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,first", [(300, 150), (129, 128), (600, 33)])
@pytest.mark.parametrize("poison", [float("nan"), float("-inf"), float("inf")])
def test_prompt_weights_never_look_at_queries_before_the_first(ops, kind, T, first, poison):
    """Queries in front of first_query, and their lse, may hold anything."""
    q, k, lse = prompt(kind, 1, T, 2, 2, 32, 32 ** -0.5, T)
    mode = "tf32" if kind == "tf32" else None
    clean = ops.key_weights(q, k, lse, first_query=first, dtype=mode)
    q[:, :first], lse[:, :, :first] = float("nan"), poison
    got = ops.key_weights(q, k, lse, first_query=first, dtype=mode)
    assert bool(torch.isfinite(clean).all()) and torch.equal(got, clean)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("poison", [float("nan"), float("-inf")])
def test_prompt_weights_of_a_bad_query_stay_before_it(ops, kind, poison):
    """A query whose lse is not finite poisons the keys that it sees, and none behind it."""
    T, at = 300, 141
    q, k, lse = prompt(kind, 1, T, 2, 2, 32, 32 ** -0.5, 5)
    mode = "tf32" if kind == "tf32" else None
    clean = ops.key_weights(q, k, lse, dtype=mode)
    q[0, at, 1], lse[0, 1, at] = float("nan"), poison
    got = ops.key_weights(q, k, lse, dtype=mode)
    assert torch.equal(got[0, 0], clean[0, 0]) and torch.equal(got[0, 1, at + 1:], clean[0, 1, at + 1:])
    assert not bool(torch.isfinite(got[0, 1, :at + 1]).any())


@pytest.mark.parametrize("D", [32, 64, 128])
def test_tf32_module_weights_match_its_forward(pkg, ops, D):
    """Every query's tracked weights add up to one against the lse of the module's own forward.

    p = exp(z - lse): z and the forward's scores are float32 sums of D products below A = scale sum |q||k| (each off by
    at most u (D + 16) A, the forward's tf32 products at head_dim 32 being the same as these), the approximate
    exponentials are off by 2^-21 each side with their argument's 2 u (A + |lse|), the sums by (T / 16 + 64) u."""
    B, T, NH = 1, 400, 2
    C = NH * D
    np.random.seed(7)
    attn = pkg.MultiHeadAttention(pkg.GPTConfig(vocab_size=50, embedding_dim=C, num_heads=NH, attention_precision="tf32"))
    attn.c_attn_w.weights.mul_(300.0 / math.sqrt(C))  # scores up to about 100
    cache = attn.new_kv_cache(B, T, bits=4, track_weights=True)
    x = torch.randn((B, T, C), generator=torch.Generator().manual_seed(3)).cuda()
    attn.forward(x.view(-1), B, T, kv_cache=cache)
    qkv = attn._cache["qkv"].view(B, T, 3, NH, D).double()
    A = torch.einsum("bihd,bjhd->bhij", qkv[:, :, 0].abs(), qkv[:, :, 1].abs()).tril_().amax(-1) / math.sqrt(D)
    rho = 2 * U * (D + 16) * A + 4 * U * (2 * A + 1) + 2.0 ** -20 + 2 * (T / 16 + 64) * U
    total = cache.weights[:, :, :T].double().sum(-1)
    assert bool(((total - T).abs() <= rho.sum(-1)).all()), (total - T, rho.sum(-1))


# ------------------------------------------------------------------------------------ decode
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,NH,NKV,L", [(2, 2, 1, 300), (1, 1, 1, 20000), (70, 16, 8, 600), (2, 18, 2, 40), (2, 18, 2, 9000)])
def test_bad_queries_leave_the_weights_behind_the_rows(ops, dtype, B, NH, NKV, L):
    """Slots from a sequence's length on keep their weights whatever the queries hold (one launch, clusters, the
    combine kernel, several CTAs of query heads)."""
    codes, params = make_cache(ops, B, NKV, L, 64, seed=L)
    q = torch.randn((B, NH, 64), generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    q[0, 0, 5] = float("nan")
    q[-1, -1, 0] = float("inf")
    w = torch.rand((B, NKV, codes.shape[3]), generator=torch.Generator().manual_seed(3)).cuda()
    before = w.clone()
    lens = [(L // 3 + 13 * b) % L for b in range(B)]
    ops.kv4_decode(q, codes, params, L, lengths=i32(lens), weights=w)
    for b in range(B):
        assert torch.equal(w[b, :, lens[b]:], before[b, :, lens[b]:]), b
    assert bool(torch.isnan(w[0, 0, :lens[0]]).all()) and bool(torch.isnan(w[-1, -1, :lens[-1]]).all())


def spread_cache(ops, B, NKV, L, D, seed, wild):
    """Small value scales everywhere but in the rows ``wild`` of every head, whose keys point away from q = ones."""
    gen = torch.Generator().manual_seed(seed)
    codes, params = ops.kv4_empty(B, NKV, L, D)
    codes.copy_(torch.randint(0, 256, codes.shape, dtype=torch.uint8, generator=gen))
    p = torch.zeros(params.shape)
    p[0, ..., 0], p[0, ..., 1] = 0.01, 0.02 * torch.randn(p[0, ..., 1].shape, generator=gen)
    p[1, ..., 0], p[1, ..., 1] = 2.0 ** -20, 0.0
    for j, (low, scale) in wild.items():
        p[0, :, :, j, :, 1] = low
        p[1, :, :, j, :, 0] = scale
    params.copy_(p)
    return codes, params


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("NH,NKV,D", [(2, 2, 64), (8, 2, 64), (3, 3, 16), (2, 2, 32), (8, 2, 128), (7, 1, 128)])
@pytest.mark.parametrize("L,at", [(600, 3), (600, 400), (700, 699), (9000, 70)])
def test_decode_with_one_wild_value_scale(ops, dtype, NH, NKV, D, L, at):
    """A row of a value scale 2^35 times the others', which hardly any weight falls on, takes no digits from the
    others' part of the output."""
    codes, params = spread_cache(ops, 2, NKV, L, D, L + at, {at: (-2.0, 32768.0)})
    q = torch.ones((2, NH, D), device="cuda") * (60.0 / math.sqrt(D))  # the wild row's score: about 120 below
    q += 0.01 * torch.randn((2, NH, D), generator=torch.Generator().manual_seed(1)).cuda()
    q = q.to(dtype)
    o, l, _, eo, el, _ = decode_plain(q, codes, params, [L] * 2, 1 / math.sqrt(D), dtype)
    lse = torch.empty((2, NH), device="cuda")
    within(ops.kv4_decode(q, codes, params, L, lse=lse), o, eo, "o")
    within(lse, l, el, "lse")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_with_a_wild_value_scale_that_leads_at_first(ops, dtype):
    """The wild row holds the largest score until a later tile's scores leave it 100 and more below (so many sequences
    that one CTA takes all rows of a head)."""
    B, NKV, L, D = 300, 4, 1500, 64
    codes, params = spread_cache(ops, B, NKV, L, D, 4, {5: (0.5, 32768.0)})
    params[0, :, :, 1000:, :, 1] = 2.0
    q = (torch.ones((B, NKV, D)) * 12.0).to(dtype).cuda()
    got = ops.kv4_decode(q, codes, params, L)
    pick = [0, 144, 299]
    o, _, _, eo, _, _ = decode_plain(q[pick], codes[:, pick], params[:, pick], [L] * 3, 1 / math.sqrt(D), dtype)
    within(got[pick], o, eo, "o")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_where_heads_see_different_value_scales(ops, dtype, D):
    """Two query heads of one cached head: one looks at rows of large value scales, the other at small ones."""
    L = 500
    codes, params = spread_cache(ops, 1, 1, L, D, 8, {j: (-2.0, 32768.0) for j in range(200, 232)})
    q = torch.ones((1, 2, D), device="cuda") * (60.0 / math.sqrt(D))
    q[:, 1] *= -1.0
    q = q.to(dtype)
    o, _, _, eo, _, _ = decode_plain(q, codes, params, [L], 1 / math.sqrt(D), dtype)
    within(ops.kv4_decode(q, codes, params, L), o, eo, "o")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_with_groups_of_different_value_scales(ops, dtype):
    """head_dim 128: the second group's scales 2^35 times the first's; every element keeps the digits of its group."""
    L = 300
    codes, params = spread_cache(ops, 2, 2, L, 128, 9, {})
    params[1, ..., 1, 0] = 32768.0
    q = torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    o, _, _, eo, _, _ = decode_plain(q, codes, params, [L] * 2, 0.1, dtype)
    within(ops.kv4_decode(q, codes, params, L, scale=0.1), o, eo, "o")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_with_a_value_group_that_is_not_finite(ops, dtype):
    """head_dim 128: a NaN among one group's scales reaches that group's outputs only, not the other's, the lse or the
    weights."""
    L = 400
    codes, params = make_cache(ops, 1, 2, L, 128, seed=12)
    q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    for group in (0, 1):
        bad = params.clone()
        bad[1, :, :, 77, group, 0] = float("nan")
        lse, w = torch.empty((1, 8), device="cuda"), torch.empty((1, 2, L), device="cuda")
        got = ops.kv4_decode(q, codes, bad, L, lse=lse, weights_out=w)
        o, l, wp, eo, el, ew = decode_plain(q, codes, params, [L], 128 ** -0.5, dtype)
        fine = slice(64, 128) if group == 0 else slice(0, 64)
        within(got[..., fine], o[..., fine], eo[..., fine], "o")
        within(lse, l, el, "lse")
        within(w, wp[..., :L], ew[..., :L] + U * wp[..., :L], "weights")
        gone = slice(0, 64) if group == 0 else slice(64, 128)
        assert bool(torch.isnan(got[..., gone].float()).all())


# ------------------------------------------------------------------------------------ arguments
def test_numbers_past_32_bits_are_refused(ops):
    """(They reach C as an int, whose upper bits would be dropped: position 2^32 would be slot 0.)"""
    codes, params = make_cache(ops, 1, 1, 16, 64, seed=1)
    x = torch.randn((1, 2, 1, 64), device="cuda")
    q = x[:, 0]
    w = torch.zeros((1, 1, 16), device="cuda")
    marks = torch.zeros((1, 1, 16), dtype=torch.int32, device="cuda")
    held = codes.clone()
    for call in (lambda: ops.kv4_store(x, x, codes, params, 1 << 32), lambda: ops.kv4_store(x, x, codes, params, 0, seen=1 << 31),
                 lambda: ops.kv4_store(x, x, codes, params, 0, positions=marks, seen=(1 << 31) - 1),
                 lambda: ops.kv4_store(x, x, codes, params, -(1 << 32)), lambda: ops.kv4_load(codes, params, 1 << 32, 1),
                 lambda: ops.kv4_decode(q, codes, params, (1 << 32) + 4),
                 lambda: ops.key_weights(x, x, torch.zeros((1, 1, 2), device="cuda"), first_query=1 << 32),
                 lambda: ops.kv4_evict(codes, params, w, None, (1 << 32) + 9, 4),
                 lambda: ops.kv4_evict(codes, params, w, None, 9, 4, recent=1 << 32),
                 lambda: ops.kv4_evict(codes, params, w, None, 9, 4, seen=1 << 32)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.kv4_store(x, x, codes, params, 1.5)
    assert torch.equal(codes, held)


def test_lengths_and_counts_are_device_arrays(ops):
    """A plain number where a device array belongs is refused, not passed over."""
    codes, params = make_cache(ops, 1, 1, 16, 64, seed=1)
    x = torch.randn((1, 2, 1, 64), device="cuda")
    w = torch.zeros((1, 1, 16), device="cuda")
    held = codes.clone()
    for call in (lambda: ops.kv4_store(x, x, codes, params, 0, counts=1), lambda: ops.kv4_load(codes, params, 0, 2, counts=1),
                 lambda: ops.kv4_decode(x[:, 0], codes, params, 16, lengths=3),
                 lambda: ops.key_weights(x, x, torch.zeros((1, 1, 2), device="cuda"), lengths=1),
                 lambda: ops.kv4_evict(codes, params, w, None, 9, 4, lengths=5)):
        with pytest.raises(TypeError):
            call()
    assert torch.equal(codes, held)


def test_batches_of_none(ops):
    """No sequences: nothing to do, as the store and the load have it."""
    codes, params = ops.kv4_empty(0, 2, 16, 64)
    none = torch.zeros((0, 3, 2, 64), device="cuda")
    w = torch.zeros((0, 2, 16), device="cuda")
    ops.kv4_store(none, none, codes, params, 0)
    assert ops.kv4_load(codes, params, 0, 3)[0].shape == (0, 3, 2, 64)
    out = torch.empty((0, 4, 64), device="cuda")
    assert ops.kv4_decode(torch.zeros((0, 4, 64), device="cuda"), codes, params, 5, weights=w, out=out) is out
    assert ops.kv4_evict(codes, params, w, None, 9, 4).shape == (0, 2, 4)
    assert ops.key_weights(none, none, torch.zeros((0, 2, 3), device="cuda")).shape == (0, 2, 3)
    assert ops.key_weights(none[:, :0], none[:, :0], torch.zeros((0, 2, 0), device="cuda")).shape == (0, 2, 0)


def test_prompt_weights_of_no_tokens(ops):
    """T = 0: no weights; sums that are there stay."""
    x = torch.zeros((2, 0, 3, 64), device="cuda")
    have = torch.ones((2, 3, 5), device="cuda")
    assert ops.key_weights(x, x, torch.zeros((2, 3, 0), device="cuda")).shape == (2, 3, 0)
    ops.key_weights(x, x, torch.zeros((2, 3, 0), device="cuda"), weights=have)
    assert bool((have == 1).all())


def test_calls_through_torchs_public_names(ops, monkeypatch):
    """On a side stream, without the private names: the same stream, the same numbers."""
    codes, params = make_cache(ops, 2, 3, 500, 64, seed=4)
    q = torch.randn((2, 3, 64), generator=torch.Generator().manual_seed(4)).cuda()
    want = ops.kv4_decode(q, codes, params, 500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert ops._public_raw_stream(0) == ops._raw_stream(0) == side.cuda_stream
        monkeypatch.setattr(ops, "_raw_stream", ops._public_raw_stream)
        monkeypatch.setattr(ops, "_current_device", torch.cuda.current_device)
        got = ops.kv4_decode(q, codes, params, 500)
    side.synchronize()
    assert torch.equal(got, want)
