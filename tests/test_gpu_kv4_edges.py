"""The 4-bit cache operators where they went wrong once: numbers that are not finite in places a mask
leaves out, scales of zero and below, the tf32 module's prompt weights.

Bounds on errors are those derived in test_gpu_kv4.py (u = 2^-24), or stand beside the test."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv4 import U, make_cache, prompt_plain, within

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
