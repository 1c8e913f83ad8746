"""Cases of the 4-bit key/value cache operators: store and load, decode attention, the prompt's
accumulated attention weights, eviction.

``run`` computes each in plain torch (float32, rounded once at the end) or, with ``own`` set, through
this package.  A cached row of D values is held as 4-bit codes in groups of g = min(D, 64): with
s = float16((max - min) / 15) and m = float16(min), x becomes n = round((x - m) / s) in 0..15 (half to
even) and stands for n * s + m.  ``codes`` is uint8 [2, B, NH, cap, D / 2] (index 0 keys, 1 values; the
even element in the low nibble), ``params`` float16 [2, B, NH, cap, D / g, 2] (s, m).
"""

import importlib
import math

import torch

own = False

DEV = "cuda"
F16_MAX = 65504.0


def _ops():
    return importlib.import_module("llm-gpu-5_b200").mha_ops


def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


# ------------------------------------------------------------------------------------ the cases
def _store(name, B, T, NH, D, dtype, cap, pos, ragged):
    return dict(name=name, op="store", B=B, T=T, NH=NH, D=D, dtype=dtype, cap=cap, pos=pos, ragged=ragged)


def _decode(name, B, NH, NKV, D, L, dtype, weights, ragged):
    return dict(name=name, op="decode", B=B, NH=NH, NKV=NKV, D=D, L=L, dtype=dtype, weights=weights, ragged=ragged)


def _weights(name, B, NH, NKV, T, D, dtype, first, ragged):
    return dict(name=name, op="weights", B=B, NH=NH, NKV=NKV, T=T, D=D, dtype=dtype, first=first, ragged=ragged)


def _evict(name, B, NH, D, L, keep, recent, ragged):
    return dict(name=name, op="evict", B=B, NH=NH, D=D, L=L, keep=keep, recent=recent, ragged=ragged)


def listed():
    return [
        # one generated token of one sequence enters the cache: the latency of the smallest call
        _store("store one token", 1, 1, 12, 64, "bf16", 2048, 777, False),
        # the prompts of the long-context configuration, 32 x 1,024 tokens, 8 heads of 64
        _store("store prompts bf16", 32, 1024, 8, 64, "bf16", 1088, 0, False),
        # padded prompts of the training-batch configuration's heads in float32, behind a shared prefix
        _store("store ragged prompts f32", 64, 127, 8, 32, "f32", 256, 33, True),
        # one sequence just past its prompt: the latency of the smallest call, weights kept
        _decode("decode one short sequence", 1, 12, 12, 64, 129, "bf16", True, False),
        # the decode configuration: 64 sequences over 2,048 cached tokens
        _decode("decode batch", 64, 8, 8, 64, 2048, "bf16", False, False),
        # four query heads to a cached head, sequences of every length from none to 8,191
        _decode("decode shared heads ragged", 16, 32, 8, 128, 8191, "bf16", True, True),
        # the float32 module's arithmetic at the training-batch configuration's heads
        _decode("decode f32", 8, 8, 8, 32, 4099, "f32", True, False),
        # many long sequences, weights kept: the largest
        _decode("decode long", 32, 12, 12, 64, 16384, "bf16", True, False),
        # prompt weights of the small float32 configuration
        _weights("prompt weights f32", 8, 4, 4, 128, 16, "f32", 0, False),
        # prompt weights of the long-context configuration
        _weights("prompt weights bf16", 32, 8, 8, 1024, 64, "bf16", 0, False),
        # one sequence at its budget gives up one row per head: the latency of the smallest call
        _evict("evict one row", 1, 12, 64, 513, 512, 64, False),
        # a batch of long prompts cut to half
        _evict("evict half", 32, 8, 64, 8192, 4096, 256, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    """Sizes over the listed cases' ranges, no more work than the largest listed case of the operator."""
    op = rng.choice(["store", "decode", "decode", "weights", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    ragged = rng.random() < 0.4
    D = rng.choice([16, 32, 64, 64, 128])
    NH = rng.choice([1, 4, 5, 8, 12])
    if op == "store":
        T = _log(rng, 1, 1024)
        B = max(1, min(_log(rng, 1, 64), 32 * 1024 * 8 * 64 // (T * NH * D)))
        pos = rng.randrange(0, 100)
        return dict(op=op, B=B, T=T, NH=NH, D=D, dtype=dtype, cap=(pos + T + 15) // 16 * 16, pos=pos, ragged=ragged)
    if op == "decode":
        L = _log(rng, 1, 32768)
        G = rng.choice([1, 1, 2, 4, 7])
        B = max(1, min(_log(rng, 1, 64), 32 * 12 * 16384 * 64 // (L * NH * G * D)))
        return dict(op=op, B=B, NH=NH * G, NKV=NH, D=D, L=L, dtype=dtype, weights=rng.random() < 0.6, ragged=ragged)
    if op == "weights":
        D = rng.choice([16, 32, 64]) if dtype == "bf16" else D
        T = _log(rng, 2, 4096)
        G = rng.choice([1, 1, 3])
        most = 32 * 8 * 1024 * 1024 if dtype == "bf16" else 32 * 8 * 1024 * 64
        if dtype == "f32":
            T = min(T, 1024)
        while T * T * NH * G > most:
            NH, G = max(1, NH // 2), 1
            if NH == 1 and T * T > most:
                T //= 2
        B = max(1, min(_log(rng, 1, 32), most // (T * T * NH * G)))
        first = 0 if rng.random() < 0.5 else rng.randrange(0, T)
        return dict(op=op, B=B, NH=NH * G, NKV=NH, T=T, D=D, dtype=dtype, first=first, ragged=ragged)
    L = _log(rng, 2, 16384)
    B = max(1, min(_log(rng, 1, 32), 32 * 8 * 8192 * 64 // (L * NH * D)))
    keep = max(1, int(L * rng.uniform(0.1, 1.0)))
    return dict(op=op, B=B, NH=NH, D=D, L=L, keep=keep, recent=rng.randrange(0, keep + 1), ragged=ragged)


def _lengths(case, most):
    """Ragged lengths: from none to all of ``most``, evenly, in a fixed mixed order."""
    B = case["B"]
    if not case["ragged"]:
        return [most] * B
    if B == 1:
        return [(most + 1) // 2]
    return [most * ((b * 7 + 3) % B) // (B - 1) for b in range(B)]


# ------------------------------------------------------------------------------------ the inputs
def _group(D):
    return min(D, 64)


def _keys_like(shape, gen):
    """Keys or values as a projection gives them: unit noise about a per-channel offset."""
    return torch.randn(shape, generator=gen, device=DEV) + 0.7 * torch.randn(shape[-2:], generator=gen, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))
    B, D, dt = case["B"], case["D"], _dt(case) if "dtype" in case else None
    s = dict(case=case)
    if case["op"] == "store":
        T, NH, cap = case["T"], case["NH"], case["cap"]
        # keys and values stand in the fused projection's output, as the module holds them
        qkv = _keys_like((B, T, 3 * NH, D), gen).to(dt)
        s["k"], s["v"] = qkv[:, :, NH:2 * NH], qkv[:, :, 2 * NH:]
        s["codes"] = torch.zeros((2, B, NH, cap, D // 2), dtype=torch.uint8, device=DEV)
        s["params"] = torch.zeros((2, B, NH, cap, D // _group(D), 2), dtype=torch.float16, device=DEV)
        s["counts"] = torch.tensor(_lengths(case, T), dtype=torch.int32, device=DEV) if case["ragged"] else None
    elif case["op"] == "decode":
        NH, NKV, L = case["NH"], case["NKV"], case["L"]
        cap = (L + 15) // 16 * 16
        s["q"] = torch.randn((B, NH, D), generator=gen, device=DEV).mul_(1.5).to(dt)
        s["codes"] = torch.zeros((2, B, NKV, cap, D // 2), dtype=torch.uint8, device=DEV)
        s["params"] = torch.zeros((2, B, NKV, cap, D // _group(D), 2), dtype=torch.float16, device=DEV)
        for b in range(B):
            for i in range(2):
                x = _keys_like((L, NKV, D), gen).transpose(0, 1)
                s["codes"][i, b, :, :L], s["params"][i, b, :, :L] = _quantise(x)
        s["lengths"] = torch.tensor(_lengths(case, L), dtype=torch.int32, device=DEV) if case["ragged"] else None
        s["lse"] = torch.empty((B, NH), dtype=torch.float32, device=DEV)
        if case["weights"]:
            s["weights"] = torch.rand((B, NKV, cap), generator=gen, device=DEV)
            s["weights_out"] = torch.zeros((B, NKV, cap), dtype=torch.float32, device=DEV)
    elif case["op"] == "weights":
        NH, NKV, T = case["NH"], case["NKV"], case["T"]
        qkv = _keys_like((B, T, NH + 2 * NKV, D), gen).to(dt)
        s["q"], s["k"] = qkv[:, :, :NH], qkv[:, :, NH:NH + NKV]
        s["lse"] = torch.empty((B, NH, T), dtype=torch.float32, device=DEV)
        causal = torch.ones((T, T), dtype=torch.bool, device=DEV).tril_()
        for b in range(B):
            sc = _scores(s["q"][b:b + 1].float(), s["k"][b:b + 1].float(), D)[0]
            s["lse"][b] = sc.masked_fill_(~causal, -math.inf).logsumexp(-1).view(NH, T)
        s["lengths"] = torch.tensor(_lengths(case, T), dtype=torch.int32, device=DEV) if case["ragged"] else None
    else:
        NH, L, keep = case["NH"], case["L"], case["keep"]
        cap, cap_out = (L + 15) // 16 * 16, (keep + 15) // 16 * 16
        g = D // _group(D)
        s["codes"] = torch.randint(0, 256, (2, B, NH, cap, D // 2), dtype=torch.uint8, generator=gen, device=DEV)
        s["params"] = torch.randn((2, B, NH, cap, g, 2), generator=gen, device=DEV).half()
        # accumulated weights as decoding leaves them: a few large, most small, some never attended to
        w = torch.rand((B, NH, cap), generator=gen, device=DEV).pow_(6)
        s["weights"] = w.masked_fill_(w < 1e-4, 0.0)
        # earlier evictions have mixed the order: a slot's token position is no longer its index
        s["seen"] = L + L // 2
        order = torch.rand((B, NH, s["seen"]), generator=gen, device=DEV).argsort(-1)
        s["positions"] = torch.zeros((B, NH, cap), dtype=torch.int32, device=DEV)
        s["positions"][:, :, :L] = order[:, :, :L]
        s["lengths"] = torch.tensor(_lengths(case, L), dtype=torch.int32, device=DEV) if case["ragged"] else None
        s["out"] = (torch.zeros((2, B, NH, cap_out, D // 2), dtype=torch.uint8, device=DEV),
                    torch.zeros((2, B, NH, cap_out, g, 2), dtype=torch.float16, device=DEV),
                    torch.zeros((B, NH, cap_out), dtype=torch.float32, device=DEV),
                    torch.zeros((B, NH, cap_out), dtype=torch.int32, device=DEV))
    return s


# ------------------------------------------------------------------------------------ the plain forms
def _quantise(x):
    """Codes and params of float rows [..., D]: scale and minimum in float32, the codes in 64 bits,
    where a value lies next to the border of two codes."""
    D = x.shape[-1]
    x = x.float().reshape(*x.shape[:-1], D // _group(D), _group(D))
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) / 15).clamp(max=F16_MAX).half()
    m = lo.clamp(-F16_MAX, F16_MAX).half()
    n = ((x.double() - m.double()[..., None]) / s.double()[..., None]).round().clamp(0, 15)
    n = torch.where(s[..., None] > 0, n, torch.zeros_like(n)).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.stack((s, m), -1)


def _dequantise(codes, params):
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    n = n.reshape(*params.shape[:-1], -1).float()
    return (n * params[..., :1].float() + params[..., 1:].float()).flatten(-2)


def _scores(q, k, D):
    """scale q.k of q [B, T, NH, D], k [B, S, NKV, D] -> [B, NKV, NH / NKV, T, S]."""
    B, T, NH, _ = q.shape
    q = q.reshape(B, T, k.shape[2], NH // k.shape[2], D).permute(0, 2, 3, 1, 4)
    return q @ k.permute(0, 2, 3, 1)[:, :, None] * (1.0 / math.sqrt(D))


def _plain_store(s):
    case = s["case"]
    B, T, pos, dt = case["B"], case["T"], case["pos"], _dt(case)
    put = torch.arange(T, device=DEV).expand(B, T)
    put = (put < s["counts"][:, None])[:, None, :, None] if s["counts"] is not None else (put >= 0)[:, None, :, None]
    x = torch.stack((s["k"], s["v"])).transpose(2, 3)
    codes, params = _quantise(x)
    at = slice(pos, pos + T)
    s["codes"][:, :, :, at] = torch.where(put, codes, s["codes"][:, :, :, at])
    s["params"][:, :, :, at] = torch.where(put[..., None], params, s["params"][:, :, :, at])
    kv = torch.where(put, _dequantise(s["codes"][:, :, :, at], s["params"][:, :, :, at]), 0.0)
    kv = kv.transpose(2, 3).to(dt)
    return kv[0].contiguous(), kv[1].contiguous()


def _plain_decode(s):
    case = s["case"]
    B, NH, NKV, D, L = case["B"], case["NH"], case["NKV"], case["D"], case["L"]
    kv = _dequantise(s["codes"][:, :, :, :L], s["params"][:, :, :, :L])
    q = s["q"].float().view(B, NKV, NH // NKV, D)
    sc = q @ kv[0].transpose(-1, -2) * (1.0 / math.sqrt(D))
    if s["lengths"] is not None:
        seen = torch.arange(L, device=DEV) < s["lengths"][:, None]
        sc = torch.where(seen[:, None, None], sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (sc - top).exp()
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    out = [(p @ kv[1]).view(B, NH, D).to(_dt(case)), (total.log() + top).view(B, NH)]
    if case["weights"]:
        s["weights_out"][:, :, :L] = s["weights"][:, :, :L] + p.sum(2)
        out.append(s["weights_out"])
    return out


def _plain_weights(s):
    case = s["case"]
    B, NH, NKV, T, D = case["B"], case["NH"], case["NKV"], case["T"], case["D"]
    p = (_scores(s["q"].float(), s["k"].float(), D) - s["lse"].view(B, NKV, NH // NKV, T, 1)).exp()
    i = torch.arange(T, device=DEV)
    use = ((i[:, None] >= i) & (i[:, None] >= case["first"])).expand(B, T, T)
    if s["lengths"] is not None:
        use = use & (i[:, None] < s["lengths"][:, None, None])
    return torch.where(use[:, None, None], p, 0.0).sum((2, 3))


def _plain_evict(s):
    case = s["case"]
    L, keep = case["L"], case["keep"]
    i = torch.arange(L, device=DEV)
    w, pos = s["weights"][:, :, :L], s["positions"][:, :, :L]
    n = s["lengths"][:, None, None] if s["lengths"] is not None else torch.tensor(L, device=DEV)
    order = torch.where(pos >= s["seen"] - case["recent"], math.inf, w)
    order = torch.where(i < n, order, -math.inf)
    best = order.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros(w.shape, dtype=torch.bool, device=DEV).scatter_(-1, best, True) & (i < n)
    # rows kept from slot `keep` on fill, in order, the slots below `keep` that were given up
    spare = torch.where(kept & (i >= keep), i, L).sort(-1).values
    hole = ~kept[..., :keep]
    at = (hole.cumsum(-1) - 1).clamp(min=0, max=L - 1)
    slots = torch.where(hole, spare.gather(-1, at), i[:keep])
    valid = i[:keep] < n
    slots = torch.where(valid, slots, -1)
    src = slots.clamp(min=0)
    codes, params, weights, positions = s["out"]
    src2, ok2 = src[None, ..., None], valid[..., None]
    c = s["codes"].gather(3, src2.expand(2, -1, -1, -1, s["codes"].shape[-1]))
    codes[:, :, :, :keep] = torch.where(ok2, c, codes[:, :, :, :keep])
    flat = s["params"].flatten(-2)
    c = flat.gather(3, src2.expand(2, -1, -1, -1, flat.shape[-1])).view_as(params[:, :, :, :keep])
    params[:, :, :, :keep] = torch.where(ok2[..., None], c, params[:, :, :, :keep])
    weights[:, :, :keep] = torch.where(valid, w.gather(-1, src), weights[:, :, :keep])
    positions[:, :, :keep] = torch.where(valid, pos.gather(-1, src), positions[:, :, :keep])
    # rows are moved, not computed: their bytes have to be the same ones
    return slots.to(torch.int32), codes, params, weights, positions


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        ops = _ops()
        if op == "store":
            ops.kv4_store(s["k"], s["v"], s["codes"], s["params"], case["pos"], counts=s["counts"])
            return ops.kv4_load(s["codes"], s["params"], case["pos"], case["T"], dtype=_dt(case), counts=s["counts"])
        if op == "decode":
            o = ops.kv4_decode(s["q"], s["codes"], s["params"], case["L"], lengths=s["lengths"], lse=s["lse"],
                               weights=s.get("weights"), weights_out=s.get("weights_out"))
            return [o, s["lse"]] + ([s["weights_out"]] if case["weights"] else [])
        if op == "weights":
            return ops.key_weights(s["q"], s["k"], s["lse"], first_query=case["first"], lengths=s["lengths"])
        slots = ops.kv4_evict(s["codes"], s["params"], s["weights"], s["positions"], case["L"], case["keep"],
                              recent=case["recent"], seen=s["seen"], lengths=s["lengths"], out=s["out"])
        return (slots,) + s["out"]
    return {"store": _plain_store, "decode": _plain_decode, "weights": _plain_weights, "evict": _plain_evict}[op](s)


# ------------------------------------------------------------------------------------ work and exact values
def _row_bytes(D):
    return D // 2 + 4 * (D // _group(D))


def work(case):
    B, D = case["B"], case["D"]
    esz = 2 if case.get("dtype") == "bf16" else 4
    if case["op"] == "store":
        rows = 2 * sum(_lengths(case, case["T"])) * case["NH"]
        # read once and held once by the store; read back and written once by the load
        return dict(bytes=rows * (2 * D * esz + 2 * _row_bytes(D)), flops=rows * D * 6)
    if case["op"] == "decode":
        rows = sum(_lengths(case, case["L"])) * case["NKV"]
        extra = 8 * rows if case["weights"] else 0
        return dict(bytes=rows * 2 * _row_bytes(D) + extra + 2 * B * case["NH"] * D * esz,
                    flops=4 * rows * (case["NH"] // case["NKV"]) * D)
    if case["op"] == "weights":
        pairs = sum(n * (n + 1) // 2 - min(n, case["first"]) * (min(n, case["first"]) + 1) // 2
                    for n in _lengths(case, case["T"])) * case["NH"]
        T = case["T"]
        return dict(bytes=B * T * ((case["NH"] + case["NKV"]) * D * esz + 4 * case["NH"] + 4 * case["NKV"]),
                    flops=2 * D * pairs + 4 * pairs)
    n = _lengths(case, case["L"])
    kept = sum(min(x, case["keep"]) for x in n) * case["NH"]
    return dict(bytes=8 * sum(n) * case["NH"] + kept * (4 * _row_bytes(D) + 8 + 4), flops=0)


def _levels(x):
    """The values that 4-bit groups of x stand for, by trying all sixteen codes in 64 bits; the scale
    and minimum are float16 by definition, from float32 arithmetic."""
    D = x.shape[-1]
    g = _group(D)
    xf = x.to(torch.float32).unflatten(-1, (D // g, g))
    lo = xf.min(dim=-1, keepdim=True).values
    hi = xf.max(dim=-1, keepdim=True).values
    s = torch.clamp((hi - lo) / 15.0, max=F16_MAX).to(torch.float16).double()
    m = torch.clamp(lo, -F16_MAX, F16_MAX).to(torch.float16).double()
    best = torch.full(xf.shape, math.inf, dtype=torch.float64, device=x.device)
    value = torch.zeros_like(best)
    for n in list(range(0, 16, 2)) + list(range(1, 16, 2)):  # even codes first: they win a tie
        far = (xf.double() - (m + n * s)).abs()
        nearer = far < best
        best = torch.where(nearer, far, best)
        value = torch.where(nearer, m + n * s, value)
    return value.flatten(-2)


def _held(codes, params):
    """The 64-bit values of held rows."""
    lo, hi = codes.bitwise_and(15).double(), codes.div(16, rounding_mode="floor").double()
    D = 2 * codes.shape[-1]
    n = torch.empty((*codes.shape[:-1], D), dtype=torch.float64, device=codes.device)
    n[..., 0::2], n[..., 1::2] = lo, hi
    p = params.double().repeat_interleave(_group(D), dim=-2)
    return n * p[..., 0] + p[..., 1]


def exact(case, seed):
    s = prepare(case, seed)
    B, D = case["B"], case["D"]
    lens = None
    if case["op"] == "store":
        lens = _lengths(case, case["T"])
        out = []
        for x in (s["k"], s["v"]):
            y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
            for b in range(B):
                if lens[b]:
                    y[b, :lens[b]] = _levels(x[b, :lens[b]])
            out.append(y)
        return tuple(out)
    if case["op"] == "decode":
        NH, NKV, L = case["NH"], case["NKV"], case["L"]
        G = NH // NKV
        o = torch.zeros((B, NH, D), dtype=torch.float64, device=DEV)
        lse = torch.full((B, NH), -math.inf, dtype=torch.float64, device=DEV)
        w = torch.zeros((B, NKV, s["codes"].shape[3]), dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lengths(case, L)):
            if case["weights"]:
                w[b, :, :L] = s["weights"][b, :, :L].double()
            if n == 0:
                continue
            k = _held(s["codes"][0, b, :, :n], s["params"][0, b, :, :n])
            v = _held(s["codes"][1, b, :, :n], s["params"][1, b, :, :n])
            z = torch.einsum("hgd,hnd->hgn", s["q"][b].double().view(NKV, G, D), k) / math.sqrt(D)
            total = torch.logsumexp(z, -1)
            p = torch.exp(z - total[..., None])
            o[b] = torch.einsum("hgn,hnd->hgd", p, v).reshape(NH, D)
            lse[b] = total.reshape(NH)
            w[b, :, :n] += p.sum(1)
        return [o, lse] + ([w] if case["weights"] else [])
    if case["op"] == "weights":
        NH, NKV, T = case["NH"], case["NKV"], case["T"]
        G = NH // NKV
        w = torch.zeros((B, NKV, T), dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lengths(case, T)):
            lo = case["first"]
            if n <= lo:
                continue
            for h in range(NH):
                z = s["q"][b, lo:n, h].double() @ s["k"][b, :n, h // G].double().T / math.sqrt(D)
                p = torch.exp(z - s["lse"][b, h, lo:n].double()[:, None])
                w[b, h // G, :n] += torch.tril(p, diagonal=lo).sum(0)
        return w
    return None  # an eviction computes no numbers: its outputs are whole numbers and moved bytes
