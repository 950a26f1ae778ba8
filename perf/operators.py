"""The 4-bit decode operators, as a user calls them and in plain form.

Three operators that together are one decode step over 4-bit data:

  gemv       y = x W^T (+ residual) for a few tokens, W held as 4-bit codes with a
             scale and a zero point for every `group` columns of a row
  append     new tokens' q and k rotated by position, k and v written into a paged
             cache that holds 4-bit codes with a scale and a zero point for every
             (token, head); the held values are read back
  attention  softmax attention of the new tokens' q over such a cache

The plain forms are elementary torch operations in 32 bits (angles in 64).
"""
import math

import torch

own = False

FP16, BF16 = 0, 1
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
DT_CODE = {"fp16": FP16, "bf16": BF16}


# ------------------------------------------------------------------ cases

def _gemv(name, M, N, K, group, zeros, residual):
    return {"name": name, "op": "gemv", "M": M, "N": N, "K": K, "group": group, "zeros": zeros, "residual": residual}


def _append(name, seqs, q_len, kv_len, heads, kv_heads, head_dim, page, dtype):
    return {"name": name, "op": "append", "seqs": seqs, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}


def _attn(name, seqs, q_len, kv_len, heads, kv_heads, head_dim, page, dtype, causal):
    return {"name": name, "op": "attention", "seqs": seqs, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "causal": causal}


def listed():
    return [
        # one token, the 0.5B shape's output projection: all latency
        _gemv("gemv 896x896 m1", 1, 896, 896, 64, False, True),
        # one token, the 7B shape's gate and up projections: all bandwidth
        _gemv("gemv 37888x3584 m1", 1, 37888, 3584, 128, True, False),
        # a small batch through the 7B down projection: few rows, a long sum, fine groups
        _gemv("gemv 3584x18944 m7", 7, 3584, 18944, 32, True, True),
        # a batch of answers through the 7B vocabulary projection
        _gemv("gemv 152064x3584 m16", 16, 152064, 3584, 128, False, False),
        # decode: 33 sequences, one token each
        _append("append decode 33", 33, 1, 20011, 28, 4, 128, 16, "fp16"),
        # prompts of five lengths, in one call
        _append("append prompts 5x2900", 5, 2900, 2900, 28, 4, 128, 64, "bf16"),
        # the 0.5B shape: one short sequence, one token
        _attn("attn 1x517 d64", 1, 1, 517, 14, 2, 64, 16, "fp16", True),
        # decode: 64 sequences of mixed lengths
        _attn("attn 64x8192", 64, 1, 8192, 28, 4, 128, 64, "fp16", True),
        # decode: one very long sequence
        _attn("attn 1x131071", 1, 1, 131071, 28, 4, 128, 32, "bf16", True),
        # a few drafted tokens checked at once
        _attn("attn 9x3x6000", 9, 3, 6000, 28, 4, 128, 16, "fp16", True),
        # two prompts, most of their keys their own
        _attn("attn prompts 2x1800", 2, 1800, 1900, 14, 2, 64, 128, "fp16", True),
        # a chunk of a long prompt: 2048 new tokens behind 14000 held ones
        _attn("attn chunk 2048x16048", 1, 2048, 16048, 28, 4, 128, 64, "fp16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemv", "append", "attention", "attention"])
    if op == "gemv":
        M = rng.choice([1, 1, 2, 3, 5, 8, 11, 16])
        group = rng.choice([32, 64, 128])
        while True:
            N, K = _log(rng, 200, 152064), group * _log(rng, max(1, 512 // group), 18944 // group)
            if N * K <= 152064 * 3584:
                break
        c = _gemv("", M, N, K, group, rng.random() < 0.5, rng.random() < 0.5)
    else:
        heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (28, 4, 128), (28, 4, 128), (8, 8, 64), (16, 1, 128),
                                                (12, 4, 128), (7, 1, 64)])
        page = rng.choice([16, 32, 64, 128])
        dtype = rng.choice(["fp16", "bf16"])
        if op == "append":
            q_len = rng.choice([1, 1, _log(rng, 2, 4000)])
            seqs = min(_log(rng, 1, 200), max(1, 14000 // q_len))
            c = _append("", seqs, q_len, q_len + _log(rng, 1, 20000) - 1, heads, kv_heads, head_dim, page, dtype)
        else:
            q_len = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 2048)])
            while True:
                seqs, past = _log(rng, 1, 96), _log(rng, 1, 131071) - 1
                pairs = seqs * q_len * (q_len + past) * heads * head_dim
                if seqs * (q_len + past) * kv_heads <= 64 * 8192 * 4 and pairs <= 2048 * 16048 * 28 * 128:
                    break
            c = _attn("", seqs, q_len, q_len + past, heads, kv_heads, head_dim, page, dtype, rng.random() < 0.8)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, tokens held after the call) of each sequence: the first has the case's own, the others fewer."""
    out = []
    for b in range(case["seqs"]):
        f = 1.0 - (b * 0.6180339887498949) % 1.0 * 0.75
        n = max(1, round(case["q_len"] * f))
        past = round((case["kv_len"] - case["q_len"]) * f)
        out.append((n, n + past))
    return out


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _weights(case, seed):
    g = _gen(seed)
    M, N, K, G = case["M"], case["N"], case["K"], case["group"]
    x = _randn(g, M, K)
    x[:, torch.randint(0, K, (max(1, K // 512),), generator=g, device="cuda")] *= 12.0  # a few large channels
    hi = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = {
        "case": case,
        "x": x.half(),
        "codes": hi,  # two columns a byte, the even one in the low half
        "scales": (0.002 + 0.006 * torch.rand(N, K // G, generator=g, device="cuda")).half(),
        "zeros": torch.randint(5, 11, (N, K // G), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None,
        "res": _randn(g, M, N).half() if case["residual"] else None,
    }
    return s


def _batch(case, seed):
    """Where each sequence's tokens are: first row, tokens held, pages (in no order)."""
    g = _gen(seed + 1)
    lens = _lengths(case)
    per = [-(-kv // case["page"]) for _, kv in lens]
    pages = sum(per)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([0] + per, device="cuda").cumsum(0)[:-1]
    at = first[:, None] + torch.arange(max(per), device="cuda")[None, :]
    table = torch.where(torch.arange(max(per), device="cuda")[None, :] < torch.tensor(per, device="cuda")[:, None],
                        order[at.clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    return {
        "case": case,
        "pages": pages,
        "tokens": starts[-1],
        "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
        "kv_len": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda"),
        "table": table.contiguous(),
        "max_q": max(n for n, _ in lens),
        "max_kv": max(kv for _, kv in lens),
    }


def _heads_in(g, case, tokens, heads, dtype, outliers):
    x = _randn(g, tokens, heads, case["head_dim"])
    if outliers:  # keys have a few channels with a large mean
        x[:, :, 3] += 4.0
        x[:, :, case["head_dim"] // 2 + 5] -= 6.0
    return x.to(dtype)


def _held(case, s, seed):
    """The keys and values that the attention cases' caches hold, as they came."""
    g = _gen(seed + 2)
    total = int(sum(kv for _, kv in _lengths(case)))
    k = _heads_in(g, case, total, case["kv_heads"], torch.float16, True)
    v = _heads_in(g, case, total, case["kv_heads"], torch.float16, False)
    return k, v


def _kv_batch(s, q_start=None, max_q=None, tokens=None):
    from mruntime_b200 import capi

    q_start = s["q_start"] if q_start is None else q_start
    return capi.KvBatch(s["case"]["seqs"], s["tokens"] if tokens is None else tokens, max_q or s["max_q"], s["max_kv"],
                        q_start.data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1])


def _quantise(x):
    """4-bit codes, scale and zero point of the last axis, range widened to hold 0."""
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    s = ((hi - lo) * (1.0 / 15.0)).half().clamp(min=2.0 ** -24)
    inv = torch.reciprocal(s.to(x.dtype))
    z = torch.round(-lo * inv).clamp(0, 15)
    c = (torch.round(x * inv) + z).clamp(0, 15)
    return c.to(torch.uint8), s, z.to(torch.uint8)


def _pack(c):
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _unpack(p):
    return torch.stack((p & 15, p >> 4), -1).flatten(-2)


def prepare(case, seed):
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "gemv":
        s = _weights(case, seed)
        if own:
            from mruntime_b200 import capi

            s["w"] = capi.WeightQ4.from_codes(s["codes"].data_ptr(), s["scales"].data_ptr(), capi.FP16,
                                              s["zeros"].data_ptr() if case["zeros"] else None, True, case["N"],
                                              case["K"], case["group"], stream)
            s["codes"] = s["scales"] = s["zeros"] = None
            s["y"] = torch.empty(case["M"], case["N"], dtype=torch.float16, device="cuda")
        return s
    dtype, D = DT[case["dtype"]], case["head_dim"]
    s = _batch(case, seed)
    g = _gen(seed)
    T = s["tokens"]
    s["q"] = _heads_in(g, case, T, case["heads"], dtype, False)
    if case["op"] == "append":
        s["k"] = _heads_in(g, case, T, case["kv_heads"], dtype, True)
        s["v"] = _heads_in(g, case, T, case["kv_heads"], dtype, False)
        theta = s["theta"] = 1000000.0
    else:
        theta = 0.0
    if own:
        from mruntime_b200 import capi

        kv = s["kv"] = capi.KvQ4(s["pages"], case["page"], case["kv_heads"], D, theta)
        s["batch"] = _kv_batch(s)
        if case["op"] == "append":
            s["q_out"] = torch.empty_like(s["q"])
            s["k_held"] = torch.empty(T, case["kv_heads"], D, dtype=torch.float16, device="cuda")
            s["v_held"] = torch.empty_like(s["k_held"])
        else:
            k, v = _held(case, s, seed)
            all_start = torch.cat([s["kv_len"].new_zeros(1), s["kv_len"].cumsum(0).to(torch.int32)])
            kv.append(_kv_batch(s, all_start, s["max_kv"], k.shape[0]), capi.FP16, None, 0, 0, None, 0, k.data_ptr(),
                      k.shape[1] * D, v.data_ptr(), v.shape[1] * D, stream)
            capi.sync(stream)
            s["out"] = torch.empty_like(s["q"])
            n = kv.attention_workspace(s["batch"], case["heads"])
            s["ws"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    else:  # the plain cache: [page, token of the page, head] rows of packed codes, scale and zero point
        rows = s["pages"] * case["page"]
        shape = (rows, case["kv_heads"])
        for n in ("k", "v"):
            s[n + "_codes"] = torch.zeros(*shape, D // 2, dtype=torch.uint8, device="cuda")
            s[n + "_scale"] = torch.zeros(*shape, 1, dtype=torch.float16, device="cuda")
            s[n + "_zero"] = torch.zeros(*shape, 1, dtype=torch.uint8, device="cuda")
        if case["op"] == "attention":
            k, v = _held(case, s, seed)
            seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), s["kv_len"].long())
            pos = torch.arange(k.shape[0], device="cuda") - (s["kv_len"].long().cumsum(0) - s["kv_len"].long())[seq]
            _store(s, seq, pos, k.float(), v.float())
    return s


# ------------------------------------------------------------------ plain forms

def _rows(s, seq, pos):
    return s["table"][seq, pos // s["case"]["page"]].long() * s["case"]["page"] + pos % s["case"]["page"]


def _store(s, seq, pos, k, v):
    at = _rows(s, seq, pos)
    c, sc, z = _quantise(k)
    s["k_codes"][at], s["k_scale"][at], s["k_zero"][at] = _pack(c), sc, z
    c, sc, z = _quantise(v)
    s["v_codes"][at], s["v_scale"][at], s["v_zero"][at] = _pack(c), sc, z
    return at


def _values(s, n, at):
    c = _unpack(s[n + "_codes"][at]).float() - s[n + "_zero"][at].float()
    return c * s[n + "_scale"][at].float()


def _new_tokens(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), t, right=True) - 1
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    return seq, (s["kv_len"].long() - n)[seq] + t - s["q_start"].long()[seq]


def _rotate(x, pos, theta):
    half = x.shape[-1] // 2
    freq = theta ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    a = pos.double()[:, None] * freq
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    x0, x1 = x[..., :half], x[..., half:]
    return torch.cat((x0 * c - x1 * s, x0 * s + x1 * c), -1)


def _plain_gemv(s):
    case, x = s["case"], s["x"].float()
    N, K, G = case["N"], case["K"], case["group"]
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None]
    w = (_unpack(s["codes"]).view(N, K // G, G).float() - zero) * s["scales"].float()[:, :, None]
    y = (x @ w.view(N, K).t()).half()
    if s["res"] is not None:
        y = (s["res"].float() + y.float()).half()
    return {"y": y}


def _plain_append(s):
    seq, pos = _new_tokens(s)
    q = _rotate(s["q"].float(), pos, s["theta"]).to(s["q"].dtype)
    at = _store(s, seq, pos, _rotate(s["k"].float(), pos, s["theta"]), s["v"].float())
    return {"q": q, "k": _values(s, "k", at).half(), "v": _values(s, "v", at).half()}


def _plain_attention(s):
    case = s["case"]
    B, H, Hk, D = case["seqs"], case["heads"], case["kv_heads"], case["head_dim"]
    seq, pos = _new_tokens(s)
    t = torch.arange(s["max_kv"], device="cuda")
    held = t[None, :] < s["kv_len"][:, None]
    at = _rows(s, torch.arange(B, device="cuda")[:, None], torch.where(held, t[None, :], 0))
    k = _values(s, "k", at).permute(0, 2, 3, 1)  # [B, Hk, D, L]
    v = _values(s, "v", at).permute(0, 2, 1, 3)  # [B, Hk, L, D]
    i = torch.arange(s["tokens"], device="cuda") - s["q_start"].long()[seq]
    q = torch.zeros(B, s["max_q"], H, D, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(B, -1, Hk, H // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)  # rows: token, head of the group
    p = torch.matmul(q, k).mul_(D ** -0.5).view(B, Hk, s["max_q"], H // Hk, -1)
    last = torch.full((B, s["max_q"]), -1, dtype=torch.long, device="cuda")
    last[seq, i] = pos if case["causal"] else (s["kv_len"].long() - 1)[seq]
    p.masked_fill_((t[None, None, :] > last[:, :, None])[:, None, :, None, :], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.view(B, Hk, -1, s["max_kv"]), v).view(B, Hk, s["max_q"], H // Hk, D) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(B, s["max_q"], H, D)
    return {"out": o[seq, i].to(s["q"].dtype)}


def run(s):
    case = s["case"]
    if not own:
        return {"gemv": _plain_gemv, "append": _plain_append, "attention": _plain_attention}[case["op"]](s)
    from mruntime_b200 import capi

    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "gemv":
        res = s["res"]
        capi.gemv_q4(s["w"], s["x"].data_ptr(), case["K"], s["y"].data_ptr(), case["N"], case["M"],
                     res_ptr=None if res is None else res.data_ptr(), ldr=case["N"], stream=stream)
        return {"y": s["y"]}
    H, Hk, D, dt = case["heads"], case["kv_heads"], case["head_dim"], DT_CODE[case["dtype"]]
    if case["op"] == "append":
        s["kv"].append(s["batch"], dt, s["q"].data_ptr(), H * D, H, s["q_out"].data_ptr(), H * D, s["k"].data_ptr(),
                       Hk * D, s["v"].data_ptr(), Hk * D, stream)
        s["kv"].read(s["batch"], capi.FP16, s["k_held"].data_ptr(), Hk * D, s["v_held"].data_ptr(), Hk * D, stream)
        return {"q": s["q_out"], "k": s["k_held"], "v": s["v_held"]}
    s["kv"].attention(s["batch"], dt, s["q"].data_ptr(), H * D, H, s["out"].data_ptr(), H * D, D ** -0.5,
                      case["causal"], s["ws"].data_ptr(), s["ws"].numel(), stream)
    return {"out": s["out"]}


def work(case):
    if case["op"] == "gemv":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        b = N * K // 2 + N * (K // G) * (2.5 if case["zeros"] else 2) + M * K * 2 + M * N * (4 if case["residual"] else 2)
        return {"bytes": b, "flops": 2.0 * M * N * K}
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    T = sum(n for n, _ in lens)
    row = D / 2 + 2.5  # a held row: codes, 16-bit scale, 4-bit zero point
    if case["op"] == "append":  # q in and out, k and v in, their rows written and read, their values out
        return {"bytes": T * (4 * H * D + 8 * Hk * D + 4 * Hk * row), "flops": T * (H + Hk) * D * 3.0 + T * Hk * D * 8.0}
    pairs = sum(n * (kv - n) + (n * (n + 1) // 2 if case["causal"] else n * n) for n, kv in lens)
    return {"bytes": sum(kv for _, kv in lens) * Hk * 2 * row + T * H * D * 4, "flops": 4.0 * D * H * pairs}


# ------------------------------------------------------------------ 64 bits

def _exact_gemv(case, seed):
    s = _weights(case, seed)
    N, K, G = case["N"], case["K"], case["group"]
    x = s["x"].double()
    y = torch.empty(case["M"], N, dtype=torch.float64, device="cuda")
    for a in range(0, N, 16384):
        c = s["codes"][a:a + 16384]
        w = torch.empty(c.shape[0], K, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (c % 16).double(), (c // 16).double()
        z = s["zeros"][a:a + 16384].double() if case["zeros"] else torch.full((c.shape[0], K // G), 8.0, dtype=torch.float64, device="cuda")
        w = (w - z.repeat_interleave(G, 1)) * s["scales"][a:a + 16384].double().repeat_interleave(G, 1)
        y[:, a:a + 16384] = torch.einsum("mk,nk->mn", x, w)
    return {"y": y + s["res"].double() if case["residual"] else y}


def _exact_append(case, seed):
    s = prepare_inputs(case, seed)
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    pos = torch.cat([torch.arange(kv - n, kv, device="cuda") for n, kv in _lengths(case)]).double()
    half = case["head_dim"] // 2
    a = torch.outer(pos, torch.tensor([s["theta"] ** (-j / half) for j in range(half)], dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.ones_like(a), a)[:, None, :]

    def rotated(x):
        y = torch.complex(x[..., :half], x[..., half:]) * turn
        return torch.cat((y.real, y.imag), -1)

    def held(x):
        lo, hi = torch.minimum(x.min(-1)[0], x.new_zeros(())), torch.maximum(x.max(-1)[0], x.new_zeros(()))
        step = torch.maximum(((hi - lo) / 15).half().double(), x.new_tensor(2.0 ** -24))[..., None]
        z = torch.round(-lo[..., None] / step).clamp(0, 15)
        return ((torch.round(x / step) + z).clamp(0, 15) - z) * step

    return {"q": rotated(q), "k": held(rotated(k)), "v": held(v)}


def prepare_inputs(case, seed):
    """An append case's inputs alone."""
    g = _gen(seed)
    T, dtype = sum(n for n, _ in _lengths(case)), DT[case["dtype"]]
    q = _heads_in(g, case, T, case["heads"], dtype, False)
    k = _heads_in(g, case, T, case["kv_heads"], dtype, True)
    return {"q": q, "k": k, "v": _heads_in(g, case, T, case["kv_heads"], dtype, False), "theta": 1000000.0}


def _exact_attention(case, seed):
    H, Hk, D, dtype = case["heads"], case["kv_heads"], case["head_dim"], DT[case["dtype"]]
    lens = _lengths(case)
    q = _heads_in(_gen(seed), case, sum(n for n, _ in lens), H, dtype, False)
    k, v = _held(case, None, seed)
    out, row, tok = torch.empty_like(q, dtype=torch.float64), 0, 0
    for n, kv in lens:
        c, s, z = _quantise(k[tok:tok + kv].float())
        kd = (c.double() - z.double()) * s.double()
        c, s, z = _quantise(v[tok:tok + kv].float())
        vd = (c.double() - z.double()) * s.double()
        for a in range(0, n, 512):
            m = min(512, n - a)
            qd = q[row + a:row + a + m].double().view(m, Hk, H // Hk, D)
            w = torch.einsum("mhgd,thd->hgmt", qd, kd) / math.sqrt(D)
            if case["causal"]:
                w += torch.full((m, kv), -math.inf, dtype=torch.float64, device="cuda").triu(kv - n + a + 1)
            out[row + a:row + a + m] = torch.einsum("hgmt,thd->mhgd", w.softmax(-1), vd).reshape(m, H, D)
        row, tok = row + n, tok + kv
    return {"out": out}


def exact(case, seed):
    return {"gemv": _exact_gemv, "append": _exact_append, "attention": _exact_attention}[case["op"]](case, seed)
