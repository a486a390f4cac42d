"""Cases for the ragged-batch operators: keys and values appended to a paged cache (coda_paged_append), attention of a chunk
of new tokens over that cache (coda_paged_attn), and low-rank adapters of many requests beside a shared projection
(coda_lora_bf16).  Sizes are the decoder's (hidden 2048, MLP 6144, 16 query heads, 8 key/value heads of 128) and the
batches, block lengths and context lengths that the sampler, its benchmark and its tests run, plus other head counts and
odd sizes around them."""
import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
D = 128
BF = torch.bfloat16
F8 = torch.float8_e4m3fn
K_SCALE, V_SCALE = 1.0 / 32, 1.0 / 64  # e4m3 caches: value = scale * stored


def listed():
    # mask: 0 = every key of the sequence, m = blocks of m positions (1: causal)
    return [
        # one token for each of a batch of requests: the launch-latency end of the cache write
        dict(name="append_token_b32", op="append", B=32, lo=1, hi=1, past=383, page=16, n_q=16, n_kv=8, cache="bf16"),
        # a denoise block of 32 positions for 128 requests, written as e4m3
        dict(name="append_block_b128_e4m3", op="append", B=128, lo=32, hi=32, past=512, page=64, n_q=16, n_kv=8, cache="e4m3"),
        # prompts of very different lengths on their way into an empty cache
        dict(name="append_prompts_b32", op="append", B=32, lo=1, hi=1024, past=0, page=64, n_q=16, n_kv=8, cache="bf16"),
        # one request, one token: nothing but latency
        dict(name="attn_token_b1", op="attn", B=1, lo=1, hi=1, past=383, page=16, n_q=16, n_kv=8, cache="bf16", mask=1),
        # the benchmark's batch: a denoise block of 32 sees the whole 384-token sequence, later positions included
        dict(name="attn_block32_b32", op="attn", B=32, lo=32, hi=32, past=352, page=16, n_q=16, n_kv=8, cache="bf16", mask=0),
        # many requests of unequal length, one token each, e4m3 cache
        dict(name="attn_token_b128_e4m3", op="attn", B=128, lo=1, hi=1, past=2047, page=64, n_q=16, n_kv=8, cache="e4m3", mask=1),
        # few requests at the model's longest context: the work has to be split over the keys
        dict(name="attn_token_b4_40k", op="attn", B=4, lo=1, hi=1, past=40959, page=64, n_q=16, n_kv=8, cache="bf16", mask=1),
        # the long-form setting: blocks of 64 behind a 1024..2048-token prefix, block-causal
        dict(name="attn_block64_b16", op="attn", B=16, lo=64, hi=64, past=1984, page=32, n_q=16, n_kv=8, cache="bf16", mask=64),
        # ragged prompt chunks, causal, behind what is already cached: the matrix-product end
        dict(name="attn_prompts_b8", op="attn", B=8, lo=700, hi=2048, past=1000, page=64, n_q=16, n_kv=8, cache="bf16", mask=1),
        # one token for each of 32 requests, an adapter each, beside the fused q|k|v projection
        dict(name="lora_token_b32_r16", op="lora", B=32, lo=1, hi=1, K=2048, N=4096, rank=16, adapters=32),
        # denoise blocks beside the down projection, fewer adapters than requests
        dict(name="lora_block_b32_r64", op="lora", B=32, lo=32, hi=32, K=6144, N=2048, rank=64, adapters=8),
        # prompts beside the gate projection
        dict(name="lora_prompts_b32_r32", op="lora", B=32, lo=1, hi=1024, K=2048, N=6144, rank=32, adapters=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "lora"])
    if op == "lora":
        K, N = rng.choice([(2048, 4096), (2048, 2048), (6144, 2048), (2048, 6144), (256, 512), (512, 1056), (1088, 264)])
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 16384 // B))
        rank = rng.choice([8, 16, 24, 32, 64, 128])
        return dict(op=op, B=B, lo=rng.choice([0, 1, hi]), hi=hi, K=K, N=N, rank=rank, adapters=_log(rng, 1, min(48, 1024 // rank)))
    n_q, n_kv = rng.choice([(16, 8), (16, 8), (16, 16), (16, 2), (8, 1), (12, 4), (6, 2), (2, 1)])
    page = rng.choice([1, 8, 16, 24, 32, 64, 100, 128, 256])
    cache = rng.choice(["bf16", "bf16", "e4m3"])
    if op == "append":
        B = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, 16384 // B))
        past = rng.choice([0, _log(rng, 1, 4096)])
        return dict(op=op, B=B, lo=rng.choice([0, 1, hi]), hi=hi, past=past, page=page, n_q=n_q, n_kv=n_kv, cache=cache)
    mask = rng.choice([0, 1, 1, 4, 32, 64])
    B = _log(rng, 1, 160)
    hi = rng.choice([1, 1, 32, _log(rng, 2, max(2, min(2048, 8192 // B)))])
    lo = rng.choice([0, 1, hi])
    past = _log(rng, 1, max(1, min(40000, 1280000 // (n_kv * B)) if hi < 64 else min(3800, 16000 // B)))
    return dict(op=op, B=B, lo=lo, hi=hi, past=past, page=page, n_q=n_q, n_kv=n_kv, cache=cache, mask=mask)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """New tokens of each sequence: between lo and hi, fixed by the case alone.  The first sequence has hi."""
    r = random.Random("%(op)s %(B)d %(lo)d %(hi)d" % case)
    return [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["B"] - 1)]


def _past(case):
    """Positions already in the cache: the first sequence has all of `past`, the others down to a quarter of it."""
    r = random.Random("past %(B)d %(past)d" % case)
    return [case["past"]] + [r.randint(case["past"] // 4, case["past"]) for _ in range(case["B"] - 1)]


def _starts(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lengths(case)
    starts = _starts(lens)
    T, B = starts[-1], case["B"]
    s = dict(op=case["op"], T=T, B=B, lens=lens, seq_start=_i32(starts))

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * std

    # token -> its sequence and its place in it (the plain form's indexes)
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(lens, device=DEV))
    s["seq"] = seq
    s["place"] = torch.arange(T, device=DEV) - s["seq_start"].long()[seq]
    if case["op"] == "lora":
        K, N, r, n = case["K"], case["N"], case["rank"], case["adapters"]
        s.update(K=K, N=N, rank=r, n=n, x=normal(T, K).to(BF), resid=normal(T, N).to(BF),
                 a=normal(n, r, K, std=K ** -0.5).to(BF), b=normal(n, N, r, std=r ** -0.5).to(BF),
                 scale=torch.rand(n, generator=g, device=DEV) + 0.5,
                 # about one request in eight runs without an adapter
                 adapter=torch.where(torch.rand(B, generator=g, device=DEV) < 0.125, -1,
                                     torch.randint(0, n, (B,), generator=g, device=DEV)).to(torch.int32))
        s["out"] = torch.empty(T, N, device=DEV, dtype=BF)
    else:
        n_q, n_kv, page = case["n_q"], case["n_kv"], case["page"]
        past = _past(case)
        total = [p + n for p, n in zip(past, lens)]
        max_pages = max(1, -(-max(total) // page))
        pages = sum(-(-t // page) for t in total)
        pool = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros(B, max_pages, dtype=torch.int32, device=DEV)
        used = torch.tensor([-(-t // page) for t in total], device=DEV)
        inside = torch.arange(max_pages, device=DEV)[None, :] < used[:, None]
        table[inside] = pool
        f8 = case["cache"] == "e4m3"
        shape = (max(1, pages), n_kv, page, D)
        if case["op"] == "append":            # what is in the other slots does not matter to the call: zeros show that they stay
            k, v = torch.zeros(2, *shape, device=DEV, dtype=BF)
        else:
            k, v = normal(*shape, std=1.5), normal(*shape)
        if f8:
            k, v = (k / K_SCALE).to(F8), (v / V_SCALE).to(F8)
        s.update(n_q=n_q, n_kv=n_kv, page=page, f8=f8, table=table, max_pages=max_pages, num_pages=shape[0], max_kv=max(total),
                 pos0=_i32(past), kv_len=_i32(total), k=k.to(F8 if f8 else BF), v=v.to(F8 if f8 else BF))
        if case["op"] == "append":
            inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D))
            ang = torch.arange(s["max_kv"], dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
            ang = torch.cat((ang, ang), dim=-1)
            s.update(cos=ang.cos().to(BF), sin=ang.sin().to(BF), qkv=normal(T, (n_q + 2 * n_kv) * D).to(BF),
                     qw=(normal(D, std=0.2) + 1).to(BF), kw=(normal(D, std=0.2) + 1).to(BF), eps=1e-6,
                     q_out=torch.empty(T, n_q * D, device=DEV, dtype=BF))
        else:
            s.update(q=normal(T, n_q * D, std=1.5).to(BF), out=torch.empty(T, n_q * D, device=DEV, dtype=BF), mask=case["mask"],
                     sm=1.0 / math.sqrt(D))
    if own:
        from coda_amd import _lib
        s["call"] = _lib.call
        size = 0
        if case["op"] == "attn":
            size = _lib.load().coda_paged_attn_workspace_bytes(T, B, s["max_kv"], s["n_q"], s["n_kv"])
        elif case["op"] == "lora":
            size = _lib.load().coda_lora_workspace_bytes(T, B, s["N"], s["K"], s["rank"])
        s["ws"], s["ws_bytes"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV), size
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "append":
        return _own_append(s) if own else _plain_append(s)
    if s["op"] == "attn":
        return _own_attn(s) if own else _plain_attn(s)
    return _own_lora(s) if own else _plain_lora(s)


def _own_append(s):
    qkv, q_out, k, v = s["qkv"], s["q_out"], s["k"], s["v"]
    s["call"]("coda_paged_append", qkv.data_ptr(), qkv.stride(0), q_out.data_ptr(), q_out.stride(0), s["qw"].data_ptr(),
              s["kw"].data_ptr(), s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], s["seq_start"].data_ptr(),
              s["pos0"].data_ptr(), s["B"], s["T"], s["table"].data_ptr(), s["table"].stride(0), s["max_pages"], k.data_ptr(),
              v.data_ptr(), k.stride(0), s["num_pages"], s["page"], int(s["f8"]), K_SCALE, V_SCALE, s["n_q"], s["n_kv"], s["eps"], 0,
              torch.cuda.current_stream().cuda_stream)
    return {"q": q_out, "k": k, "v": v}


def _own_attn(s):
    q, out, k = s["q"], s["out"], s["k"]
    s["call"]("coda_paged_attn", q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), s["seq_start"].data_ptr(),
              s["pos0"].data_ptr(), s["kv_len"].data_ptr(), s["B"], s["T"], s["table"].data_ptr(), s["table"].stride(0),
              s["max_pages"], k.data_ptr(), s["v"].data_ptr(), k.stride(0), s["num_pages"], s["page"], int(s["f8"]), K_SCALE, V_SCALE,
              s["max_kv"], s["n_q"], s["n_kv"], s["sm"], s["mask"], s["ws"].data_ptr(), s["ws_bytes"],
              torch.cuda.current_stream().cuda_stream)
    return out


def _own_lora(s):
    x, resid, out = s["x"], s["resid"], s["out"]
    s["call"]("coda_lora_bf16", x.data_ptr(), x.stride(0), s["a"].data_ptr(), s["b"].data_ptr(), s["scale"].data_ptr(),
              s["seq_start"].data_ptr(), s["adapter"].data_ptr(), s["B"], s["T"], s["n"], s["rank"], resid.data_ptr(),
              resid.stride(0), out.data_ptr(), out.stride(0), s["N"], s["K"], s["ws"].data_ptr(), s["ws_bytes"],
              torch.cuda.current_stream().cuda_stream)
    return out


def _norm_rotate(x, w, cos, sin, eps):
    """x [T, heads, 128] in fp32 -> normalised over the head, times w, rotated."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = torch.cat((-x[..., D // 2:], x[..., :D // 2]), dim=-1)
    return x * cos[:, None, :] + half * sin[:, None, :]


def _plain_append(s):
    T, n_q, n_kv = s["T"], s["n_q"], s["n_kv"]
    pos = s["pos0"].long()[s["seq"]] + s["place"]
    cos, sin = s["cos"][pos].float(), s["sin"][pos].float()
    x = s["qkv"].float().view(T, n_q + 2 * n_kv, D)
    q = _norm_rotate(x[:, :n_q], s["qw"].float(), cos, sin, s["eps"])
    k = _norm_rotate(x[:, n_q:n_q + n_kv], s["kw"].float(), cos, sin, s["eps"])
    v = x[:, n_q + n_kv:]
    page, slot = s["table"].long()[s["seq"], pos // s["page"]], pos % s["page"]
    if s["f8"]:
        # 8-bit values are written through their bytes: indexed writes of the type itself are not offered everywhere
        s["k"].view(torch.uint8)[page, :, slot] = (k * (1 / K_SCALE)).clamp(-448, 448).to(F8).view(torch.uint8)
        s["v"].view(torch.uint8)[page, :, slot] = (v * (1 / V_SCALE)).clamp(-448, 448).to(F8).view(torch.uint8)
    else:
        s["k"][page, :, slot] = k.to(BF)
        s["v"][page, :, slot] = v.to(BF)
    s["q_out"].copy_(q.reshape(T, n_q * D))
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_attn(s):
    B, n_q, n_kv, longest, most = s["B"], s["n_q"], s["n_kv"], max(s["lens"]), s["max_kv"]
    group = n_q // n_kv
    table = s["table"].long()

    def dense(cache, scale):                  # pages -> [B, n_kv, keys, 128] in fp32
        x = cache.view(torch.uint8)[table].view(F8).float() * scale if s["f8"] else cache[table].float()
        return x.permute(0, 2, 1, 3, 4).reshape(B, n_kv, -1, D)[:, :, :most]

    q = s["q"].new_zeros(B, longest, n_kv, group, D)
    q[s["seq"], s["place"]] = s["q"].view(-1, n_kv, group, D)
    q = q.float().permute(0, 2, 3, 1, 4).reshape(B, n_kv, group * longest, D)
    scores = torch.matmul(q, dense(s["k"], K_SCALE).transpose(-1, -2).contiguous()).mul_(s["sm"])
    place = torch.arange(longest, device=DEV)
    limit = s["kv_len"].long()[:, None].expand(B, longest)
    if s["mask"]:
        pos = s["pos0"].long()[:, None] + place[None, :]
        limit = torch.minimum(limit, (pos // s["mask"] + 1) * s["mask"])
    seen = torch.arange(most, device=DEV)[None, None, :] < limit[:, :, None]
    scores.view(B, n_kv, group, longest, most).masked_fill_(~seen[:, None, None], float("-inf"))
    scores = (scores - scores.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(scores, dense(s["v"], V_SCALE)) / scores.sum(-1, keepdim=True)
    out = out.view(B, n_kv, group, longest, D).permute(0, 3, 1, 2, 4)[s["seq"], s["place"]]
    s["out"].copy_(out.reshape(-1, n_q * D))
    return s["out"]


def _plain_lora(s):
    # every adapter's down projection of every token, the token's own one kept: no gather of whole weight matrices
    T, n, r, N = s["T"], s["n"], s["rank"], s["N"]
    who = s["adapter"].long()[s["seq"]]
    u = torch.matmul(s["x"].float(), s["a"].float().view(n * r, -1).t()).view(T, n, r)
    mine = torch.nn.functional.one_hot(who.clamp(min=0), n).float() * ((who >= 0).float() * s["scale"][who.clamp(min=0)])[:, None]
    u = (u * mine[:, :, None]).view(T, n * r)
    w = s["b"].float().permute(0, 2, 1).reshape(n * r, N)
    s["out"].copy_(s["resid"].float() + torch.matmul(u, w))
    return s["out"]


# ------------------------------------------------------------------------------------------------ work, exact values
def work(case):
    lens = _lengths(case)
    T = sum(lens)
    if case["op"] == "lora":
        K, N, r = case["K"], case["N"], case["rank"]
        used = min(case["adapters"], case["B"])
        return {"bytes": 2 * (T * K + 2 * T * N + used * r * (K + N)), "flops": 2 * T * r * (K + N)}
    n_q, n_kv, size = case["n_q"], case["n_kv"], 1 if case["cache"] == "e4m3" else 2
    past = _past(case)
    if case["op"] == "append":
        return {"bytes": T * D * (2 * (n_q + 2 * n_kv) + 2 * n_q + 2 * n_kv * size) + 4 * T * D, "flops": 10 * T * (n_q + n_kv) * D}
    keys = pairs = 0
    m = case["mask"]
    for p, n in zip(past, lens):
        if not n:
            continue
        if not m:
            keys, pairs = keys + p + n, pairs + n * (p + n)
        else:
            seen = [min(p + n, (x // m + 1) * m) for x in range(p, p + n)]
            keys, pairs = keys + seen[-1], pairs + sum(seen)
    return {"bytes": 4 * T * n_q * D + 2 * keys * n_kv * D * size, "flops": 4 * D * n_q * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    starts = _starts(s["lens"])
    f64 = torch.float64
    if case["op"] == "lora":
        out = s["resid"].to(f64)
        for b, a in enumerate(s["adapter"].tolist()):
            rows = slice(starts[b], starts[b + 1])
            if a >= 0 and s["lens"][b]:
                low = s["x"][rows].to(f64) @ s["a"][a].to(f64).t().contiguous()
                out[rows] += float(s["scale"][a]) * (low @ s["b"][a].to(f64).t().contiguous())
        return out
    n_q, n_kv, page = s["n_q"], s["n_kv"], s["page"]
    past = s["pos0"].tolist()

    def stored(cache, scale):
        return cache.to(f64) * scale if s["f8"] else cache.to(f64)

    if case["op"] == "append":
        # the cache as it is returned: stored values, for e4m3 before the scale and within the type's range
        q, k, v = torch.empty(s["T"], n_q * D, device=DEV, dtype=f64), stored(s["k"], 1.0), stored(s["v"], 1.0)
        for b, n in enumerate(s["lens"]):
            if not n:
                continue
            x = s["qkv"][starts[b]:starts[b + 1]].to(f64).view(n, -1, D)
            at = torch.arange(past[b], past[b] + n, device=DEV)
            c, z = s["cos"][at].to(f64)[:, None, :64], s["sin"][at].to(f64)[:, None, :64]

            def turned(h, w):
                h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / D + s["eps"]) * w.to(f64)
                lo, hi = h[..., :64], h[..., 64:]
                return torch.cat((lo * c - hi * z, hi * c + lo * z), dim=-1)

            q[starts[b]:starts[b + 1]] = turned(x[:, :n_q], s["qw"]).reshape(n, -1)
            kk, vv = turned(x[:, n_q:n_q + n_kv], s["kw"]), x[:, n_q + n_kv:]
            if s["f8"]:
                kk, vv = (kk / K_SCALE).clamp(-448, 448), (vv / V_SCALE).clamp(-448, 448)
            row = s["table"][b].long()[at // page]
            k[row, :, at % page], v[row, :, at % page] = kk, vv
        return {"q": q, "k": k, "v": v}
    if work(case)["flops"] > 2e12:
        return None
    out = torch.zeros(s["T"], n_q, D, device=DEV, dtype=f64)
    for b, n in enumerate(s["lens"]):
        if not n:
            continue
        keys = past[b] + n
        at = torch.arange(keys, device=DEV)
        row = s["table"][b].long()[at // page]
        raw = (lambda c: c.view(torch.uint8)[row, :, at % page].view(F8)) if s["f8"] else (lambda c: c[row, :, at % page])
        k, v = stored(raw(s["k"]), K_SCALE), stored(raw(s["v"]), V_SCALE)
        q = s["q"][starts[b]:starts[b + 1]].to(f64).view(n, n_q, D)
        pos = torch.arange(past[b], keys, device=DEV)
        seen = at[None, :] < (keys if not s["mask"] else (pos // s["mask"] + 1) * s["mask"])[:, None] if s["mask"] else None
        for h in range(n_q):
            z = q[:, h] @ k[:, h // (n_q // n_kv)].t().contiguous() * s["sm"]
            if seen is not None:
                z = z.masked_fill(~seen, float("-inf"))
            out[starts[b]:starts[b + 1], h] = torch.softmax(z, dim=-1) @ v[:, h // (n_q // n_kv)].contiguous()
    return out.view(s["T"], n_q * D)
