"""The serving operators on a paged key-value cache, and the log probabilities of an answer's tokens: cases to measure.

Each case is one call of one operator.  ``run`` computes it in its plain form (elementary torch operations in fp32, rounded
once at the end) or, where ``own`` is true, through this package's entry points; ``exact`` computes it again in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a prompt of one request just answered, and the step of a middling batch, each on the vocabulary of the 250M model
        # (rows padded to 64 columns as the output projection writes them)
        dict(name="logprobs_1row", op="logprobs", rows=1, vocab=50257, dtype="bf16", top=5, temperature=1.0, masked=False),
        dict(name="logprobs_step64", op="logprobs", rows=64, vocab=50257, dtype="bf16", top=20, temperature=0.8, masked=True),
        # scoring whole prompts (four sequences of 2048 tokens): every position's token, entropy and best alternative
        dict(name="logprobs_prompt", op="logprobs", rows=8192, vocab=50257, dtype="bf16", top=1, temperature=1.0, masked=False),
        # one decode step of 64 running requests, and a batch of prompts that is admitted at once
        dict(name="plan_decode64", op="plan", batch=64, page=16, new=1, context=8192, width=513, room=64),
        dict(name="plan_prefill", op="plan", batch=250, page=16, new=511, context=0, width=64, room=65536),
        # the 250M model's heads (8 query, 2 key-value, size 32) in the model's own [B, H, S, hd] order, interleaved pairs
        dict(name="norm_rope_model", op="norm_rope", batch=4, seq=2048, hq=8, hkv=2, hd=32, rot=32, layout="interleaved",
             norm="l2", dtype="bf16", order="bhsd"),
        # a ragged odd size: packed tokens out of one qkv projection, part of the head rotated, half-precision storage
        dict(name="norm_rope_ragged", op="norm_rope", batch=1, seq=4099, hq=20, hkv=5, hd=80, rot=40, layout="half",
             norm="rms", dtype="f16", order="thd"),
        # one decode step of 64 requests (three rows of padding) and a long prefill chunk, into the cache
        dict(name="append_decode64", op="append", tokens=64, pad=3, hq=32, hkv=8, hd=128, rot=128, layout="half", norm="rms",
             dtype="bf16", page=16),
        dict(name="append_prefill", op="append", tokens=32768, pad=0, hq=32, hkv=8, hd=128, rot=128, layout="half", norm="rms",
             dtype="bf16", page=16),
        # attention of one token: a short chat, a mixed batch (lengths spread from a few to 8192), one very long document
        dict(name="attn_chat", op="attention", batch=1, hq=32, hkv=8, hd=128, page=16, longest=1500, spread=0.0, dtype="bf16",
             order="hnd"),
        dict(name="attn_batch64", op="attention", batch=64, hq=32, hkv=4, hd=64, page=16, longest=8192, spread=1.0, dtype="bf16",
             order="nhd"),
        dict(name="attn_long", op="attention", batch=1, hq=32, hkv=8, hd=128, page=64, longest=131072, spread=0.0, dtype="f16",
             order="hnd"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "plan", "norm_rope", "append", "attention"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 160000)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = 8192 * 50257 // (2 if dtype == "f32" else 1)
        return dict(op=op, rows=max(1, min(_log(rng, 1, 8192), most // (vocab + 64))), vocab=vocab, dtype=dtype,
                    top=rng.choice([0, 1, 3, 5, 8, 20, 32]), temperature=rng.choice([1.0, 0.7, 1.3]), masked=rng.random() < 0.3)
    if op == "plan":
        page = rng.choice([1, 8, 16, 16, 24, 32, 64])
        batch = _log(rng, 1, 1024)
        if rng.random() < 0.5:  # a decode step
            context = _log(rng, 16, 16384)
            return dict(op=op, batch=batch, page=page, new=1, context=context, width=context // page + 2, room=batch + rng.randrange(32))
        new = max(1, min(_log(rng, 16, 8192), 120000 // batch))
        context = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(op=op, batch=batch, page=page, new=new, context=context, width=(context + new) // page + 2,
                    room=max(new, batch * new // 2 + batch) + rng.randrange(512))
    if op in ("norm_rope", "append"):
        hkv = rng.choice([1, 2, 3, 4, 5, 8])
        hq = hkv * rng.choice([1, 2, 3, 4, 6, 8])
        hd = rng.choice([8, 16, 32, 48, 64, 80, 96, 128, 192, 256])
        rot = rng.choice([hd, hd, hd // 2, 2 * rng.randrange(1, hd // 2 + 1)])
        most = 32768 * 40 * 128 // ((hq + 2 * hkv) * hd)
        tokens = max(1, min(_log(rng, 1, 65536), most))
        case = dict(op=op, hq=hq, hkv=hkv, hd=hd, rot=rot, layout=rng.choice(["half", "interleaved"]),
                    norm=rng.choice(["rms", "rms", "l2", "none"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        if case["dtype"] == "f32":
            tokens = max(1, tokens // 2)
        if op == "append":
            return dict(case, tokens=tokens, pad=rng.randrange(0, 1 + min(7, tokens - 1)), page=rng.choice([1, 16, 24, 64]))
        batch = rng.choice([1, 1, 2, 3])
        return dict(case, batch=batch, seq=max(1, tokens // batch), order=rng.choice(["bhsd", "bshd"]) if batch > 1 else "thd")
    hkv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([8, 16, 32, 64, 64, 80, 128, 128, 256])
    batch = _log(rng, 1, 256)
    spread = rng.choice([0.0, 0.5, 1.0, 2.0])
    most = 131072 * 8 * 128 // (hkv * hd * batch)
    return dict(op=op, batch=batch, hq=hkv * rng.choice([1, 2, 4, 5, 8, 16, 20]), hkv=hkv, hd=hd, page=rng.choice([1, 16, 16, 24, 64, 128]),
                longest=max(1, min(_log(rng, 1, 131072), most)), spread=spread, dtype=rng.choice(["bf16", "bf16", "f16"]),
                order=rng.choice(["hnd", "nhd"]))


def _lengths(case):
    """Lengths of a batch before they are shuffled: all `longest`, or spread from a few tokens to `longest` (a few of a large
    spread batch are empty: rows that a captured step keeps for requests to come)."""
    B, top = case["batch"], case["longest"]
    if case["spread"] == 0.0:
        return [top] * B
    return [int(top * ((i + 1) / B) ** case["spread"]) for i in range(B)]


def _new_lengths(case):
    """New tokens of a batch of requests: one each, or one to `new` spread evenly."""
    B, new = case["batch"], case["new"]
    return [1 + i * (new - 1) // (B - 1) for i in range(B)] if B > 1 else [new]


# -------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"logprobs": _prepare_logprobs, "plan": _prepare_plan, "norm_rope": _prepare_norm_rope, "append": _prepare_append,
            "attention": _prepare_attention}[case["op"]](dict(case), g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _prepare_logprobs(case, g):
    """Logits with a few likely tokens in every row; the given token is one of those in three rows of four; where a grammar
    masks, seven of ten columns are -inf."""
    N, V = case["rows"], case["vocab"]
    x = torch.empty(N, -(-V // 64) * 64, dtype=DTYPES[case["dtype"]], device="cuda")
    for i in range(0, N, 1024):
        x[i:i + 1024] = 2.0 * _randn(g, *x[i:i + 1024].shape)
    tokens = _ints(g, 0, V, N)
    likely = _ints(g, 0, V, N, 4)
    likely[:, 0] = torch.where(_ints(g, 0, 4, N) > 0, tokens, likely[:, 0])
    x.scatter_(1, likely, (6.0 + 3.0 * _randn(g, N, 4)).to(x.dtype))
    if case["masked"]:
        for i in range(0, N, 1024):
            n = min(1024, N - i)
            keep = _ints(g, 0, 10, n, x.shape[1]) < 3
            keep.scatter_(1, likely[i:i + n], True)
            x[i:i + n].masked_fill_(~keep, float("-inf"))
    if N > 8:
        tokens[_ints(g, 0, N, 1)] = -100  # a position whose token is not scored
    return dict(case, logits=x, tokens=tokens)


def _prepare_plan(case, g):
    """Requests with `context` tokens at most in their pages, which lie anywhere in the cache, and a list of free pages."""
    B, P, W = case["batch"], case["page"], case["width"]
    order = torch.randperm(B, generator=g, device="cuda")
    new = torch.tensor(_new_lengths(case), dtype=torch.int32, device="cuda")[order]
    context = _ints(g, 0, case["context"] + 1, B).to(torch.int32) if case["context"] else torch.zeros(B, dtype=torch.int32, device="cuda")
    pages = torch.randperm(2 * B * W + 64, generator=g, device="cuda").to(torch.int32)
    table = pages[:B * W].view(B, W).clone()
    held = (context + P - 1) // P
    table[torch.arange(W, device="cuda")[None] >= held[:, None]] = -1
    return dict(case, context_lens=context, new_lens=new, table=table, free=pages[B * W:].clone())


def _tables(rows, rot):
    """cos and sin of position / 10000^(2i / rot), in 64 bits, held in 32."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-2.0 * i / rot)[None]
    return a.cos().float(), a.sin().float()


def _weights(case, g):
    if case["norm"] != "rms":
        return None, None
    return 1 + 0.1 * _randn(g, case["hd"]), 1 + 0.1 * _randn(g, case["hd"])


def _prepare_norm_rope(case, g):
    """q and k: views of one projection's rows (packed tokens, or [B, S, H, hd]), or contiguous [B, H, S, hd]."""
    B, S, hq, hkv, hd, dt = (case[k] for k in ("batch", "seq", "hq", "hkv", "hd", "dtype"))
    cos, sin = _tables(max(4096, S + 1000), case["rot"])
    wq, wk = _weights(case, g)
    if case["order"] == "bhsd":
        q, k = _randn(g, B, hq, S, hd).to(DTYPES[dt]), _randn(g, B, hkv, S, hd).to(DTYPES[dt])
    else:
        rows = _randn(g, B, S, hq + 2 * hkv, hd).to(DTYPES[dt])
        q, k = rows[:, :, :hq], rows[:, :, hq:hq + hkv]
        q, k = (q[0], k[0]) if case["order"] == "thd" else (q.transpose(1, 2), k.transpose(1, 2))
    first = _ints(g, 0, 1000, B, 1)
    positions = (first + torch.arange(S, device="cuda")[None]).to(torch.int32)
    return dict(case, q=q, k=k, cos=cos, sin=sin, wq=wq, wk=wk, positions=positions[0] if case["order"] == "thd" else positions)


def _prepare_append(case, g):
    """A projection's rows of packed tokens, the slots that they go to, and a cache that holds other tokens already.  The last
    `pad` rows are those of a batch that is not full: position and slot -1."""
    T, pad, hq, hkv, hd, P = (case[k] for k in ("tokens", "pad", "hq", "hkv", "hd", "page"))
    dt = DTYPES[case["dtype"]]
    cos, sin = _tables(8192, case["rot"])
    wq, wk = _weights(case, g)
    rows = _randn(g, T, hq + 2 * hkv, hd).to(dt)
    pages = -(-T // P) + 4
    kc, vc = _randn(g, pages, hkv, P, hd).to(dt), _randn(g, pages, hkv, P, hd).to(dt)
    slots = torch.randperm(pages * P, generator=g, device="cuda")[:T].clone()
    if T > 256:  # a prompt's tokens lie side by side in their pages
        n = torch.arange(T, device="cuda")
        slots = torch.randperm(pages, generator=g, device="cuda")[n // P] * P + n % P
    positions = _ints(g, 0, 8192, T).to(torch.int32)
    slots[T - pad:], positions[T - pad:] = -1, -1
    return dict(case, q=rows[:, :hq], k=rows[:, hq:hq + hkv], v=rows[:, hq + hkv:], cos=cos, sin=sin, wq=wq, wk=wk,
                kc=kc, vc=vc, slots=slots, positions=positions)


def _prepare_attention(case, g):
    """Queries and keys of unit-norm heads times their size's root, as after a norm; pages anywhere in the cache, what lies
    behind a request's length is whatever was there."""
    B, hq, hkv, hd, P = (case[k] for k in ("batch", "hq", "hkv", "hd", "page"))
    dt = DTYPES[case["dtype"]]
    lens = torch.tensor(_lengths(case), device="cuda")[torch.randperm(B, generator=g, device="cuda")]
    W = -(-case["longest"] // P)
    pages = sum(-(-n // P) for n in _lengths(case)) + 3
    shape = (pages, hkv, P, hd) if case["order"] == "hnd" else (pages, P, hkv, hd)
    kc, vc = torch.empty(shape, dtype=dt, device="cuda"), torch.empty(shape, dtype=dt, device="cuda")
    step = max(1, (1 << 26) // max(1, hkv * P * hd))
    for c in (kc, vc):
        for i in range(0, pages, step):
            c[i:i + step] = _randn(g, *c[i:i + step].shape)
    if case["order"] == "nhd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    need = (lens + P - 1) // P
    here = torch.arange(W, device="cuda")[None] < need[:, None]
    table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = (here.flatten().cumsum(0) - 1).clamp(min=0).view(B, W)
    table = torch.where(here, order[at], table)
    return dict(case, q=(1.5 * _randn(g, B, hq, hd)).to(dt), kc=kc, vc=vc, table=table, lens=lens.to(torch.int32), scale=hd ** -0.5)


# ----------------------------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return _run_own(s)
    return {"logprobs": _plain_logprobs, "plan": _plain_plan, "norm_rope": _plain_norm_rope, "append": _plain_append,
            "attention": _plain_attention}[s["op"]](s)


def _run_own(s):
    from hydra_b200 import kernels, paged, sampling
    if s["op"] == "logprobs":
        r = sampling.token_logprobs(s["logits"], s["tokens"], top=s["top"], temperature=s["temperature"], vocab=s["vocab"])
        return dict(logprobs=r.logprobs, entropy=r.entropy, top_logprobs=r.top_logprobs, top_ids=r.top_ids)
    if s["op"] == "plan":
        p = paged.paged_plan(s["context_lens"], s["new_lens"], s["table"], s["free"], s["page"], s["room"])
        return dict(table=s["table"], kv_lens=p.kv_lens, cu_new=p.cu_new, positions=p.positions, slots=p.slots,
                    free_start=p.free_start, status=p.status)
    norm = None if s["op"] == "attention" or s["norm"] == "none" else s["norm"]
    if s["op"] == "norm_rope":
        q, k = kernels.fused_qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], q_weight=s["wq"], k_weight=s["wk"],
                                          norm=norm, eps=1e-6, layout=s["layout"])
        return dict(q=q, k=k)
    if s["op"] == "append":
        q = paged.paged_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["cos"], s["sin"], s["positions"],
                               q_weight=s["wq"], k_weight=s["wk"], norm=norm, eps=1e-6, layout=s["layout"])
        return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])
    out, lse = paged.paged_decode_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], scale=s["scale"], return_lse=True)
    return dict(out=out, lse=lse)


def _plain_logprobs(s):
    V, top, tokens = s["vocab"], s["top"], s["tokens"]
    x = s["logits"][:, :V].float()
    z = x / s["temperature"]
    d = z - z.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    lz = total.log()
    entropy = lz[:, 0] - (torch.where(e > 0, d, 0.0) * e).sum(1) / total[:, 0]
    given = d.gather(1, tokens.clamp(min=0)[:, None]) - lz
    logprobs = torch.where(tokens == -100, 0.0, given[:, 0])
    if not top:
        return dict(logprobs=logprobs, entropy=entropy, top_logprobs=x[:, :0], top_ids=tokens[:, None][:, :0])
    # the largest, of equal ones the lowest index: the value's bits in an order of whole numbers, then the index from behind
    b = (x + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(b < 0, -(b & 0x7FFFFFFF), b) * (1 << 20) + ((1 << 20) - 1 - torch.arange(V, device=x.device))
    ids = order.topk(top, dim=1).indices
    return dict(logprobs=logprobs, entropy=entropy, top_logprobs=d.gather(1, ids) - lz, top_ids=ids)


def _plain_plan(s):
    context, new, table, free, P, room = s["context_lens"].long(), s["new_lens"].long(), s["table"], s["free"], s["page"], s["room"]
    W = table.shape[1]
    total = context + new
    held, want = (context + P - 1) // P, (total + P - 1) // P
    more = want - held
    first = more.cumsum(0) - more
    j = torch.arange(W, device=table.device)[None]
    fresh = (j >= held[:, None]) & (j < want[:, None])
    at = (first - held)[:, None] + j
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    i = torch.arange(room, device=table.device)
    b = (torch.searchsorted(cu, i, right=True) - 1).clamp(max=new.numel() - 1)
    real = i < cu[-1]
    pos = torch.where(real, context[b] + i - cu[b], 0)
    slot = table[b, pos // P].long() * P + pos % P
    return dict(table=table, kv_lens=total.int(), cu_new=cu.int(), positions=torch.where(real, pos, -1).int(),
                slots=torch.where(real, slot, -1), free_start=more.sum()[None].int(), status=more.new_zeros(1).int())


def _plain_norm(x, norm, w):
    x = x.float()
    if norm == "rms":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    elif norm == "l2":
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)
    return x


def _plain_rotate(x, c, n, layout):
    """x [..., hd] in 32 bits, its first 2 * c.shape[-1] values turned by the angles whose cosines and sines c and n are."""
    r = c.shape[-1]
    rest = x[..., 2 * r:]
    if layout == "half":
        a, b = x[..., :r], x[..., r:2 * r]
        return torch.cat([a * c - b * n, a * n + b * c, rest], -1)
    a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
    return torch.cat([torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2), rest], -1)


def _plain_norm_rope(s):
    pos = s["positions"].long()
    c, n = s["cos"][pos], s["sin"][pos]
    heads = 1 if s["order"] == "thd" else -3  # [T, 1, r], or [B, 1, S, r]
    c, n = c.unsqueeze(heads), n.unsqueeze(heads)
    return dict(q=_plain_rotate(_plain_norm(s["q"], s["norm"], s["wq"]), c, n, s["layout"]).to(s["q"].dtype),
                k=_plain_rotate(_plain_norm(s["k"], s["norm"], s["wk"]), c, n, s["layout"]).to(s["k"].dtype))


def _plain_append(s):
    pos, slots, P, dt = s["positions"].long(), s["slots"], s["page"], s["q"].dtype
    c, n = s["cos"][pos.clamp(min=0)][:, None], s["sin"][pos.clamp(min=0)][:, None]
    q = _plain_rotate(_plain_norm(s["q"], s["norm"], s["wq"]), c, n, s["layout"])
    k = _plain_rotate(_plain_norm(s["k"], s["norm"], s["wk"]), c, n, s["layout"])
    q = torch.where((pos >= 0)[:, None, None], q, 0.0).to(dt)
    real = slots >= 0
    at = slots[real]
    s["kc"][at // P, :, at % P] = k[real].to(dt)
    s["vc"][at // P, :, at % P] = s["v"][real]
    return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])


def _plain_attention(s):
    q, lens, table = s["q"], s["lens"], s["table"].clamp(min=0).long()
    B, hq, hd = q.shape
    hkv = s["hkv"]
    q4 = q.float().view(B, hkv, hq // hkv, hd)
    k = s["kc"][table].transpose(1, 2).flatten(2, 3).float()  # [B, hkv, W * P, hd]
    there = torch.arange(k.shape[2], device=q.device)[None] < lens[:, None]
    sc = torch.where(there[:, None, None], (q4 @ k.transpose(2, 3)) * s["scale"], float("-inf"))
    del k
    m = sc.amax(-1, keepdim=True)
    p = (sc - m.clamp(min=-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    v = torch.where(there[:, None, :, None], s["vc"][table].transpose(1, 2).flatten(2, 3).float(), 0.0)
    out = (p @ v) / total.clamp(min=1e-30)
    return dict(out=out.view(B, hq, hd).to(q.dtype), lse=(m + total.log()).view(B, hq))


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    if op == "plan":
        new, P = _new_lengths(case), case["page"]
        return {"bytes": 24 * len(new) + 8 * sum(-(-n // P) for n in new) + 12 * case["room"], "flops": 0}
    if op in ("norm_rope", "append"):
        tokens = case["batch"] * case["seq"] if op == "norm_rope" else case["tokens"] - case["pad"]
        heads = case["hq"] + case["hkv"]
        moved = heads + (case["hkv"] if op == "append" else 0)
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": tokens * (2 * moved * case["hd"] * size + 12) + 8 * min(tokens, 8192) * case["rot"] // 2,
                "flops": 8 * tokens * heads * case["hd"]}
    total = sum(_lengths(case))
    return {"bytes": total * case["hkv"] * case["hd"] * 4 + case["batch"] * case["hq"] * (case["hd"] * 4 + 4),
            "flops": 4 * total * case["hq"] * case["hd"]}


# --------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "plan": _exact_plan, "norm_rope": _exact_norm_rope, "append": _exact_append,
            "attention": _exact_attention}[s["op"]](s)


def _exact_logprobs(s):
    """Row block by row block: log softmax by logsumexp, entropy as the expectation of -log p, order by a stable sort."""
    parts = []
    for i in range(0, s["rows"], 512):
        x, t = s["logits"][i:i + 512, :s["vocab"]], s["tokens"][i:i + 512]
        lp = x.double() / s["temperature"]
        lp = lp - torch.logsumexp(lp, 1, keepdim=True)
        h = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
        given = lp[torch.arange(len(t), device=t.device), t.clamp(min=0)]
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        parts.append((given.masked_fill(t == -100, 0.0), h, torch.take_along_dim(lp, ids, 1), ids))
    a = [torch.cat(p) for p in zip(*parts)]
    return dict(logprobs=a[0], entropy=a[1], top_logprobs=a[2], top_ids=a[3])


def _exact_plan(s):
    """Request by request, with the free pages handed out one by one."""
    P, table, free = s["page"], s["table"].cpu().clone(), s["free"].tolist()
    taken, cu, lens, pos, slots = 0, [0], [], [], []
    for b, (c, n) in enumerate(zip(s["context_lens"].tolist(), s["new_lens"].tolist())):
        row = table[b].tolist()
        for t in range(c, c + n):
            if t % P == 0:
                row[t // P] = free[taken]
                taken += 1
            pos.append(t)
            slots.append(row[t // P] * P + t % P)
        table[b] = torch.tensor(row, dtype=torch.int32)
        cu.append(cu[-1] + n)
        lens.append(c + n)
    pad = [-1] * (s["room"] - len(pos))
    i32 = torch.int32
    return dict(table=table, kv_lens=torch.tensor(lens, dtype=i32), cu_new=torch.tensor(cu, dtype=i32),
                positions=torch.tensor(pos + pad, dtype=i32), slots=torch.tensor(slots + pad), free_start=torch.tensor([taken], dtype=i32),
                status=torch.zeros(1, dtype=i32))


def _exact_turned(x, w, cos, sin, s):
    """x [..., hd] in 64 bits, normed, its pairs taken as complex numbers and multiplied by cos + i sin."""
    x = x.double()
    if s["norm"] != "none":
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / (x.shape[-1] if s["norm"] == "rms" else 1) + 1e-6)
    if w is not None:
        x = x * w.double()
    rot = s["rot"]
    head = x[..., :rot]
    pairs = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if s["layout"] == "half" else head.unflatten(-1, (rot // 2, 2))
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.complex(cos.double(), sin.double()))
    turned = turned.transpose(-1, -2) if s["layout"] == "half" else turned
    return torch.cat([turned.reshape(head.shape), x[..., rot:]], -1)


def _exact_norm_rope(s):
    pos = s["positions"].long()
    cos, sin = (t[pos][:, None] for t in (s["cos"], s["sin"]))  # thd: [T, 1, r]; else [B, 1, S, r]
    return dict(q=_exact_turned(s["q"], s["wq"], cos, sin, s), k=_exact_turned(s["k"], s["wk"], cos, sin, s))


def _exact_append(s):
    n, P = s["tokens"] - s["pad"], s["page"]
    pos = s["positions"][:n].long()
    cos, sin = (t[pos][:, None] for t in (s["cos"], s["sin"]))
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    q[:n] = _exact_turned(s["q"][:n], s["wq"], cos, sin, s)
    page, row = torch.div(s["slots"][:n], P, rounding_mode="floor"), s["slots"][:n] % P
    kc, vc = s["kc"].double(), s["vc"].double()
    kc[page, :, row] = _exact_turned(s["k"][:n], s["wk"], cos, sin, s)
    vc[page, :, row] = s["v"][:n].double()
    return dict(q=q, k_cache=kc, v_cache=vc)


def _exact_attention(s):
    """Request by request over its own pages."""
    B, hq, hd = s["q"].shape
    P, group = s["page"], hq // s["hkv"]
    out = torch.zeros(B, hq, hd, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((B, hq), float("-inf"), dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["lens"].tolist()):
        if not n:
            continue
        at = s["table"][b, :-(-n // P)].long()
        for h in range(s["hkv"]):
            k = s["kc"][at, h].reshape(-1, hd)[:n].double()
            v = s["vc"][at, h].reshape(-1, hd)[:n].double()
            mine = slice(h * group, (h + 1) * group)
            a = (s["q"][b, mine].double() * s["scale"]) @ k.T
            lse[b, mine] = torch.logsumexp(a, -1)
            out[b, mine] = torch.softmax(a, -1) @ v
    return dict(out=out, lse=lse)
