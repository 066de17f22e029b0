"""Operators of a server's step over paged caches, and what one call of each costs.

    listed()             the cases with names               draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program has before the call run(state)           one pass, its outputs
    work(case)           bytes and operations of one pass   exact(case, seed)    the outputs in 64 bits

``own`` False: the operators in elementary torch operations; True: this package's calls.  ``kind`` of a case:

    attention   queries of one new token per sequence, or of a few drafted ones, over a paged cache (``paged_attention``)
    append      rotation of the new tokens' queries and keys, keys and values into the pages (``paged_rotary_append``)
    verify      drafted tokens against the target's probabilities (``verify_draft``)

Sequences of a batch have lengths of their own, spread evenly from ``low`` to ``high``; which sequence has which length is up to the seed.  Of
``tokens`` new tokens a sequence has all, or with ``ragged`` between one and all of them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BASE = 500000.0


def listed():
    return [
        # one chat at the start: nothing but latency
        dict(name="attention_one_short", kind="attention", batch=1, heads=32, kv=8, dim=128, page=16, low=300, high=300, tokens=1, ragged=False,
             window=0, sinks=0, cap=0.0, dtype="bf16"),
        # the serving step that the repository's benchmark reports, on pages
        dict(name="attention_8b_b32", kind="attention", batch=32, heads=32, kv=8, dim=128, page=64, low=2048, high=2048, tokens=1, ragged=False,
             window=0, sinks=0, cap=0.0, dtype="bf16"),
        # one very long document
        dict(name="attention_one_long", kind="attention", batch=1, heads=32, kv=8, dim=128, page=128, low=131071, high=131071, tokens=1, ragged=False,
             window=0, sinks=0, cap=0.0, dtype="f16"),
        # a mixed batch of a small model: from a first token to long chats
        dict(name="attention_mixed_b96", kind="attention", batch=96, heads=32, kv=4, dim=64, page=16, low=1, high=6000, tokens=1, ragged=False,
             window=0, sinks=0, cap=0.0, dtype="f16"),
        # up to four drafted tokens behind the last one
        dict(name="attention_drafts_b16", kind="attention", batch=16, heads=32, kv=8, dim=128, page=32, low=1500, high=4500, tokens=5, ragged=True,
             window=0, sinks=0, cap=0.0, dtype="bf16"),
        # endless conversations: first tokens and a window; pages in between have been given back; capped scores
        dict(name="attention_window_b48", kind="attention", batch=48, heads=16, kv=8, dim=128, page=24, low=900, high=90000, tokens=1, ragged=False,
             window=1000, sinks=4, cap=50.0, dtype="bf16"),
        # an unquantised model in 32 bits with a key head per query head, heads of an odd size, small pages
        dict(name="attention_f32_odd", kind="attention", batch=7, heads=12, kv=12, dim=80, page=10, low=1, high=1501, tokens=1, ragged=False,
             window=0, sinks=0, cap=0.0, dtype="f32"),
        # the new token of each sequence of a step
        dict(name="append_step_b32", kind="append", batch=32, heads=32, kv=8, dim=128, page=64, low=200, high=700, tokens=1, ragged=False,
             rot=128, halves=True, norm=False, dtype="bf16"),
        # prompts of odd length, part of each head rotated, heads normed
        dict(name="append_prompts_b6", kind="append", batch=6, heads=32, kv=8, dim=128, page=24, low=777, high=1100, tokens=777, ragged=True,
             rot=64, halves=False, norm=True, dtype="f16"),
        # one user's drafts, a small vocabulary
        dict(name="verify_one", kind="verify", batch=1, drafts=4, vocab=32000, draft=True, dtype="f32"),
        # a batch's drafts over the benchmark's large vocabulary
        dict(name="verify_b64", kind="verify", batch=64, drafts=7, vocab=128256, draft=True, dtype="f32"),
        # drafts that were looked up rather than drawn, odd vocabulary, 16-bit probabilities
        dict(name="verify_lookup_b200", kind="verify", batch=200, drafts=3, vocab=50257, draft=False, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_attention(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128, 80, 96, 192, 256, 40])
    kv = rng.choice([1, 2, 4, 8, 8, 12])
    heads = kv * rng.choice([1, 2, 4, 4, 7, 8])
    tokens = rng.choice([1, 1, 1, 1, 2, 3, 5, 8])
    window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    batch = _log(rng, 1, 256)
    row = kv * dim * BYTES[dtype] * 2  # bytes of a position
    # at most a third of the largest listed case's cache, and of the rows that its plain form lays out (as long as the longest sequence, 32 bits)
    most = min((1 << 29) // (3 * row), (1 << 29) // (3 * kv * dim * 4)) // batch
    high = min(_log(rng, 1, 131072), max(most, tokens))
    low = rng.choice([high, 1, max(1, high // 3)])
    return dict(kind="attention", batch=batch, heads=heads, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256, 1, 10, 24]), low=max(low, tokens),
                high=max(high, tokens), tokens=tokens, ragged=tokens > 1 and rng.random() < 0.7, window=window,
                sinks=rng.choice([0, 1, 4, 64]) if window else 0, cap=rng.choice([0.0, 0.0, 30.0]), dtype=dtype)


def _draw_append(rng):
    dim = rng.choice([64, 128, 128, 96, 80, 256])
    kv = rng.choice([1, 2, 4, 8])
    batch = _log(rng, 1, 256)
    tokens = min(_log(rng, 1, 900), max(1, 4000 // batch))
    high = tokens + _log(rng, 1, 600)
    return dict(kind="append", batch=batch, heads=kv * rng.choice([1, 2, 4, 7]), kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 10, 24]), low=tokens, high=high,
                tokens=tokens, ragged=tokens > 1 and rng.random() < 0.5, rot=rng.choice([dim, dim, dim // 2, 0]), halves=rng.random() < 0.7,
                norm=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))


def _draw_verify(rng):
    drafts = rng.choice([1, 2, 3, 4, 5, 7, 8])
    vocab = _log(rng, 500, 200000)
    batch = _log(rng, 1, max(1, min(256, 64 * 8 * 128256 // ((drafts + 1) * vocab))))
    return dict(kind="verify", batch=batch, drafts=drafts, vocab=vocab, draft=rng.random() < 0.7, dtype=rng.choice(["f32", "f32", "bf16", "f16"]))


def draw(rng):
    return rng.choice([_draw_attention, _draw_attention, _draw_append, _draw_verify])(rng)


# ---- inputs ----
def _lengths(case):
    """(length, new tokens) of every sequence, shortest first."""
    b, low, high, t = case["batch"], case["low"], case["high"], case["tokens"]
    out = []
    for i in range(b):
        n = high if b == 1 else low + (high - low) * i // (b - 1)
        c = 1 + (5 * i) % t if case["ragged"] else t
        out.append((max(n, c), c))
    return out


def _first_visible(length, count, window):
    return max(0, length - count - window + 1) if window else 0


def _cache(case, gen, order):
    """Pages of random rows in random order, the table of the pages that are held (-1: none), lengths and counts."""
    page, kv, dim, dt = case["page"], case["kv"], case["dim"], DTYPES[case["dtype"]]
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    both = _lengths(case)
    both = [both[i] for i in order.tolist()]
    width = -(-max(n for n, _ in both) // page) + 1
    held = []
    for b, (n, c) in enumerate(both):
        lo = _first_visible(n, c, window)
        for i in range(-(-n // page)):
            if (i + 1) * page > lo or i * page < sinks:
                held.append(b * width + i)
    total = len(held) + 3
    pages = torch.randperm(total, generator=gen, device="cuda")[:len(held)].int()
    table = torch.full((len(both) * width,), -1, dtype=torch.int32, device="cuda")
    table[torch.tensor(held, device="cuda")] = pages
    shape = (total, kv, page, dim)
    return dict(k_pages=torch.randn(shape, generator=gen, device="cuda", dtype=dt), v_pages=torch.randn(shape, generator=gen, device="cuda", dtype=dt),
                table=table.view(len(both), width), lengths=torch.tensor([n for n, _ in both], dtype=torch.int32, device="cuda"),
                counts=torch.tensor([c for _, c in both], dtype=torch.int32, device="cuda") if case["ragged"] else None)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    if case["kind"] == "verify":
        b, k, v, dt = case["batch"], case["drafts"], case["vocab"], DTYPES[case["dtype"]]
        # a distribution whose mass is on some hundred tokens, and a draft model's that overlaps with three quarters of it
        z = 3.0 * torch.randn(b, k + 1, v, generator=gen, device="cuda")
        target = torch.softmax(z, -1).to(dt)
        near = torch.softmax(z[:, :k] + 0.6 * torch.randn(b, k, v, generator=gen, device="cuda"), -1)
        tokens = torch.multinomial(near.view(b * k, v), 1, generator=gen).view(b, k).int()
        return dict(kind="verify", target=target, draft=near.to(dt) if case["draft"] else None, tokens=tokens,
                    accept=torch.rand(b, k, generator=gen, device="cuda"), sample=torch.rand(b, generator=gen, device="cuda"))
    b, h, g, d, t, dt = case["batch"], case["heads"], case["kv"], case["dim"], case["tokens"], DTYPES[case["dtype"]]
    state = _cache(case, gen, torch.randperm(b, generator=host))
    state["kind"] = case["kind"]
    if case["kind"] == "attention":
        state.update(q=1.5 * torch.randn(b, h, t, d, generator=gen, device="cuda", dtype=dt), scale=d ** -0.5, window=case["window"], sinks=case["sinks"],
                     cap=case["cap"])
        return state
    angle = None
    if case["rot"]:
        inv = BASE ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        angle = torch.arange(case["high"] + 1, dtype=torch.float64, device="cuda")[:, None] * inv
    state.update(proj=torch.randn(b, t, (h + 2 * g) * d, generator=gen, device="cuda", dtype=dt), heads=h, halves=case["halves"], norm=case["norm"], eps=1e-5,
                 cos=None if angle is None else angle.cos().float(), sin=None if angle is None else angle.sin().float())
    return state


# ---- the operators in elementary operations, 32 bits ----
def _plain_attention(s):
    q, table, lengths = s["q"], s["table"].long(), s["lengths"].long()
    B, H, T, D = q.shape
    G, page = s["k_pages"].shape[1], s["k_pages"].shape[2]
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, T)
    window, sinks = s["window"], s["sinks"]
    if window:  # the first tokens, and what the windows of the new ones cover
        start = (lengths - counts - window + 1).clamp(min=0)
        head = torch.arange(sinks, device=q.device).expand(B, sinks)
        body = start[:, None] + torch.arange(window + T - 1, device=q.device)
        pos = torch.cat([torch.where(head < start[:, None], head, lengths[:, None]), body], 1)
    else:
        pos = torch.arange(table.shape[1] * page, device=q.device).expand(B, -1)
    there = pos < lengths[:, None]
    pos = torch.where(there, pos, 0)
    rows = table.gather(1, pos // page).clamp(min=0)
    k = s["k_pages"][rows, :, pos % page].float()  # [B, N, G, D]
    v = s["v_pages"][rows, :, pos % page].float()
    at = lengths[:, None] - counts[:, None] + torch.arange(T, device=q.device)  # [B, T]
    seen = there[:, None] & (pos[:, None] <= at[:, :, None]) & (torch.arange(T, device=q.device) < counts[:, None])[:, :, None]
    if window:
        seen &= (at[:, :, None] - pos[:, None] < window) | (pos[:, None] < sinks)
    qf = q.float().view(B, G, H // G * T, D)
    x = torch.matmul(qf, k.permute(0, 2, 3, 1)) * s["scale"]
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    mask = seen[:, None, None].expand(B, G, H // G, T, -1).reshape(x.shape)
    x = torch.where(mask, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    return o.view(B, H, T, D).transpose(1, 2).to(q.dtype).contiguous()


def _plain_append(s):
    proj, table, lengths = s["proj"], s["table"].long(), s["lengths"].long()
    B, T, _ = proj.shape
    G, page, D = s["k_pages"].shape[1:]
    H = s["heads"]
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, T)
    pos = lengths[:, None] - counts[:, None] + torch.arange(T, device=proj.device)
    real = torch.arange(T, device=proj.device) < counts[:, None]
    x = proj.view(B, T, H + 2 * G, D)
    qk = x[:, :, :H + G].float()
    if s["cos"] is not None:
        half = s["cos"].shape[1]
        c, n = s["cos"][torch.where(real, pos, 0)][:, :, None], s["sin"][torch.where(real, pos, 0)][:, :, None]
        rot, rest = qk[..., :2 * half], qk[..., 2 * half:]
        if s["halves"]:
            a, b = rot[..., :half], rot[..., half:]
            rot = torch.cat([a * c - b * n, b * c + a * n], -1)
        else:
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
        qk = torch.cat([rot, rest], -1)
    if s["norm"]:
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + s["eps"])
    qk = qk.to(proj.dtype)
    q = torch.where(real[:, :, None, None], qk[:, :, :H], 0).transpose(1, 2).contiguous()
    b, t = real.nonzero(as_tuple=True)
    at = pos[b, t]
    row = table[b, at // page]
    s["k_pages"][row, :, at % page] = qk[b, t, H:]
    s["v_pages"][row, :, at % page] = x[b, t, H + G:]
    return q, s["k_pages"], s["v_pages"]


def _plain_verify(s):
    p, q, x, u, r = s["target"], s["draft"], s["tokens"].long(), s["accept"].double(), s["sample"].double()
    B, K = x.shape
    px = p[:, :K].gather(2, x[..., None])[..., 0].double()
    qx = q.gather(2, x[..., None])[..., 0].double() if q is not None else torch.ones_like(px)
    n = torch.cumprod((u * qx < px).int(), 1).sum(1)  # drafts that stand
    b = torch.arange(B, device=p.device)
    w = p[b, n].double()
    short = (n < K)[:, None]
    last = n.clamp(max=K - 1)
    if q is not None:
        left = (w - q[b, last].double()).clamp(min=0)
    else:
        left = torch.where(torch.arange(w.shape[1], device=p.device) == x[b, last][:, None], 0.0, w)
    left = torch.where(short, left, w)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, w)
    total = left.cumsum(1)
    pick = (total > (r * total[:, -1])[:, None]).int().argmax(1)
    out = torch.cat([x, torch.full_like(x[:, :1], -1)], 1)
    place = torch.arange(K + 1, device=p.device)
    out = torch.where(place < n[:, None], out, torch.where(place == n[:, None], pick[:, None], -1))
    return out.int(), n.int()


def run(state):
    kind = state["kind"]
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "verify": _plain_verify}[kind](state)
    from my_nn_engine_b200 import ops
    if kind == "attention":
        return ops.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["table"], state["lengths"], state["scale"], counts=state["counts"],
                                   window=state["window"], sinks=state["sinks"], softcap=state["cap"])
    if kind == "append":
        q = ops.paged_rotary_append(state["proj"], state["lengths"], state["table"], state["k_pages"], state["v_pages"], state["heads"], state["cos"], state["sin"],
                                    counts=state["counts"], halves=state["halves"], qk_norm=state["norm"], eps=state["eps"])
        return q, state["k_pages"], state["v_pages"]
    return ops.verify_draft(state["target"], state["tokens"], state["accept"], state["sample"], draft=state["draft"])


# ---- what a pass cannot do without ----
def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "verify":
        # the row that the token behind the accepted ones comes from, and the draft's row beside it
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        rows = b * (2 if case["draft"] else 1)
        return {"bytes": rows * v * size + b * k * (4 + 4 + 2 * size) + b * (4 + 4 * (k + 2)), "flops": 3 * rows * v}
    h, g, d, both = case["heads"], case["kv"], case["dim"], _lengths(case)
    if case["kind"] == "append":
        new = sum(c for _, c in both)
        return {"bytes": new * 2 * (h + 2 * g) * d * size + new * case["rot"] * 4 + 4 * len(both), "flops": new * (h + g) * (3 * case["rot"] + (3 * d if case["norm"] else 0))}
    cached, pairs = 0, 0
    for n, c in both:
        lo = _first_visible(n, c, case["window"])
        cached += n - lo + min(case["sinks"], lo)
        for s in range(c):
            p = n - c + s
            first = max(0, p - case["window"] + 1) if case["window"] else 0
            pairs += p + 1 - first + min(case["sinks"], first)
    new = sum(c for _, c in both)
    return {"bytes": cached * 2 * g * d * size + 2 * new * h * d * size + sum(4 * -(-n // case["page"]) for n, _ in both), "flops": 4 * pairs * h * d}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "verify": _exact_verify}[case["kind"]](s)


def _sequences(s, tokens):
    lengths = s["lengths"].tolist()
    return list(zip(lengths, s["counts"].tolist() if s["counts"] is not None else [tokens] * len(lengths)))


def _exact_attention(s):
    B, H, T, D = s["q"].shape
    G, page = s["k_pages"].shape[1:3]
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    for b, (n, c) in enumerate(_sequences(s, T)):
        for t in range(c):
            p = n - c + t
            first = max(0, p - s["window"] + 1) if s["window"] else 0
            j = torch.cat([torch.arange(0, min(s["sinks"], first), device="cuda"), torch.arange(first, p + 1, device="cuda")])
            rows = s["table"][b].long()[torch.div(j, page, rounding_mode="floor")]
            for g in range(G):
                keys, values = s["k_pages"][rows, g, j % page].double(), s["v_pages"][rows, g, j % page].double()
                x = s["q"][b, g * (H // G):(g + 1) * (H // G), t].double() @ keys.T * s["scale"]
                if s["cap"]:
                    x = s["cap"] * torch.tanh(x / s["cap"])
                out[b, t, g * (H // G):(g + 1) * (H // G)] = torch.softmax(x, -1) @ values
    return out


def _exact_append(s):
    B, T, _ = s["proj"].shape
    G, page, D = s["k_pages"].shape[1:]
    H = s["heads"]
    q = torch.zeros(B, H, T, D, dtype=torch.float64, device="cuda")
    k, v = s["k_pages"].double(), s["v_pages"].double()
    for b, (n, c) in enumerate(_sequences(s, T)):
        x = s["proj"][b, :c].double().view(c, H + 2 * G, D)
        pos = torch.arange(n - c, n, device="cuda")
        y = x[:, :H + G].clone()
        if s["cos"] is not None:
            half = s["cos"].shape[1]
            cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]
            for i in range(half):
                lo, hi = (i, i + half) if s["halves"] else (2 * i, 2 * i + 1)
                y[:, :, lo] = x[:, :H + G, lo] * cos[:, i, None] - x[:, :H + G, hi] * sin[:, i, None]
                y[:, :, hi] = x[:, :H + G, hi] * cos[:, i, None] + x[:, :H + G, lo] * sin[:, i, None]
        if s["norm"]:
            y = y / (y.pow(2).mean(-1, keepdim=True) + s["eps"]).sqrt()
        q[b, :, :c] = y[:, :H].transpose(0, 1)
        rows = s["table"][b].long()[torch.div(pos, page, rounding_mode="floor")]
        k[rows, :, pos % page] = y[:, H:]
        v[rows, :, pos % page] = x[:, H + G:]
    return q, k, v


def _exact_verify(s):
    B, K = s["tokens"].shape
    out = torch.full((B, K + 1), -1, dtype=torch.int32)
    taken = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        tokens = s["tokens"][b].tolist()
        n = 0
        while n < K:
            p = s["target"][b, n, tokens[n]].double().item()
            q = s["draft"][b, n, tokens[n]].double().item() if s["draft"] is not None else 1.0
            if not s["accept"][b, n].double().item() * q < p:
                break
            n += 1
        weight = s["target"][b, n].double()
        if n < K:
            rest = weight.clone()
            if s["draft"] is not None:
                rest = torch.relu(rest - s["draft"][b, n].double())
            else:
                rest[tokens[n]] = 0
            weight = rest if rest.sum().item() > 0 else weight
        reached = torch.cumsum(weight, 0)
        pick = torch.searchsorted(reached, s["sample"][b].double() * reached[-1], right=True).item()
        out[b, :n] = torch.tensor(tokens[:n], dtype=torch.int32)
        out[b, n] = pick
        taken[b] = n
    return out.cuda(), taken.cuda()
