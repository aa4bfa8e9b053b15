"""The latent-attention operators as a serving program calls them, for timing and comparison.

Four operators work together around one cache: ``plan_pages`` builds block tables
and slot maps from request lengths, ``latent_cache_write`` normalises, rotates and
stores one latent row a token, ``latent_attention_absorbed`` reads that cache for
decode, and ``latent_attention_expanded`` attends over expanded keys and values for
prefill.  ``run`` computes them in plain torch operations, or, where ``own`` is
true, through this package.
"""

import math

import torch

own = False

# 512 latent values and 64 rotary ones a token (the [576, 4096] latent projection),
# 64 heads of 256 output values (the [4096, 16384] output projection).
LATENT = 512
ROPE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # page planning: one new token for each of a few running requests
        {"name": "plan decode 16", "op": "plan", "requests": 16, "cached": 2000, "new": 1, "page": 64, "pad": 0},
        # page planning: a large batch, decoding requests mixed with prompt chunks, padded token count
        {"name": "plan mixed 512", "op": "plan", "requests": 512, "cached": 4000, "new": 64, "page": 16, "pad": 37},
        # one decoded token: the smallest call, where latency counts
        {"name": "write 1", "op": "write", "tokens": 1, "heads": 64, "rope": True, "page": 64, "type": "bf16"},
        # an odd chunk without positions or queries
        {"name": "write 1001 unrotated", "op": "write", "tokens": 1001, "heads": 0, "rope": False, "page": 16,
         "type": "fp16"},
        # a prompt chunk with its queries' rotary part
        {"name": "write 4096", "op": "write", "tokens": 4096, "heads": 64, "rope": True, "page": 64, "type": "bf16"},
        # one short conversation
        {"name": "absorbed 1x777", "op": "absorbed", "requests": 1, "longest": 777, "shortest": 777, "queries": 1,
         "heads": 64, "page": 64, "type": "bf16"},
        # one very long document
        {"name": "absorbed 1x100003", "op": "absorbed", "requests": 1, "longest": 100003, "shortest": 100003,
         "queries": 1, "heads": 64, "page": 64, "type": "bf16"},
        # a ragged batch with two tokens a request (one proposed), small pages
        {"name": "absorbed 24 ragged x2", "op": "absorbed", "requests": 24, "longest": 5000, "shortest": 1,
         "queries": 2, "heads": 16, "page": 16, "type": "fp16"},
        # a full serving batch
        {"name": "absorbed 64x8192", "op": "absorbed", "requests": 64, "longest": 8192, "shortest": 6000,
         "queries": 1, "heads": 64, "page": 64, "type": "bf16"},
        # one prompt chunk of the output projection's 256 rows
        {"name": "expanded 256", "op": "expanded", "requests": 1, "queries": 256, "context": 0, "ragged": False,
         "heads": 64, "nope": 192, "value": 256, "type": "bf16"},
        # several prompts of odd lengths with earlier context, smaller heads
        {"name": "expanded 5 ragged", "op": "expanded", "requests": 5, "queries": 700, "context": 300,
         "ragged": True, "heads": 16, "nope": 128, "value": 128, "type": "fp16"},
        # a 2048-token chunk of a long prompt behind 6144 tokens of context
        {"name": "expanded 2048 of 8192", "op": "expanded", "requests": 1, "queries": 2048, "context": 6144,
         "ragged": False, "heads": 64, "nope": 192, "value": 256, "type": "bf16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "absorbed", "absorbed", "expanded", "expanded"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 512), "cached": _log(rng, 1, 4000), "new": _log(rng, 1, 64),
                "page": rng.choice([16, 32, 64, 128]), "pad": rng.choice([0, rng.randint(1, 200)])}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 4096), "heads": rng.choice([0, 5, 16, 32, 64]),
                "rope": rng.random() < 0.75, "page": rng.choice([16, 48, 64]), "type": kind}
    if op == "absorbed":
        requests = _log(rng, 1, 64)
        longest = _log(rng, 1, min(100003, 8192 * 48 // requests))
        return {"op": op, "requests": requests, "longest": longest, "shortest": rng.randint(max(1, longest // 4), longest),
                "queries": rng.choice([1, 1, 1, 2, 3]) if requests <= 24 else 1, "heads": rng.choice([8, 16, 20, 32, 64, 64, 64]),
                "page": rng.choice([16, 32, 64, 128]), "type": kind}
    requests = rng.randint(1, 4)
    return {"op": op, "requests": requests, "queries": _log(rng, 1, 2048 // requests),
            "context": rng.choice([0, _log(rng, 1, 2000)]), "ragged": rng.random() < 0.5,
            "heads": rng.choice([3, 8, 16, 32, 64]), "nope": rng.choice([64, 128, 192, 192]),
            "value": rng.choice([64, 128, 256, 256]), "type": kind}


def _lengths(count, low, high, generator, device):
    """`count` lengths spread over [low, high], the longest among them."""
    n = torch.randint(low, high + 1, (count,), generator=generator, device=device, dtype=torch.int64)
    n[-1] = high
    return n


def _starts(lengths):
    return torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])


def _mean_length(case):
    return (case["shortest"] + case["longest"]) // 2


def _new_lengths(case):
    """New tokens of each request: half of them decode one, the others bring `new` at most."""
    return [1 + (i * 11 % case["new"] if i % 2 else 0) for i in range(case["requests"])]


def _expanded_lengths(case):
    """(queries, keys) of each request: odd steps below the largest where the batch is ragged."""
    out = []
    for i in range(case["requests"]):
        q = max(1, case["queries"] - (i * case["queries"] * 5 // 23 if case["ragged"] else 0))
        c = max(0, case["context"] - (i * case["context"] * 3 // 17 if case["ragged"] else 0))
        out.append((q, q + c))
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    op = case["op"]
    s = {"op": op}
    if op == "plan":
        page, b = case["page"], case["requests"]
        cached = torch.randint(0, case["cached"] + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        new = torch.tensor(_new_lengths(case), dtype=torch.int32).to(dev)
        new = new[torch.randperm(b, generator=g, device=dev)]
        width = -(-(case["cached"] + case["new"]) // page)
        pages = b * (width + 1)
        order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        held = (cached.long() + page - 1) // page
        table = torch.full((b, width), -1, dtype=torch.int32, device=dev)
        at = torch.arange(width, device=dev)
        table = torch.where(at < held[:, None], order[: b * width].view(b, width), table)
        free = torch.cat([order[b * width:], order[: b * width].view(b, width)[at >= held[:, None]]])
        count = torch.tensor([free.numel()], dtype=torch.int32, device=dev)
        tokens = sum(_new_lengths(case)) + case["pad"]
        s.update(cached=cached, new=new, table=table.contiguous(), free=free, count=count, page=page, tokens=tokens)
        return s
    dt = TYPES[case["type"]]
    if op == "write":
        t, page = case["tokens"], case["page"]
        pages = -(-t // page) + 3
        s["kv"] = normal(t, LATENT + ROPE, dtype=dt)
        s["cache"] = normal(pages, page, LATENT + ROPE, dtype=dt)
        s["slots"] = torch.randperm(pages * page, generator=g, device=dev)[:t]
        if t > 20:
            s["slots"][-3:] = -1  # rows behind the last token of a padded batch
        s["weight"] = (1 + 0.1 * torch.randn(LATENT, generator=g, device=dev)).to(dt)
        s["positions"] = s["inv_freq"] = s["queries"] = None
        if case["rope"]:
            s["positions"] = torch.randint(0, 131072, (t,), generator=g, device=dev, dtype=torch.int32)
            s["inv_freq"] = 10000.0 ** (-torch.arange(0, ROPE, 2, device=dev, dtype=torch.float64) / ROPE)
            if case["heads"]:  # the rotary part of each head's query, a view of the whole query
                s["queries"] = normal(t, case["heads"], 192 + ROPE, dtype=dt)[..., 192:]
        return s
    if op == "absorbed":
        b, page, h, nq = case["requests"], case["page"], case["heads"], case["queries"]
        lens = _lengths(b, case["shortest"], case["longest"], g, dev)
        width = -(-case["longest"] // page)
        pages = b * width + 2
        s["table"] = torch.randperm(pages, generator=g, device=dev)[: b * width].to(torch.int32).view(b, width)
        s["cache"] = normal(pages, page, LATENT + ROPE, dtype=dt)
        s["lens"] = lens.to(torch.int32)
        s["q_latent"] = normal(b * nq, h, LATENT, dtype=dt)
        s["q_rope"] = normal(b * nq, h, ROPE, dtype=dt)
        s["starts"] = None if nq == 1 else torch.arange(0, b * nq + 1, nq, device=dev, dtype=torch.int32)
        s["scale"] = (192 + ROPE) ** -0.5
        return s
    if op == "expanded":
        h, dn, dv = case["heads"], case["nope"], case["value"]
        lens = _expanded_lengths(case)
        tq, tk = sum(q for q, _ in lens), sum(k for _, k in lens)
        q = normal(tq, h, dn + ROPE, dtype=dt)
        kv = normal(tk, h, dn + dv, dtype=dt)  # the expanded latents: keys and values side by side
        latent = normal(tk, LATENT + ROPE, dtype=dt)
        s.update(q_nope=q[..., :dn], q_rope=q[..., dn:], k_nope=kv[..., :dn], values=kv[..., dn:],
                 k_rope=latent[:, LATENT:], scale=(dn + ROPE) ** -0.5)
        s["q_starts"] = _starts(torch.tensor([q for q, _ in lens])).to(torch.int32).to(dev)
        s["k_starts"] = _starts(torch.tensor([k for _, k in lens])).to(torch.int32).to(dev)
        s["most"] = (max(q for q, _ in lens), max(k for _, k in lens))
        return s
    raise ValueError(f"unknown operator {op!r}")


# --- plain forms -----------------------------------------------------------


def _plan(s):
    cached, new, page, tokens = s["cached"].long(), s["new"].long(), s["page"], s["tokens"]
    held = (cached + page - 1) // page
    wanted = (cached + new + page - 1) // page
    first = _starts(wanted - held)
    at = torch.arange(s["table"].shape[1], device=cached.device)
    taken = s["count"].long() - 1 - (first[:-1, None] + at - held[:, None])
    fresh = s["free"][taken.clamp(0, s["free"].numel() - 1)]
    s["table"].copy_(torch.where((at >= held[:, None]) & (at < wanted[:, None]), fresh, s["table"]))
    starts = _starts(new)
    t = torch.arange(tokens, device=cached.device)
    row = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=cached.numel() - 1)
    real = t < starts[-1]
    position = torch.where(real, cached[row] + t - starts[row], 0)
    slots = torch.where(real, s["table"][row, position // page].long() * page + position % page, -1)
    return {"table": s["table"], "slots": slots, "positions": position.int(), "query_starts": starts.int(),
            "seq_lens": (cached + new).int(), "free_count": (s["count"] - first[-1:]).int()}


def _rotate(x, positions, inv_freq):
    """The two halves of the last axis as (real, imaginary) parts, turned by position * inv_freq."""
    angle = positions.double()[:, None] * inv_freq
    c, n = torch.cos(angle).float(), torch.sin(angle).float()
    shape = (x.shape[0],) + (1,) * (x.dim() - 2) + (x.shape[-1] // 2,)
    a, b = x.float().chunk(2, dim=-1)
    c, n = c.view(shape), n.view(shape)
    return torch.cat([a * c - b * n, b * c + a * n], dim=-1)


def _write(s):
    x = s["kv"].float()
    c = x[:, :LATENT]
    c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    r = x[:, LATENT:]
    if s["positions"] is not None:
        r = _rotate(r, s["positions"], s["inv_freq"])
    rows = torch.cat([c, r], dim=-1).to(s["cache"].dtype)
    real = s["slots"] >= 0  # the rows behind the last token repeat the first one's store
    rows = torch.where(real[:, None], rows, rows[:1])
    slots = torch.where(real, s["slots"], s["slots"][:1])
    s["cache"].view(-1, LATENT + ROPE)[slots] = rows
    if s["queries"] is None:
        return {"cache": s["cache"]}
    q = _rotate(s["queries"], s["positions"], s["inv_freq"]).to(s["queries"].dtype)
    return {"cache": s["cache"], "queries": q}


def _absorbed(s):
    b, page = s["lens"].numel(), s["cache"].shape[1]
    h = s["q_latent"].shape[1]
    q = torch.cat([s["q_latent"], s["q_rope"]], dim=-1).float().view(b, -1, LATENT + ROPE)
    nq = q.shape[1] // h
    rows = s["cache"][s["table"].long()].view(b, -1, LATENT + ROPE).float()
    at = torch.arange(rows.shape[1], device=q.device)
    rows = rows * (at < s["lens"][:, None])[..., None]
    visible = s["lens"][:, None] - (nq - 1) + torch.arange(nq, device=q.device)  # [b, nq]
    score = torch.bmm(q, rows.transpose(1, 2)).view(b, nq, h, -1) * s["scale"]
    score = score.masked_fill(at >= visible[:, :, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(b, nq * h, -1), rows[..., :LATENT]).view(b, nq, h, LATENT)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).squeeze(-1)
    return {"out": o.reshape(b * nq, h, LATENT).to(s["q_latent"].dtype), "lse": lse.reshape(b * nq, h)}


def _expanded(s):
    qs, ks = s["q_starts"].long(), s["k_starts"].long()
    nq, nk = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    mq, mk = s["most"]
    dev = qs.device
    iq, ik = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    tq, tk = s["q_nope"].shape[0], s["k_nope"].shape[0]
    at_q = (qs[:-1, None] + iq).clamp(max=tq - 1)
    at_k = (ks[:-1, None] + ik).clamp(max=tk - 1)
    q = torch.cat([s["q_nope"], s["q_rope"]], dim=-1)[at_q].float().transpose(1, 2)  # [b, h, mq, d]
    kr = s["k_rope"][:, None].expand(-1, s["k_nope"].shape[1], -1)
    k = torch.cat([s["k_nope"], kr], dim=-1)[at_k].float().transpose(1, 2)
    v = s["values"][at_k].float().transpose(1, 2)
    v = v * (ik < nk[:, None])[:, None, :, None]
    score = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    seen = ik <= (nk - nq)[:, None, None] + iq[:, None]  # [b, mq, mk]
    score.masked_fill_(~(seen & (ik < nk[:, None, None]))[:, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(score.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).squeeze(-1)
    t = torch.arange(tq, device=dev)
    row = torch.searchsorted(qs, t, right=True) - 1
    return {"out": o[row, :, t - qs[row]].to(s["q_nope"].dtype), "lse": lse[row, :, t - qs[row]]}


def run(state):
    s = state
    if own:
        import glm53_flash_mlx_b200 as G

        if s["op"] == "plan":
            p = G.plan_pages(s["cached"], s["new"], s["table"], s["free"], s["count"], page_size=s["page"],
                             tokens=s["tokens"])
            return {"table": s["table"], "slots": p.slots, "positions": p.positions, "query_starts": p.query_starts,
                    "seq_lens": p.seq_lens, "free_count": p.free_count}
        if s["op"] == "write":
            q = G.latent_cache_write(s["kv"], s["cache"], s["slots"], rope_dim=ROPE, norm_weight=s["weight"], eps=1e-6,
                                     positions=s["positions"], inv_freq=s["inv_freq"], queries=s["queries"])
            return {"cache": s["cache"]} if q is None else {"cache": s["cache"], "queries": q}
        if s["op"] == "absorbed":
            out, lse = G.latent_attention_absorbed(s["q_latent"], s["q_rope"], s["cache"], s["table"], s["lens"],
                                                   scale=s["scale"], query_starts=s["starts"], return_lse=True)
            return {"out": out, "lse": lse}
        out, lse = G.latent_attention_expanded(s["q_nope"], s["q_rope"], s["k_nope"], s["k_rope"], s["values"],
                                               s["q_starts"], s["k_starts"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    return {"plan": _plan, "write": _write, "absorbed": _absorbed, "expanded": _expanded}[s["op"]](s)


def work(case):
    op = case["op"]
    if op == "plan":
        b, tokens = case["requests"], sum(_new_lengths(case))
        grown = tokens // case["page"]  # pages taken, on average
        return {"bytes": 8 * b + 8 * grown + 12 * (tokens + case["pad"]) + 8 * b, "flops": 0}
    width = 2 * (LATENT + ROPE)
    if op == "write":
        t = case["tokens"]
        q = t * case["heads"] * ROPE * 2 if case["rope"] else 0
        return {"bytes": 2 * t * width + 2 * q + 12 * t, "flops": 4 * t * (LATENT + ROPE) + 3 * q}
    if op == "absorbed":
        rows = case["requests"] * _mean_length(case)
        io = case["requests"] * case["queries"] * case["heads"] * (width + 2 * LATENT + 4)
        return {"bytes": rows * width + io,
                "flops": 2 * rows * case["queries"] * case["heads"] * (2 * LATENT + ROPE)}
    h, dn, dv = case["heads"], case["nope"], case["value"]
    pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in _expanded_lengths(case))
    tq = sum(q for q, _ in _expanded_lengths(case))
    tk = sum(k for _, k in _expanded_lengths(case))
    return {"bytes": 2 * tq * h * (dn + ROPE + dv) + 4 * tq * h + 2 * tk * (h * (dn + dv) + ROPE),
            "flops": 2 * pairs * h * (dn + ROPE + dv)}


# --- 64-bit values ---------------------------------------------------------


def _turn64(x, positions, inv_freq):
    z = torch.complex(x[..., : ROPE // 2].double(), x[..., ROPE // 2:].double())
    turn = torch.exp(1j * positions.double().view(-1, *[1] * (x.dim() - 1)) * inv_freq)
    z = z * turn
    return torch.cat([z.real, z.imag], dim=-1)


def _attend64(q, k, v, first, scale):
    """softmax(q k^T scale) v and its log-sum, query j seeing keys 0..first + j, over one head's rows."""
    score = (q @ k.T) * scale
    hidden = torch.ones_like(score, dtype=torch.bool).triu(first + 1)
    score[hidden] = -math.inf
    lse = torch.logsumexp(score, dim=-1)
    weights = torch.exp(score - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    return weights @ v, lse


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "plan":
        return None  # whole numbers only
    if s["op"] == "write":
        cache = s["cache"].double()
        x = s["kv"].double()
        norm = (x[:, :LATENT].pow(2).sum(-1) / LATENT + 1e-6).sqrt()
        x[:, :LATENT] = x[:, :LATENT] / norm[:, None] * s["weight"].double()
        if s["positions"] is not None:
            x[:, LATENT:] = _turn64(x[:, LATENT:], s["positions"], s["inv_freq"])
        real = (s["slots"] >= 0).nonzero().flatten()
        cache.view(-1, LATENT + ROPE).index_copy_(0, s["slots"][real], x[real])
        if s["queries"] is None:
            return {"cache": cache}
        return {"cache": cache, "queries": _turn64(s["queries"], s["positions"], s["inv_freq"])}
    if s["op"] == "absorbed":
        nq, h = case["queries"], case["heads"]
        flat = s["cache"].view(-1, LATENT + ROPE)
        page = s["cache"].shape[1]
        outs, logs = [], []
        for i, n in enumerate(s["lens"].tolist()):
            at = torch.arange(n, device=flat.device)
            k = flat[s["table"][i].long()[at // page] * page + at % page].double()
            for j in range(nq):
                t = i * nq + j
                q = torch.cat([s["q_latent"][t], s["q_rope"][t]], dim=-1).double()
                seen = max(0, n - (nq - 1) + j)
                o, lse = _attend64(q, k[:seen], k[:seen, :LATENT], seen, s["scale"])
                outs.append(o)
                logs.append(lse)
        return {"out": torch.stack(outs), "lse": torch.stack(logs)}
    h = case["heads"]
    out = torch.empty(s["q_nope"].shape[0], h, case["value"], dtype=torch.float64, device=s["q_nope"].device)
    lse = torch.empty(out.shape[:2], dtype=torch.float64, device=out.device)
    qa = ka = 0
    for nq, nk in _expanded_lengths(case):
        for i in range(h):
            q = torch.cat([s["q_nope"][qa:qa + nq, i], s["q_rope"][qa:qa + nq, i]], dim=-1).double()
            k = torch.cat([s["k_nope"][ka:ka + nk, i], s["k_rope"][ka:ka + nk]], dim=-1).double()
            o, l = _attend64(q, k, s["values"][ka:ka + nk, i].double(), nk - nq, s["scale"])
            out[qa:qa + nq, i] = o
            lse[qa:qa + nq, i] = l
        qa, ka = qa + nq, ka + nk
    return {"out": out, "lse": lse}
