"""Batched serving over a paged 8-bit cache: what one step of it costs.

The operators, in the order a serving step calls them: block tables and slot maps from request lengths (`plan`), new keys
and values into an 8-bit cache with one scale for a page and key-value head, read back as values (`append`), attention of
single tokens over that cache (`attend`), attention of a prompt's chunks over it (`prefill`), and penalties, biases and
grammar masks on a batch of logits (`logits`).

`own` False computes each in elementary torch operations in 32 bits; `own` True calls the framework.  `exact` restates each
definition in 64 bits, request by request.
"""
import math
import random

import torch

own = False

DEV = "cuda"
ENDS = -1  # 0xffffffff as int32: the request has ended


# ---- cases --------------------------------------------------------------------------------------------------------


def listed():
    return [
        # A decode step of 64 conversations: one token each, a few idle, a few that ended since the last step.
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "page": 64, "longest": 8192, "most": 1},
        # Admission of a large mixed batch: prompts' chunks beside single tokens, odd page counts.
        {"name": "plan_mixed_1000", "op": "plan", "requests": 1000, "page": 16, "longest": 4096, "most": 257},
        # The keys and values of a decode step, f32 as the projections leave them.
        {"name": "append_decode_64", "op": "append", "requests": 64, "page": 64, "longest": 8192, "most": 1, "kv_heads": 8, "head_dim": 128, "f16": False},
        # A prompt chunk of 2048 tokens of the benchmark's model shape, cut over ragged requests, f16.
        {"name": "append_chunk_8k", "op": "append", "requests": 5, "page": 32, "longest": 8192, "most": 2048, "kv_heads": 2, "head_dim": 256, "f16": True},
        # One conversation in the benchmark's shape (8 query heads on 2 key-value heads of 256), context 4096: latency.
        {"name": "attend_one_4096", "op": "attend", "requests": 1, "page": 64, "longest": 4096, "most": 1, "heads": 8, "kv_heads": 2, "head_dim": 256, "window": 0,
         "f16": False},
        # Its sliding layers: window 512.
        {"name": "attend_window_512", "op": "attend", "requests": 33, "page": 16, "longest": 4001, "most": 1, "heads": 8, "kv_heads": 2, "head_dim": 256, "window": 512,
         "f16": True},
        # A full decode batch at ragged lengths, heads of 128.
        {"name": "attend_batch_96", "op": "attend", "requests": 96, "page": 64, "longest": 16384, "most": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "f16": True},
        # One very long context, heads of 512 (the global layers), two drafted tokens checked at once.
        {"name": "attend_long_131k", "op": "attend", "requests": 2, "page": 128, "longest": 131071, "most": 2, "heads": 8, "kv_heads": 2, "head_dim": 512, "window": 0,
         "f16": False},
        # Prompt chunks of the benchmark's model shape late in a long prompt.
        {"name": "prefill_256", "op": "prefill", "requests": 2, "page": 64, "longest": 8192, "most": 2048, "heads": 8, "kv_heads": 2, "head_dim": 256, "window": 0},
        # Ragged chunks of many requests, heads of 128.
        {"name": "prefill_128", "op": "prefill", "requests": 7, "page": 32, "longest": 4100, "most": 1030, "heads": 16, "kv_heads": 4, "head_dim": 128, "window": 0},
        # One conversation's logits over the benchmark's vocabulary, in f32.
        {"name": "logits_one", "op": "logits", "rows": 1, "vocab": 262144, "history": 2000, "biases": 8, "masked": True, "f16": False},
        # A decode batch's, in f16, with long histories.
        {"name": "logits_64", "op": "logits", "rows": 64, "vocab": 262144, "history": 8000, "biases": 100, "masked": True, "f16": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "prefill", "logits"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 1000), "page": page, "longest": _log(rng, 1, 8192), "most": rng.choice([1, _log(rng, 1, 257)])}
    if op == "logits":
        rows = _log(rng, 1, 64)
        return {"op": op, "rows": rows, "vocab": _log(rng, 500, 262144), "history": _log(rng, 1, 8000), "biases": rng.choice([0, _log(rng, 1, 300)]),
                "masked": rng.random() < 0.7, "f16": rng.random() < 0.5}
    kv, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256, 512])
    if op == "append":
        requests, longest, most = _log(rng, 1, 64), _log(rng, 1, 8192), rng.choice([1, _log(rng, 1, 2048)])
        while requests * min(most, longest) * kv * dim > 5 * 2048 * 2 * 256 or requests * longest * kv * dim > 64 * 8192 * 8 * 128:
            requests, longest = max(1, requests // 2), max(1, longest // 2)
        return {"op": op, "requests": requests, "page": page, "longest": longest, "most": most, "kv_heads": kv, "head_dim": dim, "f16": rng.random() < 0.5}
    group = rng.choice([1, 2, 4, 4, 7, 8])
    window = rng.choice([0, 0, _log(rng, 1, 4096)])
    if op == "attend":
        requests, longest = _log(rng, 1, 96), _log(rng, 1, 131072)
        while requests * longest * kv * dim > 96 * 16384 * 8 * 128:
            requests, longest = max(1, requests // 2), max(1, longest // 2)
        return {"op": op, "requests": requests, "page": page, "longest": longest, "most": rng.choice([1, 1, 2, 16 // group if group <= 8 else 1]), "heads": kv * group,
                "kv_heads": kv, "head_dim": dim, "window": window, "f16": rng.random() < 0.5}
    requests, longest, most = _log(rng, 1, 16), _log(rng, 16, 8192), _log(rng, 2, 2048)
    while requests * kv * group * min(most, longest) * longest * dim > 2 * 8 * 2048 * 8192 * 256:
        requests, longest, kv = max(1, requests // 2), max(16, longest // 2), max(1, kv // 2)
    return {"op": op, "requests": requests, "page": page, "longest": longest, "most": most, "heads": kv * group, "kv_heads": kv, "head_dim": dim, "window": window}


# ---- inputs -------------------------------------------------------------------------------------------------------


def _requests(case, seed):
    """Lengths after this step, the new tokens among them and a draw in [0, 1) for each request: ragged, one request at the
    longest, as continuous batching has them.  The case says which there are, the seed in which order."""
    rng = random.Random("%d %d %d" % (case["requests"], case["longest"], case["most"]))
    n, longest, most = case["requests"], case["longest"], case["most"]
    after = [longest] + [_log(rng, max(1, longest // 16), longest) for _ in range(n - 1)]
    new = [min(a, most if i == 0 else rng.randint(max(1, most // 4), most)) for i, a in enumerate(after)]
    made = [(a, x, rng.random()) for a, x in zip(after, new)]
    random.Random(seed * 7919 + 17).shuffle(made)
    return tuple(list(x) for x in zip(*made))


def _ints(values):
    return torch.tensor(values, dtype=torch.int64).to(torch.int32).to(DEV)


def _wrap(v):
    return v - (1 << 32) if v >= (1 << 31) else v


def _tables(case, seed, lengths, spare=0):
    """Pages handed out in a shuffled order, as a pool that has been in use gives them.  Returns (table, pages, free)."""
    n, page = case["requests"], case["page"]
    width = max(1, -(-case["longest"] // page))
    need = [-(-x // page) for x in lengths]
    pages = sum(need) + spare
    gen = torch.Generator(device=DEV).manual_seed(seed + 5)
    order = torch.randperm(max(1, pages), generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32, device=DEV)
    need_t = torch.tensor(need, device=DEV)
    at = torch.cumsum(need_t, 0) - need_t
    col = torch.arange(width, device=DEV)[None, :].expand(n, width)
    held = col < need_t[:, None]
    table[held] = order[(at[:, None] + col)[held]]
    return table, max(1, pages), order[sum(need):].contiguous()


def _cache(case, seed, pages):
    gen = torch.Generator(device=DEV).manual_seed(seed + 6)
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    made = []
    for _ in range(2):
        codes = torch.empty(shape, dtype=torch.int8, device=DEV)
        flat = codes.view(-1)
        for i in range(0, flat.numel(), 1 << 28):
            part = flat[i:i + (1 << 28)]
            part.copy_((torch.randn(part.numel(), generator=gen, device=DEV) * 28).round_().clamp_(-127, 127))
        scale = torch.exp2(torch.randint(-6, -4, (pages, case["kv_heads"]), generator=gen, device=DEV).float())
        made += [codes, scale.contiguous()]
    return made


def _starts(new):
    at = [0]
    for x in new:
        at.append(at[-1] + x)
    return at


def prepare(case, seed):
    op = case["op"]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    if op == "plan":
        after, new, kind = _requests(case, seed)
        lengths = [a - x for a, x in zip(after, new)]
        fresh = [0 if c < 0.05 else ENDS if c < 0.12 else x for x, c in zip(new, kind)]
        table, pages, free = _tables(case, seed, lengths, spare=sum(-(-(le + max(0, f)) // case["page"]) - -(-le // case["page"]) for le, f in zip(lengths, fresh)) + 9)
        top = torch.zeros(pages, dtype=torch.int32, device=DEV)
        top[: free.numel()] = free
        tokens = sum(max(0, f) for f in fresh) + 5
        st |= {"lengths": _ints(lengths), "fresh": _ints(fresh), "table": table, "free": top, "count": _ints([free.numel()]), "pages": pages, "tokens": tokens,
               "lengths_out": torch.zeros(len(new), dtype=torch.int32, device=DEV), "count_out": _ints([0]), "refused": _ints([0]),
               "starts": torch.zeros(len(new) + 1, dtype=torch.int32, device=DEV), "slots": torch.zeros(tokens, dtype=torch.int32, device=DEV),
               "positions": torch.zeros(tokens, dtype=torch.int32, device=DEV), "scratch": torch.zeros(64, dtype=torch.uint8, device=DEV)}
        return st
    if op == "logits":
        n, vocab, hist, biases = case["rows"], case["vocab"], case["history"], case["biases"]
        kind = torch.float16 if case["f16"] else torch.float32
        rng = random.Random(seed + 4)
        total = [hist] + [rng.randint(0, hist) for _ in range(n - 1)]
        prompt = [rng.randint(0, t) for t in total]
        # Tokens repeat as in text: low ids often.
        history = (torch.rand(n, hist, generator=gen, device=DEV) ** 3 * vocab).to(torch.int32).clamp_(0, vocab - 1)
        st |= {"logits": (torch.randn(n, vocab, generator=gen, device=DEV) * 4).to(kind), "out": torch.zeros(n, vocab, dtype=kind, device=DEV),
               "history": history, "prompt": _ints(prompt), "total": _ints(total),
               "repetition": 1 + 0.3 * torch.rand(n, generator=gen, device=DEV), "frequency": 0.5 * torch.rand(n, generator=gen, device=DEV),
               "presence": 0.5 * torch.rand(n, generator=gen, device=DEV), "bias_token": None, "allowed": None}
        if biases:
            count = [biases] + [rng.randint(0, biases) for _ in range(n - 1)]
            st |= {"bias_token": torch.randint(0, vocab, (n, biases), generator=gen, device=DEV).to(torch.int32),
                   "bias": torch.randn(n, biases, generator=gen, device=DEV) * 3, "bias_count": _ints(count)}
        if case["masked"]:
            words = -(-vocab // 32)
            few = torch.randint(-(1 << 31), 1 << 31, (n, words), generator=gen, device=DEV)
            few &= torch.randint(-(1 << 31), 1 << 31, (n, words), generator=gen, device=DEV)
            # A grammar lets a sixteenth of the vocabulary through on odd rows, nearly all of it on even ones.
            open_ = torch.arange(n, device=DEV)[:, None] % 2 == 0
            st["allowed"] = torch.where(open_, few | ~(few << 3), few & (few >> 5) & (few << 7)).to(torch.int32)
        return st
    after, new, _ = _requests(case, seed)
    table, pages, _ = _tables(case, seed, after, spare=1)
    k, ks, v, vs = _cache(case, seed, pages)
    starts = _starts(new)
    tokens, kvh, dim = starts[-1], case["kv_heads"], case["head_dim"]
    st |= {"table": table, "pages": pages, "k": k, "v": v, "k_scale": ks, "v_scale": vs, "starts": _ints(starts), "lengths": _ints(after), "tokens": tokens}
    if op == "append":
        kind = torch.float16 if case["f16"] else torch.float32
        page = case["page"]
        own_of = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
        pos = torch.arange(tokens, device=DEV) - torch.tensor(starts[:-1], device=DEV)[own_of] + torch.tensor([a - x for a, x in zip(after, new)], device=DEV)[own_of]
        slots = table[own_of, pos // page].long() * page + pos % page
        first = torch.tensor([(a - x) // page * page for a, x in zip(after, new)], device=DEV)
        spans = torch.tensor(after, device=DEV) - first
        of = torch.repeat_interleave(torch.arange(len(new), device=DEV), spans)
        at = torch.arange(int(spans.sum()), device=DEV) - (torch.cumsum(spans, 0) - spans)[of] + first[of]
        wide = 1 + 3 * torch.rand(tokens, 1, 1, generator=gen, device=DEV)
        st |= {"new_k": (torch.randn(tokens, kvh, dim, generator=gen, device=DEV) * wide).to(kind), "new_v": (torch.randn(tokens, kvh, dim, generator=gen, device=DEV)).to(kind),
               "slots": slots.to(torch.int32), "seen": (table[of, at // page].long() * page + at % page).to(torch.int32)}
        count = st["seen"].numel()
        st |= {"k_values": torch.zeros(count, kvh, dim, dtype=torch.float16, device=DEV), "v_values": torch.zeros(count, kvh, dim, dtype=torch.float16, device=DEV)}
        return st
    f16 = case.get("f16", True)
    kind = torch.float16 if f16 else torch.float32
    st["q"] = (torch.randn(tokens, case["heads"], dim, generator=gen, device=DEV) * 1.5).to(kind)
    st["out"] = torch.zeros(tokens, case["heads"], dim, dtype=kind, device=DEV)
    st["scratch"] = torch.zeros(64 << 20, dtype=torch.uint8, device=DEV)  # a serving program's workspace, larger than any case needs
    return st


# ---- plain forms --------------------------------------------------------------------------------------------------


def _plan(st):
    page, pages, width = st["case"]["page"], st["pages"], st["table"].shape[1]
    n = st["lengths"].numel()
    length, fresh = st["lengths"].long(), st["fresh"].long()
    ends = fresh == ENDS
    new = torch.where(ends, torch.zeros_like(fresh), fresh)
    have = (length + page - 1) // page
    need = torch.where(ends, torch.zeros_like(have), (length + new + page - 1) // page - have)
    back = torch.where(ends, have, torch.zeros_like(have))
    cols = torch.arange(width, device=DEV)[None, :]
    table = st["table"].clone()
    returned = table[cols < back[:, None]]  # request order, then page order
    count = st["count"].long()[0]
    stack = torch.zeros(pages, dtype=torch.int32, device=DEV)
    at = torch.arange(pages, device=DEV)
    in_back = (at >= count) & (at < count + returned.numel())
    padded = torch.cat([returned, returned.new_zeros(1)])
    stack = torch.where(in_back, padded[(at - count).clamp(0, returned.numel())], st["free"])
    total, want = count + returned.numel(), need.sum()
    before = torch.cumsum(need, 0) - need
    k = cols - have[:, None]
    gets = (k >= 0) & (k < need[:, None])
    taken = stack[(total - 1 - (before[:, None] + k)).clamp(0, pages - 1)]
    table = torch.where(gets, taken, table)
    starts = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    tok = torch.arange(st["tokens"], device=DEV)
    real = tok < starts[-1]
    owner = torch.searchsorted(starts[1:].contiguous(), tok, right=True).clamp(0, n - 1)
    pos = length[owner] + tok - starts[owner]
    slot = table[owner, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    left = total - want
    free = torch.where(at < torch.maximum(left, count), stack, st["free"])
    return {"table": table, "free": free, "count": left.to(torch.int32).reshape(1), "lengths": torch.where(ends, torch.zeros_like(length), length + new).to(torch.int32),
            "starts": starts.to(torch.int32), "slots": torch.where(real, slot, torch.zeros_like(slot)).to(torch.int32),
            "positions": torch.where(real, pos, torch.zeros_like(pos)).to(torch.int32), "refused": torch.zeros(1, dtype=torch.int32, device=DEV)}


def _append_one(codes, scale, rows, slots, page):
    """One of the two caches: (codes, scale) with `rows` [tokens][heads][dim] stored at `slots`."""
    rows = rows.float()
    of, off = slots // page, slots % page
    fine = torch.isfinite(rows)
    amax = torch.where(fine, rows.abs(), torch.zeros_like(rows)).amax(-1)
    touched, which = torch.unique(of, return_inverse=True)
    top = torch.zeros(touched.numel(), rows.shape[1], device=DEV).scatter_reduce_(0, which[:, None].expand_as(amax), amax, "amax")
    first = torch.full((touched.numel(),), page, device=DEV).scatter_reduce_(0, which, off, "amin")
    part, power = torch.frexp(top)
    power = (power - 7 + (part > 127 / 128).to(power.dtype)).clamp(min=-126)
    least = torch.where(top > 0, torch.exp2(power.float()), torch.zeros_like(top))
    before = torch.where((first > 0)[:, None], scale[touched], torch.zeros_like(top))
    after = torch.maximum(before, least)
    ratio = torch.where(after > 0, before / after, torch.ones_like(after))
    old = codes[touched].float()
    kept = torch.arange(page, device=DEV)[None, None, :, None] < first[:, None, None, None]
    codes[touched] = torch.where(kept, torch.round(old * ratio[:, :, None, None]), old).to(torch.int8)
    scale[touched] = after
    s = after[which][:, :, None]
    x = torch.where(s > 0, rows / s, torch.zeros_like(rows))
    x = torch.where(torch.isnan(rows), torch.zeros_like(x), torch.round(x.clamp(-127, 127)))
    codes[of, :, off] = x.to(torch.int8)


def _append(st):
    page = st["case"]["page"]
    slots, seen = st["slots"].long(), st["seen"].long()
    _append_one(st["k"], st["k_scale"], st["new_k"], slots, page)
    _append_one(st["v"], st["v_scale"], st["new_v"], slots, page)
    of, off = seen // page, seen % page
    return {"k": (st["k"][of, :, off].float() * st["k_scale"][of][:, :, None]).half(), "v": (st["v"][of, :, off].float() * st["v_scale"][of][:, :, None]).half(),
            "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _attend(st):
    c = st["case"]
    n, page, heads, kvh, dim, most = c["requests"], c["page"], c["heads"], c["kv_heads"], c["head_dim"], c["most"]
    group, width = heads // kvh, st["table"].shape[1]
    idx = st["table"].long()
    length, starts = st["lengths"].long(), st["starts"].long()
    new = starts[1:] - starts[:-1]

    def values(codes, scale):
        x = codes[idx].float() * scale[idx][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, kvh, width * page, dim)

    i = torch.arange(most, device=DEV)
    tok = (starts[:-1, None] + i).clamp(max=st["tokens"] - 1)
    q = st["q"][tok].float().reshape(n, most, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kvh, most * group, dim)
    s = torch.matmul(q, values(st["k"], st["k_scale"]).transpose(-1, -2)) * (1 / math.sqrt(dim))
    pos = (length - new)[:, None] + i  # [n, most]
    j = torch.arange(width * page, device=DEV)
    sees = (j[None, None, :] <= pos[..., None]) & (i < new[:, None])[..., None]
    if c["window"]:
        sees &= j[None, None, :] > pos[..., None] - c["window"]
    sees = sees.repeat_interleave(group, dim=1)[:, None]
    s = s.masked_fill_(~sees, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, values(st["v"], st["v_scale"])) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(n, kvh, most, group, dim).permute(0, 2, 1, 3, 4).reshape(n, most, heads, dim)
    return o[i < new[:, None]].to(st["out"].dtype)  # request order, then token order: the packed rows


def _logits(st):
    x = st["logits"].float()
    n, vocab = x.shape
    hist = st["history"].long()
    at = torch.arange(hist.shape[1], device=DEV)
    live, said = at < st["total"][:, None], at >= st["prompt"][:, None]
    seen = torch.zeros(n, vocab, device=DEV).scatter_add_(1, hist, live.float())
    count = torch.zeros(n, vocab, device=DEV).scatter_add_(1, hist, (live & said).float())
    rep = st["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (st["frequency"][:, None] * count + st["presence"][:, None] * (count > 0))
    if st["bias_token"] is not None:
        live = torch.arange(st["bias"].shape[1], device=DEV) < st["bias_count"][:, None]
        x = x.scatter_add(1, st["bias_token"].long(), torch.where(live, st["bias"], torch.zeros_like(st["bias"])))
    if st["allowed"] is not None:
        t = torch.arange(vocab, device=DEV)
        ok = (st["allowed"].long()[:, t // 32] >> (t % 32)) & 1
        x = x.masked_fill(ok == 0, -math.inf)
    return x.to(st["out"].dtype)


# ---- the framework's calls ----------------------------------------------------------------------------------------

_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import tachyon_b200 as tb

        _ctx = tb.Context(torch.cuda.current_device())
    return _ctx


def _pages(st):
    import tachyon_b200 as tb

    c = st["case"]
    return tb.Pages(k=st["k"].data_ptr(), v=st["v"].data_ptr(), k_scale=st["k_scale"].data_ptr(), v_scale=st["v_scale"].data_ptr(), table=st["table"].data_ptr(),
                    pages=st["pages"], page=c["page"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], requests=c["requests"], width=st["table"].shape[1])


def _arguments(st):
    """The descriptors a serving loop fills once and keeps."""
    import tachyon_b200 as tb

    c, p = st["case"], lambda name: None if st.get(name) is None else st[name].data_ptr()
    op = c["op"]
    if op == "plan":
        return tb.PagePlan(lengths=p("lengths"), fresh=p("fresh"), lengths_out=p("lengths_out"), table=p("table"), free_pages=p("free"), free_count=p("count"),
                           free_count_out=p("count_out"), starts=p("starts"), slots=p("slots"), positions=p("positions"), refused=p("refused"), scratch=p("scratch"),
                           requests=c["requests"], width=st["table"].shape[1], page=c["page"], pages=st["pages"], max_tokens=st["tokens"])
    if op == "append":
        kind = tb.F16 if c["f16"] else tb.F32
        dim = c["head_dim"]
        return (tb.CacheRows(cache=_pages(st), k=p("new_k"), v=p("new_v"), dtype=kind, token_stride=c["kv_heads"] * dim, head_stride=dim, slots=p("slots"),
                             tokens=st["tokens"]),
                tb.CacheRows(cache=_pages(st), k=p("k_values"), v=p("v_values"), dtype=tb.F16, token_stride=c["kv_heads"] * dim, head_stride=dim, slots=p("seen"),
                             tokens=st["seen"].numel()))
    if op == "logits":
        return tb.Logits(logits=p("logits"), out=p("out"), dtype=tb.F16 if c["f16"] else tb.F32, rows=c["rows"], vocab=c["vocab"], stride=c["vocab"],
                         out_stride=c["vocab"], history=p("history"), history_stride=c["history"], prompt=p("prompt"), total=p("total"), repetition=p("repetition"),
                         frequency=p("frequency"), presence=p("presence"), bias_token=p("bias_token"), bias=p("bias"), bias_count=p("bias_count"),
                         bias_stride=c["biases"], allowed=p("allowed"), allowed_stride=-(-c["vocab"] // 32), masks=c["rows"], mask_of=None)
    kind = tb.F16 if c.get("f16", True) else tb.F32
    row = c["heads"] * c["head_dim"]
    return tb.PagedAttend(cache=_pages(st), q=p("q"), q_dtype=kind, q_stride=row, starts=p("starts"), lengths=p("lengths"), tokens=st["tokens"], heads=c["heads"],
                          most=c["most"], window=c["window"], scale=1 / math.sqrt(c["head_dim"]), out=p("out"), out_dtype=kind, out_stride=row, scratch=p("scratch"),
                          scratch_bytes=st["scratch"].numel())


def _run_own(st):
    ctx, op = _context(), st["case"]["op"]
    if "arguments" not in st:
        st["arguments"] = _arguments(st)
    a = st["arguments"]
    if op == "plan":
        ctx.page_plan(a)
        return {"table": st["table"], "free": st["free"], "count": st["count_out"], "lengths": st["lengths_out"], "starts": st["starts"], "slots": st["slots"],
                "positions": st["positions"], "refused": st["refused"]}
    if op == "append":
        ctx.cache_append_q8(a[0])
        ctx.cache_read_q8(a[1])
        return {"k": st["k_values"], "v": st["v_values"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if op == "logits":
        ctx.logits_adjust(a)
    elif op == "attend":
        ctx.attend_paged_q8(a)
    else:
        ctx.prefill_paged_q8(a)
    return st["out"]


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "plan":
        return _plan(st)
    if op == "append":
        return _append(st)
    return _logits(st) if op == "logits" else _attend(st)


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    after, new, _ = _requests(case, 1) if op != "logits" else (None, None, None)
    if op == "plan":
        return {"bytes": 8.0 * len(new) + 8.0 * len(new) + 8.0 * sum(new) + 8.0 * sum(new) / case["page"], "flops": 0}
    if op == "logits":
        cells = case["rows"] * case["vocab"]
        size = 2 if case["f16"] else 4
        return {"bytes": cells * 2.0 * size + (cells / 8 if case["masked"] else 0) + 4.0 * case["rows"] * case["history"], "flops": 2.0 * cells}
    kvh, dim = case["kv_heads"], case["head_dim"]
    if op == "append":
        rows = sum(a - (a - x) // case["page"] * case["page"] for a, x in zip(after, new))
        return {"bytes": 2.0 * kvh * dim * (sum(new) * ((2 if case["f16"] else 4) + 1) + rows * 3), "flops": 0}
    pairs, seen = 0, 0
    for a, x in zip(after, new):
        w = case["window"] or a
        first = max(0, a - x + 1 - w)
        seen += a - first
        if case["window"]:
            pairs += sum(min(a - x + i + 1, w) for i in range(x))
        else:
            pairs += x * (a - x) + x * (x + 1) // 2
    size = 2 if case.get("f16", True) else 4
    return {"bytes": 2.0 * kvh * dim * seen + 2.0 * size * sum(new) * case["heads"] * dim, "flops": 4.0 * pairs * case["heads"] * dim}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def _exact_append(codes, scale, rows, slots, page, seen):
    """The values that the stored numbers stand for, page by page."""
    codes, scale, rows = codes.double(), scale.double(), rows.double()
    by_page = {}
    for t, s in enumerate(slots):
        by_page.setdefault(s // page, []).append((s % page, t))
    for pg, items in by_page.items():
        first = min(o for o, _ in items)
        at = torch.tensor([t for _, t in items], device=DEV)
        off = torch.tensor([o for o, _ in items], device=DEV)
        x = rows[at]  # [m, heads, dim]
        top = x.abs().amax(dim=(0, 2))
        for h, big in enumerate(top.tolist()):
            e = -math.inf if big == 0 else max(-126, math.ceil(math.log2(big / 127)))
            if big and e > -126 and math.ldexp(127, e - 1) >= big:  # log2 rounded up across a power of two
                e -= 1
            elif big and math.ldexp(127, e) < big:
                e += 1
            was = float(scale[pg, h]) if first else 0.0
            s = max(was, math.ldexp(1, e) if big else 0.0)
            if first and s > 0:
                codes[pg, h, :first] = torch.round(codes[pg, h, :first] * (was / s))
            scale[pg, h] = s
            codes[pg, h, off] = torch.round(x[:, h] / s).clamp(-127, 127) if s > 0 else 0.0
    of, off = seen // page, seen % page
    return codes[of, :, off] * scale[of][:, :, None], scale


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    st = prepare(case, seed)
    if op == "append":
        slots, seen = st["slots"].tolist(), st["seen"].long()
        if len(slots) * case["kv_heads"] > 40000:
            return None
        k, ks = _exact_append(st["k"], st["k_scale"], st["new_k"], slots, case["page"], seen)
        v, vs = _exact_append(st["v"], st["v_scale"], st["new_v"], slots, case["page"], seen)
        return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}
    if op == "logits":
        rows = []
        for r in range(case["rows"]):
            x = st["logits"][r].double()
            total, prompt = int(st["total"][r]), int(st["prompt"][r])
            h = st["history"][r, :total].long()
            seen = torch.bincount(h, minlength=case["vocab"]) > 0
            count = torch.bincount(h[prompt:], minlength=case["vocab"]).double()
            rep = st["repetition"][r].double()
            x[seen] = torch.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
            x = x - st["frequency"][r].double() * count - st["presence"][r].double() * (count > 0).double()
            if st["bias_token"] is not None:
                m = int(st["bias_count"][r])
                x.index_add_(0, st["bias_token"][r, :m].long(), st["bias"][r, :m].double())
            if st["allowed"] is not None:
                bits = (st["allowed"][r].long()[:, None] >> torch.arange(32, device=DEV)) & 1
                x[bits.reshape(-1)[: case["vocab"]] == 0] = -math.inf
            rows.append(x)
        return torch.stack(rows)
    kvh, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // kvh
    starts, lengths = st["starts"].tolist(), st["lengths"].tolist()
    out = torch.zeros(st["tokens"], case["heads"], dim, dtype=torch.float64, device=DEV)
    for r, length in enumerate(lengths):
        t0, t1 = starts[r], starts[r + 1]
        ids = st["table"][r, : -(-length // page)].long()
        for h in range(kvh):
            k = (st["k"][ids, h].double() * st["k_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[:length]
            v = (st["v"][ids, h].double() * st["v_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[:length]
            pos = length - (t1 - t0) + torch.arange(t1 - t0, device=DEV)
            j = torch.arange(length, device=DEV)
            hidden = j[None] > pos[:, None]
            if case["window"]:
                hidden |= j[None] <= pos[:, None] - case["window"]
            for g in range(h * group, (h + 1) * group):
                s = st["q"][t0:t1, g].double() @ k.T / math.sqrt(dim)
                out[t0:t1, g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
    return out
