"""Restatements in 64 bits of the operators on the paged 8-bit cache, request by request, for the tests."""
import numpy as np

ENDS = 0xFFFFFFFF


def plan(lengths, fresh, table, free, count, page, pages, max_tokens):
    """tb_page_plan: a dict of what it leaves, `refused` not 0 when nothing changes."""
    n, width = table.shape
    table, free = table.copy(), free.copy()
    have = [-(-int(x) // page) for x in lengths]
    add = [0 if f == ENDS else int(f) for f in fresh]
    need = [0 if f == ENDS else -(-(int(x) + a) // page) - h for x, f, a, h in zip(lengths, fresh, add, have)]
    back = sum(h for h, f in zip(have, fresh) if f == ENDS)
    refused = 0
    if any(int(x) + a > width * page for x, a in zip(lengths, add)):
        refused |= 2
    if count > pages or count + back > pages:
        refused |= 8
    if sum(need) > count + back:
        refused |= 1
    if sum(add) > max_tokens:
        refused |= 4
    if refused:
        return {"refused": refused, "table": table, "free": free, "count": count, "lengths": lengths.copy(), "starts": np.zeros(n + 1, np.uint32), "slots": [], "positions": []}
    stack = list(free[:count])
    for r in range(n):
        if fresh[r] == ENDS:
            stack += list(table[r, : have[r]])
    slots, positions, out, starts = [], [], [], [0]
    for r in range(n):
        for i in range(need[r]):
            table[r, have[r] + i] = stack.pop()
        for i in range(add[r]):
            p = int(lengths[r]) + i
            positions.append(p)
            slots.append(int(table[r, p // page]) * page + p % page)
        out.append(0 if fresh[r] == ENDS else int(lengths[r]) + add[r])
        starts.append(starts[-1] + add[r])
    if len(stack) > count:
        free[count: len(stack)] = stack[count:]
    return {"refused": 0, "table": table, "free": free, "count": len(stack), "lengths": np.array(out, np.uint32), "starts": np.array(starts, np.uint32), "slots": slots,
            "positions": positions}


def append(codes, scale, rows, slots, page):
    """tb_cache_append_q8 on one of the two caches: codes [pages][heads][page][D], rows [tokens][heads][D]; in place."""
    pages = codes.shape[0]
    by_page = {}
    for t, s in enumerate(slots):
        if s // page < pages:
            by_page.setdefault(int(s) // page, []).append((int(s) % page, t))
    for pg, items in by_page.items():
        first = min(o for o, _ in items)
        for h in range(codes.shape[1]):
            x = np.stack([rows[t, h] for _, t in items]).astype(np.float64)
            fine = np.abs(x[np.isfinite(x)])
            top = float(fine.max()) if fine.size else 0.0
            least = 0.0
            if top > 0:
                e = -126
                while 127 * 2.0**e < top:
                    e += 1
                least = 2.0**e
            was = float(scale[pg, h]) if first > 0 else 0.0
            s = max(was, least)
            if first and s != was:
                codes[pg, h, :first] = np.rint(codes[pg, h, :first] * (was / s))
            for (o, _), row in zip(items, x):
                with np.errstate(invalid="ignore", over="ignore"):
                    y = row / s if s > 0 else np.zeros_like(row)
                codes[pg, h, o] = np.where(np.isnan(y), 0, np.rint(np.clip(y, -127, 127)))
            scale[pg, h] = s


def attend(q, codes_k, k_scale, codes_v, v_scale, table, starts, lengths, window, scale, page):
    """q [tokens][heads][D] f64 -> (out [tokens][heads][D], largest sum of |q||k| scale, largest |v|) in f64; rows that no request owns are NaN."""
    heads, D = q.shape[1:]
    pages, kvh = codes_k.shape[:2]
    out = np.full(q.shape, np.nan)
    size, vmax = 0.0, 0.0
    for r, length in enumerate(lengths):
        length = int(length)
        t0, t1 = int(starts[r]), int(starts[r + 1])
        j = np.arange(length)
        ids = table[r][j // page].astype(np.int64) if length else np.zeros(0, np.int64)
        real = ids < pages
        ids = np.where(real, ids, 0)
        for h in range(heads):
            g = h // (heads // kvh)
            k = codes_k[ids, g, j % page].astype(np.float64) * k_scale[ids, g][:, None].astype(np.float64)
            v = codes_v[ids, g, j % page].astype(np.float64) * v_scale[ids, g][:, None].astype(np.float64)
            for t in range(t0, t1):
                p = length - (t1 - t0) + (t - t0)
                sees = real & (j <= p) & ((j > p - window) if window else True)
                if not sees.any():
                    out[t, h] = 0
                    continue
                s = scale * (k[sees] @ q[t, h])
                w = np.exp(s - s.max())
                out[t, h] = (w / w.sum()) @ v[sees]
                size = max(size, float((scale * (np.abs(k[sees]) @ np.abs(q[t, h]))).max()))
                vmax = max(vmax, float(np.abs(v[sees]).max()))
    return out, size, vmax


def logits(x, history, prompt, total, rep, freq, pres, bias_token, bias, bias_count, allowed, mask_of):
    """tb_logits_adjust in f64; None for what is not given."""
    y = x.astype(np.float64).copy()
    n, vocab = y.shape
    for r in range(n):
        if history is not None:
            h = history[r, : min(int(total[r]), history.shape[1])].astype(np.int64)
            said = h[min(int(prompt[r]), len(h)):]
            seen = np.bincount(h[h < vocab], minlength=vocab) > 0
            count = np.bincount(said[said < vocab], minlength=vocab)
            if rep is not None:
                y[r] = np.where(seen, np.where(y[r] > 0, y[r] / float(rep[r]), y[r] * float(rep[r])), y[r])
            f, p = (0.0 if freq is None else float(freq[r])), (0.0 if pres is None else float(pres[r]))
            y[r] = np.where(count > 0, y[r] - (f * count + p), y[r])
        if bias_token is not None:
            for i in range(min(int(bias_count[r]), bias_token.shape[1])):
                if bias_token[r, i] < vocab:
                    y[r, bias_token[r, i]] += float(bias[r, i])
        if allowed is not None:
            m = r if mask_of is None else int(mask_of[r])
            if m < allowed.shape[0]:
                t = np.arange(vocab)
                y[r, (allowed[m, t // 32] >> (t % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return y
