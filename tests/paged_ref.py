"""Plain restatements of the operators over pages, one sequence at a time, and of beam search's choice in 64 bits."""
import math

import numpy as np

from tests import attention_ref

TOP = 1 << 30


def plan(lens, n_new, table, free, count, n_pages, page, tokens, refs=None):
    """What PagedPlan gives: dict of lens, starts, slots, positions, free_count, refused, table, refs."""
    lens, n_new, table = [int(x) for x in lens], [int(x) for x in n_new], table.copy()
    refs = None if refs is None else refs.copy()
    n, width = table.shape
    count = min(max(int(count), 0), n_pages)
    slots, positions, starts = np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32), np.zeros(n + 1, np.int64)
    most = min(width * page, TOP)
    at, off, taken, refused, out = 0, 0, 0, 0, list(lens)
    for i in range(n):
        starts[i] = at
        begin, at = at, min(at + min(max(n_new[i], 0), TOP), TOP)
        fits = lens[i] >= 0 and n_new[i] >= 0 and lens[i] <= most and n_new[i] <= most - lens[i] and at <= tokens
        have, need = -(-lens[i] // page), 0
        if fits:
            need = -(-(lens[i] + n_new[i]) // page) - have
        first, off = off, off + need
        if not fits or (need and off > count):
            refused += 1
            continue
        pages = [int(free[count - 1 - first - j]) for j in range(need)]
        taken += need
        table[i, have:have + need] = pages
        for p in pages:
            if refs is not None and 0 <= p < n_pages:
                refs[p] = 1
        out[i] = lens[i] + n_new[i]
        for t in range(n_new[i]):
            pos = lens[i] + t
            p = int(table[i, pos // page])
            positions[begin + t] = pos
            if 0 <= p < n_pages:
                slots[begin + t] = p * page + pos % page
    starts[n] = at
    return {"lens": np.array(out, np.int32), "starts": starts.astype(np.int32), "slots": slots, "positions": positions, "free_count": np.array([count - taken], np.int32),
            "refused": np.array([refused], np.int32), "table": table, "refs": refs}


def append(rows, pages, slots):
    """`pages` [n_pages, H, P, D] with rows [tokens, H, D] stored at their slots."""
    pages = pages.copy()
    n_pages, _, page, _ = pages.shape
    for t, s in enumerate(slots):
        if 0 <= s < n_pages * page:
            pages[s // page, :, s % page] = rows[t]
    return pages


def reorder(parents, table, lens, refs, free, count, page):
    """What PagedReorder gives: dict of table, lens, refs, free_pages, free_count, copies, missing."""
    n, width = table.shape
    n_pages = len(refs)
    count = min(max(int(count), 0), n_pages)
    hold = lambda s: (0, 0) if not 0 <= lens[s] <= min(width * page, TOP) else divmod(int(lens[s]), page)  # noqa: E731
    here = lambda p: 0 <= p < n_pages  # noqa: E731
    first, copies = {}, np.tile(np.array([-1, -1, 0], np.int32), (n, 1))
    for j in range(n):
        p = int(parents[j])
        if not 0 <= p < n:
            continue
        eldest = p not in first
        first.setdefault(p, j)
        full, part = hold(p)
        if part and here(table[p, full]) and not (eldest and refs[table[p, full]] == 1):
            copies[j] = table[p, full], -1, part
    asked = [j for j in range(n) if copies[j, 0] >= 0]
    stack = [int(x) for x in free[:count]]
    if len(asked) > count:
        kept = np.full(n_pages, -1, np.int32)
        kept[:count] = stack
        return {"table": table.copy(), "lens": lens.copy(), "refs": refs.copy(), "free_pages": kept, "free_count": np.array([count], np.int32),
                "copies": np.tile(np.array([-1, -1, 0], np.int32), (n, 1)), "missing": np.array([len(asked) - count], np.int32)}
    new_refs, new_table, new_lens = refs.astype(np.int64), np.full_like(table, -1), np.zeros_like(lens)
    for j in asked:
        copies[j, 1] = stack.pop()
    for s in range(n):
        full, part = hold(s)
        for p in table[s, :full + (part > 0)]:
            if here(p):
                new_refs[p] -= 1
    for j in range(n):
        p = int(parents[j])
        if not 0 <= p < n:
            continue
        full, part = hold(p)
        new_lens[j] = lens[p]
        new_table[j, :full + (part > 0)] = table[p, :full + (part > 0)]
        if copies[j, 0] >= 0:
            new_table[j, full] = copies[j, 1]
        for q in new_table[j, :full + (part > 0)]:
            if here(q):
                new_refs[q] += 1
    stack += [p for p in range(n_pages) if new_refs[p] <= 0 and refs[p] > 0]
    out = np.full(n_pages, -1, np.int32)
    out[:len(stack)] = stack[:n_pages]
    return {"table": new_table, "lens": new_lens, "refs": new_refs.astype(np.int32), "free_pages": out, "free_count": np.array([len(stack)], np.int32), "copies": copies,
            "missing": np.array([0], np.int32)}


def copy(pool, copies):
    """`pool` after the copies."""
    out = pool.copy()
    for src, dst, tokens in copies:
        if 0 <= src < len(pool) and 0 <= dst < len(pool) and tokens > 0:
            out[dst, :, :tokens] = pool[src, :, :tokens]
    return out


def attend(q, k_pages, v_pages, table, lens, scale=None, causal=True):
    """(result, bound) of PagedSdpa; holes are not seen."""
    n, hq, sq, d = q.shape
    n_pages, hkv, page, _ = k_pages.shape
    out, bound = np.zeros(q.shape), np.full(q.shape, 1e-30)
    for i in range(n):
        length = min(max(int(lens[i]), 0), table.shape[1] * page)
        ids = table[i, :-(-length // page)]
        place = np.arange(length)
        there = ((ids >= 0) & (ids < n_pages))[place // page] if length else np.zeros(0, bool)
        place = place[there]
        sees = place[None, :] <= (length - sq + np.arange(sq) if causal else np.full(sq, length))[:, None]
        for h in range(hq):
            kv = h // (hq // hkv)
            keys, values = (x[ids[place // page], kv, place % page] if len(place) else np.zeros((0, d)) for x in (k_pages, v_pages))
            out[i, h], bound[i, h] = attention_ref.attend(q[i, h], keys, values, q.dtype, scale=scale, sees=sees)
    return out, bound


def select(logits, scores, keep, ended=None, eos=-1):
    """What BeamSelect gives, in 64 bits: dict of scores, parents, tokens, ended."""
    b, w, n = logits.shape
    out = {"scores": np.zeros((b, keep)), "parents": np.zeros((b, keep), np.int32), "tokens": np.zeros((b, keep), np.int32), "ended": np.zeros((b, keep), np.int32)}
    for i in range(b):
        c = np.full((w, n), -np.inf)
        for j in range(w):
            s = float(scores[i, j])
            if not math.isfinite(s):
                continue
            if ended is not None and ended[i, j]:
                c[j, eos] = s
                continue
            x = logits[i, j].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            top = x.max()
            if np.isfinite(top):
                c[j] = s + ((x - top) - math.log(math.fsum(np.exp(x - top))))
        order = np.argsort(-c.reshape(-1), kind="stable")[:keep]
        out["scores"][i], out["parents"][i], out["tokens"][i] = c.reshape(-1)[order], i * w + order // n, order % n
        out["ended"][i] = (order % n == eos) | (False if ended is None else ended[i][order // n] != 0)
    return out
