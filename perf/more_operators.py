"""What serving over pages of keys and values is timed on: the tables of a step, the append through them, the attention over them,
and beam search's selection and reordering of sequences.

A case is a dict of plain values.  Its "kind" is the operator:

* ``plan``     pages for the tokens that a step adds to every sequence, and where each of them goes
* ``append``   new rows of keys and values into their pages
* ``attend``   attention of one or a few new tokens per sequence over its pages
* ``select``   the best continuations of a request's beams over the whole vocabulary
* ``reorder``  sequences that go on from other sequences: tables, counts of holders, copies of pages in all layers

Plain forms compute in 32 bits and round once; the values that beams are chosen by are of 64 bits, since the order of two of them counts.
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f16": torch.float16, "f32": torch.float32}
_NP = {torch.float16: np.float16, torch.float32: np.float32, torch.int32: np.int32}
_EOS = 2


def _plan(name, seqs, shortest, longest, least, most, page):
    """Sequences of shortest..longest tokens, to which a step adds least..most each."""
    return {"name": name, "kind": "plan", "seqs": seqs, "shortest": shortest, "longest": longest, "least": least, "most": most, "page": page}


def _append(name, dtype, tokens, heads, kv_heads, dim, page, fused):
    """fused: the rows are views into the rows of one projection to queries, keys and values."""
    return {"name": name, "kind": "append", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "fused": fused}


def _attend(name, dtype, seqs, shortest, longest, queries, heads, kv_heads, dim, page):
    return {"name": name, "kind": "attend", "dtype": dtype, "seqs": seqs, "shortest": shortest, "longest": longest, "queries": queries, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _select(name, dtype, batch, beams, vocab, keep, ended):
    """keep: continuations per request; ended: some beams are complete."""
    return {"name": name, "kind": "select", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab, "keep": keep, "ended": ended}


def _reorder(name, dtype, batch, beams, shortest, longest, kv_heads, dim, page, layers):
    return {"name": name, "kind": "reorder", "dtype": dtype, "batch": batch, "beams": beams, "shortest": shortest, "longest": longest, "kv_heads": kv_heads,
            "dim": dim, "page": page, "layers": layers}


def listed():
    return [
        # a serving batch's next tokens
        _plan("plan_step", 256, 1, 8192, 1, 1, 16),
        # prompts in chunks beside next tokens and idle places
        _plan("plan_chunks", 500, 0, 4000, 0, 130, 32),
        # the next tokens of a batch, cut out of a fused projection
        _append("append_step", "f16", 64, 32, 8, 128, 16, True),
        # chunks of prompts, an odd number of tokens in all
        _append("append_chunks", "f16", 16001, 32, 8, 128, 16, True),
        # one user's next token, not far into a conversation, through a small model
        _attend("attend_token", "f16", 1, 777, 777, 1, 14, 2, 64, 16),
        # a serving batch, each conversation of its own length
        _attend("attend_batch", "f16", 64, 64, 8192, 1, 32, 8, 128, 16),
        # a few tokens to verify behind two long documents
        _attend("attend_verify_long", "f16", 2, 90000, 100001, 3, 32, 8, 128, 64),
        # samples from an f32 model with a key head for every query head, some without a token yet
        _attend("attend_f32", "f32", 16, 0, 3000, 1, 32, 32, 64, 32),
        # one request
        _select("select_request", "f32", 1, 4, 32000, 4, False),
        # a batch of requests over a large vocabulary, twice the beams kept so that those which end can be put aside
        _select("select_batch", "f16", 32, 8, 128256, 16, True),
        # a request of four beams through a small model
        _reorder("reorder_request", "f32", 1, 4, 100, 400, 2, 64, 16, 4),
        # a batch of requests, eight layers' pages
        _reorder("reorder_batch", "f16", 32, 8, 20, 700, 8, 128, 16, 8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "select", "select", "reorder"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 64), (14, 2, 64), (32, 32, 128)])
    dtype = rng.choice(["f16", "f16", "f32"])
    page = rng.choice([16, 16, 32, 64, 128])
    size = 4 if dtype == "f32" else 2
    if kind == "plan":
        least = rng.choice([0, 1])
        case = _plan("", _log(rng, 1, 1000), rng.choice([0, 1, 100]), _log(rng, 200, 16000), least, rng.choice([1, _log(rng, 2, 200)]), page)
        if case["most"] == 1:
            case["least"] = 1
    elif kind == "append":
        tokens = min(_log(rng, 1, 16000), 16000 * 8 * 128 * 2 // (kv_heads * dim * size))
        case = _append("", dtype, tokens, heads, kv_heads, dim, page, rng.random() < 0.7)
    elif kind == "attend":
        seqs, longest = _log(rng, 1, 200), _log(rng, 30, 60000)
        longest = max(30, min(longest, 64 * 8192 * 8 * 128 * 2 // (seqs * kv_heads * dim * size)))
        queries = rng.choice([1, 1, 1, rng.randint(2, 6)])
        case = _attend("", dtype, seqs, rng.choice([0, 1, longest // 2, longest]), longest, queries, heads, kv_heads, dim, page)
    elif kind == "select":
        beams, vocab = rng.randint(1, 8), _log(rng, 1000, 128256)
        batch = min(_log(rng, 1, 64), 32 * 8 * 128256 * 2 // (beams * vocab * size))
        case = _select("", dtype, batch, beams, vocab, beams * rng.choice([1, 2]), rng.random() < 0.5)
    else:
        batch, beams, layers = _log(rng, 1, 32), rng.randint(2, 8), rng.choice([1, 2, 4])
        longest = _log(rng, 50, 700)
        case = _reorder("", dtype, batch, beams, longest // rng.choice([1, 2, 8]), longest, min(kv_heads, 8), dim, min(page, 32), layers)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(gen, shape, dtype, scale=1.0):
    out = torch.randn(tuple(shape), generator=gen, device="cuda", dtype=_TORCH[dtype])
    return out if scale == 1.0 else out.mul_(scale)


def _ints(values):
    return torch.tensor(np.ascontiguousarray(values, dtype=np.int32), device="cuda")


def _lengths(case):
    """How many tokens each sequence holds: the case's, not the seed's."""
    lens = np.random.default_rng(21).integers(case["shortest"], case["longest"], size=case["seqs"], endpoint=True)
    lens[case["seqs"] // 2] = case["longest"]
    return lens


def _added(case):
    new = np.random.default_rng(22).integers(case["least"], case["most"], size=case["seqs"], endpoint=True)
    new[case["seqs"] // 2] = case["most"]
    return new


def _table(rng, lens, page, width, n_pages):
    """Pages of the sequences in any order, and the others: (table, -1 behind each sequence's pages; the free ones)."""
    order = rng.permutation(n_pages)
    held = -(-lens // page)
    there = np.arange(width)[None, :] < held[:, None]
    table = np.full(there.shape, -1, np.int64)
    table[there] = order[: held.sum()]
    return table, order[held.sum() :]


def _prepare_plan(case, seed):
    rng = np.random.default_rng(seed)
    lens, new, page = _lengths(case), _added(case), case["page"]
    width = -(-(case["longest"] + case["most"]) // page) + 1
    more = int((-(-(lens + new) // page) - -(-lens // page)).sum())
    n_pages = int((-(-lens // page)).sum()) + more + case["seqs"]
    table, free = _table(rng, lens, page, width, n_pages)
    refs = np.zeros(n_pages, np.int64)
    refs[table[table >= 0]] = 1
    stack = np.full(n_pages, -1)
    stack[: len(free)] = free
    tokens = int(new.sum()) + int(new.sum()) % 7     # a few places more than are filled
    s = {"lens": _ints(lens), "new": _ints(new), "table": _ints(table), "free": _ints(stack), "count": _ints([len(free)]), "refs": _ints(refs), "tokens": tokens, "page": page}
    s["out"] = {"lens": _ints(lens), "starts": _ints(np.zeros(case["seqs"] + 1)), "slots": _ints(np.zeros(tokens)), "positions": _ints(np.zeros(tokens)),
                "free_count": _ints([0]), "refused": _ints([0])}
    return s


def _prepare_append(case, seed):
    t, hq, hkv, d, dt, page = (case[x] for x in ("tokens", "heads", "kv_heads", "dim", "dtype", "page"))
    gen, rng = _generator(seed), np.random.default_rng(seed)
    n_pages = t // page + 64
    if case["fused"]:
        rows = _normal(gen, (t, (hq + 2 * hkv) * d), dt)
        k, v = rows[:, hq * d : (hq + hkv) * d].view(t, hkv, d), rows[:, (hq + hkv) * d :].view(t, hkv, d)
    else:
        k, v = _normal(gen, (t, hkv, d), dt), _normal(gen, (t, hkv, d), dt)
    # runs of tokens go to consecutive places of a page, as a chunk's do; next tokens go anywhere
    first = rng.permutation(n_pages)[: -(-t // page)] * page
    slots = (first[:, None] + np.arange(page)[None, :]).reshape(-1)[:t]
    if t <= 64:
        slots = rng.permutation(n_pages * page)[:t]
    return {"k": k, "v": v, "slots": _ints(slots), "page": page, "k_pages": _normal(gen, (n_pages, hkv, page, d), dt), "v_pages": _normal(gen, (n_pages, hkv, page, d), dt)}


def _prepare_attend(case, seed):
    n, hq, hkv, d, dt, page, m = (case[x] for x in ("seqs", "heads", "kv_heads", "dim", "dtype", "page", "queries"))
    gen, rng, lens = _generator(seed), np.random.default_rng(seed), _lengths(case)
    n_pages = int((-(-lens // page)).sum()) + 16
    table, _ = _table(rng, lens, page, max(1, -(-case["longest"] // page)), n_pages)
    return {"q": _normal(gen, (n, hq, m, d), dt, 2.0), "k_pages": _normal(gen, (n_pages, hkv, page, d), dt), "v_pages": _normal(gen, (n_pages, hkv, page, d), dt),
            "table": _ints(table), "lens": _ints(lens), "out": torch.empty((n, hq, m, d), device="cuda", dtype=_TORCH[dt])}


def _prepare_select(case, seed):
    b, w, n, dt, keep = (case[x] for x in ("batch", "beams", "vocab", "dtype", "keep"))
    gen = _generator(seed)
    s = {"logits": _normal(gen, (b, w, n), dt, 3.0), "scores": -20.0 * torch.rand((b, w), generator=gen, device="cuda"), "ended": None, "keep": keep,
         "out": {"scores": torch.empty((b, keep), device="cuda")}}
    if case["ended"]:
        s["ended"] = (torch.rand((b, w), generator=gen, device="cuda") < 0.2).int()
        s["ended"][:, 0] = 0     # (a request with nothing left to go on is done)
    for name in ("parents", "tokens", "ended"):
        s["out"][name] = torch.empty((b, keep), device="cuda", dtype=torch.int32)
    return s


def _prepare_reorder(case, seed):
    b, w, hkv, d, dt, page, layers = (case[x] for x in ("batch", "beams", "kv_heads", "dim", "dtype", "page", "layers"))
    gen, rng, n = _generator(seed), np.random.default_rng(seed), case["batch"] * case["beams"]
    # a request's beams have one length, share the pages of its prompt and hold the others alone
    of_request = np.random.default_rng(23).integers(case["shortest"], case["longest"], size=b, endpoint=True)
    lens = np.repeat(of_request, w)
    width = -(-case["longest"] // page) + 2
    n_pages = int((-(-lens // page)).sum()) + n
    table, _ = _table(rng, lens, page, width, n_pages)
    prompt = np.repeat(of_request * 2 // 3 // page, w)
    shared = np.arange(width)[None, :] < prompt[:, None]
    table = np.where(shared, np.repeat(table[::w], w, axis=0), table)
    refs = np.bincount(table[table >= 0], minlength=n_pages)
    free = rng.permutation(np.flatnonzero(refs == 0))
    stack = np.full(n_pages, -1)
    stack[: len(free)] = free
    parents = (np.arange(b)[:, None] * w + rng.integers(0, w, size=(b, w))).reshape(-1)
    pools = torch.empty((2 * layers, n_pages, hkv, page, d), device="cuda", dtype=_TORCH[dt]).normal_(generator=gen)
    s = {"parents": _ints(parents), "table": _ints(table), "lens": _ints(lens), "refs": _ints(refs), "free": _ints(stack), "count": _ints([len(free)]), "page": page,
         "pools": pools}
    s["out"] = {"table": torch.empty_like(s["table"]), "lens": torch.empty_like(s["lens"]), "refs": torch.empty_like(s["refs"]), "free_pages": torch.empty_like(s["free"]),
                "free_count": _ints([0]), "copies": _ints(np.zeros((n, 3))), "missing": _ints([0])}
    return s


_PREPARE = {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend, "select": _prepare_select, "reorder": _prepare_reorder}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, seed)
    state["kind"] = case["kind"]
    torch.cuda.synchronize()
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------


def _plain_plan(s):
    lens, new, table, page, tokens = s["lens"].long(), s["new"].long(), s["table"].long(), s["page"], s["tokens"]
    n, width = table.shape
    ends = new.cumsum(0)
    starts = ends - new
    have = (lens + page - 1) // page
    fits = (ends <= tokens) & (lens + new <= width * page)
    need = torch.where(fits, (lens + new + page - 1) // page - have, 0)
    off = need.cumsum(0) - need
    admitted = fits & ((need == 0) | (off + need <= s["count"]))
    need = torch.where(admitted, need, 0)
    p = torch.arange(width, device="cuda")[None, :] - have[:, None]
    is_new = (p >= 0) & (p < need[:, None])
    pages = s["free"].long()[(s["count"] - 1 - off[:, None] - p).clamp(0, len(s["free"]) - 1)]
    table = torch.where(is_new, pages, table)
    refs = torch.cat([s["refs"], s["refs"].new_zeros(1)])     # (a place behind the last for those that are not new)
    refs[torch.where(is_new, pages, len(refs) - 1)] = 1
    t = torch.arange(tokens, device="cuda")
    of = torch.searchsorted(ends, t, right=True)
    there = of < n
    of = of.clamp(max=n - 1)
    there = there & admitted[of]
    at = lens[of] + t - starts[of]
    slots = table[of, (at // page).clamp(max=width - 1)] * page + at % page
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    return {"lens": whole(torch.where(admitted, lens + new, lens)), "starts": whole(torch.cat([starts, ends[-1:]])), "slots": whole(torch.where(there, slots, -1)),
            "positions": whole(torch.where(there, at, -1)), "free_count": whole(s["count"] - need.sum()), "refused": whole((~admitted).sum()[None]), "table": whole(table),
            "refs": refs[:-1]}


def _plain_append(s):
    slots, page = s["slots"].long(), s["page"]
    s["k_pages"][slots // page, :, slots % page] = s["k"]
    s["v_pages"][slots // page, :, slots % page] = s["v"]
    return [s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    n, hq, m, d = s["q"].shape
    hkv = s["k_pages"].shape[1]
    table, lens = s["table"].clamp(min=0).long(), s["lens"].long()
    k, v = (s[x][table].transpose(1, 2).reshape(n, hkv, -1, d).float() for x in ("k_pages", "v_pages"))
    scores = torch.matmul(s["q"].float().view(n, hkv, -1, d) * (1.0 / math.sqrt(d)), k.transpose(2, 3)).view(n, hq, m, -1)
    last = lens[:, None] - m + torch.arange(m, device="cuda")[None, :]
    scores = scores.masked_fill((torch.arange(scores.shape[-1], device="cuda") > last[:, :, None])[:, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(dim=-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    return torch.matmul(w.view(n, hkv, -1, w.shape[-1]), v).view(n, hq, m, d).to(s["q"].dtype)


def _plain_select(s):
    b, w, n = s["logits"].shape
    x = s["logits"].double()
    top = x.amax(dim=-1, keepdim=True)
    x = x - top
    x = s["scores"].double()[..., None] + (x - x.exp().sum(dim=-1, keepdim=True).log())
    if s["ended"] is not None:
        alone = torch.full((n,), -math.inf, device="cuda", dtype=torch.float64)
        alone[_EOS] = 0.0
        x = torch.where(s["ended"][..., None] != 0, s["scores"].double()[..., None] + alone, x)
    x, at = torch.sort(x.view(b, w * n), dim=-1, descending=True, stable=True)
    x, at = x[:, : s["keep"]], at[:, : s["keep"]]
    ended = at % n == _EOS
    if s["ended"] is not None:
        ended = ended | (s["ended"].gather(1, at // n) != 0)
    return {"scores": x.float(), "parents": (at // n + w * torch.arange(b, device="cuda")[:, None]).int(), "tokens": (at % n).int(), "ended": ended.int()}


def _plain_reorder(s):
    parents, table, lens, refs, page = s["parents"].long(), s["table"].long(), s["lens"].long(), s["refs"].long(), s["page"]
    n, width = table.shape
    rows = torch.arange(n, device="cuda")
    new_table, new_lens = table[parents], lens[parents]
    # the partial page stays with the first of the children and is copied for the others
    first = torch.full((n,), n, device="cuda").scatter_reduce(0, parents, rows, "amin")
    at = (new_lens // page).clamp(max=width - 1)
    partial = new_table.gather(1, at[:, None])[:, 0]
    copied = (new_lens % page > 0) & ((first[parents] != rows) | (refs[partial.clamp(min=0)] != 1))
    order = copied.long().cumsum(0) - copied.long()
    fresh = s["free"].long()[(s["count"] - 1 - order).clamp(min=0)]
    new_table = new_table.scatter(1, at[:, None], torch.where(copied, fresh, new_table.gather(1, at[:, None])[:, 0])[:, None])
    taken = copied.sum()
    spare = torch.cat([refs, refs.new_zeros(1)])     # (a place behind the last for what is not a page)
    for t, by in ((table, -1), (new_table, 1)):
        spare = spare.scatter_add(0, torch.where(t >= 0, t, len(refs)).view(-1), torch.full((n * width,), by, device="cuda"))
    new_refs = spare[:-1]
    freed = (new_refs == 0) & (refs > 0)
    left = s["count"].long() - taken
    place = torch.arange(len(refs), device="cuda")
    stack = torch.where(place < left, s["free"].long(), -1)
    to = torch.where(freed, left + freed.long().cumsum(0) - 1, len(refs))
    stack = torch.cat([stack, stack.new_zeros(1)]).scatter(0, to, place)[:-1]
    stack = torch.where(place < left + freed.sum(), stack, -1)
    copies = torch.where(copied[:, None], torch.stack([partial, fresh, new_lens % page], dim=1), torch.tensor([-1, -1, 0], device="cuda"))
    # rows of the copied pages, in all layers
    hits = copies[:, 0].clamp(min=0)
    old, to = s["pools"][:, hits], torch.where(copied, fresh, hits)
    keep = (torch.arange(page, device="cuda")[None, :] < copies[:, 2:])[None, :, None, :, None]
    s["pools"][:, to] = torch.where(keep, old, s["pools"][:, to])
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    return {"table": whole(new_table), "lens": whole(new_lens), "refs": whole(new_refs), "free_pages": whole(stack), "free_count": whole(left + freed.sum()), "copies": whole(copies),
            "missing": whole((taken - s["count"]).clamp(min=0)), "pools": s["pools"]}


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}


# ---- the framework's -------------------------------------------------------------------------------------------


def _handles(s):
    """The tensors as the library's own over the same memory, the operator and its workspace: what a program makes once."""
    import tract_amd as ta

    if "handles" not in s:
        ta.runtime_for_name("rocm")
        over = lambda t: ta.DeviceTensor(t.shape, _NP[t.dtype], ptr=t.data_ptr(), owner=t)  # noqa: E731
        h = {name: over(t) for name, t in s.items() if isinstance(t, torch.Tensor)}
        if isinstance(s.get("out"), dict):
            h["out"] = {name: over(t) for name, t in s["out"].items()}
        if s["kind"] == "plan":
            h["op"] = ta.PagedPlan(s["page"])
        elif s["kind"] == "append":
            h["op"] = ta.PagedAppend()
            h["strides"] = s["k"].stride(), s["v"].stride()
        elif s["kind"] == "attend":
            h["op"] = ta.PagedSdpa()
        elif s["kind"] == "select":
            h["op"] = ta.BeamSelect(s["keep"], eos=_EOS)
        else:
            h["op"], h["copy"] = ta.PagedReorder(s["page"]), ta.PagedCopy()
            h["pools"] = [over(t) for t in s["pools"]]
        s["handles"] = h
    return s["handles"]


def _own_plan(s):
    h = _handles(s)
    h["op"].eval(h["lens"], h["new"], h["table"], h["free"], h["count"], s["tokens"], refs=h["refs"], out=h["out"])
    return {**s["out"], "table": s["table"], "refs": s["refs"]}


def _own_append(s):
    h = _handles(s)
    h["op"].eval(h["k"], h["v"], h["slots"], h["k_pages"], h["v_pages"], k_strides=h["strides"][0], v_strides=h["strides"][1])
    return [s["k_pages"], s["v_pages"]]


def _own_attend(s):
    h = _handles(s)
    h["op"].eval(h["q"], h["k_pages"], h["v_pages"], h["table"], h["lens"], out=h["out"])
    return s["out"]


def _own_select(s):
    h = _handles(s)
    h["op"].eval(h["logits"], h["scores"], ended=h.get("ended"), out=h["out"])
    return s["out"]


def _own_reorder(s):
    h = _handles(s)
    h["op"].eval(h["parents"], h["table"], h["lens"], h["refs"], h["free"], h["count"], out=h["out"])
    h["copy"].eval(h["out"]["copies"], h["pools"])
    return {**s["out"], "pools": s["pools"]}


_OWN = {"plan": _own_plan, "append": _own_append, "attend": _own_attend, "select": _own_select, "reorder": _own_reorder}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---- the same in 64 bits -----------------------------------------------------------------------------------


def _exact_append(case, s):
    where = [divmod(int(x), case["page"]) for x in s["slots"].cpu()]
    outs = []
    for rows, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        flat = pages.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        flat = flat.index_copy(0, torch.tensor([p * case["page"] + r for p, r in where], device="cuda"), rows.contiguous())
        outs.append(flat.view(-1, case["page"], case["kv_heads"], case["dim"]).transpose(1, 2).double())
    return outs


def _exact_attend(case, s):
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    group, m, d = case["heads"] // case["kv_heads"], case["queries"], case["dim"]
    for i, n in enumerate(_lengths(case)):
        pages = s["table"][i, : -(-int(n) // case["page"])].long()
        for r in range(m):
            sees = int(n) - m + r + 1
            if sees <= 0:
                continue
            q = s["q"][i, :, r].double().view(-1, group, d)
            for h in range(case["kv_heads"]):
                k, v = (s[x][pages, h].reshape(-1, d)[:sees].double() for x in ("k_pages", "v_pages"))
                w = torch.softmax((k @ q[h].t().contiguous()).t() / math.sqrt(d), dim=-1)
                out[i, h * group : (h + 1) * group, r] = w @ v
    return out


def _exact_select(case, s):
    scores = torch.empty((case["batch"], case["keep"]), device="cuda", dtype=torch.float64)
    for i in range(case["batch"]):
        all_of = []
        for j in range(case["beams"]):
            score = s["scores"][i, j].double()
            if s["ended"] is not None and int(s["ended"][i, j]):
                all_of.append(score[None])
            else:
                all_of.append(score + torch.log_softmax(s["logits"][i, j].double(), dim=-1))
        all_of = torch.cat(all_of)
        scores[i] = -math.inf
        best = torch.topk(all_of, min(case["keep"], len(all_of))).values
        scores[i, : len(best)] = best
    return {"scores": scores, "parents": None, "tokens": None, "ended": None}


def _exact_reorder(case, s):
    """The pages after the copies, walked through one sequence at a time; the tables are whole numbers."""
    page, parents, lens, table, refs, free = case["page"], *(s[x].tolist() for x in ("parents", "lens", "table", "refs", "free"))
    free = free[: int(s["count"])]
    begun = set()
    for p in parents:
        partial = lens[p] % page
        if partial:
            old = table[p][lens[p] // page]
            if p in begun or refs[old] != 1:
                s["pools"][:, free.pop(), :, :partial] = s["pools"][:, old, :, :partial]
        begun.add(p)
    return {"pools": s["pools"]}


def exact(case, seed):
    if case["kind"] == "plan":
        return None     # whole numbers
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](case, prepare(case, seed))


# ---- what a pass cannot do without ---------------------------------------------------------------------------


def work(case):
    size = {"f16": 2, "f32": 4}[case.get("dtype", "f32")]
    if case["kind"] == "plan":
        lens, new, page = _lengths(case), _added(case), case["page"]
        pages = int((-(-(lens + new) // page) - -(-lens // page)).sum())
        return {"bytes": 4 * (4 * case["seqs"] + 2 * int(new.sum()) + 3 * pages), "flops": 2 * int(new.sum()) + 8 * case["seqs"]}
    if case["kind"] == "append":
        return {"bytes": case["tokens"] * (4 * case["kv_heads"] * case["dim"] * size + 4), "flops": 0}
    if case["kind"] == "attend":
        lens, m = _lengths(case), case["queries"]
        pairs = sum(max(0, int(n) - m + r + 1) for n in lens for r in range(m))
        held = int((-(-lens // case["page"])).sum())
        return {"bytes": (2 * int(lens.sum()) * case["kv_heads"] + 2 * case["seqs"] * m * case["heads"]) * case["dim"] * size + 4 * held, "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["kind"] == "select":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * size + 16 * case["batch"] * case["keep"], "flops": 4 * n}
    # a request's beams go on from random ones: of w children 1 - (1 - 1 / w)^w of w parents have a first one, which keeps its page
    w, page = case["beams"], case["page"]
    of_request = np.random.default_rng(23).integers(case["shortest"], case["longest"], size=case["batch"], endpoint=True)
    rows = int((of_request % page).sum() * w * (1 - 1 / w) ** w)
    n_pages = int((-(-of_request // page)).sum()) * w + case["batch"] * w
    width = -(-case["longest"] // page) + 2
    return {"bytes": 4 * rows * case["layers"] * case["kv_heads"] * case["dim"] * size + 4 * (4 * n_pages + 2 * case["batch"] * w * width), "flops": 4 * case["batch"] * w * width}
