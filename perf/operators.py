"""What the operators around a decoder's attention are timed on: the norms of queries and keys with their rotation, decode
attention over a prefix that all sequences share, and attention whose scores are capped, biased or cut into documents.

A case is a dict of plain values.  Its "kind" is the operator:

* ``norm_rope``  RMS norm of every query and key head, scaled by a weight per feature, then the rotation by position
* ``shared``     one query per sequence over the keys of one prefix, kept once, and over the sequence's own keys after it
* ``scored``     attention with a tanh cap, a slope per head times the distance, documents packed into one row of tokens, and a
                 prefix that every query sees

Plain forms compute in 32 bits and round once.
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f16": torch.float16, "f32": torch.float32}
_NP = {torch.float16: np.float16, torch.float32: np.float32, torch.int32: np.int32}
_EPS = 1e-6


def _norm_rope(name, dtype, batch, n, heads, kv_heads, dim, fused):
    """fused: queries and keys are views into the rows of one projection to queries, keys and values."""
    return {"name": name, "kind": "norm_rope", "dtype": dtype, "batch": batch, "n": n, "heads": heads, "kv_heads": kv_heads, "dim": dim, "fused": fused}


def _shared(name, dtype, seqs, prefix, shortest, longest, heads, kv_heads, dim):
    return {"name": name, "kind": "shared", "dtype": dtype, "seqs": seqs, "prefix": prefix, "shortest": shortest, "longest": longest,
            "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _scored(name, dtype, batch, n, keys, heads, kv_heads, dim, cap, slopes, documents, prefix):
    """cap: 0 for none; documents: how many are packed into a row, 0 for none; prefix: keys that every query sees, up to so many."""
    return {"name": name, "kind": "scored", "dtype": dtype, "batch": batch, "n": n, "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "cap": cap, "slopes": slopes, "documents": documents, "prefix": prefix}


def listed():
    return [
        # one user's next token: the launch is all there is
        _norm_rope("norm_rope_token", "f16", 1, 1, 32, 8, 128, True),
        # a serving batch's next tokens
        _norm_rope("norm_rope_batch", "f16", 64, 1, 40, 8, 128, True),
        # two prompts of 4096 tokens
        _norm_rope("norm_rope_prompt", "f16", 2, 4096, 32, 8, 128, True),
        # a prompt of odd length through a small f32 model
        _norm_rope("norm_rope_prompt_f32", "f32", 1, 1777, 14, 2, 64, False),
        # a few answers to one short instruction, just begun
        _shared("shared_few", "f16", 4, 777, 1, 40, 14, 2, 64),
        # 64 users behind one long system prompt, each with a conversation of its own
        _shared("shared_batch", "f16", 64, 8192, 64, 512, 32, 8, 128),
        # many short requests over one document, some of them without a token of their own yet
        _shared("shared_wide", "f16", 200, 1500, 0, 300, 64, 8, 64),
        # samples of one prompt from an f32 model with a key head for every query head
        _shared("shared_f32", "f32", 16, 4096, 1, 600, 32, 32, 64),
        # the next tokens of a batch through a model that caps its scores
        _scored("scored_token", "f16", 8, 1, 8193, 32, 8, 128, 50.0, False, 0, 0),
        # a prompt through the same
        _scored("scored_prompt", "f16", 1, 4096, 4096, 32, 8, 128, 30.0, False, 0, 0),
        # rows of documents packed one behind the other, through a model whose scores fall with the distance
        _scored("scored_documents", "f16", 2, 4096, 4096, 14, 2, 64, 0.0, True, 9, 0),
        # a chunk of an f32 prompt behind a prefix that all of its tokens see, with everything that scores can have
        _scored("scored_chunk_f32", "f32", 1, 333, 1333, 32, 8, 128, 20.0, True, 3, 500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "shared", "shared", "scored", "scored"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 64), (14, 2, 64), (32, 32, 128)])
    dtype = rng.choice(["f16", "f16", "f32"])
    if kind == "norm_rope":
        batch = _log(rng, 1, 64)
        n = rng.choice([1, _log(rng, 2, 4096)])
        n = max(1, min(n, 8192 * 40 * 256 // (batch * (heads + kv_heads) * dim * (4 if dtype == "f32" else 2))))
        case = _norm_rope("", dtype, batch, n, heads, kv_heads, dim, rng.random() < 0.7)
    elif kind == "shared":
        prefix = _log(rng, 100, 12000)
        seqs = _log(rng, 2, 200)
        room = (1 << 31) // (heads * dim)      # as many products as the largest listed case has
        prefix = min(prefix, max(100, room // seqs))
        longest = _log(rng, 10, 2000)
        longest = max(8, min(longest, 40000 * 8 // (seqs * kv_heads)))
        if dtype == "f32":
            prefix, longest = min(prefix, 4096), min(longest, 600)
            seqs = min(seqs, 32)
        case = _shared("", dtype, seqs, prefix, rng.choice([0, 1, longest // 2]), longest, heads, kv_heads, dim)
    else:
        cap = rng.choice([0.0, 20.0, 50.0])
        slopes = rng.random() < 0.4
        documents = rng.choice([0, 0, rng.randint(2, 12)])
        if cap == 0.0 and not slopes and documents == 0:
            cap = 30.0
        if rng.random() < 0.4:      # the next token, or a few to verify
            batch, n = _log(rng, 1, 16), rng.choice([1, 1, rng.randint(2, 12)])
            keys = n + _log(rng, 100, 16000)
            keys = max(n + 100, min(keys, 65536 * 8 // (batch * kv_heads)))
        else:
            batch, n = rng.choice([1, 1, 2, 3]), _log(rng, 30, 4096)
            keys = n + rng.choice([0, 0, _log(rng, 10, 2000)])
            most = (1 << 29) * 16 // 17 if dtype == "f16" else 1 << 25
            while batch * heads * n * keys > most:
                n, keys = n * 3 // 4, keys * 3 // 4
            keys = max(keys, n)
        prefix = rng.choice([0, 0, keys // 3])
        case = _scored("", dtype, batch, n, keys, heads, kv_heads, dim, cap, slopes, documents, prefix)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(tuple(shape), generator=gen, device="cuda", dtype=torch.float32) * scale).to(_TORCH[dtype])


def _lengths(case):
    """How many keys each sequence has of its own: the case's, not the seed's."""
    rng = np.random.default_rng(11)
    return [int(n) for n in rng.integers(case["shortest"], case["longest"], size=case["seqs"], endpoint=True)]


def _documents(case):
    """The document of every token, [batch, keys]: packed one behind the other, the last row's tail of padding (-1)."""
    rng = np.random.default_rng(12)
    ids = np.empty((case["batch"], case["keys"]), np.int32)
    for row in ids:
        ends = np.sort(rng.integers(0, case["keys"], size=case["documents"] - 1))
        row[:] = np.searchsorted(ends, np.arange(case["keys"]), side="right")
    ids[-1, case["keys"] - case["keys"] // 50 :] = -1
    return ids


def _prefixes(case):
    rng = np.random.default_rng(13)
    return rng.integers(case["prefix"] // 2, case["prefix"], size=case["batch"], endpoint=True).astype(np.int32)


def _prepare_norm_rope(case, seed):
    b, n, hq, hkv, d, dt = (case[x] for x in ("batch", "n", "heads", "kv_heads", "dim", "dtype"))
    gen = _generator(seed)
    if case["fused"]:
        rows = _normal(gen, (b, n, (hq + 2 * hkv) * d), dt)
        rows[..., ::96] *= 8.0     # a few channels are larger, as projections have them
        q = rows[..., : hq * d].view(b, n, hq, d).transpose(1, 2)
        k = rows[..., hq * d : (hq + hkv) * d].view(b, n, hkv, d).transpose(1, 2)
    else:
        q, k = _normal(gen, (b, hq, n, d), dt), _normal(gen, (b, hkv, n, d), dt)
    wq, wk = (torch.rand(d, generator=gen, device="cuda") + 0.5 for _ in range(2))
    start = torch.randint(0, 30000, (b, 1), generator=gen, device="cuda")
    angle = (start + torch.arange(n, device="cuda"))[:, :, None].double() * 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.cat([angle, angle], dim=-1)
    return {"q": q, "k": k, "wq": wq.to(_TORCH[dt]), "wk": wk.to(_TORCH[dt]), "cos": angle.cos().to(_TORCH[dt])[:, None], "sin": angle.sin().to(_TORCH[dt])[:, None],
            "out": [torch.empty((b, h, n, d), device="cuda", dtype=_TORCH[dt]) for h in (hq, hkv)]}


def _prepare_shared(case, seed):
    n, p, hq, hkv, d, dt = (case[x] for x in ("seqs", "prefix", "heads", "kv_heads", "dim", "dtype"))
    gen, lens = _generator(seed), _lengths(case)
    room = max(1, max(lens))
    return {"q": _normal(gen, (n, hq, 1, d), dt, 2.0), "prefix_k": _normal(gen, (1, hkv, p, d), dt), "prefix_v": _normal(gen, (1, hkv, p, d), dt),
            "k": _normal(gen, (n, hkv, room, d), dt), "v": _normal(gen, (n, hkv, room, d), dt), "lens": lens,
            "lens_on_device": torch.tensor(lens, device="cuda"), "out": torch.empty((n, hq, 1, d), device="cuda", dtype=_TORCH[dt])}


def _prepare_scored(case, seed):
    b, n, t, hq, hkv, d, dt = (case[x] for x in ("batch", "n", "keys", "heads", "kv_heads", "dim", "dtype"))
    gen = _generator(seed)
    s = {"q": _normal(gen, (b, hq, n, d), dt, 6.0 if case["cap"] else 2.0), "k": _normal(gen, (b, hkv, t, d), dt), "v": _normal(gen, (b, hkv, t, d), dt),
         "cap": case["cap"], "slopes": None, "documents": None, "prefix": None, "out": torch.empty((b, hq, n, d), device="cuda", dtype=_TORCH[dt])}
    if case["slopes"]:
        s["slopes"] = (2.0 ** (-8.0 * (torch.arange(hq, device="cuda", dtype=torch.float64) + 1) / hq)).float()
    if case["documents"]:
        s["documents"] = torch.from_numpy(_documents(case)).cuda()
    if case["prefix"]:
        s["prefix"] = torch.from_numpy(_prefixes(case)).cuda()
    return s


_PREPARE = {"norm_rope": _prepare_norm_rope, "shared": _prepare_shared, "scored": _prepare_scored}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, seed)
    state["kind"] = case["kind"]
    torch.cuda.synchronize()
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------


def _plain_norm_rope_one(x, w, cos, sin):
    f = x.float()
    y = f * torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + _EPS) * w.float()
    half = y.shape[-1] // 2
    turned = torch.cat([-y[..., half:], y[..., :half]], dim=-1)
    return (y * cos.float() + turned * sin.float()).to(x.dtype)


def _plain_norm_rope(s):
    return [_plain_norm_rope_one(s["q"], s["wq"], s["cos"], s["sin"]), _plain_norm_rope_one(s["k"], s["wk"], s["cos"], s["sin"])]


def _weights(scores):
    """Softmax of scores whose hidden places hold -inf; a row that sees nothing weighs nothing."""
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_shared(s):
    n, hq, _, d = s["q"].shape
    hkv, p = s["prefix_k"].shape[1:3]
    room = s["k"].shape[2]
    q = s["q"].float().view(n, hkv, hq // hkv, d) * (1.0 / math.sqrt(d))
    by_head = q.transpose(0, 1).reshape(hkv, -1, d)
    over_prefix = torch.matmul(by_head, s["prefix_k"][0].float().transpose(1, 2)).view(hkv, n, hq // hkv, p).transpose(0, 1)
    over_own = torch.matmul(q, s["k"].float().transpose(2, 3))
    over_own = over_own.masked_fill((torch.arange(room, device="cuda")[None, :] >= s["lens_on_device"][:, None])[:, None, None, :], -math.inf)
    w = _weights(torch.cat([over_prefix, over_own], dim=-1))
    out = torch.matmul(w[..., :p].transpose(0, 1).reshape(hkv, -1, p), s["prefix_v"][0].float()).view(hkv, n, hq // hkv, d).transpose(0, 1)
    return (out + torch.matmul(w[..., p:], s["v"].float())).reshape(n, hq, 1, d).to(s["q"].dtype)


def _plain_scored(s):
    b, hq, n, d = s["q"].shape
    hkv, t = s["k"].shape[1:3]
    scores = torch.matmul(s["q"].float().view(b, hkv, -1, d) * (1.0 / math.sqrt(d)), s["k"].float().transpose(2, 3)).view(b, hq, n, t)
    if s["cap"]:
        scores = s["cap"] * torch.tanh(scores / s["cap"])
    at = torch.arange(t - n, t, device="cuda")[:, None]
    j = torch.arange(t, device="cuda")[None, :]
    if s["slopes"] is not None:
        scores = scores - s["slopes"][None, :, None, None] * (at - j).abs()
    sees = (j <= at)[None]
    if s["prefix"] is not None:
        sees = sees | (j[None] < s["prefix"][:, None, None])
    if s["documents"] is not None:
        docs = s["documents"]
        sees = sees & (docs[:, None, :] == docs[:, t - n :, None]) & (docs >= 0)[:, None, :]
    w = _weights(scores.masked_fill(~sees[:, None], -math.inf))
    return torch.matmul(w.view(b, hkv, -1, t), s["v"].float()).view(b, hq, n, d).to(s["q"].dtype)


_PLAIN = {"norm_rope": _plain_norm_rope, "shared": _plain_shared, "scored": _plain_scored}


# ---- the framework's -------------------------------------------------------------------------------------------


def _handles(s):
    """The tensors as the library's own over the same memory, the operator and its workspace: what a program makes once."""
    import tract_amd as ta

    if "handles" not in s:
        ta.runtime_for_name("rocm")
        h = {name: ta.DeviceTensor(t.shape, _NP[t.dtype], ptr=t.data_ptr(), owner=t) for name, t in s.items() if isinstance(t, torch.Tensor) and t.dtype in _NP}
        if s["kind"] == "norm_rope":
            h["op"] = ta.QkNormRope(eps=_EPS)
            h["out"] = [ta.DeviceTensor(t.shape, _NP[t.dtype], ptr=t.data_ptr(), owner=t) for t in s["out"]]
            h["strides"] = [s["q"].stride(), s["k"].stride()]
        else:
            h["op"] = ta.SharedPrefixSdpa() if s["kind"] == "shared" else ta.ScoredSdpa(softcap=s["cap"], is_causal=True)
        s["handles"] = h
    return s["handles"]


def _own_norm_rope(s):
    h = _handles(s)
    h["op"].eval(h["q"], h["k"], h["wq"], h["wk"], h["cos"], h["sin"], q_strides=h["strides"][0], k_strides=h["strides"][1], q_out=h["out"][0], k_out=h["out"][1])
    return s["out"]


def _own_shared(s):
    h = _handles(s)
    h["op"].eval(h["q"], h["prefix_k"], h["prefix_v"], h["k"], h["v"], s["lens"], out=h["out"])
    return s["out"]


def _own_scored(s):
    h = _handles(s)
    h["op"].eval(h["q"], h["k"], h["v"], slopes=h.get("slopes"), documents=h.get("documents"), prefix_lens=h.get("prefix"), out=h["out"])
    return s["out"]


_OWN = {"norm_rope": _own_norm_rope, "shared": _own_shared, "scored": _own_scored}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---- the same in 64 bits -----------------------------------------------------------------------------------


def _exact_norm_rope(case, s):
    outs = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        x = w.double() * x / torch.sqrt(x.pow(2).sum(dim=-1, keepdim=True) / case["dim"] + _EPS)
        first, second = x.chunk(2, dim=-1)
        (c1, c2), (s1, s2) = (t.double().chunk(2, dim=-1) for t in (s["cos"], s["sin"]))
        outs.append(torch.cat([first * c1 - second * s1, second * c2 + first * s2], dim=-1))
    return outs


def _exact_shared(case, s):
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    group = case["heads"] // case["kv_heads"]
    pk, pv = s["prefix_k"][0].double(), s["prefix_v"][0].double()
    for i, n in enumerate(s["lens"]):
        k = torch.cat([pk, s["k"][i, :, :n].double()], dim=1)
        v = torch.cat([pv, s["v"][i, :, :n].double()], dim=1)
        q = s["q"][i, :, 0].double().view(case["kv_heads"], group, -1)
        w = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(case["dim"]), dim=-1)
        out[i, :, 0] = torch.matmul(w, v).reshape(case["heads"], -1)
    return out


def _exact_scored(case, s):
    b, n, t, hq = case["batch"], case["n"], case["keys"], case["heads"]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    place = torch.arange(t, device="cuda")
    for i in range(b):
        hidden = place[None, :] > place[t - n :, None]
        if case["prefix"]:
            hidden &= place[None, :] >= int(_prefixes(case)[i])
        if case["documents"]:
            ids = torch.from_numpy(_documents(case)[i]).cuda()
            hidden |= (ids[None, :] != ids[t - n :, None]) | (ids < 0)[None, :]
        for h in range(hq):
            kv = h * case["kv_heads"] // hq
            x = torch.matmul(s["q"][i, h].double(), s["k"][i, kv].double().t().contiguous()) / math.sqrt(case["dim"])
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - s["slopes"][h].double() * (place[t - n :, None] - place[None, :]).abs()
            x = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1)
            out[i, h] = torch.matmul(torch.nan_to_num(x, nan=0.0), s["v"][i, kv].double())
    return out


_EXACT = {"norm_rope": _exact_norm_rope, "shared": _exact_shared, "scored": _exact_scored}


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))


# ---- what a pass cannot do without ---------------------------------------------------------------------------


def _pairs(case):
    """(query, key) pairs that see each other, of one head and all of the batch."""
    b, n, t = case["batch"], case["n"], case["keys"]
    if not case["documents"] and not case["prefix"]:
        return b * (n * (t - n) + n * (n + 1) // 2)
    at, j, total = np.arange(t - n, t)[:, None], np.arange(t)[None, :], 0
    for i in range(b):
        sees = j <= at
        if case["prefix"]:
            sees = sees | (j < _prefixes(case)[i])
        if case["documents"]:
            ids = _documents(case)[i]
            sees = sees & (ids[None, :] == ids[t - n :, None]) & (ids >= 0)[None, :]
        total += int(sees.sum())
    return total


def work(case):
    size, hq, hkv, d = {"f16": 2, "f32": 4}[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "norm_rope":
        rows = case["batch"] * case["n"]
        return {"bytes": rows * d * size * (2 * (hq + hkv) + 2) + 2 * d * size, "flops": rows * (hq + hkv) * d * 8}
    if case["kind"] == "shared":
        lens = _lengths(case)
        keys = case["prefix"] + sum(lens)
        return {"bytes": (2 * keys * hkv + 2 * case["seqs"] * hq) * d * size, "flops": 4 * hq * d * (case["seqs"] * case["prefix"] + sum(lens))}
    b, n, t = case["batch"], case["n"], case["keys"]
    return {"bytes": b * (2 * t * hkv + 2 * n * hq) * d * size + (4 * b * t if case["documents"] else 0), "flops": 4 * _pairs(case) * hq * d}
