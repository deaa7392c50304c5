"""The serving operators around the decoder, as a program calls them, and what they cost at least.

Three groups that a decode step uses one after the other:
  process / select   penalties for repeated tokens, biases and grammar masks on logits, written out or
                     followed by log-softmax and the k best tokens
  append / attend    a paged cache of keys and values in 8 bits with one scale for each block of 16
                     tokens and head, and causal attention over it
  advance / compact  forking, freeing, growing (copy on write) and compacting the pages of such a cache

`run` computes them in elementary torch operations, or, where `own` is true, through vokra_b200."""
import json
import math
import zlib

import numpy as np
import torch

own = False
BLOCK = 16  # tokens of a page: one scale for each page and head

F = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # one stream's greedy step with the decoder's vocabulary: suppressed tokens as a bias row, a repetition penalty
        {"name": "process_one", "op": "process", "rows": 1, "vocab": 51866, "dtype": "f32", "history": 224, "n_bias": 1, "n_mask": 0, "ngram": 0},
        # a full batch with every rule on, a grammar state for each row
        {"name": "process_batch", "op": "process", "rows": 128, "vocab": 51866, "dtype": "f32", "history": 448, "n_bias": 4, "n_mask": 64, "ngram": 3},
        # the beams of one clip: the candidates of each beam
        {"name": "select_beams", "op": "select", "rows": 5, "vocab": 51866, "dtype": "f32", "history": 100, "n_bias": 1, "n_mask": 2, "ngram": 3, "k": 5},
        # a large batch over a large, odd vocabulary in 16 bits (many ties): the candidates a sampler takes
        {"name": "select_batch", "op": "select", "rows": 256, "vocab": 131071, "dtype": "f16", "history": 2048, "n_bias": 1, "n_mask": 256, "ngram": 0, "k": 40},
        # a decode step of the batched session: one token a stream
        {"name": "append_decode", "op": "append", "n_seq": 64, "max_q": 1, "max_len": 448, "n_kv_head": 20, "d_head": 64, "dtype": "f32"},
        # prompts of several streams, ragged, some continuing in the middle of a page
        {"name": "append_prompt", "op": "append", "n_seq": 8, "max_q": 2047, "max_len": 4000, "n_kv_head": 8, "d_head": 128, "dtype": "f16"},
        # the batched session's self-attention, a head of its own for each query head, in 32 bits
        {"name": "attend_batch", "op": "attend", "n_seq": 64, "max_q": 1, "max_len": 448, "group": 1, "n_kv_head": 20, "d_head": 64, "dtype": "f32", "idle": False},
        # one stream with a long cache
        {"name": "attend_long", "op": "attend", "n_seq": 1, "max_q": 1, "max_len": 131071, "group": 4, "n_kv_head": 8, "d_head": 128, "dtype": "f16", "idle": False},
        # a ragged batch in which each stream has up to four tokens to check, one stream without any key
        {"name": "attend_ragged", "op": "attend", "n_seq": 48, "max_q": 4, "max_len": 8191, "group": 4, "n_kv_head": 8, "d_head": 128, "dtype": "f16", "idle": True},
        # a chunk of four long prompts behind what the cache holds of them
        {"name": "attend_prompt", "op": "attend", "n_seq": 4, "max_q": 2047, "max_len": 12000, "group": 4, "n_kv_head": 8, "d_head": 128, "dtype": "f16", "idle": False},
        # one beam-search step over all layers: streams reordered, freed and grown, shared last pages copied
        {"name": "advance_beams", "op": "advance", "n_seq": 64, "max_len": 447, "n_layer": 32, "n_kv_head": 20, "d_head": 64, "spare": 1.3},
        # a cache after many streams came and went: its pages moved to the front
        {"name": "compact_half", "op": "compact", "n_seq": 256, "max_len": 4096, "n_layer": 2, "n_kv_head": 8, "d_head": 128, "spare": 2.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["process", "select", "append", "attend", "attend", "advance", "compact"])
    if op in ("process", "select"):
        rows = _log(rng, 1, 256 if op == "select" else 128)
        vocab = _log(rng, 1000, 131071) if op == "select" else _log(rng, 1000, 51866)
        c = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "f16"]), "history": rng.choice([0, _log(rng, 1, 2048)]),
             "n_bias": rng.choice([0, 1, 3]), "n_mask": rng.choice([0, 1, rows]), "ngram": rng.choice([0, 2, 3])}
        if op == "select":
            if c["dtype"] == "f32":
                c["rows"] = min(rows, 128)
            c["k"] = _log(rng, 1, 40)
        return c
    if op == "append":
        return {"op": op, "n_seq": _log(rng, 1, 64), "max_q": rng.choice([1, _log(rng, 1, 255)]), "max_len": _log(rng, 300, 4000),
                "n_kv_head": rng.randint(1, 20) if rng.random() < 0.5 else 8, "d_head": 64, "dtype": rng.choice(["f32", "f16"])}
    if op == "attend":
        kind = rng.choice(["step", "check", "chunk"])
        d_head = rng.choice([64, 128])
        n_kv_head = rng.randint(1, 8) if d_head == 128 else rng.randint(1, 20)
        group = rng.choice([1, 2, 4, 8]) if n_kv_head <= 8 else 1
        dtype = rng.choice(["f32", "f16"])
        if kind == "step":
            c = {"n_seq": _log(rng, 1, 48), "max_q": 1, "max_len": _log(rng, 16, 8191)}
        elif kind == "check":
            c = {"n_seq": _log(rng, 1, 48), "max_q": rng.randint(2, 8), "max_len": _log(rng, 16, 4095)}
        else:
            max_q = _log(rng, 9, 1000)
            c = {"n_seq": rng.randint(1, 4), "max_q": max_q, "max_len": max_q + _log(rng, 1, 3000)}
            group = min(group, 4)
        return {"op": op, **c, "group": group, "n_kv_head": n_kv_head, "d_head": d_head, "dtype": dtype, "idle": rng.random() < 0.3}
    d_head = rng.choice([64, 128])
    return {"op": op, "n_seq": _log(rng, 1, 64), "max_len": _log(rng, 16, 900), "n_layer": _log(rng, 1, 16), "n_kv_head": rng.randint(1, 8),
            "d_head": d_head, "spare": rng.choice([1.2, 1.5, 2.0])}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed)), np.random.default_rng(int(seed))


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _plain_case_logits(c, seed):
    g, r = _gen(seed)
    rows, vocab, hist = c["rows"], c["vocab"], c["history"]
    s = {"logits": (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(F[c["dtype"]]), "ngram": c["ngram"], "k": c.get("k", 0)}
    s["history"] = s["history_len"] = s["bias"] = s["bias_row"] = s["mask"] = s["mask_row"] = None
    if hist:
        # tokens repeat, and loops of a few tokens come up again
        h = (r.random((rows, hist)) ** 4 * vocab).astype(np.int32)
        loop = r.integers(2, 9)
        h[:, hist // 2:] = np.where(r.random((rows, 1)) < 0.5, np.resize(h[:, :loop], (rows, hist - hist // 2)), h[:, hist // 2:])
        n = r.integers(0, hist + 1, rows)
        n[0] = hist
        s["history"], s["history_len"] = _ints(h), _ints(n)
    s["repetition"] = torch.rand(rows, generator=g, device="cuda") * 0.3 + 1.0
    s["frequency"] = torch.rand(rows, generator=g, device="cuda") * 0.5
    s["presence"] = torch.rand(rows, generator=g, device="cuda") * 0.5
    if c["n_bias"]:
        b = torch.randn(c["n_bias"], vocab, generator=g, device="cuda") * (torch.rand(c["n_bias"], vocab, generator=g, device="cuda") < 0.01)
        s["bias"] = torch.where(torch.rand(c["n_bias"], vocab, generator=g, device="cuda") < 0.002, torch.full_like(b, -math.inf), b)
        s["bias_row"] = _ints(r.integers(-1 if rows > 1 else 0, c["n_bias"], rows))
    if c["n_mask"]:
        words = (vocab + 31) // 32
        m = torch.randint(-2**31, 2**31, (c["n_mask"], words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        if c["n_mask"] > 2:
            m[2] = 0  # a grammar state that allows nothing
        s["mask"], s["mask_row"] = m, _ints(r.integers(-1, c["n_mask"], rows))
    return s


def _case_rng(c):
    """What a case's sizes are drawn from: the case alone, so that every seed has the same shapes."""
    return np.random.default_rng(zlib.crc32(json.dumps({k: v for k, v in c.items() if k != "name"}, sort_keys=True).encode()))


def _streams(c):
    """Lengths of the streams (new tokens counted) and how many tokens of each are new."""
    n, r = c["n_seq"], _case_rng(c)
    new = r.integers(1, c["max_q"] + 1, n)
    new[r.integers(0, n)] = c["max_q"]
    lens = np.maximum(new, r.integers(max(1, c["max_len"] // 8) if n > 1 else c["max_len"], c["max_len"] + 1, n))
    if c.get("idle") and n > 1:
        lens[r.integers(0, n)] = 0  # a stream without any key: its rows are zero
    return lens, new


def _beams(c):
    """Lengths of the streams of an earlier state, which streams were forked from the one before them, each one's parent now and its new tokens."""
    n, r = c["n_seq"], _case_rng(c)
    lens = r.integers(1, c["max_len"] + 1, n)
    lens[r.integers(0, n)] = c["max_len"]
    fork = np.zeros(n, bool)
    parent, new = np.arange(n), np.zeros(n, np.int64)
    if c["op"] == "advance":
        fork[1::3] = True
        lens[fork] = lens[np.flatnonzero(fork) - 1]
        parent = r.integers(0, n, n)
        parent[r.random(n) < 0.1] = -1  # finished streams are freed
        new = (r.random(n) < 0.95).astype(np.int64)
    pages = int((-(-lens // BLOCK))[~fork].sum())
    return lens, fork, parent, new, int(pages * c["spare"]) + 2 * n


def _tables(lens, r, n_pages=0):
    """Pages for the streams, in random order, and how many pages there are."""
    need = -(-lens // BLOCK)
    n_pages = n_pages or int(need.sum()) + 1
    ids = r.permutation(n_pages)
    table = np.full((len(lens), int(need.max()) + 2), -1, np.int32)
    at = 0
    for i, p in enumerate(need):
        table[i, :p] = ids[at:at + p]
        at += p
    return table, n_pages


def _arena(c, n_pages, g, layers=1):
    h, d = c["n_kv_head"], c["d_head"]
    k = torch.empty(layers, n_pages, h, BLOCK, d, dtype=torch.int8, device="cuda")
    v = torch.empty(layers, n_pages, h, d, BLOCK, dtype=torch.int8, device="cuda")
    for x in (k, v):  # quants of normal values whose largest in a block is about three deviations
        for at in range(0, n_pages, 4096):
            y = torch.randn(x[:, at:at + 4096].shape, generator=g, device="cuda", dtype=torch.float16) * 42
            x[:, at:at + 4096] = y.clamp_(-127, 127).to(torch.int8)
    ks = (torch.rand(layers, n_pages, h, generator=g, device="cuda") + 0.5) * (3.0 / 127)
    vs = (torch.rand(layers, n_pages, h, generator=g, device="cuda") + 0.5) * (3.0 / 127)
    return k, v, ks, vs


def prepare(case, seed):
    c = dict(case)
    if c["op"] in ("process", "select"):
        return {"case": c, **_plain_case_logits(c, seed)}
    g, r = _gen(seed)
    h, d = c["n_kv_head"], c["d_head"]
    if c["op"] in ("append", "attend"):
        lens, new = _streams(c)
        table, n_pages = _tables(lens, r)
        k, v, ks, vs = _arena(c, n_pages, g)
        start = np.concatenate([[0], np.cumsum(new)])
        s = {"case": c, "k": k, "v": v, "ks": ks, "vs": vs, "table": _ints(table), "len": _ints(lens), "start": _ints(start), "n_tok": int(start[-1]),
             "max_q": int(new.max())}
        dt = F[c["dtype"]]
        if c["op"] == "attend":
            s["q"] = torch.randn(s["n_tok"], h * c["group"], d, generator=g, device="cuda").to(dt)
            s["scale"] = d ** -0.5
        else:
            s["new_k"] = torch.randn(s["n_tok"], h, d, generator=g, device="cuda").to(dt)
            s["new_v"] = torch.randn(s["n_tok"], h, d, generator=g, device="cuda").to(dt)
            back = lens - (lens - new) // BLOCK * BLOCK  # the positions of the pages that the new tokens touch
            row = np.concatenate([[0], np.cumsum(back)])
            s["row"], s["n_row"], s["max_back"] = _ints(row), int(row[-1]), int(back.max())
        return s
    lens, fork, parent, new, n_pages = _beams(c)
    table, n_pages = _tables(np.where(fork, 0, lens), r, n_pages)
    # a forked stream shares all pages of the one before it, a partly filled last page among them
    table[fork] = table[np.flatnonzero(fork) - 1]
    k, v, ks, vs = _arena(c, n_pages, g, c["n_layer"])
    refs = np.bincount(table[table >= 0], minlength=n_pages)
    s = {"case": c, "k": k, "v": v, "ks": ks, "vs": vs, "table": _ints(table), "len": _ints(lens), "refs": _ints(refs)}
    s["to"] = {"table": torch.empty_like(s["table"]), "len": torch.empty_like(s["len"]), "refs": torch.empty_like(s["refs"])}
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if c["op"] == "advance":
        s["parent"], s["new"] = _ints(parent), _ints(new)
    else:
        s["used"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _rules(s, dt):
    """The logits after every rule, in `dt`."""
    x = s["logits"].to(dt)
    rows, vocab = x.shape
    banned = torch.zeros(rows, vocab + 1, dtype=torch.bool, device=x.device)
    if s["history"] is not None:
        h, n = s["history"].long(), s["history_len"].long()
        live = torch.arange(h.shape[1], device=x.device) < n[:, None]
        ids = torch.where(live & (h >= 0) & (h < vocab), h, vocab)
        count = torch.zeros(rows, vocab + 1, dtype=dt, device=x.device).scatter_add_(1, ids, torch.ones_like(ids, dtype=dt))[:, :vocab]
        rep, freq, pres = (s[w].to(dt)[:, None] for w in ("repetition", "frequency", "presence"))
        y = torch.where(x > 0, x / rep, x * rep) - (freq * count + pres)
        x = torch.where(count > 0, y, x)
        m = s["ngram"]
        if m > 1 and h.shape[1] >= m:
            w = h.unfold(1, m, 1)  # [rows, places, m]
            at = (n[:, None] - (m - 1) + torch.arange(m - 1, device=x.device)).clamp_min(0)
            same = (w[:, :, :-1] == h.gather(1, at)[:, None]).all(2) & (torch.arange(w.shape[1], device=x.device) + m <= n[:, None])
            last = w[:, :, -1]
            last = torch.where(same & (last >= 0) & (last < vocab), last, vocab)
            banned = banned.scatter(1, last, True)
            banned[:, vocab] = False
    if s["bias"] is not None:
        b = s["bias_row"].long()
        x = x + torch.where((b >= 0)[:, None], s["bias"].to(dt)[b.clamp_min(0)], torch.zeros((), dtype=dt, device=x.device))
    stop = banned[:, :vocab]
    if s["mask"] is not None:
        m = s["mask_row"].long()
        word = s["mask"][m.clamp_min(0)]
        j = torch.arange(vocab, device=x.device)
        stop = stop | ((((word[:, j // 32] >> (j % 32)) & 1) == 0) & (m >= 0)[:, None])
    return torch.where(stop, torch.full((), -math.inf, dtype=dt, device=x.device), x)


def _select(x, k):
    m = x.amax(1, keepdim=True)
    lse = torch.where(m > -math.inf, m, torch.zeros_like(m)) + (x - torch.where(m > -math.inf, m, torch.zeros_like(m))).exp().sum(1, keepdim=True).log()
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    none = top == -math.inf
    return torch.where(none, -1, ids).to(torch.int32), torch.where(none, top, top - lse)


def _rows_of(start, n_seq, max_n, n_tok):
    """For each stream the rows that it has, padded: indexes and which of them are real."""
    i = start[:n_seq, None].long() + torch.arange(max_n, device=start.device)
    return i.clamp_max(n_tok - 1), i < start[1:, None]


def _attend(s, dt):
    c, n, h, d = s["case"], s["len"].shape[0], s["case"]["n_kv_head"], s["case"]["d_head"]
    t = s["table"].clamp_min(0).long()
    L = t.shape[1] * BLOCK
    k = (s["k"][0][t].to(dt) * s["ks"][0][t].to(dt)[..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, h, L, d)
    v = (s["v"][0][t].to(dt) * s["vs"][0][t].to(dt)[..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, h, L, d)
    at, real = _rows_of(s["start"], n, s["max_q"], s["n_tok"])
    q = s["q"].to(dt)[at].reshape(n, s["max_q"], h, c["group"], d).permute(0, 2, 3, 1, 4).reshape(n, h, c["group"] * s["max_q"], d)
    score = (q @ k.transpose(2, 3)).mul_(s["scale"]).reshape(n, h, c["group"], s["max_q"], L)
    new = (s["start"][1:] - s["start"][:-1]).long()
    pos = s["len"].long()[:, None] - new[:, None] + torch.arange(s["max_q"], device=q.device)
    score.masked_fill_((torch.arange(L, device=q.device) > pos[..., None])[:, None, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_().reshape(n, h, -1, L)
    z = p.sum(-1, keepdim=True)
    o = (p @ v / torch.where(z > 0, z, torch.ones_like(z))).reshape(n, h, c["group"], s["max_q"], d).permute(0, 3, 1, 2, 4)
    out = torch.empty(s["n_tok"], h * c["group"], d, dtype=dt, device=q.device)
    out[at[real]] = o.reshape(n, s["max_q"], h * c["group"], d)[real]
    return out


def _append(s, dt):
    """Stores the new tokens: (quants, scales) of the touched pages for both sides, and the values of their rows."""
    n, h, d = s["len"].shape[0], s["case"]["n_kv_head"], s["case"]["d_head"]
    new = (s["start"][1:] - s["start"][:-1]).long()
    first = (s["len"].long() - new) // BLOCK  # page of the first new token
    pages = -(-s["max_back"] // BLOCK)
    at = first[:, None] + torch.arange(pages, device=new.device)
    live = at * BLOCK < s["len"].long()[:, None]
    ids = s["table"].long().gather(1, at.clamp_max(s["table"].shape[1] - 1))[live]
    pos = at[..., None] * BLOCK + torch.arange(BLOCK, device=new.device)  # [n, pages, 16]
    is_new = ((pos >= (s["len"].long() - new)[:, None, None]) & (pos < s["len"].long()[:, None, None]))
    is_old = pos < (s["len"].long() - new)[:, None, None]
    src = (s["start"][:-1].long()[:, None, None] + pos - (s["len"].long() - new)[:, None, None]).clamp(0, s["n_tok"] - 1)
    where_new, where_old = is_new[live], is_old[live]
    back = _rows_of(s["row"], n, pages * BLOCK, s["n_row"])
    got = {}
    for side in ("k", "v"):
        x = torch.where(where_new[..., None, None], s["new_" + side].to(dt)[src[live]], torch.zeros((), dtype=dt, device=new.device))  # [pages, 16, h, d]
        old_q = (s[side][0][ids] if side == "k" else s[side][0][ids].transpose(2, 3)).transpose(1, 2)  # [pages, 16, h, d]
        old_s = torch.where(where_old.any(1)[:, None], s[side + "s"][0][ids].to(dt), torch.zeros((), dtype=dt, device=new.device))
        new_s = torch.maximum(old_s, x.abs().amax((1, 3)) / 127)
        some = new_s > 0
        inv = torch.where(some, 1 / new_s, torch.zeros_like(new_s))[:, None, :, None]
        ratio = torch.where(some, old_s / new_s, torch.zeros_like(new_s))[:, None, :, None]
        q = torch.where(where_old[..., None, None], (old_q.to(dt) * ratio).round(), old_q.to(dt))
        q = torch.where(where_new[..., None, None], (x * inv).round().clamp(-127, 127), q)
        got[side] = (ids, q, new_s)
        val = torch.zeros(n, pages, BLOCK, h, d, dtype=dt, device=new.device)
        val[live] = q * new_s[:, None, :, None]
        out = torch.empty(s["n_row"], h, d, dtype=dt, device=new.device)
        out[back[0][back[1]]] = val.reshape(n, pages * BLOCK, h, d)[back[1]]
        got["value_" + side] = out
    return got


def _append_plain(s):
    got = _append(s, torch.float32)
    for side in ("k", "v"):
        ids, q, scale = got[side]
        q = q.to(torch.int8).transpose(1, 2)
        s[side][0][ids] = q if side == "k" else q.transpose(2, 3)
        s[side + "s"][0][ids] = scale
    return {"k": got["value_k"], "v": got["value_v"]}


def _advance_plain(s):
    table, lens, refs = s["table"].long(), s["len"].long(), s["refs"]
    n, ld = table.shape
    par = s["parent"].long()
    live = par >= 0
    t = torch.where(live[:, None], table[par.clamp_min(0)], -1)
    ln = torch.where(live, lens[par.clamp_min(0)], 0)
    col = torch.arange(ld, device=t.device)
    have, want = (ln + BLOCK - 1) // BLOCK, (ln + torch.where(live, s["new"].long(), 0) + BLOCK - 1) // BLOCK
    t = torch.where(col < have[:, None], t, -1)
    count = torch.zeros(refs.shape[0] + 1, dtype=torch.int64, device=t.device)
    held = count.index_add(0, torch.where(t >= 0, t, refs.shape[0]).reshape(-1), torch.ones_like(t).reshape(-1))
    last = t.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0]
    writes = live & (s["new"] > 0) & (ln % BLOCK > 0)
    cow = writes & (held[last.clamp_min(0)] > 1)
    # pages that a stream takes: the copy of its last page, then the new ones; the lowest pages that no stream held before or holds now
    takes = (col >= have[:, None]) & (col < want[:, None]) | cow[:, None] & (col == (have - 1)[:, None])
    free = ((held[:-1] == 0) & (refs == 0)).nonzero()[:, 0]
    order = takes.reshape(-1).cumsum(0).reshape(n, ld) - 1
    fresh = free[order.clamp(0, free.shape[0] - 1)]
    out = torch.where(takes, fresh, t)
    src, dst = last[cow], out.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0][cow]
    for a in ("k", "v", "ks", "vs"):
        s[a][:, dst] = s[a][:, src]
    held = count.index_add(0, torch.where(out >= 0, out, refs.shape[0]).reshape(-1), torch.ones_like(out).reshape(-1))
    return out.to(torch.int32), (ln + torch.where(live, s["new"].long(), 0)).to(torch.int32), held[:-1].to(torch.int32)


def _compact_plain(s):
    refs = s["refs"]
    held = refs > 0
    used = held.sum()
    i = torch.arange(refs.shape[0], device=refs.device)
    src = (held & (i >= used)).nonzero()[:, 0]
    dst = (~held & (i < used)).nonzero()[:, 0]
    for a in ("k", "v", "ks", "vs"):
        s[a][:, dst] = s[a][:, src]
    to = i.clone()
    to[src] = dst
    t = s["table"].long()
    table = torch.where(t >= 0, to[t.clamp_min(0)], -1).to(torch.int32)
    out = torch.where(i < used, refs, 0)
    out[dst] = refs[src]
    return table, s["len"].clone(), out, used.to(torch.int32).reshape(1)


# ---- the calls a program makes ----------------------------------------------------------------------------------------

_ctx = None


def _own(s):
    """The handles that a program makes once: the context, the rules or the cache, the streams of the step."""
    global _ctx
    from vokra_b200 import blockkv, logits, ops
    if _ctx is None:
        _ctx = ops.Context(0)
    c, o = s["case"], {}
    if c["op"] in ("process", "select"):
        o["rules"] = logits.LogitsRules(history=s["history"], history_len=s["history_len"], repetition=s["repetition"], frequency=s["frequency"],
                                        presence=s["presence"], no_repeat_ngram=s["ngram"], bias=s["bias"], bias_row=s["bias_row"], mask=s["mask"],
                                        mask_row=s["mask_row"])
        o["process"], o["topk"] = logits.process, logits.topk
    else:
        o["cache"] = blockkv.BlockKvCache(_ctx, s["k"], s["v"], s["ks"], s["vs"])
        if c["op"] in ("append", "attend"):
            o["batch"] = blockkv.Batch(s["start"], s["len"], s["table"], s["n_tok"], s["max_q"])
        if c["op"] == "append":
            o["rows"] = blockkv.Batch(s["row"], s["len"], s["table"], s["n_row"], s["max_back"])
        if c["op"] in ("advance", "compact"):
            o["pages"] = o["cache"].pages(s["status"])
            o["state"] = blockkv.PageState(s["table"], s["len"], s["refs"])
            o["to"] = blockkv.PageState(**s["to"])
    return o


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        if "own" not in s:
            s["own"] = _own(s)
        o = s["own"]
        if op == "process":
            return o["process"](_ctx, s["logits"], o["rules"])
        if op == "select":
            return o["topk"](_ctx, s["logits"], s["k"], o["rules"])
        if op == "append":
            o["cache"].append(0, o["batch"], s["new_k"], s["new_v"])
            k, v = o["cache"].read(0, o["rows"])
            return {"k": k, "v": v}
        if op == "attend":
            return o["cache"].attention(0, o["batch"], s["q"], scale=s["scale"])
        if op == "advance":
            o["pages"].advance(o["state"], o["to"], parent=s["parent"], n_new=s["new"])
            table, lens, refs = s["to"]["table"], s["to"]["len"], s["to"]["refs"]
            used = None
        else:
            o["pages"].compact(o["state"], o["to"], n_used=s["used"])
            table, lens, refs, used = s["to"]["table"], s["to"]["len"], s["to"]["refs"], s["used"]
    else:
        if op == "process":
            return _rules(s, torch.float32).to(s["logits"].dtype)
        if op == "select":
            return _select(_rules(s, torch.float32), s["k"])
        if op == "append":
            return _append_plain(s)
        if op == "attend":
            return _attend(s, torch.float32).to(s["q"].dtype)
        if op == "advance":
            table, lens, refs = _advance_plain(s)
            used = None
        else:
            table, lens, refs, used = _compact_plain(s)
    # pages are moved as bytes, so they come back as bytes
    return {"table": table, "len": lens, "refs": refs, "used": used, "k": s["k"].view(torch.int32), "v": s["v"].view(torch.int32), "k_scale": s["ks"],
            "v_scale": s["vs"]}


# ---- the least that a pass reads, writes and computes -----------------------------------------------------------------


def work(case):
    c = dict(case)
    if c["op"] in ("process", "select"):
        rows, vocab, size = c["rows"], c["vocab"], 4 if c["dtype"] == "f32" else 2
        b = rows * vocab * size + min(rows, c["n_bias"]) * vocab * 4 + min(rows, c["n_mask"]) * vocab / 8 + rows * c["history"] * 2
        b += rows * vocab * size if c["op"] == "process" else rows * c["k"] * 8
        return {"bytes": b, "flops": rows * vocab * (2 if c["op"] == "process" else 5)}
    h, d = c["n_kv_head"], c["d_head"]
    page = h * (2 * BLOCK * d + 8)  # both sides of a page of one layer, with its scales
    size = 4 if c.get("dtype") == "f32" else 2
    if c["op"] in ("append", "attend"):
        lens, new = _streams(c)
        if c["op"] == "attend":
            # query i of a stream sees len - new + i + 1 keys
            seen = sum(float(np.maximum(0, n - m + 1 + np.arange(m)).sum()) for n, m in zip(lens, new)) * h * c["group"]
            return {"bytes": float((-(-lens // BLOCK)).sum()) * page + 2.0 * new.sum() * h * c["group"] * d * size, "flops": 4 * seen * d}
        back = lens - (lens - new) // BLOCK * BLOCK
        return {"bytes": 2.0 * h * d * (new.sum() * (size + 1) + back.sum() * 4), "flops": 6.0 * new.sum() * h * d}
    lens, fork, parent, new, n_pages = _beams(c)
    have = -(-lens // BLOCK)
    meta = 8.0 * have.sum() + 8.0 * n_pages
    if c["op"] == "advance":
        # the partly filled last pages that more than one stream holds and writes
        par = parent[parent >= 0]
        root = np.where(fork, np.arange(len(lens)) - 1, np.arange(len(lens)))  # a fork holds the pages of the stream before it
        shared = np.bincount(root[par], minlength=len(lens))[root[par]] > 1
        moved = float((shared & (lens[par] % BLOCK > 0) & (new[parent >= 0] > 0)).sum())
    else:
        held = float(have.sum())
        moved = held * (1 - held / n_pages)  # the held pages that lie behind the first `held` ones
    return {"bytes": meta + 2 * moved * page * c["n_layer"], "flops": 0.0}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("advance", "compact"):
        return None  # nothing is computed but whole numbers, and pages moved as they are
    if op in ("process", "select"):
        return _exact_logits(s, op)
    if op == "attend":
        return _exact_attend(s)
    return _exact_append(s)


def _exact_logits(s, op):
    """Row by row on the host, from the rules' definition."""
    x = s["logits"].double().cpu().numpy()
    host = {w: (None if s[w] is None else s[w].cpu().numpy()) for w in ("history", "history_len", "bias", "bias_row", "mask", "mask_row")}
    rep, freq, pres = (s[w].double().cpu().numpy() for w in ("repetition", "frequency", "presence"))
    rows, vocab = x.shape
    ids = np.full((rows, max(1, s["k"])), -1)
    prob = np.full((rows, max(1, s["k"])), -np.inf)
    for r in range(rows):
        y = x[r]
        stop = np.zeros(vocab, bool)
        if host["history"] is not None:
            h = host["history"][r, :host["history_len"][r]]
            token, times = np.unique(h[(h >= 0) & (h < vocab)], return_counts=True)
            z = y[token]
            y[token] = np.where(z > 0, z / rep[r], z * rep[r]) - freq[r] * times - pres[r]
            m = s["ngram"]
            if m > 1 and len(h) >= m:
                tail = h[len(h) - m + 1:]
                for i in range(len(h) - m + 1):
                    if np.array_equal(h[i:i + m - 1], tail) and 0 <= h[i + m - 1] < vocab:
                        stop[h[i + m - 1]] = True
        if host["bias"] is not None and host["bias_row"][r] >= 0:
            y += host["bias"][host["bias_row"][r]]
        if host["mask"] is not None and host["mask_row"][r] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_row"][r]].view(np.uint8), bitorder="little")
            stop |= bits[:vocab] == 0
        y[stop] = -np.inf
        if op == "select" and np.max(y) > -np.inf:
            best = np.argsort(-y, kind="stable")[:s["k"]]
            best = best[y[best] > -np.inf]
            top = np.max(y)
            ids[r, :len(best)] = best
            prob[r, :len(best)] = y[best] - top - np.log(np.exp(y - top).sum())
    return x if op == "process" else (None, prob)


def _exact_attend(s):
    """Stream by stream and head by head."""
    c = s["case"]
    out = torch.zeros(s["n_tok"], c["n_kv_head"] * c["group"], c["d_head"], dtype=torch.float64, device="cuda")
    start, lens = s["start"].tolist(), s["len"].tolist()
    for i, n in enumerate(lens):
        a, b = start[i], start[i + 1]
        ids = s["table"][i, :-(-n // BLOCK)].long()
        seen = torch.arange(n, device="cuda")[None, :] <= (n - (b - a) + torch.arange(b - a, device="cuda"))[:, None]
        some = seen.any(1)
        if n == 0 or not bool(some.any()):
            continue
        for h in range(c["n_kv_head"]):
            k = (s["k"][0, ids, h].double() * s["ks"][0, ids, h].double()[:, None, None]).reshape(-1, c["d_head"])[:n]
            v = (s["v"][0, ids, h].double() * s["vs"][0, ids, h].double()[:, None, None]).transpose(1, 2).reshape(-1, c["d_head"])[:n]
            for j in range(h * c["group"], (h + 1) * c["group"]):
                w = torch.einsum("qd,kd->qk", s["q"][a:b, j].double(), k) * s["scale"]
                w = torch.softmax(w.masked_fill(~seen, -math.inf)[some], 1)
                out[a:b, j][some] = w @ v
    return out


def _exact_append(s):
    """Page by page on the host: the largest value of a page and head sets its scale, earlier tokens are rounded anew."""
    c = s["case"]
    h, d = c["n_kv_head"], c["d_head"]
    start, lens, table = s["start"].tolist(), s["len"].tolist(), s["table"].tolist()
    out = {"k": [], "v": []}
    for side in ("k", "v"):
        new = s["new_" + side].double()
        for i, n in enumerate(lens):
            a, b = start[i], start[i + 1]
            first = n - (b - a)
            for page in range(first // BLOCK, -(-n // BLOCK)):
                lo, hi = page * BLOCK, min(n, (page + 1) * BLOCK)
                x = new[a + max(lo, first) - first:a + hi - first]  # [new tokens, h, d]
                scale = x.abs().amax((0, 2)) / 127
                rows = []
                if first > lo:
                    q = s[side][0, table[i][page]].double()
                    q = (q if side == "k" else q.transpose(1, 2))[:, :first - lo].transpose(0, 1)  # [old tokens, h, d]
                    was = s[side + "s"][0, table[i][page]].double()
                    scale = torch.maximum(scale, was)
                    rows.append((q * (was / scale)[None, :, None]).round() * scale[None, :, None])
                rows.append((x / scale[None, :, None]).round().clamp(-127, 127) * scale[None, :, None])
                out[side] += rows
    return {side: torch.cat(v) for side, v in out.items()}
