"""The operators around a paged cache of keys and values, as timed cases: what writes it, what reads it, what forks it.

  rope      rotary positions of rows of heads (Rope.apply)
  append    head norms and rotary positions of new tokens, keys and values into their pages (KvCache.append)
  attn      attention of chunks of new tokens over the pages (KvCache.attention)
  select    beam search's choice over beams and vocabulary (beam_select)
  reorder   page tables of the beams that go on, half-filled pages copied (KvCache.reorder)

A pool of pages is one tensor [layers][pages][2: keys, values][kv heads][planes][page][128] of fp16: one plane, or two whose
sum is the value. Head counts, layers and vocabulary are those of `synth.SPECS`. Sequences of a batch have fixed ragged lengths;
the seed gives values, the placement of the pages and beam scores.
"""
import math

import torch

own = False

F16, PAIR = 1, 2
D = 128
VOCAB = 151936
HEADS = {"0.6b": (16, 8, 28), "1.7b": (16, 8, 28), "4b": (32, 8, 36), "32b": (64, 8, 64)}  # query heads, kv heads, layers


def listed():
    return [
        # positions of the queries of a short document; the whole head, pairs half a head apart
        {"name": "rope-1999x16-half", "kind": "rope", "n": 1999, "heads": 16, "dim": 128, "layout": 0, "scaling": 0, "far": 4000},
        # half of every head rotated, neighbouring pairs, positions far behind the trained context
        {"name": "rope-4096x32-interleaved-far", "kind": "rope", "n": 4096, "heads": 32, "dim": 64, "layout": 1, "scaling": 2, "far": 900000},
        # a server's step: one token of each of 64 sequences
        {"name": "append-step-64", "kind": "append", "shape": "4b", "seqs": 64, "q_lo": 1, "q_hi": 1, "len_lo": 40, "len_hi": 4000, "page": 16,
         "scaling": 0},
        # the benchmark's long prompt
        {"name": "append-prompt-2048", "kind": "append", "shape": "32b", "seqs": 1, "q_lo": 2048, "q_hi": 2048, "len_lo": 2048, "len_hi": 2048,
         "page": 64, "scaling": 2},
        # the first words of an answer from the smallest model: latency
        {"name": "attn-one-41", "kind": "attn", "shape": "0.6b", "seqs": 1, "q_lo": 1, "q_hi": 1, "len_lo": 41, "len_hi": 41, "page": 16, "type": PAIR},
        # a server's step over contexts of very different lengths
        {"name": "attn-step-64-f16", "kind": "attn", "shape": "4b", "seqs": 64, "q_lo": 1, "q_hi": 1, "len_lo": 100, "len_hi": 8000, "page": 16,
         "type": F16},
        # one answer behind a very long document: the keys must be cut over the whole GPU
        {"name": "attn-one-100003-pair", "kind": "attn", "shape": "32b", "seqs": 1, "q_lo": 1, "q_hi": 1, "len_lo": 100003, "len_hi": 100003,
         "page": 64, "type": PAIR},
        # next turns of several conversations, ragged
        {"name": "attn-turns-9-pair", "kind": "attn", "shape": "1.7b", "seqs": 9, "q_lo": 3, "q_hi": 77, "len_lo": 203, "len_hi": 4100, "page": 32,
         "type": PAIR},
        # prompts of two users in one pass
        {"name": "attn-prompts-2-f16", "kind": "attn", "shape": "4b", "seqs": 2, "q_lo": 2048, "q_hi": 4096, "len_lo": 2048, "len_hi": 4097, "page": 64,
         "type": F16},
        # a small beam search's step
        {"name": "select-1x4", "kind": "select", "groups": 1, "beams": 4, "k": 8, "vocab": VOCAB, "mask": 0},
        # the beams of a batch, under a grammar
        {"name": "select-16x4-masked", "kind": "select", "groups": 16, "beams": 4, "k": 8, "vocab": VOCAB, "mask": 1},
        # their states
        {"name": "reorder-64-pair", "kind": "reorder", "shape": "4b", "rows": 64, "beams": 4, "len_lo": 30, "len_hi": 200, "page": 32, "type": PAIR,
         "layers": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attn", "attn", "attn", "select", "reorder"])
    shape = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 64, 128])
    if kind == "rope":
        return {"kind": kind, "n": _log_int(rng, 1, 4096), "heads": rng.choice([8, 16, 32]), "dim": rng.choice([32, 64, 96, 128]),
                "layout": rng.choice([0, 1]), "scaling": rng.choice([0, 1, 2, 3]), "far": _log_int(rng, 100, 1000000)}
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 2048 // seqs))
        lo = rng.randint(1, hi)
        return {"kind": kind, "shape": shape, "seqs": seqs, "q_lo": lo, "q_hi": hi, "len_lo": hi, "len_hi": hi + _log_int(rng, 1, 2000), "page": page,
                "scaling": rng.choice([0, 1, 2, 3])}
    if kind == "attn":
        t = rng.choice([F16, PAIR])
        if rng.random() < 0.5:  # a step
            seqs = _log_int(rng, 1, 64)
            hi = _log_int(rng, 1, 100000 // seqs)
            return {"kind": kind, "shape": shape, "seqs": seqs, "q_lo": 1, "q_hi": rng.choice([1, 1, 4]), "len_lo": min(hi, _log_int(rng, 1, 400)),
                    "len_hi": hi, "page": page, "type": t}
        seqs = _log_int(rng, 1, 16)  # chunks
        hi = _log_int(rng, 2, 2048 // seqs)
        lo = rng.randint(1, hi)
        most = min(32000 // seqs, 4000000 // (seqs * hi))
        return {"kind": kind, "shape": shape, "seqs": seqs, "q_lo": lo, "q_hi": hi, "len_lo": hi, "len_hi": max(hi, _log_int(rng, 1, max(2, most))),
                "page": page, "type": t}
    if kind == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return {"kind": kind, "groups": _log_int(rng, 1, 64 // beams), "beams": beams, "k": rng.choice([beams, 2 * beams]),
                "vocab": rng.choice([VOCAB, VOCAB, _log_int(rng, 1000, 200000)]), "mask": rng.choice([0, 0, 1])}
    beams = rng.choice([2, 3, 4, 8])
    return {"kind": kind, "shape": shape, "rows": beams * _log_int(rng, 1, 64 // beams), "beams": beams, "len_lo": 1, "len_hi": _log_int(rng, 2, 300),
            "page": page, "type": rng.choice([F16, PAIR]), "layers": rng.choice([2, 5, 8])}


# ---------------------------------------------------------------- what a program has in hand

def _spread(lo, hi, count, salt):
    """`count` fixed whole numbers between lo and hi, the ends among them when there is room."""
    if count == 1:
        return [hi]
    mid = [lo + (i * 7919 + salt * 104729) % (hi - lo + 1) for i in range(count - 2)]
    return [lo] + mid + [hi]


def _lengths(case):
    """New tokens and cached positions (the new ones included) of every sequence."""
    nq = _spread(case["q_lo"], case["q_hi"], case["seqs"], 1)
    ln = _spread(case["len_lo"], case["len_hi"], case["seqs"], 2)
    return nq, [max(a, b) for a, b in zip(nq, ln)]


def _rope_config(scaling):
    """base and scaling of the positions; the factors are the usual ones of a context four times the trained one."""
    return {"base": 1e6, "scaling": scaling, "factor": 4.0, "orig_ctx": 32768.0, "beta_fast": 32.0, "beta_slow": 1.0, "attn_factor": 0.0,
            "low_freq": 1.0, "high_freq": 4.0}


def _frequencies(dim, c):
    """Angle per position of every pair, and the factor on the rotated values (64 bits)."""
    freq, mscale = [], 1.0
    if c["scaling"] == 2:
        mscale = c["attn_factor"] or 0.1 * math.log(c["factor"]) + 1.0
        turns = lambda beta: dim * math.log(c["orig_ctx"] / (2 * math.pi * beta)) / (2 * math.log(c["base"]))
        low, high = max(math.floor(turns(c["beta_fast"])), 0), min(math.ceil(turns(c["beta_slow"])), dim - 1)
        high = high + 0.001 if high == low else high
    for i in range(dim // 2):
        f = c["base"] ** (-2.0 * i / dim)
        if c["scaling"] == 1:
            f /= c["factor"]
        elif c["scaling"] == 2:
            r = min(max((i - low) / (high - low), 0.0), 1.0)
            f = f / c["factor"] * r + f * (1 - r)
        elif c["scaling"] == 3:
            turned = c["orig_ctx"] * f / (2 * math.pi)  # full turns within the trained context
            if turned < c["low_freq"]:
                f /= c["factor"]
            elif turned <= c["high_freq"]:
                r = (turned - c["low_freq"]) / (c["high_freq"] - c["low_freq"])
                f = (1 - r) * f / c["factor"] + r * f
        freq.append(f)
    return freq, mscale


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _pages_of(lens, page):
    return [(n + page - 1) // page for n in lens]


def _fill_pool(gen, layers, pages, hkv, planes, page, layer=None):
    """A pool with values of both signs, of the spread that normed keys and values have, in one layer or in all."""
    pool = torch.zeros((layers, pages, 2, hkv, planes, page, D), dtype=torch.half, device="cuda")
    for i in range(layers) if layer is None else [layer]:
        x = torch.randn((pages, 2, hkv, page, D), generator=gen, device="cuda")
        pool[i, :, :, :, 0] = x.half()
        if planes == 2:
            pool[i, :, :, :, 1] = (x - x.half().float()).half()
    return pool


def _tables(gen, counts, pages, width):
    """Page tables with the pages of the pool in random order; unused entries are -1."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((len(counts), width), -1, dtype=torch.int32), 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    return table.cuda(), order[at:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    st = {"case": case}
    if own:
        import exactinfer_b200 as e
    if kind == "rope":
        n, width = case["n"], case["heads"] * D
        st["x"] = torch.randn((n, width), generator=gen, device="cuda")
        st["pos"] = torch.randint(0, case["far"], (n,), generator=gen, device="cuda", dtype=torch.int32)
        st["y"] = torch.empty_like(st["x"])
        st["cfg"] = _rope_config(case["scaling"])
        if own:
            st["rope"] = e.Rope(D, dim=case["dim"], layout=case["layout"], **st["cfg"])
        return st
    if kind in ("append", "attn"):
        h, hkv, _ = HEADS[case["shape"]]
        planes = case.get("type", F16)
        nq, lens = _lengths(case)
        counts = _pages_of(lens, case["page"])
        pages, width = sum(counts) + 3, max(counts)
        st["nq"], st["lens"] = nq, lens
        st["table"], _ = _tables(gen, counts, pages, width)
        start = [0]
        for a in nq:
            start.append(start[-1] + a)
        st["start"] = start
        st["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        st["len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        n = start[-1]
        if kind == "append":  # rows q|k|v as a joint projection leaves them
            st["qkv"] = torch.randn((n, (h + 2 * hkv) * D), generator=gen, device="cuda")
            st["pool"] = torch.zeros((2, pages, 2, hkv, planes, case["page"], D), dtype=torch.half, device="cuda")
            st["q_norm"] = torch.randn(D, generator=gen, device="cuda").mul_(0.01).add_(1)
            st["k_norm"] = torch.randn(D, generator=gen, device="cuda").mul_(0.01).add_(1)
            st["cfg"] = _rope_config(case["scaling"])
            st["q_out"] = torch.empty((n, h * D), device="cuda")
        else:
            st["pool"] = _fill_pool(gen, 2, pages, hkv, planes, case["page"], layer=1)
            st["q"] = torch.randn((n, h * D), generator=gen, device="cuda")
            st["out"] = torch.empty((n, h * D), device="cuda")
        if own:
            st["kv"] = e.KvCache(2, hkv, case["page"], pages, planes, mem=st["pool"])
            st["batch"] = e.KvBatch(len(lens), n, max(nq), max(lens), st["q_start"], st["len"], st["table"], width)
            if kind == "append":
                st["rope"] = e.Rope(D, **st["cfg"])
            else:
                st["work"] = torch.empty(st["kv"].attention_work(st["batch"], h), dtype=torch.uint8, device="cuda")
        return st
    if kind == "select":
        rows, v, k = case["groups"] * case["beams"], case["vocab"], case["k"]
        st["logits"] = torch.randn((rows, v), generator=gen, device="cuda").mul_(3)
        st["scores"] = torch.randn(rows, generator=gen, device="cuda", dtype=torch.float64).mul_(2).sub_(20)
        if case["mask"]:
            words = torch.randint(-2**31, 2**31, (rows, (v + 31) // 32), generator=gen, device="cuda").to(torch.int32)
            st["allowed"] = words
        st["parent"], st["token"] = (torch.empty((case["groups"], k), dtype=torch.int32, device="cuda") for _ in range(2))
        st["score"] = torch.empty((case["groups"], k), dtype=torch.float64, device="cuda")
        if own:
            st["work"] = torch.empty(e.beam_select_work(v, case["groups"], case["beams"], k), dtype=torch.uint8, device="cuda")
        return st
    _, hkv, _ = HEADS[case["shape"]]
    rows, page, planes = case["rows"], case["page"], case["type"]
    lens = [n for g in _spread(case["len_lo"], case["len_hi"], rows // case["beams"], 3) for n in [g] * case["beams"]]
    counts = _pages_of(lens, page)
    pages, width = sum(counts) + rows, max(counts) + 1
    st["pool"] = _fill_pool(gen, case["layers"], pages, hkv, planes, page)
    st["table"], rest = _tables(gen, counts, pages, width)
    st["lens"] = lens
    st["len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["spare"] = rest[:rows].clone().cuda()
    base = torch.arange(rows, device="cuda", dtype=torch.int32) // case["beams"] * case["beams"]
    st["parent"] = base + torch.randint(0, case["beams"], (rows,), generator=gen, device="cuda", dtype=torch.int32)
    st["table_out"], st["len_out"], st["taken"] = torch.empty_like(st["table"]), torch.empty_like(st["len"]), torch.empty_like(st["len"])
    if own:
        st["kv"] = e.KvCache(case["layers"], hkv, page, pages, planes, mem=st["pool"])
    return st


# ---------------------------------------------------------------- plain forms

def _rotate(x, pos, dim, layout, cfg, work=torch.float32):
    """x[n][heads][D] at positions pos[n]; angles in 64 bits."""
    freq, mscale = _frequencies(dim, cfg)
    a = pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = (a.cos() * mscale).to(work)[:, None], (a.sin() * mscale).to(work)[:, None]
    y = x.clone()
    first, second = (slice(0, dim // 2), slice(dim // 2, dim)) if layout == 0 else (slice(0, dim, 2), slice(1, dim, 2))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    return y


def _head_norm(x, w, eps):
    return x * torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + eps).to(x.dtype) * w.to(x.dtype)


def _positions(st):
    """Sequence and position of every new token."""
    seq = torch.repeat_interleave(torch.arange(len(st["nq"]), device="cuda"), torch.tensor(st["nq"], device="cuda"))
    first = torch.tensor([n - a - b for n, a, b in zip(st["lens"], st["nq"], st["start"])], device="cuda")
    return seq, torch.arange(seq.numel(), device="cuda") + first[seq]


def _append_plain(st):
    case = st["case"]
    h, hkv, _ = HEADS[case["shape"]]
    qkv = st["qkv"].view(-1, h + 2 * hkv, D)
    seq, pos = _positions(st)
    turn = lambda x, w: _rotate(_head_norm(x, w, 1e-6), pos, D, 0, st["cfg"])
    q, k, v = turn(qkv[:, :h], st["q_norm"]), turn(qkv[:, h:h + hkv], st["k_norm"]), qkv[:, h + hkv:]
    page = st["table"][seq, pos // case["page"]].long()
    st["pool"][1, page, 0, :, 0, pos % case["page"]] = k.half()
    st["pool"][1, page, 1, :, 0, pos % case["page"]] = v.half()
    return q.reshape(st["q_out"].shape)


def _sequence(st, s, work):
    """Keys and values of a sequence, [2][kv heads][len][D]."""
    pages = st["table"][s, :(st["lens"][s] + st["case"]["page"] - 1) // st["case"]["page"]].long()
    x = st["pool"][1, pages].to(work).sum(3)  # [pages][2][kv heads][page][D]
    return x.permute(1, 2, 0, 3, 4).reshape(2, x.shape[2], -1, D)[:, :, :st["lens"][s]]


def _attention_plain(st):
    h, hkv, _ = HEADS[st["case"]["shape"]]
    out = torch.empty_like(st["out"])
    for s, (nq, n) in enumerate(zip(st["nq"], st["lens"])):
        rows = slice(st["start"][s], st["start"][s] + nq)
        kv = _sequence(st, s, torch.float32)
        hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - nq, n, device="cuda")[:, None]
        q = st["q"][rows].view(nq, hkv, h // hkv, D)
        o = out[rows].view(nq, hkv, h // hkv, D)
        for j in range(hkv):
            x = torch.matmul(q[:, j].transpose(0, 1), kv[0, j].T) * (1.0 / math.sqrt(D))  # [group][nq][n]
            x.masked_fill_(hidden, -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o[:, j] = (torch.matmul(x, kv[1, j]) / x.sum(-1, keepdim=True)).transpose(0, 1)
    return out


def _select_plain(st):
    case = st["case"]
    v, k, beams = case["vocab"], case["k"], case["beams"]
    x = st["logits"].double()
    m = x.amax(-1, keepdim=True)
    lse = m + (x - m).exp().sum(-1, keepdim=True).log()
    if case["mask"]:
        bits = st["allowed"][:, torch.arange(v, device="cuda") // 32] >> (torch.arange(v, device="cuda") % 32) & 1
        x = x.masked_fill(bits == 0, -math.inf)
    best, ids = torch.sort(x, dim=-1, descending=True, stable=True)  # (logit, token) within a beam
    best, ids = best[:, :k], ids[:, :k]
    score = (st["scores"][:, None] + (best - lse)).reshape(case["groups"], -1)
    score, at = torch.sort(score, dim=-1, descending=True, stable=True)  # then (score, beam)
    score, at = score[:, :k], at[:, :k]
    parent = at // best.shape[1] + torch.arange(case["groups"], device="cuda")[:, None] * beams
    return parent.to(torch.int32), ids.reshape(case["groups"], -1).gather(1, at).to(torch.int32), score


def _reorder_plain(st):
    page, rows = st["case"]["page"], st["parent"].numel()
    parent = st["parent"].long()
    index = torch.arange(rows, device="cuda")
    first = (parent[:, None] == parent[None, :]).long().argmax(1) == index  # the first row that goes on from this parent
    table, length = st["table"][parent], st["len"][parent]
    width = torch.arange(table.shape[1], device="cuda")[None, :]
    table = torch.where(width < ((length + page - 1) // page)[:, None], table, -1)
    copy = ~first & (length % page != 0)
    r = index[copy]
    last = (length[copy] // page).long()
    st["pool"][:, st["spare"][r].long()] = st["pool"][:, table[r, last].long()]
    table[r, last] = st["spare"][r]
    return table, length, copy.to(torch.int32)


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "rope":
        if not own:
            n = case["n"]
            return _rotate(st["x"].view(n, case["heads"], D), st["pos"], case["dim"], case["layout"], st["cfg"]).view(n, -1)
        st["rope"].apply(st["x"], st["pos"], st["y"], case["n"], case["heads"], stream=_stream())
        return st["y"]
    if kind == "append":
        if not own:
            return _append_plain(st), st["pool"][1]
        h, hkv, _ = HEADS[case["shape"]]
        ld = (h + 2 * hkv) * D
        q = st["qkv"].data_ptr()
        st["kv"].append(1, st["batch"], q + 4 * h * D, q + 4 * (h + hkv) * D, ld, ld, rope=st["rope"], k_norm=st["k_norm"], eps=1e-6, q=q, ldq=ld,
                        n_head=h, q_norm=st["q_norm"], q_out=st["q_out"], ldqo=h * D, stream=_stream())
        return st["q_out"], st["pool"][1]
    if kind == "attn":
        if not own:
            return _attention_plain(st)
        h = HEADS[case["shape"]][0]
        st["kv"].attention(1, st["batch"], st["q"], st["out"], h, 1.0 / math.sqrt(D), st["work"], st["work"].numel(), stream=_stream())
        return st["out"]
    if kind == "select":
        if not own:
            return _select_plain(st)
        from exactinfer_b200 import beam_select
        beam_select(st["logits"], case["vocab"], case["groups"], case["beams"], st["scores"], case["k"], st["parent"], st["token"], st["score"],
                    st["work"], st["work"].numel(), allowed=st.get("allowed"), allowed_ld=(case["vocab"] + 31) // 32 if case["mask"] else 0,
                    stream=_stream())
        return st["parent"], st["token"], st["score"]
    if not own:
        return (*_reorder_plain(st), st["pool"])
    st["kv"].reorder(case["rows"], st["parent"], st["len"], st["table"], st["table"].shape[1], st["spare"], st["len_out"], st["table_out"],
                     st["taken"], stream=_stream())
    return st["table_out"], st["len_out"], st["taken"], st["pool"]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "rope":
        values = case["n"] * case["heads"] * D
        return {"bytes": 8 * values + 4 * case["n"], "flops": 3 * case["n"] * case["heads"] * case["dim"]}
    if kind in ("append", "attn"):
        h, hkv, _ = HEADS[case["shape"]]
        nq, lens = _lengths(case)
        n = sum(nq)
        if kind == "append":
            return {"bytes": n * D * (8 * h + 2 * hkv * (4 + 2)) + 4 * n, "flops": n * D * (7 * (h + hkv) + hkv)}
        seen = sum(a * (m - a) + a * (a + 1) // 2 for a, m in zip(nq, lens))
        return {"bytes": sum(lens) * hkv * D * 4 * case["type"] + 8 * n * h * D, "flops": 4 * D * h * seen}
    if kind == "select":
        rows, v = case["groups"] * case["beams"], case["vocab"]
        return {"bytes": rows * (4 * v + 8) + (rows * ((v + 31) // 32) * 4 if case["mask"] else 0) + 16 * case["groups"] * case["k"], "flops": 2 * rows * v}
    _, hkv, _ = HEADS[case["shape"]]
    lens = _spread(case["len_lo"], case["len_hi"], case["rows"] // case["beams"], 3)
    # of `beams` rows with random parents, beams (1 - 1/beams)^beams parents have no child: as many pages are copied
    copies = sum(case["beams"] * (1 - 1 / case["beams"]) ** case["beams"] for n in lens if n % case["page"])
    page = 2 * hkv * case["type"] * case["page"] * D * 2
    width = (max(lens) + case["page"] - 1) // case["page"] + 1
    return {"bytes": int(2 * copies * case["layers"] * page) + 8 * case["rows"] * (width + 2), "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    if case["kind"] == "reorder":
        return None  # whole numbers and copies
    st = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "rope":
        return _turned(st["x"].to(f64).view(case["n"], case["heads"], D), st["pos"], case["dim"], case["layout"], st["cfg"]).reshape(st["x"].shape)
    if case["kind"] == "append":
        h, hkv, _ = HEADS[case["shape"]]
        x = st["qkv"].to(f64).view(-1, h + 2 * hkv, D)
        x[:, :h + hkv] /= (x[:, :h + hkv].square().sum(-1, keepdim=True) / D + 1e-6).sqrt()
        x[:, :h] *= st["q_norm"].to(f64)
        x[:, h:h + hkv] *= st["k_norm"].to(f64)
        pos = torch.cat([torch.arange(n - a, n) for a, n in zip(st["nq"], st["lens"])]).cuda()
        x[:, :h + hkv] = _turned(x[:, :h + hkv], pos, D, 0, st["cfg"])
        pool = st["pool"][1].to(f64)
        table, row = st["table"].tolist(), 0
        for s, (a, n) in enumerate(zip(st["nq"], st["lens"])):
            p = n - a
            while p < n:  # page by page
                m = min(case["page"] - p % case["page"], n - p)
                for which, head in ((0, h), (1, h + hkv)):
                    pool[table[s][p // case["page"]], which, :, 0, p % case["page"]:p % case["page"] + m] = x[row:row + m, head:head + hkv].transpose(0, 1)
                p, row = p + m, row + m
        return x[:, :h].reshape(st["q_out"].shape), pool
    if case["kind"] == "select":
        k = case["k"]
        logp = (st["logits"].to(f64) - st["logits"].to(f64).logsumexp(-1, keepdim=True)) + st["scores"][:, None]
        if case["mask"]:
            on = torch.stack([(st["allowed"] >> b) & 1 for b in range(32)], -1).flatten(1)[:, :case["vocab"]]
            logp[on == 0] = -math.inf
        return None, None, logp.view(case["groups"], -1).topk(k).values
    if work(case)["flops"] > 4e12:
        return None
    h, hkv, _ = HEADS[case["shape"]]
    out = []
    for s, (a, n) in enumerate(zip(st["nq"], st["lens"])):
        x = st["pool"][1, st["table"][s, :-(-n // case["page"])].long()].to(f64)
        x = x.sum(3).transpose(1, 2)  # [pages][kv heads][2][page][D]
        k = torch.cat(list(x[:, :, 0].unbind(0)), 1)[:, :n]
        v = torch.cat(list(x[:, :, 1].unbind(0)), 1)[:, :n]
        q = st["q"][st["start"][s]:st["start"][s] + a].to(f64).view(a, h, D)
        for lo in range(0, a, 256):  # rows at a time
            part = q[lo:lo + 256]
            last = torch.arange(n - a + lo, n - a + lo + part.shape[0], device="cuda")
            see = torch.arange(n, device="cuda")[None, :] <= last[:, None]
            heads = []
            for i in range(h):
                w = (part[:, i] @ k[i // (h // hkv)].T) / math.sqrt(D)
                w = torch.where(see, w, -math.inf).softmax(-1)
                heads.append(w @ v[i // (h // hkv)])
            out.append(torch.cat(heads, 1))
    return torch.cat(out)


def _turned(x, pos, dim, layout, cfg):
    """The rotation as a product of complex numbers."""
    freq, mscale = _frequencies(dim, cfg)
    a = pos.to(torch.float64)[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    head = x[..., :dim]
    pairs = head.unflatten(-1, (dim // 2, 2)) if layout else head.unflatten(-1, (2, dim // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(a, mscale), a)
    z = torch.view_as_real(z)
    z = z.flatten(-2) if layout else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., dim:]], -1)
