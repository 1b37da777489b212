"""What the operators for several hypotheses of one prompt are measured on.

Five operators that n-best decoding, rescoring and many sessions behind one text
prompt are made of: the pages of a KV cache forked to new hypotheses (with room
for their next rows, copies of last pages that are no longer common, and what
nobody holds set free) and compacted, the write of K and V into pages, the
attention over them with a prefix that the members of a group share, and the log
probabilities of given tokens with entropy and top alternatives.

Sizes are those of this repository's decoders (16 query heads and 8 KV heads of
128, 28 layers, a vocabulary of 151936) and of its workloads: prompts of 404 rows
(30 s of audio), 1337 rows (a long recording), 32 streams, heads of other widths.

`own` false: plain forms in elementary torch operations.  `own` true: the calls
of `qwenasr_amd.kernels`, on torch tensors (a program may hold its buffers in any
device allocation).

A pool is pages [n_pages][heads][page][dim] in bf16; K and V of every layer are a
pool each, one behind another in one allocation.  table[j][s] is the page that
holds positions s * page .. of sequence j.
"""
import functools
import math

import torch

own = False


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # eight hypotheses of one 30 s prompt go on from three of them: the step between two tokens, every layer's pools
        {"name": "fork_8", "kind": "fork", "groups": 1, "beams": 8, "shared": 404, "past": 30, "rows": 1, "page": 64,
         "heads": 8, "dim": 128, "pools": 56},
        # 32 recordings with four hypotheses each, small pages
        {"name": "fork_32x4", "kind": "fork", "groups": 32, "beams": 4, "shared": 600, "past": 200, "rows": 1, "page": 16,
         "heads": 8, "dim": 128, "pools": 56},
        # sessions that have ended left holes: a small pool drawn together
        {"name": "compact_32", "kind": "compact", "seqs": 32, "past": 200, "live": 0.5, "page": 16, "heads": 8, "dim": 128,
         "pools": 56},
        # the same of a large pool of long recordings
        {"name": "compact_64x900", "kind": "compact", "seqs": 64, "past": 900, "live": 0.5, "page": 64, "heads": 8, "dim": 128,
         "pools": 56},
        # one new position of each of 32 streams: latency
        {"name": "write_step_32", "kind": "write", "seqs": 32, "rows": 1, "ragged": False, "past": 1000, "page": 64,
         "heads": 8, "dim": 128, "bf16": False},
        # ragged prompts of eight sessions behind what they hold
        {"name": "write_8_prompts_bf16", "kind": "write", "seqs": 8, "rows": 1337, "ragged": True, "past": 300, "page": 16,
         "heads": 8, "dim": 128, "bf16": True},
        # the token of eight hypotheses of one 30 s prompt: the smallest attention
        {"name": "attn_8_hypotheses", "kind": "attn", "groups": 1, "beams": 8, "shared": 384, "past": 50, "rows": 1,
         "ragged": False, "page": 64, "heads": 8, "ratio": 2, "dim": 128, "bf16": False},
        # four long text prompts, sixteen sessions behind each
        {"name": "attn_4x16_shared_4000_bf16", "kind": "attn", "groups": 4, "beams": 16, "shared": 4000, "past": 300, "rows": 1,
         "ragged": False, "page": 16, "heads": 8, "ratio": 2, "dim": 128, "bf16": True},
        # one token of each of 32 streams that share nothing, sessions of different age
        {"name": "attn_32x4000_bf16", "kind": "attn", "groups": 32, "beams": 1, "shared": 0, "past": 4000, "rows": 1,
         "ragged": False, "page": 64, "heads": 8, "ratio": 2, "dim": 128, "bf16": True},
        # the prompts of six long recordings behind one text prompt
        {"name": "attn_6_prompts_1337", "kind": "attn", "groups": 1, "beams": 6, "shared": 512, "past": 0, "rows": 1337,
         "ragged": True, "page": 64, "heads": 8, "ratio": 2, "dim": 128, "bf16": False},
        # the candidates of eight hypotheses' next token, whole vocabulary
        {"name": "score_8x151936", "kind": "score", "rows": 8, "cols": 151936, "pad": 0, "k": 16, "bf16": False},
        # the confidence of every token of a 30 s prompt's rows
        {"name": "score_375x151936", "kind": "score", "rows": 375, "cols": 151936, "pad": 0, "k": 5, "bf16": False},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["fork", "compact", "write", "attn", "attn", "attn", "score", "score"])
    heads, dim, page = rng.choice([8, 8, 4, 14]), rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128, 256])
    bf16 = rng.random() < 0.5
    if kind == "fork":
        groups, pools = _log(rng, 1, 32), rng.choice([2, 8, 32])
        beams = _log(rng, 1, max(1, 128 // groups))
        return {"kind": kind, "groups": groups, "beams": beams, "shared": _log(rng, 20, 600), "past": _log(rng, 1, 200),
                "rows": rng.choice([1, 1, rng.randint(2, 20)]), "page": min(page, 128), "heads": min(heads, 8), "dim": dim, "pools": pools}
    if kind == "compact":
        return {"kind": kind, "seqs": _log(rng, 2, 64), "past": _log(rng, 16, 600), "live": round(rng.uniform(0.2, 0.9), 2),
                "page": min(page, 64), "heads": min(heads, 8), "dim": dim, "pools": rng.choice([2, 8, 32])}
    if kind == "write":
        seqs = _log(rng, 1, 32)
        return {"kind": kind, "seqs": seqs, "rows": rng.choice([1, _log(rng, 2, max(2, 4 * 1337 // seqs))]),
                "ragged": rng.random() < 0.5, "past": _log(rng, 1, 1500), "page": page, "heads": min(heads, 8), "dim": dim,
                "bf16": bf16}
    if kind == "score":
        cols = _log(rng, 50, 151936)
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(4000, 375 * 151936 // cols))), "cols": cols,
                "pad": rng.choice([0, 0, 8, 3]), "k": min(cols, rng.choice([1, 5, _log(rng, 1, 32)])), "bf16": bf16}
    heads, ratio = min(heads, 8), rng.choice([2, 2, 1, 3, 4])
    c = {"kind": kind, "page": page, "heads": heads, "ratio": ratio, "dim": dim, "bf16": bf16, "ragged": rng.random() < 0.3}
    if rng.random() < 0.75:
        c["groups"] = _log(rng, 1, 8)
        c["beams"] = _log(rng, 1, 64 // c["groups"])
        c["rows"] = rng.choice([1, 1, 1, rng.randint(2, 6)])
        n = c["groups"] * c["beams"] * c["rows"]
        c["shared"] = rng.choice([0, _log(rng, 16, max(16, min(8000, 100000 // n)))])
        c["past"] = _log(rng, 1, max(1, min(8000, 60000 // n)))
    else:
        c["rows"] = _log(rng, 9, 1337)
        c["groups"], c["beams"] = 1, rng.randint(1, max(1, min(6, 4000 // (c["rows"] * ratio))))
        c["shared"] = rng.choice([0, _log(rng, 16, 600)])
        c["past"] = rng.choice([0, _log(rng, 1, 600)])
    return c


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------

class _Buf:
    """A torch tensor as an argument of the operators."""
    __slots__ = ("t", "ptr", "shape")

    def __init__(self, t):
        self.t, self.ptr, self.shape = t, t.data_ptr(), tuple(t.shape)

    @property
    def dev(self):
        return _device()


@functools.lru_cache(maxsize=None)
def _device():
    from qwenasr_amd import Device
    return Device(0)


class _Rng:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator("cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype) * std

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _type(c):
    return torch.bfloat16 if c["bf16"] else torch.float32


def _prefix(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _some(n, key):
    """n numbers in [0, 1) that go with `key` alone."""
    g = torch.Generator()
    g.manual_seed(key)
    return torch.rand(n, generator=g).tolist()


def _turned(v, seed):
    t = seed % len(v)
    return v[t:] + v[:t]


def _pages(n, page):
    return (n + page - 1) // page


def _tables(r, lengths, shared, beams, page, spare, width):
    """(table, n_pages): a random page for every position in use; the members of a group (`beams` sequences that follow
    one another) name the same pages for the whole pages of their first shared positions."""
    n = len(lengths)
    need = [_pages(m, page) for m in lengths]
    whole = [shared[j // beams] // page for j in range(n)]
    first = [j // beams * beams for j in range(n)]
    count, table = 0, []
    for j in range(n):
        common = min(whole[j], need[j], need[first[j]]) if j != first[j] else 0
        row = table[first[j]][:common] if common else []
        row = row + list(range(count, count + need[j] - len(row)))
        count = max(count, (row[-1] + 1) if row else 0)
        table.append(row)
    n_pages = count + spare
    flat = torch.full((n, width), -1, dtype=torch.int64)
    for j, row in enumerate(table):
        flat[j, :len(row)] = torch.tensor(row, dtype=torch.int64)
    flat = flat.cuda()
    return torch.where(flat >= 0, r.order(n_pages)[flat.clamp(min=0)], -1).int().contiguous(), n_pages


def _pool(c, r, n_pages, *first):
    return r.normal(*first, n_pages, c["heads"], c["page"], c["dim"], dtype=torch.bfloat16)


def _fork_plan(c, seed):
    n = c["groups"] * c["beams"]
    own_part = [1 + int(c["past"] * (0.5 + 0.5 * x)) for x in _some(n, 11 * n + c["past"])]
    shared = [max(1, int(c["shared"] * (0.7 + 0.3 * x))) for x in _some(c["groups"], 13 * c["groups"] + c["shared"])]
    shared, own_part = _turned(shared, seed), _turned(own_part, seed % c["groups"] * c["beams"])
    return [shared[j // c["beams"]] + own_part[j] for j in range(n)], shared


def _fork_inputs(c, seed):
    r, page, beams = _Rng(seed), c["page"], c["beams"]
    n = c["groups"] * beams
    lengths, shared = _fork_plan(c, seed)
    width = _pages(max(lengths) + c["rows"], page) + 2
    # room for every hypothesis' next rows and copied page
    table, n_pages = _tables(r, lengths, shared, beams, page, n * (2 + c["rows"] // page), width)
    # the hypotheses that live on: a few of each group, most of them more than once
    g = torch.Generator()
    g.manual_seed(seed)
    parent = torch.randint(0, max(1, (beams + 1) // 2), (c["groups"], beams), generator=g) + torch.arange(c["groups"])[:, None] * beams
    d = {"table": table, "len": _int32(lengths), "parent": parent.reshape(-1).int().cuda(), "pool": _pool(c, r, n_pages, c["pools"])}
    return d, {"n": n, "width": width, "n_pages": n_pages}


def _compact_inputs(c, seed):
    r, page = _Rng(seed), c["page"]
    lengths = [1 + int(c["past"] * (0.3 + 0.7 * x)) for x in _some(c["seqs"], 17 * c["seqs"] + c["past"])]
    width = _pages(max(lengths), page) + 1
    table, n_pages = _tables(r, lengths, [0] * c["seqs"], 1, page, 4, width)
    gone = [x >= c["live"] for x in _some(c["seqs"], 19 * c["seqs"] + c["past"])]
    gone[0] = False
    lengths = [0 if e else m for e, m in zip(gone, lengths)]
    d = {"table": table, "len": _int32(lengths), "pool": _pool(c, r, n_pages, c["pools"])}
    return d, {"n": c["seqs"], "width": width, "n_pages": n_pages}


def _lengths(c, seed, n):
    rows = [c["rows"]] * n
    if c["ragged"]:
        rows = [c["rows"]] + [max(1, int(c["rows"] * x)) for x in _some(n - 1, n + 64 * c["rows"])]
    past = [c["past"]] + [int(c["past"] * (0.5 + 0.5 * x)) for x in _some(n - 1, n + 100003 * c["past"])]
    return _turned(rows, seed), _turned(past, seed)


def _write_inputs(c, seed):
    r, t, n, hd = _Rng(seed), _type(c), c["seqs"], c["heads"] * c["dim"]
    rows, past = _lengths(c, seed, n)
    width = _pages(max(a + b for a, b in zip(rows, past)), c["page"])
    table, n_pages = _tables(r, [a + b for a, b in zip(rows, past)], [0] * n, 1, c["page"], 2, width)
    total = sum(rows)
    # k and v inside the fused projection's rows
    kv = torch.cat([r.normal(total, hd), r.normal(total, hd, std=0.6)], 1).to(t)
    d = {"table": table, "kv": kv, "row_start": _int32(_prefix(rows)), "pos": _int32(past),
         "k_pages": _pool(c, r, n_pages), "v_pages": _pool(c, r, n_pages)}
    return d, {"n": n, "width": width, "n_pages": n_pages, "total": total, "most": max(rows)}


def _attn_inputs(c, seed):
    r, t, n, page = _Rng(seed), _type(c), c["groups"] * c["beams"], c["page"]
    rows, past = _lengths(c, seed, n)
    shared = [max(0, int(c["shared"] * (0.75 + 0.25 * x))) for x in _some(c["groups"], 23 * c["groups"] + c["shared"])]
    shared[0] = c["shared"]
    shared = _turned(shared, seed)
    past = [p + shared[j // c["beams"]] for j, p in enumerate(past)]
    width = _pages(max(a + b for a, b in zip(rows, past)), page)
    table, n_pages = _tables(r, [a + b for a, b in zip(rows, past)], shared, c["beams"], page, 2, width)
    total = sum(rows)
    d = {"table": table, "k_pages": _pool(c, r, n_pages), "v_pages": _pool(c, r, n_pages).mul_(0.6),
         "q": r.normal(total, c["heads"] * c["ratio"], c["dim"]).to(t), "row_start": _int32(_prefix(rows)), "pos": _int32(past),
         "shared": _int32(shared)}
    # a shared prefix that ends inside a page: every member holds a copy of that part
    for j in range(n):
        s, first = shared[j // c["beams"]], j // c["beams"] * c["beams"]
        if s % page and j != first:
            at = torch.stack([table[j, s // page], table[first, s // page]]).long()
            for pool in (d["k_pages"], d["v_pages"]):
                pool[at[0], :, :s % page] = pool[at[1], :, :s % page]
    return d, {"n": n, "width": width, "n_pages": n_pages, "total": total, "most": max(rows),
               "longest": max(a + b for a, b in zip(rows, past)),
               "alone": max(a + b - shared[j // c["beams"]] for j, (a, b) in enumerate(zip(rows, past)))}


def _score_inputs(c, seed):
    r, rows, cols = _Rng(seed), c["rows"], c["cols"]
    x = r.normal(rows, cols + c["pad"], std=2.0)
    # most rows are sure of their token, some are not; the given token is the likeliest of most rows
    at = torch.randint(0, cols, (2, rows), generator=r.g, device="cuda")
    sure = 24.0 * torch.rand(rows, generator=r.g, device="cuda") - 2.0
    x[torch.arange(rows, device="cuda"), at[0]] += sure
    given = torch.where(torch.rand(rows, generator=r.g, device="cuda") < 0.8, at[0], at[1])
    return {"logits": x.to(_type(c)), "targets": given.int()}


def _empty(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    c, kind = case, case["kind"]
    s = {"case": c, "kind": kind}
    if kind == "fork":
        d, s["at"] = _fork_inputs(c, seed)
        n = s["at"]["n"]
        d.update(table_out=_empty(n, s["at"]["width"], dtype=torch.int32), pos_out=_empty(n, dtype=torch.int32),
                 len_out=_empty(n, dtype=torch.int32), status=_empty(2, dtype=torch.int32))
    elif kind == "compact":
        d, s["at"] = _compact_inputs(c, seed)
        d.update(table_out=_empty(s["at"]["n"], s["at"]["width"], dtype=torch.int32), status=_empty(2, dtype=torch.int32))
    elif kind == "write":
        d, s["at"] = _write_inputs(c, seed)
        s["v_rows"] = _Buf(d["kv"][:, c["heads"] * c["dim"]:])
    elif kind == "attn":
        d, s["at"] = _attn_inputs(c, seed)
        d["out"] = torch.zeros_like(d["q"])
    elif kind == "score":
        d = _score_inputs(c, seed)
        d.update(logp=_empty(c["rows"]), entropy=_empty(c["rows"]), ids=_empty(c["rows"], c["k"], dtype=torch.int32),
                 top=_empty(c["rows"], c["k"]))
    else:
        raise ValueError(kind)
    s.update({n: _Buf(t) for n, t in d.items()})
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _run_own(s):
    from qwenasr_amd import kernels as K
    c, kind, at = s["case"], s["kind"], s.get("at")
    if kind == "fork":
        K.kvp_fork(s["table_out"], s["pos_out"], s["len_out"], s["status"], s["table"], s["len"], at["n"], at["n"], at["width"],
                   s["pool"], c["pools"], at["n_pages"], c["heads"], c["page"], 2 * c["dim"], parent=s["parent"],
                   max_rows=c["rows"])
        return {"table": s["table_out"].t, "pos": s["pos_out"].t, "len": s["len_out"].t, "status": s["status"].t, "pool": s["pool"].t}
    if kind == "compact":
        K.kvp_compact(s["table_out"], s["status"], s["table"], s["len"], at["n"], at["width"], s["pool"], c["pools"],
                      at["n_pages"], c["heads"], c["page"], 2 * c["dim"])
        return {"table": s["table_out"].t, "status": s["status"].t, "pool": s["pool"].t}
    if kind == "write":
        K.kvp_write(s["k_pages"], s["v_pages"], at["n_pages"], s["kv"], s["v_rows"], s["table"], at["width"], s["pos"],
                    at["total"], at["n"], at["most"], c["heads"], c["dim"], c["page"], row_start=s["row_start"],
                    ld=2 * c["heads"] * c["dim"], bf16=c["bf16"])
        return {"k": s["k_pages"].t, "v": s["v_pages"].t}
    if kind == "attn":
        K.attention_kvp(s["out"], s["q"], s["k_pages"], s["v_pages"], at["n_pages"], s["table"], at["width"], s["pos"],
                        at["total"], at["n"], at["most"], c["heads"] * c["ratio"], c["heads"], c["dim"], c["page"],
                        c["dim"] ** -0.5, row_start=s["row_start"], max_len=at["longest"], group=c["beams"],
                        shared=s["shared"] if c["beams"] > 1 else None, max_own=at["alone"], bf16=c["bf16"])
        return s["out"].t
    K.token_logprobs(s["logits"], c["rows"], c["cols"], ld=c["cols"] + c["pad"], targets=s["targets"], logp=s["logp"],
                     entropy=s["entropy"], top_ids=s["ids"], top_logp=s["top"], k=c["k"], bf16=c["bf16"])
    return {"logp": s["logp"].t, "entropy": s["entropy"].t, "ids": s["ids"].t, "top": s["top"].t}


def _named(ids, flags, n_pages):
    """Truth values of the pages: whether an entry of `ids` whose flag is set names one."""
    hit = torch.zeros(n_pages + 1, dtype=torch.bool, device="cuda")
    hit[torch.where(flags, ids, n_pages).reshape(-1)] = True
    return hit[:n_pages]


def _plain_fork(s, c):
    n, width, n_pages, page = s["at"]["n"], s["at"]["width"], s["at"]["n_pages"], c["page"]
    parent = s["parent"].t.long()
    length = s["len"].t.long()[parent]
    ids = s["table"].t.long()[parent]                                       # [n, width]
    slot = torch.arange(width, device="cuda")
    held = (length + page - 1) // page
    live = slot < held[:, None]
    fill = length % page
    last = (slot == held[:, None] - 1) & (fill > 0)[:, None]                # a last page with room behind its positions
    used, full = _named(ids, live, n_pages), _named(ids, live & ~last, n_pages)
    tail = torch.where(fill > 0, ids.gather(1, (held - 1).clamp(min=0)[:, None])[:, 0], -1 - torch.arange(n, device="cuda"))
    goes_on = fill > 0 if c["rows"] > 0 else torch.zeros_like(fill, dtype=torch.bool)
    # who holds the same last page: the first that goes on among those with the most positions in it keeps it
    same = tail[:, None] == tail
    most = torch.where(same, fill, 0).amax(1)
    keeps = same & goes_on & (fill == most[:, None])
    first = torch.where(keeps, torch.arange(n, device="cuda"), n).amin(1)
    copies = goes_on & (full[tail.clamp(min=0)] | (first != torch.arange(n, device="cuda")))
    fresh = (length + c["rows"] + page - 1) // page - held
    need = copies.long() + fresh
    base = need.cumsum(0) - need
    free = torch.argsort(used.to(torch.int8), stable=True)                  # the free pages first, in order
    at = (base + copies)[:, None] + slot - held[:, None]
    grown = (slot >= held[:, None]) & (slot < (held + fresh)[:, None])
    copied = free[base.clamp(max=n_pages - 1)]
    table = torch.where(live, ids, torch.where(grown, free[at.clamp(0, n_pages - 1)], -1))
    table = torch.where(last & copies[:, None], copied[:, None], table)
    # the copied positions: those of a last page that others keep
    pool = s["pool"].t
    position = torch.arange(page, device="cuda")
    moved = (copies[:, None] & (position < fill[:, None])).nonzero()
    j, p = moved[:, 0], moved[:, 1]
    pool[:, copied[j], :, p] = pool[:, tail[j], :, p]
    s["table_out"].t.copy_(table)
    s["pos_out"].t.copy_(length)
    s["len_out"].t.copy_(length + c["rows"])
    s["status"].t.copy_(torch.stack([torch.zeros_like(base[0]), used.sum() + need.sum()]))
    return {"table": s["table_out"].t, "pos": s["pos_out"].t, "len": s["len_out"].t, "status": s["status"].t, "pool": pool}


def _plain_compact(s, c):
    width, n_pages, page = s["at"]["width"], s["at"]["n_pages"], c["page"]
    ids = s["table"].t.long()
    live = torch.arange(width, device="cuda") < ((s["len"].t.long() + page - 1) // page)[:, None]
    used = _named(ids, live, n_pages)
    count = used.sum()
    page_id = torch.arange(n_pages, device="cuda")
    src, dst = (used & (page_id >= count)).nonzero()[:, 0], (~used & (page_id < count)).nonzero()[:, 0]
    to = page_id.clone()
    to[src] = dst
    pool = s["pool"].t
    pool[:, dst] = pool[:, src]
    s["table_out"].t.copy_(torch.where(live, to[ids.clamp(min=0)], -1))
    s["status"].t.copy_(torch.stack([torch.full_like(count, len(src)), count]))
    return {"table": s["table_out"].t, "status": s["status"].t, "pool": pool}


def _row_places(s, c):
    """(sequence, position) of every row of the batch."""
    start, pos = s["row_start"].t.long(), s["pos"].t.long()
    i = torch.arange(s["at"]["total"], device="cuda")
    of = torch.searchsorted(start, i, right=True) - 1
    return of, pos[of] + i - start[of]


def _plain_write(s, c):
    of, p = _row_places(s, c)
    pages = s["table"].t.long()[of, p // c["page"]]
    hd = c["heads"] * c["dim"]
    s["k_pages"].t[pages, :, p % c["page"]] = s["kv"].t[:, :hd].view(-1, c["heads"], c["dim"]).to(torch.bfloat16)
    s["v_pages"].t[pages, :, p % c["page"]] = s["kv"].t[:, hd:].reshape(-1, c["heads"], c["dim"]).to(torch.bfloat16)
    return {"k": s["k_pages"].t, "v": s["v_pages"].t}


def _plain_attn(s, c):
    n, h, g, d, page = s["at"]["n"], c["heads"], c["ratio"], c["dim"], c["page"]
    most, total, width = s["at"]["most"], s["at"]["total"], s["at"]["width"]
    start, pos = s["row_start"].t.long(), s["pos"].t.long()
    i = torch.arange(most, device="cuda")
    row = start[:-1][:, None] + i                                                    # [n, most]
    row = torch.where(row < start[1:][:, None], row, total)                          # `total`: no row of this sequence
    q = s["q"].t.float()[row.clamp(max=total - 1)].view(n, most, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * most, d)
    ids = s["table"].t.long().clamp(min=0)
    length = width * page
    k = s["k_pages"].t[ids].float().permute(0, 2, 1, 3, 4).reshape(n, h, length, d)
    scores = (q @ k.transpose(-1, -2)).view(n, h, g, most, length) * d ** -0.5
    seen = torch.arange(length, device="cuda") <= (pos[:, None] + i)[..., None]      # [n, most, length]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    v = s["v_pages"].t[ids].float().permute(0, 2, 1, 3, 4).reshape(n, h, length, d)
    o = (e.view(n, h, g * most, length) @ v).view(n, h, g, most, d) / e.sum(-1, keepdim=True)
    out = torch.zeros((total + 1, h * g, d), dtype=_type(c), device="cuda")
    out[row] = o.permute(0, 3, 1, 2, 4).reshape(n, most, h * g, d).to(_type(c))
    return out[:total]


def _plain_score(s, c):
    x = s["logits"].t[:, :c["cols"]].float()
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    logp = (d.gather(1, s["targets"].t.long()[:, None]) - log_total)[:, 0]
    entropy = (log_total - (e * d).sum(1, keepdim=True) / total)[:, 0]
    # whole numbers in the order of the values, ties by the lowest index
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32 + torch.arange(c["cols"] - 1, -1, -1, device="cuda")
    ids = c["cols"] - 1 - (torch.topk(key, c["k"], 1).values & 0xFFFFFFFF)
    return {"logp": logp, "entropy": entropy, "ids": ids.int(), "top": d.gather(1, ids) - log_total}


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    return {"fork": _plain_fork, "compact": _plain_compact, "write": _plain_write, "attn": _plain_attn,
            "score": _plain_score}[s["kind"]](s, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind == "score":
        e = c["rows"] * c["cols"]
        return {"bytes": e * (2 if c["bf16"] else 4) + c["rows"] * (12 + 8 * c["k"]), "flops": 6 * e}
    hd, page = c["heads"] * c["dim"], c["page"]
    if kind == "fork":
        n = c["groups"] * c["beams"]
        lengths, shared = _fork_plan(c, 0)
        # of each group all but the parents themselves copy what their last page holds
        kept = sum(min(c["beams"], (c["beams"] + 1) // 2) for _ in shared)
        fill = sum(m % page for m in lengths) / n
        return {"bytes": 8 * sum(_pages(m, page) for m in lengths) + 2 * (n - kept) * fill * 2 * hd * c["pools"], "flops": n}
    if kind == "compact":
        lengths = [1 + int(c["past"] * (0.3 + 0.7 * x)) for x in _some(c["seqs"], 17 * c["seqs"] + c["past"])]
        gone = [x >= c["live"] for x in _some(c["seqs"], 19 * c["seqs"] + c["past"])]
        every = sum(_pages(m, page) for m in lengths) + 4
        used = sum(_pages(m, page) for k, (m, e) in enumerate(zip(lengths, gone)) if k == 0 or not e)
        return {"bytes": 8 * used + 2 * used * (1 - used / every) * page * 2 * hd * c["pools"], "flops": used}
    if kind == "write":
        rows = sum(_lengths(c, 0, c["seqs"])[0])
        return {"bytes": 2 * hd * rows * ((2 if c["bf16"] else 4) + 2), "flops": 2 * hd * rows}
    n = c["groups"] * c["beams"]
    rows, past = _lengths(c, 0, n)
    shared = [c["shared"]] + [max(0, int(c["shared"] * (0.75 + 0.25 * x))) for x in _some(c["groups"], 23 * c["groups"] + c["shared"])][1:]
    keys = sum(shared) + sum(a + b for a, b in zip(rows, past))
    seen = sum(a * (shared[j // c["beams"]] + b + (a + 1) / 2) for j, (a, b) in enumerate(zip(rows, past)))
    return {"bytes": keys * 2 * hd * 2 + 2 * (2 if c["bf16"] else 4) * sum(rows) * hd * c["ratio"],
            "flops": 4 * hd * c["ratio"] * seen}


# ---------------------------------------------------------------------------
# the same results in 64 bits, and the tables by lists
# ---------------------------------------------------------------------------

def _exact_fork(c, seed):
    d, at = _fork_inputs(c, seed)
    page, rows = c["page"], c["rows"]
    table, lengths, parent = d["table"].tolist(), d["len"].tolist(), d["parent"].tolist()
    length = [lengths[p] for p in parent]
    held = [table[p][:_pages(lengths[p], page)] for p in parent]
    used = {p for row in held for p in row}
    free = iter([p for p in range(at["n_pages"]) if p not in used])
    holders = {}
    for j, row in enumerate(held):
        for k, p in enumerate(row):
            in_it = min(page, length[j] - k * page)
            holders.setdefault(p, []).append((-in_it, j))
    out, pool = [], d["pool"].clone()
    for j, row in enumerate(held):
        row, part = list(row), length[j] % page
        if part and rows and min(holders[row[-1]]) != (-part, j):
            new = next(free)
            pool[:, new, :, :part] = d["pool"][:, row[-1], :, :part]
            row[-1] = new
        row += [next(free) for _ in range(_pages(length[j] + rows, page) - len(row))]
        out.append(row + [-1] * (at["width"] - len(row)))
    return {"table": _int32(out), "pos": _int32(length), "len": _int32([m + rows for m in length]),
            "status": _int32([0, at["n_pages"] - len(list(free))]), "pool": pool}


def _exact_compact(c, seed):
    d, at = _compact_inputs(c, seed)
    held = [row[:_pages(m, c["page"])] for row, m in zip(d["table"].tolist(), d["len"].tolist())]
    used = sorted({p for row in held for p in row})
    n = len(used)
    moved = dict(zip([p for p in used if p >= n], sorted(set(range(n)) - set(used))))
    pool = d["pool"].clone()
    for a, b in moved.items():
        pool[:, b] = d["pool"][:, a]
    return {"table": _int32([[moved.get(p, p) for p in row] + [-1] * (at["width"] - len(row)) for row in held]),
            "status": _int32([len(moved), n]), "pool": pool}


def _exact_write(c, seed):
    d, at = _write_inputs(c, seed)
    rows, past = _lengths(c, seed, c["seqs"])
    table, hd, r0 = d["table"].tolist(), c["heads"] * c["dim"], 0
    out = {"k": d["k_pages"].double(), "v": d["v_pages"].double()}
    for j, (m, p) in enumerate(zip(rows, past)):
        for i in range(0, m):
            if i == 0 or (p + i) % c["page"] == 0:                          # a page at a time
                n = min(m - i, c["page"] - (p + i) % c["page"])
                for name, x in out.items():
                    new = d["kv"][r0 + i:r0 + i + n, (hd if name == "v" else 0):][:, :hd].double()
                    x[table[j][(p + i) // c["page"]], :, (p + i) % c["page"]:(p + i) % c["page"] + n] = \
                        new.view(n, c["heads"], c["dim"]).transpose(0, 1)
        r0 += m
    return out


def _exact_attn(c, seed):
    d, at = _attn_inputs(c, seed)
    h, g, dim = c["heads"], c["ratio"], c["dim"]
    start, pos, out = d["row_start"].tolist(), d["pos"].tolist(), []
    for j in range(at["n"]):
        m = start[j + 1] - start[j]
        length = pos[j] + m
        ids = d["table"][j, :_pages(length, c["page"])].long()
        seen = torch.arange(length, device="cuda")[None] < torch.arange(pos[j] + 1, length + 1, device="cuda")[:, None]
        o = torch.empty((m, h * g, dim), dtype=torch.float64, device="cuda")
        for a in range(h):
            k = d["k_pages"][ids, a].reshape(-1, dim)[:length].double()
            v = d["v_pages"][ids, a].reshape(-1, dim)[:length].double()
            for e in range(a * g, a * g + g):
                w = (d["q"][start[j]:start[j + 1], e].double() @ k.T) / math.sqrt(dim)
                o[:, e] = w.masked_fill(~seen, -math.inf).softmax(1) @ v
        out.append(o)
    return torch.cat(out)


def _exact_score(c, seed):
    d = _score_inputs(c, seed)
    out = {"logp": [], "entropy": [], "ids": [], "top": []}
    for at in range(0, c["rows"], 64):
        x = d["logits"][at:at + 64, :c["cols"]].double()
        lp = x.log_softmax(1)
        v, i = x.sort(dim=1, descending=True, stable=True)
        out["logp"].append(lp.gather(1, d["targets"][at:at + 64].long()[:, None])[:, 0])
        out["entropy"].append(-(lp.exp() * lp).sum(1))
        out["ids"].append(i[:, :c["k"]].int())
        out["top"].append(lp.gather(1, i[:, :c["k"]]))
    return {n: torch.cat(v) for n, v in out.items()}


def exact(case, seed):
    return {"fork": _exact_fork, "compact": _exact_compact, "write": _exact_write, "attn": _exact_attn,
            "score": _exact_score}[case["kind"]](case, seed)
