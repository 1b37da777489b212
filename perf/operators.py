"""What the operators of an 8-bit decoder layer are measured on.

Five operators that one layer is made of when it runs wholly in 8 bits, over
many rows or many sequences: the residual's addition with RMSNorm into int8
rows, the int8 x int8 product with a scale for each row and each column, the
write of K and V into a cache held in int8 with one scale for 64 positions of a
head and its reading back, and the attention over that cache.

Sizes are those of this repository's decoders (`synth.DEC_0_6B`, `DEC_1_7B`:
16 query heads and 8 KV heads of 128, hidden 1024 and 2048) and of its
workloads: 32 streams decoded as one batch, prompts of 404 rows (30 s of
audio), 1337 rows (a long recording), streaming chunks of some tens of rows.

`own` false: plain forms in elementary torch operations.  `own` true: the calls
of `qwenasr_amd.kernels`, on torch tensors (a program may hold its buffers in
any device allocation).

The cache (both forms use its layout): K [seq][head][position][dim] int8; V in
blocks of 64 positions, [seq][head][block][dim][64], where byte 16 g + 4 t + r
of a dim's 64 is position 16 t + 4 g + r of the block; scales [seq][head][block]
f32.  A stored value stands for int8 x scale of its block.
"""
import functools
import math

import torch

own = False

EPS = 1e-6
BLOCK = 64                 # positions with one scale


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the residual rows of 32 streams decoded as one batch, before a projection: latency
        {"name": "norm8_32x1024", "kind": "norm", "rows": 32, "hidden": 1024, "pad": 0, "res": True, "norm": True,
         "bf16": False},
        # the prompts of thirty sessions at once, a bf16 residual stream of the larger decoder
        {"name": "norm8_12120x2048_bf16", "kind": "norm", "rows": 12120, "hidden": 2048, "pad": 0, "res": True,
         "norm": True, "bf16": True},
        # gate_up with SwiGLU of the larger decoder, one token of each of 32 streams: weights stream, few rows
        {"name": "w8a8_swiglu_32x12288x2048", "kind": "gemm", "m": 32, "n": 12288, "k": 2048, "mode": "swiglu",
         "bias": False, "bf16": False},
        # q, k and v of the small decoder for a prompt of 30 s
        {"name": "w8a8_404x4096x1024", "kind": "gemm", "m": 404, "n": 4096, "k": 1024, "mode": "plain", "bias": False,
         "bf16": False},
        # a biased head of odd width (a forced aligner's) over the prompts of five sessions, bf16 out
        {"name": "w8a8_2021x4999x1024_bf16", "kind": "gemm", "m": 2021, "n": 4999, "k": 1024, "mode": "plain",
         "bias": True, "bf16": True},
        # the LM head over all rows of 30 s: the largest product
        {"name": "w8a8_lm_head_375", "kind": "gemm", "m": 375, "n": 151936, "k": 1024, "mode": "plain", "bias": False,
         "bf16": False},
        # one new position in each of 32 caches, blocks partly filled, and the touched blocks read back
        {"name": "kv8_step_32", "kind": "kv", "seqs": 32, "rows": 1, "ragged": False, "past": 2000, "heads": 8, "dim": 128,
         "bf16": False},
        # ragged prompts of eight sessions written behind what they hold, and read back
        {"name": "kv8_8_prompts_bf16", "kind": "kv", "seqs": 8, "rows": 1337, "ragged": True, "past": 300, "heads": 8,
         "dim": 128, "bf16": True},
        # greedy decoding after a 30 s prompt, one session: the smallest attention
        {"name": "attn8_decode_404", "kind": "attn", "seqs": 1, "rows": 1, "ragged": False, "past": 404, "heads": 8,
         "group": 2, "dim": 128, "window": 0, "sinks": 0, "bf16": False},
        # one token of each of 32 streams, sessions of different age
        {"name": "attn8_decode_32x4000_bf16", "kind": "attn", "seqs": 32, "rows": 1, "ragged": False, "past": 4000,
         "heads": 8, "group": 2, "dim": 128, "window": 0, "sinks": 0, "bf16": True},
        # the prompt of a long recording
        {"name": "attn8_prompt_1337", "kind": "attn", "seqs": 1, "rows": 1337, "ragged": False, "past": 0, "heads": 8,
         "group": 2, "dim": 128, "window": 0, "sinks": 0, "bf16": False},
        # chunks of four streams that have run for an hour: the last 8192 positions and four sinks stay visible
        {"name": "attn8_chunk_window_4x40000", "kind": "attn", "seqs": 4, "rows": 67, "ragged": True, "past": 40000,
         "heads": 8, "group": 2, "dim": 128, "window": 8192, "sinks": 4, "bf16": True},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "gemm", "gemm", "kv", "attn", "attn"])
    bf16 = rng.random() < 0.5
    if kind == "norm":
        hidden = rng.choice([64 * _log(rng, 2, 64), _log(rng, 100, 4096)])
        return {"kind": kind, "rows": _log(rng, 1, min(12120, 12120 * 2048 // hidden)), "hidden": hidden,
                "pad": rng.choice([0, 0, 8, 3]), "res": rng.random() < 0.7, "norm": rng.random() < 0.8, "bf16": bf16}
    if kind == "gemm":
        k = rng.choice([64 * _log(rng, 4, 96), 64 * _log(rng, 4, 96), _log(rng, 100, 6144)])
        m = _log(rng, 1, 2000)
        n = _log(rng, 256, min(151936, 375 * 151936 * 1024 // (m * max(k, 1024))))
        mode = rng.choice(["plain", "plain", "add", "swiglu"])
        return {"kind": kind, "m": m, "n": n + n % 2 if mode == "swiglu" else n, "k": k, "mode": mode,
                "bias": rng.random() < 0.3, "bf16": bf16}
    heads, dim = rng.choice([8, 8, 4, 14]), rng.choice([128, 128, 64])
    if kind == "kv":
        seqs = _log(rng, 1, 32)
        rows = rng.choice([1, _log(rng, 2, max(2, 4 * 1337 // seqs))])
        return {"kind": kind, "seqs": seqs, "rows": rows, "ragged": rng.random() < 0.5, "past": _log(rng, 1, 4000),
                "heads": heads, "dim": dim, "bf16": bf16}
    heads = min(heads, 8)
    group, window = rng.choice([2, 2, 1, 3, 4]), rng.choice([0, 0, _log(rng, 16, 4096)])
    if rng.random() < 0.5:
        seqs, rows = _log(rng, 1, 32), rng.choice([1, 1, rng.randint(2, 8)])
        past = _log(rng, 30, min(100000, 32 * 4000 // (seqs * rows)))
    else:
        rows = _log(rng, 9, 1337)
        seqs = rng.randint(1, max(1, min(4, 1337 // rows)))
        past = rng.choice([0, _log(rng, 1, max(1, 1337 * 700 // (seqs * rows)))])
    return {"kind": kind, "seqs": seqs, "rows": rows, "ragged": rng.random() < 0.5, "past": past, "heads": heads,
            "group": group, "dim": dim, "window": window, "sinks": rng.choice([0, 4, 70]) if window else 0, "bf16": bf16}


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

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * std

    def int8(self, *shape, std=32.0):
        """Rows as the quantiser leaves them: normal, the largest of many at 127."""
        return (torch.randn(shape, generator=self.g, device="cuda") * std).round_().clamp_(-127, 127).to(torch.int8)

    def uniform(self, n, lo, hi):
        return lo + (hi - lo) * torch.rand(n, generator=self.g, device="cuda")


def _type(c):
    return torch.bfloat16 if c["bf16"] else torch.float32


def _lengths(c, seed):
    """Rows and first positions of every sequence (host lists): a case's own, in an order that the seed turns."""
    n, s = c["rows"], c["seqs"]
    g = torch.Generator()
    g.manual_seed(s + 64 * n + 100003 * c["past"])
    rows = [n] * s
    if c["ragged"]:
        rows = [n] + [max(1, int(n * x)) for x in torch.rand(s - 1, generator=g).tolist()]
    past = [c["past"]] + [int(c["past"] * (0.5 + 0.5 * x)) for x in torch.rand(s - 1, generator=g).tolist()]
    past = past[-1:] + past[:-1]
    turn = seed % s
    return rows[turn:] + rows[:turn], past[turn:] + past[:turn]


def _prefix(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _capacity(n):
    return (n + 255) // 256 * 256


def _norm_inputs(c, seed):
    r, t = _Rng(seed), _type(c)
    ld = c["hidden"] + c["pad"]
    d = {"x": r.normal(c["rows"], ld).to(t)}
    if c["res"]:
        d["res"] = r.normal(c["rows"], ld, std=0.3).to(t)
    if c["norm"]:
        d["w"] = 1 + r.normal(c["hidden"], std=0.05)
    return d


def _gemm_inputs(c, seed):
    r, m, n, k = _Rng(seed), c["m"], c["n"], c["k"]
    d = {"a": r.int8(m, k), "sa": r.uniform(m, 0.02, 0.03), "w": r.int8(n, k), "sw": r.uniform(n, 0.0004, 0.0006)}
    if c["bias"]:
        d["bias"] = r.normal(n, std=0.1)
    if c["mode"] == "add":
        d["y0"] = r.normal(m, n).to(_type(c))
    return d


def _cache(c, r, cap):
    s, h, d = c["seqs"], c["heads"], c["dim"]
    return {"k8": r.int8(s, h, cap, d), "v8": r.int8(s, h, cap // BLOCK, d, BLOCK),
            "ks": r.uniform((s, h, cap // BLOCK), 0.028, 0.034), "vs": r.uniform((s, h, cap // BLOCK), 0.016, 0.020)}


def _kv_inputs(c, seed):
    r, t = _Rng(seed), _type(c)
    rows, past = _lengths(c, seed)
    cap = _capacity(max(a + b for a, b in zip(rows, past)))
    d = _cache(c, r, cap)
    # k as its per-head norm leaves it, v as projected; both inside the fused projection's rows
    total = sum(rows)
    qkv = torch.cat([r.normal(total, c["heads"] * c["dim"]), r.normal(total, c["heads"] * c["dim"], std=0.6)], 1).to(t)
    d.update(kv=qkv, row_start=_int32(_prefix(rows)), pos=_int32(past))
    # what is read back: from the start of the first block that the write touches
    first = [p // BLOCK * BLOCK for p in past]
    back = [p - f + n for p, f, n in zip(past, first, rows)]
    d.update(back_start=_int32(_prefix(back)), back_pos=_int32(first))
    return d, {"total": total, "cap": cap, "most": max(rows), "back_total": sum(back), "back_most": max(back)}


def _attn_inputs(c, seed):
    r, t = _Rng(seed), _type(c)
    rows, past = _lengths(c, seed)
    cap = _capacity(max(a + b for a, b in zip(rows, past)))
    d = _cache(c, r, cap)
    total = sum(rows)
    d.update(q=r.normal(total, c["heads"] * c["group"], c["dim"]).to(t), row_start=_int32(_prefix(rows)), pos=_int32(past))
    return d, {"total": total, "cap": cap, "most": max(rows), "longest": max(a + b for a, b in zip(rows, past))}


def _empty(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    c, kind = case, case["kind"]
    s = {"case": c, "kind": kind}
    if kind == "norm":
        d = _norm_inputs(c, seed)
        d.update(q=_empty(c["rows"], c["hidden"], dtype=torch.int8), scales=_empty(c["rows"]))
        if c["res"]:
            d["sum"] = torch.zeros_like(d["x"])
    elif kind == "gemm":
        d = _gemm_inputs(c, seed)
        d["y"] = _empty(c["m"], c["n"] // 2 if c["mode"] == "swiglu" else c["n"], dtype=_type(c))
    elif kind == "kv":
        d, s["at"] = _kv_inputs(c, seed)
        d.update(k=_empty(s["at"]["back_total"], c["heads"], c["dim"]), v=_empty(s["at"]["back_total"], c["heads"], c["dim"]))
        hd = c["heads"] * c["dim"]
        s["v_rows"] = _Buf(d["kv"][:, hd:])
    elif kind == "attn":
        d, s["at"] = _attn_inputs(c, seed)
        d["out"] = torch.zeros_like(d["q"])
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
    c, kind = s["case"], s["kind"]
    if kind == "norm":
        K.add_rms_norm_int8(s["q"], s["scales"], s["x"], s.get("w"), c["rows"], c["hidden"], res=s.get("res"),
                            sum_out=s.get("sum"), ld=c["hidden"] + c["pad"], eps=EPS, bf16=c["bf16"])
        out = {"q": s["q"].t, "scales": s["scales"].t}
        if c["res"]:
            out["sum"] = s["sum"].t[:, :c["hidden"]]
        return out
    if kind == "gemm":
        if c["mode"] == "add":
            _device().copy(s["y"], s["y0"], s["y"].t.nbytes)       # the residual rows
        K.gemm_w8a8(s["y"], s["a"], s["sa"], s["w"], s["sw"], c["m"], c["n"], c["k"], bias=s.get("bias"),
                    accumulate=c["mode"] == "add", swiglu=c["mode"] == "swiglu", bf16=c["bf16"])
        return s["y"].t
    at = s["at"]
    if kind == "kv":
        hd = c["heads"] * c["dim"]
        K.kv8_write(s["k8"], s["v8"], s["ks"], s["vs"], s["kv"], s["v_rows"], s["pos"], at["total"], c["seqs"], at["most"],
                    c["heads"], c["dim"], at["cap"], row_start=s["row_start"], ld=2 * hd, bf16=c["bf16"])
        K.kv8_read(s["k"], s["v"], s["k8"], s["v8"], s["ks"], s["vs"], s["back_pos"], at["back_total"], c["seqs"],
                   at["back_most"], c["heads"], c["dim"], at["cap"], row_start=s["back_start"])
        return {"k": s["k"].t, "v": s["v"].t}
    K.attention_kv8(s["out"], s["q"], s["k8"], s["v8"], s["ks"], s["vs"], s["pos"], at["total"], c["seqs"], at["most"],
                    c["heads"] * c["group"], c["heads"], c["dim"], at["cap"], c["dim"] ** -0.5, row_start=s["row_start"],
                    max_len=at["longest"], window=c["window"], sinks=c["sinks"], bf16=c["bf16"])
    return s["out"].t


def _away(x):
    """To the nearest whole number, halves away from zero, within int8's range."""
    return torch.sign(x) * torch.floor(x.abs() + 0.5).clamp(max=127)


def _plain_norm(s, c):
    # in 64 bits: the int8 values are decided next to borders
    h = c["hidden"]
    x = s["x"].t[:, :h].double()
    out = {}
    if c["res"]:
        x = x + s["res"].t[:, :h].double()
        out["sum"] = x.to(_type(c))
    t, rms = x, 1.0
    if c["norm"]:
        t = x * s["w"].t.double()
        rms = torch.rsqrt((x * x).mean(1) + EPS)
    most = t.abs().amax(1)
    out["q"] = _away(t * 127.0 / most[:, None]).to(torch.int8)
    out["scales"] = (most * rms / 127.0).float()
    return out


def _plain_gemm(s, c):
    y = s["a"].t.float() @ s["w"].t.float().T
    y = y * s["sa"].t[:, None] * s["sw"].t
    if c["bias"]:
        y = y + s["bias"].t
    if c["mode"] == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    if c["mode"] == "add":
        y = y + s["y0"].t.float()
    return y.to(_type(c))


def _to_rows(v):
    """[..., blocks, dim, 64] as stored -> [..., blocks, 64, dim]."""
    b, d = v.shape[-3], v.shape[-2]
    v = v.reshape(*v.shape[:-1], 4, 4, 4).movedim(-4, -1)           # [..., blocks, g, t, r, dim]
    return v.transpose(-4, -3).reshape(*v.shape[:-5], b, BLOCK, d)


def _to_stored(v):
    """The way back."""
    b, d = v.shape[-3], v.shape[-1]
    v = v.reshape(*v.shape[:-2], 4, 4, 4, d).transpose(-4, -3)      # [..., blocks, g, t, r, dim]
    return v.movedim(-1, -4).reshape(*v.shape[:-5], b, d, BLOCK)


def _store(old, so, new, live, fresh):
    """int8 blocks [s, h, b, 64, d] with scales [s, h, b] after the rows `new`; `live` and `fresh` [s, 1, b, 64, 1] say
    which positions hold a value already and which get one."""
    most = torch.where(fresh, new, 0.0).abs().amax((-2, -1))
    sn = (most.double() / 127.0).float()                            # what is stored decides the borders: rounded once
    sn = torch.where(live.any(-2)[..., 0], torch.maximum(sn, so), sn)
    sd = torch.where(sn > 0, sn, 1.0).double()[..., None, None]
    again = _away(old.double() * so.double()[..., None, None] / sd)
    q = torch.where(fresh, _away(new.double() / sd), torch.where(live, again, old.double()))
    return q.to(torch.int8), sn


def _plain_kv(s, c):
    n, h, d, cap = c["seqs"], c["heads"], c["dim"], s["at"]["cap"]
    start, pos = s["row_start"].t.long(), s["pos"].t.long()
    first = pos // BLOCK
    # the blocks that the write touches: `blocks` slots per sequence, those past its last row are left as they are
    blocks = (s["at"]["most"] + BLOCK - 2) // BLOCK + 1
    slot = first[:, None] + torch.arange(blocks, device="cuda")                      # [n, blocks]
    p = slot[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")                 # [n, blocks, 64] positions
    row = p - pos[:, None, None]
    count = (start[1:] - start[:-1])[:, None, None]
    fresh, live = ((row >= 0) & (row < count))[:, None, ..., None], (row < 0)[:, None, ..., None]
    at = (start[:-1][:, None, None] + row.clamp(min=0)).clamp(max=s["at"]["total"] - 1)
    slot = torch.where(slot * BLOCK < pos[:, None] + count[..., 0], slot, first[:, None])   # unused slots: the first block's
    used = (slot == first[:, None] + torch.arange(blocks, device="cuda"))
    seq, head = torch.arange(n, device="cuda")[:, None, None], torch.arange(h, device="cuda")[None, :, None]
    where = (seq, head, slot[:, None])
    hd = h * d
    out = {}
    b0, bn = s["back_start"].t.long(), s["back_pos"].t.long()
    i = torch.arange(s["at"]["back_total"], device="cuda")
    of = torch.searchsorted(b0, i, right=True) - 1                                   # the sequence of each row read back
    bp = bn[of] + i - b0[of]
    k8 = s["k8"].t.view(n, h, cap // BLOCK, BLOCK, d)
    for name, x8, sc, new in (("k", k8, s["ks"].t, s["kv"].t[:, :hd]), ("v", s["v8"].t, s["vs"].t, s["kv"].t[:, hd:])):
        new = new.float()[at].view(n, blocks, BLOCK, h, d).permute(0, 3, 1, 2, 4)
        old = x8[where]
        rows = old if name == "k" else _to_rows(old)
        q, sn = _store(rows, sc[where], new, live, fresh)
        q = q if name == "k" else _to_stored(q)
        # unused slots write the first block's own result again
        u = used[:, None, :]
        x8[where] = torch.where(u[..., None, None], q, q[:, :, :1])
        sc[where] = torch.where(u, sn, sn[:, :, :1])
        if name == "k":
            got = x8[of, :, bp // BLOCK, bp % BLOCK]
        else:
            b = bp % BLOCK
            got = x8[of, :, bp // BLOCK, :, b % 16 // 4 * 16 + b // 16 * 4 + b % 4]
        out[name] = got.float() * sc[of, :, bp // BLOCK][..., None]
    return out


def _plain_attn(s, c):
    n, h, g, d, cap = c["seqs"], c["heads"], c["group"], c["dim"], s["at"]["cap"]
    most, total = s["at"]["most"], s["at"]["total"]
    length = (s["at"]["longest"] + BLOCK - 1) // BLOCK * BLOCK
    nb = length // BLOCK
    start, pos = s["row_start"].t.long(), s["pos"].t.long()
    i = torch.arange(most, device="cuda")
    row = start[:-1][:, None] + i                                                    # [n, most]
    row = torch.where(row < start[1:][:, None], row, total)                          # `total`: no row of this sequence
    q = s["q"].t.float()[row.clamp(max=total - 1)].view(n, most, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * most, d)
    k = (s["k8"].t.view(n, h, -1, BLOCK, d)[:, :, :nb].float() * s["ks"].t[:, :, :nb, None, None]).view(n, h, length, d)
    v = (_to_rows(s["v8"].t[:, :, :nb]).float() * s["vs"].t[:, :, :nb, None, None]).view(n, h, length, d)
    scores = (q @ k.transpose(-1, -2)).view(n, h, g, most, length) * d ** -0.5
    j, last = torch.arange(length, device="cuda"), (pos[:, None] + i)[..., None]     # [n, most, 1]
    seen = j <= last
    if c["window"]:
        seen = seen & ((j > last - c["window"]) | (j < c["sinks"]))
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (e.view(n, h, g * most, length) @ v).view(n, h, g, most, d) / e.sum(-1, keepdim=True)
    out = torch.zeros((total + 1, h * g, d), dtype=_type(c), device="cuda")
    out[row] = o.permute(0, 3, 1, 2, 4).reshape(n, most, h * g, d).to(_type(c))
    return out[:total]


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    return {"norm": _plain_norm, "gemm": _plain_gemm, "kv": _plain_kv, "attn": _plain_attn}[s["kind"]](s, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    b = 2 if c["bf16"] else 4
    if kind == "norm":
        e = c["rows"] * c["hidden"]
        return {"bytes": e * (b + 1 + (2 * b if c["res"] else 0)) + 4 * c["rows"] + 4 * c["hidden"], "flops": 8 * e}
    if kind == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        out = b * m * (n // 2 if c["mode"] == "swiglu" else n) * (2 if c["mode"] == "add" else 1)
        return {"bytes": m * k + n * k + out + 4 * (m + n) + 4 * n * c["bias"], "flops": 2 * m * n * k}
    # lengths as they come out on average
    s, hd = c["seqs"], c["heads"] * c["dim"]
    rows = s * c["rows"] * (0.5 if c["ragged"] and s > 1 else 1)
    past = c["past"] * (0.75 if s > 1 else 1)
    if kind == "kv":
        # the rows in and their bytes out; what is read back (half a block more per sequence): bytes in, f32 out
        back = rows + 32 * s
        return {"bytes": 2 * hd * (rows * (b + 1) + back * 5), "flops": 2 * hd * (6 * rows + back)}
    seen = past + c["rows"] / 2
    keys = past + c["rows"]
    if c["window"]:
        seen = min(seen, c["window"] + c["sinks"])
        keys = min(keys, c["window"] + c["sinks"] + c["rows"])
    return {"bytes": s * keys * 2 * hd * (1 + 4 / (BLOCK * c["dim"])) + 2 * b * rows * hd * c["group"],
            "flops": 4 * rows * hd * c["group"] * seen}


# ---------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------

def _half_up(v):
    """Nearest whole number, halves away from zero."""
    return torch.where(v < 0, torch.ceil(v - 0.5), torch.floor(v + 0.5)).clamp(-127, 127)


def _exact_norm(c, seed):
    d, h = _norm_inputs(c, seed), c["hidden"]
    x = d["x"].double()[:, :h]
    if c["res"]:
        x = x + d["res"].double()[:, :h]
    n = x / ((x ** 2).sum(1, keepdim=True) / h + EPS).sqrt() if c["norm"] else x
    # 1 / rms is common to a row and cancels in the ratio
    t = x * d["w"].double() if c["norm"] else x
    if c["norm"]:
        n = n * d["w"].double()
    out = {"q": _half_up(127 * t / t.abs().max(1, keepdim=True).values).to(torch.int8), "scales": n.abs().max(1).values / 127}
    if c["res"]:
        out["sum"] = x
    return out


def _exact_gemm(c, seed):
    d = _gemm_inputs(c, seed)
    parts = []
    w = d["w"].double()
    for at in range(0, c["m"], 256):
        y = (d["a"][at:at + 256].double() @ w.T) * d["sa"][at:at + 256].double()[:, None] * d["sw"].double()[None]
        if c["bias"]:
            y = y + d["bias"].double()
        if c["mode"] == "swiglu":
            y = y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
        if c["mode"] == "add":
            y = y + d["y0"][at:at + 256].double()
        parts.append(y)
    return torch.cat(parts)


def _positions(block):
    """The position inside its block that each of the 64 stored bytes holds."""
    return [16 * (b % 16 // 4) + 4 * (b // 16) + b % 4 for b in range(block)]


def _exact_kv(c, seed):
    d, at = _kv_inputs(c, seed)
    n, h, dim, hd = c["seqs"], c["heads"], c["dim"], c["heads"] * c["dim"]
    rows, past = _lengths(c, seed)
    held = {"k": d["k8"].view(n, h, -1, BLOCK, dim).double(), "v": torch.empty(0)}
    v = torch.empty_like(held["k"])
    v[:, :, :, _positions(BLOCK)] = d["v8"].double().transpose(-1, -2)
    held["v"] = v
    scale = {"k": d["ks"].double(), "v": d["vs"].double()}
    out = {"k": [], "v": []}
    r0 = 0
    for j in range(n):
        p, m = past[j], rows[j]
        for name in out:
            new = d["kv"][r0:r0 + m, (hd if name == "v" else 0):][:, :hd].double().view(m, h, dim).transpose(0, 1)
            q, sc = held[name][j], scale[name][j]
            for b in range(p // BLOCK, (p + m - 1) // BLOCK + 1):
                lo, hi = max(p, b * BLOCK), min(p + m, (b + 1) * BLOCK)
                x = new[:, lo - p:hi - p]
                # the scale is what the cache stores: 32 bits
                s1 = (x.abs().amax((1, 2)) / 127).float().double()
                keep = lo - b * BLOCK
                if keep:
                    s1 = torch.maximum(s1, sc[:, b])
                    q[:, b, :keep] = _half_up(q[:, b, :keep] * sc[:, b, None, None] / s1[:, None, None])
                q[:, b, keep:hi - b * BLOCK] = _half_up(x / s1[:, None, None])
                sc[:, b] = s1
            first = p // BLOCK
            whole = (q[:, first:] * sc[:, first:, None, None]).reshape(h, -1, dim)
            out[name].append(whole[:, :p + m - first * BLOCK].transpose(0, 1))
        r0 += m
    return {name: torch.cat(v) for name, v in out.items()}


def _exact_attn(c, seed):
    d, at = _attn_inputs(c, seed)
    n, h, g, dim = c["seqs"], c["heads"], c["group"], c["dim"]
    rows, past = _lengths(c, seed)
    out, r0, order = [], 0, _positions(BLOCK)
    for j in range(n):
        p, m = past[j], rows[j]
        length, nb = p + m, (p + m + BLOCK - 1) // BLOCK
        last = torch.arange(p, p + m, device="cuda")[:, None]
        pos = torch.arange(length, device="cuda")[None]
        seen = pos <= last
        if c["window"]:
            seen = seen & ((pos + c["window"] > last) | (pos < c["sinks"]))
        o = torch.empty((m, h * g, dim), dtype=torch.float64, device="cuda")
        for a in range(h):
            k = (d["k8"][j, a].view(-1, BLOCK, dim)[:nb].double() * d["ks"][j, a, :nb, None, None].double()).view(-1, dim)[:length]
            v = torch.empty((nb, BLOCK, dim), dtype=torch.float64, device="cuda")
            v[:, order] = d["v8"][j, a, :nb].double().transpose(1, 2)
            v = (v * d["vs"][j, a, :nb, None, None].double()).view(-1, dim)[:length]
            for e in range(g):
                q = d["q"][r0:r0 + m, a * g + e].double()
                w = ((q @ k.T) / math.sqrt(dim)).masked_fill(~seen, -math.inf).softmax(1)
                o[:, a * g + e] = w @ v
        out.append(o)
        r0 += m
    return torch.cat(out)


def exact(case, seed):
    return {"norm": _exact_norm, "gemm": _exact_gemm, "kv": _exact_kv, "attn": _exact_attn}[case["kind"]](case, seed)
