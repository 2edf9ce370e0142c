"""Timed cases of the paged-cache operators: writing a chunk's keys and values, reading them back,
attention of new tokens over the pages, and the verification of drafted tokens.

``own`` false: a pass is the operator's plain form, elementary torch operations on the inputs that
``prepare`` makes.  ``own`` true: a pass is one launch of a compiled one- or two-node plan bound to
the same device tensors.

A cache is a uint8 tensor of pages.  A page holds, for each K/V head in turn: the K rows
[page][hdp], the V rows in groups of eight tokens [page/8][hdp][8] (hdp: head_dim rounded up to 16),
and a float32 scale for each K row and each V row.  A stored value stands for itself times its
row's scale.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

ELEMENT = {"float32": torch.float32, "float16": torch.float16, "int8": torch.int8, "float8": torch.float8_e4m3fn}
TINY = 2.0 ** -126


# ---------------------------------------------------------------- the cases

def _attention(tokens, heads, kv_heads, head_dim, context, cache, page, batch=1, ragged=False, **name):
    """`tokens` new tokens a sequence over `context` earlier ones."""
    return {"op": "attention", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "context": context, "cache": cache, "page": page, "ragged": ragged, **name}


def _write(tokens, kv_heads, head_dim, context, cache, page, batch=1, ragged=False, **name):
    """A chunk written behind `context` tokens, and its rows read back."""
    return {"op": "write", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
            "context": context, "cache": cache, "page": page, "ragged": ragged, **name}


def _read(tokens, kv_heads, head_dim, cache, page, batch=1, ragged=False, **name):
    """A sequence's first `tokens` positions read back."""
    return {"op": "read", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
            "context": 0, "cache": cache, "page": page, "ragged": ragged, **name}


def _verify(drafts, vocab, batch=1, ragged=False, **name):
    return {"op": "verify", "batch": batch, "drafts": drafts, "vocab": vocab, "ragged": ragged, **name}


def listed():
    return [
        # the first token after a short prompt of a GPT-2-width model: latency
        _attention(1, 12, 12, 64, 36, "float32", 16, name="attention_first_token"),
        # one token for each of 32 conversations of every length, a 4B grouped-query model
        _attention(1, 32, 8, 128, 4096, "float16", 64, batch=32, ragged=True, name="attention_tokens_ragged"),
        # four long documents, near the end of that model's positions
        _attention(1, 32, 8, 128, 40900, "int8", 128, batch=4, name="attention_tokens_long"),
        # drafted tokens of 16 sequences checked in one call
        _attention(5, 32, 8, 128, 2048, "float8", 32, batch=16, ragged=True, name="attention_drafts"),
        # three short ragged prompts continued, sizes that are no multiple of a tile
        _attention(77, 5, 5, 80, 300, "float32", 16, batch=3, ragged=True, name="attention_chunk_odd"),
        # a prompt's second 1024 tokens, grouped heads
        _attention(1024, 32, 8, 128, 1024, "int8", 64, name="attention_chunk_grouped"),
        # half of a 7B model's 4096-token context over the other half: the largest work
        _attention(2048, 32, 32, 128, 2048, "float16", 128, name="attention_chunk_7b"),
        # a whole prompt's keys and values of one layer
        _write(4096, 8, 128, 0, "int8", 64, name="write_prompt"),
        # one token of each of 64 sequences
        _write(1, 8, 128, 2048, "float8", 16, batch=64, ragged=True, name="write_tokens"),
        # four sequences' caches taken out of the pages
        _read(4096, 12, 64, "float16", 32, batch=4, ragged=True, name="read_context"),
        # four drafted tokens of one GPT-2 sequence
        _verify(4, 50257, name="verify_one"),
        # five drafted tokens of 64 sequences, the 4B model's vocabulary
        _verify(5, 151936, batch=64, ragged=True, name="verify_batch"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    top = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in top), max(w["flops"] for w in top)
    while True:
        op = rng.choice(("attention", "attention", "attention", "write", "read", "verify"))
        ragged = rng.random() < 0.7
        if op == "verify":
            c = _verify(rng.randint(1, 8), _spread(rng, 1000, 151936), batch=_spread(rng, 1, 64), ragged=ragged)
        else:
            kv = _spread(rng, 1, 32)
            head_dim = rng.choice((16, 24, 32, 40, 64, 64, 80, 96, 128, 128))
            cache, page = rng.choice(("float32", "float16", "int8", "float8")), rng.choice((16, 32, 64, 128))
            batch = _spread(rng, 1, 48)
            if op == "attention":
                tokens = rng.choice((1, rng.randint(1, 8), _spread(rng, 1, 2048)))
                c = _attention(tokens, kv * rng.choice((1, 1, 2, 4, 8)), kv, head_dim, _spread(rng, 8, 40000), cache, page,
                               batch=batch, ragged=ragged)
            elif op == "write":
                c = _write(rng.choice((1, _spread(rng, 1, 4096))), kv, head_dim, rng.randint(0, 2048), cache, page,
                           batch=batch, ragged=ragged)
            else:
                c = _read(_spread(rng, 1, 4096), kv, head_dim, cache, page, batch=batch, ragged=ragged)
        w = work(c)
        if w["bytes"] <= bytes_ and w["flops"] <= flops and (op == "verify" or max(_held(c), _scores(c)) <= 1 << 30):
            return c


def _held(c):
    """Values of the K and V rows behind all tables, in the plain form's 32 bits: a state's size."""
    return c["batch"] * c["kv_heads"] * (c["context"] + c["tokens"] + c["page"]) * c["head_dim"] * 2


def _scores(c):
    """Values of the plain form's attention scores."""
    return c["batch"] * c.get("heads", 0) * c["tokens"] * (c["context"] + c["tokens"])


def _lengths(c):
    """(mean positions before the chunk, mean rows of it) a sequence."""
    part = 0.5 if c["ragged"] else 1.0
    return part * c["context"], max(1.0, part * c["tokens"])


def work(case):
    c = case
    if c["op"] == "verify":
        # the drafted tokens' probabilities, and the rows that the last token is drawn from
        b, d = c["batch"], c["drafts"]
        return {"bytes": b * (8 * c["vocab"] + d * (8 + 8 + 4) + 8 * (d + 1)), "flops": 4 * b * c["vocab"]}
    before, new = _lengths(c)
    rows = c["batch"] * new * c["kv_heads"]
    row = 2 * c["head_dim"] * torch.empty(0, dtype=ELEMENT[c["cache"]]).element_size() + 8
    if c["op"] == "attention":
        io = 8 * c["batch"] * c["heads"] * c["tokens"] * c["head_dim"]
        keys = c["batch"] * c["heads"] * (new * before + new * (new + 1) / 2)
        return {"bytes": io + c["batch"] * c["kv_heads"] * (before + new) * row, "flops": 4 * keys * c["head_dim"]}
    dense = 8 * c["batch"] * c["tokens"] * c["kv_heads"] * c["head_dim"]
    if c["op"] == "write":   # the rows in, stored, and read back
        return {"bytes": 2 * dense + 2 * rows * row, "flops": 6 * rows * 2 * c["head_dim"]}
    return {"bytes": dense + rows * row, "flops": rows * 2 * c["head_dim"]}


# ---------------------------------------------------------------- a state

def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _power(e):
    """2**e of whole numbers, in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _to_e4m3(y):
    """Values (in 64 bits) rounded to e4m3's: nearest, ties to even."""
    _, e = torch.frexp(y)
    step = _power((e - 4).clamp(min=-9))
    return (torch.round(y / step) * step).clamp(-448, 448)


def _stored(x, cache):
    """(stored values, scales) of rows x, in 64 bits; scales as the float32 values that are kept."""
    amax = x.abs().amax(-1, keepdim=True).double()
    if cache == "int8":
        s = (amax / 127).float().double().clamp(min=TINY)
        return torch.round(x.double() / s), s
    if cache == "float8":
        s = (amax / 448).float().double().clamp(min=TINY)
        return _to_e4m3(x.double() / s), s
    _, e = torch.frexp(amax)
    s = _power(torch.where(amax > 0, e - 15, -126).clamp(min=-126))
    return (x.double() / s).to(ELEMENT[cache]).double(), s


def _sizes(c):
    hdp = (c["head_dim"] + 15) // 16 * 16
    part = c["page"] * hdp * torch.empty(0, dtype=ELEMENT[c["cache"]]).element_size()
    return hdp, part, 2 * part + 8 * c["page"]


def _pack(k, v, ks, vs, c):
    """Pages [n, bytes] of stored K and V rows [n, kv_heads, page, head_dim] and their scales."""
    n, h, page, hd = k.shape
    hdp, _, _ = _sizes(c)
    k, v = (torch.nn.functional.pad(t, (0, hdp - hd)) for t in (k, v))
    v = v.reshape(n, h, page // 8, 8, hdp).transpose(-1, -2).contiguous()
    flat = [t.to(ELEMENT[c["cache"]]).reshape(n, h, -1).view(torch.uint8) for t in (k, v)]
    flat += [t.float().reshape(n, h, -1).contiguous().view(torch.uint8) for t in (ks, vs)]
    return torch.cat(flat, -1).reshape(n, -1)


def _unpack(pages, c):
    """Stored K and V rows [n, kv_heads, page, head_dim] and their scales [.., 1] of pages [n, bytes]."""
    n, h, page, hd = pages.shape[0], c["kv_heads"], c["page"], c["head_dim"]
    hdp, part, whole = _sizes(c)
    pages = pages.reshape(n, h, whole)
    kind = ELEMENT[c["cache"]]
    k = pages[..., :part].clone().view(kind).reshape(n, h, page, hdp)[..., :hd]
    v = pages[..., part:2 * part].clone().view(kind).reshape(n, h, page // 8, hdp, 8)
    v = v.transpose(-1, -2).reshape(n, h, page, hdp)[..., :hd]
    s = pages[..., 2 * part:].clone().view(torch.float32).reshape(n, h, 2, page, 1)
    return k, v, s[:, :, 0], s[:, :, 1]


def _make(case, seed):
    """The case's tensors, from the seed alone."""
    c, dev = case, _device()
    gen = torch.Generator(dev).manual_seed(seed * 7919 + 13)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    b = c["batch"]
    if c["op"] == "verify":
        d, vocab = c["drafts"], c["vocab"]
        logits = 3.0 * randn(b, d + 1, vocab)
        target = torch.softmax(logits, -1)
        draft = torch.softmax(logits[:, :d] + 0.5 * randn(b, d, vocab), -1)
        # the drafted tokens are drawn from the draft model's probabilities
        at = draft.reshape(b * d, vocab).double().cumsum(-1)
        tokens = torch.searchsorted(at, at[:, -1:] * rand(b * d, 1).double()).clamp(max=vocab - 1).reshape(b, d)
        count = torch.randint(0, d + 1, (b,), generator=gen, device=dev) if c["ragged"] else torch.full((b,), d, device=dev)
        return {"target": target, "draft": draft, "tokens": tokens, "uniforms": rand(b, d + 1), "count": count.int()}
    t, hd, kv, page = c["tokens"], c["head_dim"], c["kv_heads"], c["page"]
    start = torch.full((b,), c["context"], device=dev)
    count = torch.full((b,), t, device=dev)
    if c["ragged"]:
        start = (start * rand(b)).long()
        count = torch.randint(1, t + 1, (b,), generator=gen, device=dev)
    wide = -(-(c["context"] + t) // page)
    n = b * wide + 3
    table = torch.randperm(n, generator=gen, device=dev)[:b * wide].reshape(b, wide)

    def rows(*shape):   # rows of different sizes
        return randn(*shape) * torch.exp(0.3 * randn(*shape[:-1], 1))

    state = {"table": table.int(), "start": start.int(), "count": count.int()}
    if c["op"] == "write":
        state |= {"k": rows(b, kv, t, hd), "v": rows(b, kv, t, hd),
                  "cache": torch.zeros(n, kv * _sizes(c)[2], dtype=torch.uint8, device=dev)}
    else:
        # every page is full: behind a sequence's end lies what an earlier one left
        pages, step = [], max(1, (1 << 26) // (kv * page * hd))
        for at in range(0, n, step):
            m = min(step, n - at)
            k, ks = _stored(rows(m, kv, page, hd), c["cache"])
            v, vs = _stored(rows(m, kv, page, hd), c["cache"])
            pages.append(_pack(k, v, ks, vs, c))
        state["cache"] = torch.cat(pages)
    if c["op"] == "attention":
        state["q"] = 1.5 * randn(b, c["heads"], t, hd)
    return state


def prepare(case, seed):
    state = {"case": case, **_make(case, seed)}
    if own:
        state["plan"], state["out"] = _plan(case, state)
    return state


# ---------------------------------------------------------------- the framework's calls

def _plan(c, t):
    """The compiled plan of the case on the state's device tensors, and its output on the device."""
    package = os.path.join(os.getcwd(), "lets-build-a-runtime_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from runtime.ir import Graph, OpType
    from runtime.session import Session

    g = Graph()
    names = [n for n in t if n not in ("case", "cache")]
    for n in names:
        g.add_tensor(n, tuple(t[n].shape), str(t[n].dtype).replace("torch.", ""))
        g.inputs.append(n)
    b = c["batch"]
    if c["op"] == "verify":
        g.add_tensor("out", (b, c["drafts"] + 1), "int64")
        g.add_node(OpType.VERIFY_DRAFT, ["target", "draft", "tokens", "uniforms", "count"], "out")
    else:
        layout = {"kv_heads": c["kv_heads"], "head_dim": c["head_dim"], "page_size": c["page"], "cache_type": c["cache"]}
        where = ["table", "start", "count"]
        g.add_state("cache", tuple(t["cache"].shape))
        cache = "cache"
        if c["op"] == "attention":
            g.add_tensor("out", tuple(t["q"].shape))
            g.add_node(OpType.PAGED_ATTENTION, ["q", "cache", *where], "out", layout)
        else:
            if c["op"] == "write":
                g.add_tensor("written", tuple(t["cache"].shape), "uint8")
                g.add_node(OpType.CACHE_WRITE, ["cache", "k", "v", *where], "written", layout)
                cache = "written"
            g.add_tensor("out", (2, b, c["kv_heads"], c["tokens"], c["head_dim"]))
            g.add_node(OpType.CACHE_READ, [cache, *where], "out", {**layout, "length": c["tokens"]})
        names.append("cache")
    g.outputs.append("out")
    session = Session(g)
    session.create(device_tensors={n: t[n] for n in names})
    return session, torch.as_tensor(session.device_outputs()["out"], device="cuda")


# ---------------------------------------------------------------- the plain forms

def _dense(s, c):
    """K and V [batch, kv_heads, positions, head_dim] of all positions behind the tables, in 32 bits."""
    table = s["table"].long()
    b, wide = table.shape
    k, v, ks, vs = _unpack(s["cache"][table.reshape(-1)], c)
    return [(x.float() * y).reshape(b, wide, c["kv_heads"], c["page"], c["head_dim"]).transpose(1, 2)
            .reshape(b, c["kv_heads"], wide * c["page"], c["head_dim"]) for x, y in ((k, ks), (v, vs))]


def _plain_attention(s, c):
    k, v = _dense(s, c)
    b, h, t, hd = s["q"].shape
    kv, g, dev = c["kv_heads"], c["heads"] // c["kv_heads"], k.device
    q = s["q"].reshape(b, kv, g * t, hd) * (1.0 / math.sqrt(hd))
    scores = torch.matmul(q, k.transpose(-1, -2)).reshape(b, kv, g, t, -1)
    row, key = torch.arange(t, device=dev), torch.arange(k.shape[2], device=dev)
    last = s["start"].long()[:, None] + row
    scores = scores.masked_fill((key > last[..., None])[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(b, kv, g * t, -1), v).reshape(b, h, t, hd)
    return torch.where((row < s["count"].long()[:, None])[:, None, :, None], out, 0.0)


def _plain_write(s, c):
    b, t = c["batch"], c["tokens"]
    at = s["start"].long()[:, None] + torch.arange(t, device=s["k"].device)
    keep = torch.arange(t, device=at.device) < s["count"].long()[:, None]
    where = at[keep]
    seq = torch.arange(b, device=at.device)[:, None].expand(b, t)[keep]
    page = s["table"].long()[seq, where // c["page"]]
    slot = where % c["page"]
    touched, back = torch.unique(page, return_inverse=True)
    parts = list(_unpack(s["cache"][touched], c))
    for j, x in enumerate((s["k"], s["v"])):
        y, scale = _stored(x.transpose(1, 2)[keep], c["cache"])   # [rows, kv_heads, head_dim]
        parts[j] = parts[j].float()
        parts[j][back, :, slot] = y.float()
        parts[2 + j][back, :, slot] = scale.float()
    s["cache"][touched] = _pack(*parts, c)


def _plain_read(s, c):
    k, v = _dense(s, c)
    at = s["start"].long()[:, None] + torch.arange(c["tokens"], device=k.device)
    keep = (torch.arange(c["tokens"], device=k.device) < s["count"].long()[:, None])[:, None, :, None]
    at = at.clamp(max=k.shape[2] - 1)[:, None, :, None].expand(-1, c["kv_heads"], -1, c["head_dim"])
    return torch.stack([torch.where(keep, x.gather(2, at), 0.0) for x in (k, v)])


def _plain_verify(s, c):
    d, dev = c["drafts"], s["target"].device
    seq = torch.arange(c["batch"], device=dev)
    p = s["target"][:, :d].gather(2, s["tokens"][..., None])[..., 0].double()
    q = s["draft"].gather(2, s["tokens"][..., None])[..., 0].double()
    stands = (s["uniforms"][:, :d].double() * q < p) & (torch.arange(d, device=dev) < s["count"].long()[:, None])
    n = stands.long().cumprod(-1).sum(-1)
    p = s["target"][seq, n].double()
    q = s["draft"][seq, n.clamp(max=d - 1)].double() * (n < s["count"])[:, None]
    rest = (p - q).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p.clamp(min=0))
    at = rest.cumsum(-1)
    drawn = (at <= s["uniforms"][:, d:].double() * at[:, -1:]).sum(-1)
    place = torch.arange(d + 1, device=dev)
    out = torch.where(place < n[:, None], torch.nn.functional.pad(s["tokens"], (0, 1)), -1)
    return torch.where(place == n[:, None], drawn[:, None], out)


def run(state):
    if own:
        state["plan"].executor.launch()
        return state["out"]
    c = state["case"]
    if c["op"] == "attention":
        return _plain_attention(state, c)
    if c["op"] == "verify":
        return _plain_verify(state, c)
    if c["op"] == "write":
        _plain_write(state, c)
    return _plain_read(state, c)


# ---------------------------------------------------------------- the definition in 64 bits

def _position(s, c, b, at, head, which):
    """Stored row and scale of one position of one head, by its byte offsets in the page."""
    hdp, part, whole = _sizes(c)
    es = part // (c["page"] * hdp)
    d = torch.arange(c["head_dim"], device=at.device)
    slot, base = at % c["page"], which * part + head * whole
    if which == 0:
        byte = (slot[:, None] * hdp + d) * es
    else:
        byte = ((slot[:, None] // 8 * hdp + d) * 8 + slot[:, None] % 8) * es
    page = s["table"][b].long()[at // c["page"]]
    byte = base + byte[..., None] + torch.arange(es, device=at.device)
    y = s["cache"][page[:, None, None], byte].view(ELEMENT[c["cache"]])[..., 0].double()
    sc = head * whole + 2 * part + which * 4 * c["page"] + 4 * slot[:, None] + torch.arange(4, device=at.device)
    return y * s["cache"][page[:, None], sc].contiguous().view(torch.float32).double()


def exact(case, seed):
    c, s = case, _make(case, seed)
    if c["op"] == "verify":
        return _exact_verify({k: v.cpu().numpy() for k, v in s.items()})
    b, t, kv = c["batch"], c["tokens"], c["kv_heads"]
    dev = s["table"].device
    start, count = s["start"].tolist(), s["count"].tolist()
    if c["op"] == "write":   # what a stored row stands for needs no pages
        out = torch.zeros(2, b, kv, t, c["head_dim"], dtype=torch.float64, device=dev)
        for j, x in enumerate((s["k"], s["v"])):
            for i in range(b):
                out[j, i, :, :count[i]] = _exact_rows(x[i, :, :count[i]].double(), c["cache"])
        return out
    if c["op"] == "read":
        out = torch.zeros(2, b, kv, t, c["head_dim"], dtype=torch.float64, device=dev)
        for i in range(b):
            at = torch.arange(start[i], start[i] + count[i], device=dev)
            for j in range(2):
                for h in range(kv):
                    out[j, i, h, :count[i]] = _position(s, c, i, at, h, j)
        return out
    g = c["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    for i in range(b):
        n = count[i]
        at = torch.arange(start[i] + n, device=dev)
        last = start[i] + torch.arange(n, device=dev)
        for h in range(kv):
            k, v = (_position(s, c, i, at, h, j) for j in range(2))
            for r in range(h * g, (h + 1) * g):
                w = s["q"][i, r, :n].double() @ k.T / math.sqrt(c["head_dim"])
                w = torch.softmax(w.masked_fill(at[None, :] > last[:, None], -math.inf), -1)
                out[i, r, :n] = w @ v
    return out


def _exact_rows(x, cache):
    """The values that a row's stored form stands for."""
    top = x.abs().amax(-1, keepdim=True)
    if cache in ("int8", "float8"):
        s = torch.clamp((top / (127 if cache == "int8" else 448)).float().double(), min=TINY)
        y = x / s
        if cache == "int8":
            low = torch.floor(y)
            up = (y - low > 0.5) | ((y - low == 0.5) & (low % 2 != 0))
            return (low + up) * s
        # neighbours in the table of e4m3's own values, the even one where both are as near
        table = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
        a = y.abs()
        hi = torch.searchsorted(table, a).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        far = (table[hi] - a) - (a - table[lo])
        at = torch.where((far < 0) | ((far == 0) & (hi % 2 == 0)), hi, lo)
        return table[at] * y.sign() * s
    s = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(top, min=1e-300))) - 14, min=-126))
    y = x / s
    return (y.half() if cache == "float16" else y.float()).double() * s


def _exact_verify(s):
    b, d = s["tokens"].shape
    out = np.full((b, d + 1), -1, np.int64)
    for i in range(b):
        n = 0
        while n < s["count"][i]:
            t = s["tokens"][i, n]
            if not float(s["uniforms"][i, n]) * float(s["draft"][i, n, t]) < float(s["target"][i, n, t]):
                break
            out[i, n] = t
            n += 1
        p = s["target"][i, n].astype(np.float64)
        rest = np.maximum(p - s["draft"][i, n].astype(np.float64), 0.0) if n < s["count"][i] else p
        if not rest.any():
            rest = p
        at = np.cumsum(rest)
        out[i, n] = np.searchsorted(at, float(s["uniforms"][i, d]) * at[-1], side="right")
    return out
