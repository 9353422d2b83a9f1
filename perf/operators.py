"""What the 8-bit cache and the attention over shared beginnings are timed and compared on: the operators of one layer of
a serving step, from the tensors that a step has in hand to the ones that it passes on.

  write      queries and keys normed and rotated, keys and values quantised into the pages of the cache (one scale per
             token and kv head, a power of two), and the touched pages read back in bfloat16, as a prompt's attention does
  attention  rows that bring one token each, and at most one that brings a portion of its prompt, over an 8-bit cache
  shared     rows of one token whose first pages are the same ones (a system prompt, several samples of one prompt)

A page holds, per part (keys, values) and kv head, `page` rows of `dim` codes (8-bit floats with four bits of exponent and
three of fraction) and behind them one byte per row, the exponent of the row's scale plus 127: uint8
[pages, 2, kv_heads, page, dim + 1]. A value is its code times the scale. With `fp8` false a `shared` case keeps a
bfloat16 cache [pages, 2, kv_heads, page, dim].
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6
LOW, HIGH = -64, 120                            # exponents that a row's scale may have


# ---------------------------------------------------------------- the cases
def _write(name, tokens, rows, heads, kv_heads, dim, page, rotary, norm=True, before=0):
    """`tokens` new tokens of `rows` requests (portions of unequal lengths) that hold up to `before` tokens already."""
    return {"name": name, "op": "write", "tokens": tokens, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "rotary": rotary, "norm": norm, "before": before}


def _attention(name, rows, portion, length, heads, kv_heads, dim, page, window=0, sink=False, ragged=True):
    """`rows` rows of one token and, with `portion` > 0, one more that brings so many; requests hold up to `length` tokens."""
    return {"name": name, "op": "attention", "rows": rows, "portion": portion, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "sink": sink, "ragged": ragged}


def _shared(name, groups, members, prefix, tail, heads, kv_heads, dim, page, fp8, sink=False):
    """`groups` groups of `members` rows; the rows of a group share their first tokens (up to `prefix`), and each holds up
    to `tail` tokens of its own behind them."""
    return {"name": name, "op": "shared", "groups": groups, "members": members, "prefix": prefix, "tail": tail, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "fp8": fp8, "sink": sink}


def listed():
    return [
        _write("write one token", 1, 1, 16, 8, 128, 64, 128, before=700),              # one request decodes on a small model
        _write("write prompts 4096", 4096, 3, 32, 8, 128, 64, 128),                    # the engine's largest step of prompts
        _write("write 333 of dim 96", 333, 5, 6, 2, 96, 16, 48, norm=False, before=90),   # an odd head size, half of it turned
        _attention("one row 400", 1, 0, 400, 16, 8, 128, 64),                          # the start of an answer
        _attention("8 rows 8192", 8, 0, 8192, 32, 8, 128, 64, ragged=False),           # the benchmark's decode batch
        _attention("64 rows to 4096", 64, 0, 4096, 32, 8, 128, 64),                    # a full batch of unequal requests
        _attention("portion 1536 at 6144", 3, 1536, 6144, 32, 8, 128, 64),             # a prompt's portion beside decoding rows
        _attention("window, sink, dim 64", 24, 0, 2000, 8, 2, 64, 16, window=512, sink=True),
        _shared("4 on 1024", 1, 4, 1024, 130, 16, 8, 128, 64, fp8=False),              # four samples of one prompt
        _shared("64 on 8192, fp8", 1, 64, 8192, 256, 32, 8, 128, 64, fp8=True),        # a long system prompt, a full batch
        _shared("6 groups of 8 to 4096", 6, 8, 4096, 500, 32, 8, 128, 64, fp8=False),  # several prompts, eight samples each
        _shared("32 on 16384", 1, 32, 16384, 300, 32, 8, 128, 64, fp8=False, sink=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("write", "attention", "shared"))
    dim = rng.choice((32, 64, 80, 96, 128, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 6, 8))
    page = rng.choice((16, 32, 64, 64, 128))
    budget = 4096 * 8 * 128 / (kv_heads * dim)                       # tokens that cost what the largest listed case's do
    if op == "write":
        tokens = _log(rng, 1, min(4096, budget * 8 * 4 / heads))
        return {k: v for k, v in _write("", tokens, rng.randint(1, min(8, tokens)), heads, kv_heads, dim, page,
                                        rng.choice((0, dim // 2, dim, dim)), rng.random() < 0.7, rng.choice((0, 5, 700))).items() if k != "name"}
    if op == "attention":
        length = _log(rng, 1, 8192)
        rows = _log(rng, 1, max(1, min(64, 8 * budget / length)))
        most = min(1536, length, 1536 * 6144 * 4096 // (length * heads * dim))
        portion = _log(rng, 2, most) if most >= 2 and rng.random() < 0.4 else 0
        window = _log(rng, 1, length) if rng.random() < 0.25 else 0
        case = _attention("", rows, portion, length, heads, kv_heads, dim, page, window, rng.random() < 0.3, rng.random() < 0.8)
    else:
        prefix = max(page, _log(rng, 64, 16384) // page * page)
        members = _log(rng, 2, 64)
        groups = rng.randint(1, max(1, min(6, 64 // members, int(16384 // prefix))))
        while groups * members * prefix * max(heads, 4 * kv_heads) * dim > 32 * 16384 * 32 * 128 and members > 2:
            members -= 1
        case = _shared("", groups, members, prefix, _log(rng, 1, 600), heads, kv_heads, dim, page, rng.random() < 0.5, rng.random() < 0.3)
    return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------- a case's rows, from its sizes alone
def _part(i, most, ragged=True):
    """The i-th of a run of lengths up to `most`, spread unevenly over the range."""
    return max(1, round(most * (1 - 0.85 * ((i * 0.6180339887) % 1.0)))) if ragged else most


def _rows(c):
    """(tokens held after the step, new tokens, group, pages shared with the group) of each row."""
    if c["op"] == "write":
        share = [1 + (i * 0.6180339887) % 1.0 for i in range(c["rows"])]                     # one token each, the rest unevenly
        cut = [i + round((c["tokens"] - c["rows"]) * sum(share[:i]) / sum(share)) for i in range(c["rows"] + 1)]
        new = [b - a for a, b in zip(cut, cut[1:])]
        return [(n + (_part(i, c["before"]) if c["before"] else 0), n, 0, 0) for i, n in enumerate(new)]
    if c["op"] == "attention":
        rows = [(_part(i, c["length"], c["ragged"]), 1, 0, 0) for i in range(c["rows"])]
        return rows + ([(c["length"], c["portion"], 0, 0)] if c["portion"] else [])
    rows = []
    for g in range(c["groups"]):
        pages = max(1, _part(g, c["prefix"]) // c["page"])
        rows += [(pages * c["page"] + _part(g + 3 * i, c["tail"]), 1, g, pages) for i in range(c["members"])]
    return rows


def _sizes(c):
    """(query tokens, key tokens that must be read, (query, key) pairs)."""
    window, tokens, keys, pairs, seen = c.get("window", 0), 0, 0, 0, set()
    for n, new, g, pages in _rows(c):
        first = n - new
        tokens += new
        lo = max(0, first - window + 1) if window else 0
        keys += n - lo - pages * c["page"]
        if pages and g not in seen:
            seen.add(g)
            keys += pages * c["page"]
        pairs += sum(min(p + 1, window) for p in range(first, n)) if window else (first + 1 + n) * new // 2
    return tokens, keys, pairs


def work(c):
    tokens, keys, pairs = _sizes(c)
    heads, kvh, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "write":
        pages = sum(-(-n // c["page"]) for n, *_ in _rows(c))
        whole = pages * 2 * kvh * c["page"]
        moved = tokens * ((2 * heads + 2 * kvh) * dim * 2 + 4 * c["rotary"] + 2 * kvh * (dim + 1)) + whole * (dim + 1 + 2 * dim)
        return {"bytes": moved, "flops": tokens * (heads + kvh) * dim * 8 + tokens * kvh * dim * 4}
    kept = dim + 1 if c.get("fp8", True) else 2 * dim
    return {"bytes": tokens * heads * dim * 4 + keys * 2 * kvh * kept, "flops": 4 * heads * dim * pairs}


# ---------------------------------------------------------------- a step's tensors
def _power(e):
    """2^e in 32 bits, made from its bits."""
    return ((e + 127).int() << 23).view(torch.float32)


def _quantised(x):
    """Rows of 32-bit numbers as (codes uint8 [..., dim], exponents [...]): the smallest power of two that brings the
    row's largest finite magnitude to 448 or below, the largest number that a code stands for."""
    largest = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(largest)                                       # largest = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(LOW, HIGH)
    e = torch.where(largest == 0, LOW, e)
    codes = (x * _power(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), e


def _pack(codes, e):
    """[pages, 2, kv_heads, page, dim] codes and their rows' exponents in the layout of the cache's pages."""
    p, two, kvh, page, dim = codes.shape
    block = torch.cat([codes.reshape(p, two, kvh, page * dim), (e + 127).to(torch.uint8)], -1)
    return block.view(p, two, kvh, page, dim + 1)


def _values(kv):
    """The 32-bit values [pages, 2, kv_heads, page, dim] that pages stand for."""
    if kv.dtype != torch.uint8:
        return kv.float()
    p, two, kvh, page, d1 = kv.shape
    block = kv.reshape(p, two, kvh, page * d1)
    codes = block[..., :page * (d1 - 1)].contiguous().view(torch.float8_e4m3fn).view(p, two, kvh, page, d1 - 1).float()
    return codes * _power(block[..., page * (d1 - 1):].int() - 127)[..., None]


def prepare(c, seed):
    g = torch.Generator(DEVICE).manual_seed(int(seed) * 1000003 + 17)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)             # noqa: E731
    heads, kvh, dim, page, rows = c["heads"], c["kv_heads"], c["dim"], c["page"], _rows(c)
    need, first_page = [], {}
    count = 0
    for n, new, group, pages in rows:                                # pages in the order of the rows; shared ones once
        if pages and group not in first_page:
            first_page[group] = count
            count += pages
        start = first_page.get(group, 0)
        have = list(range(start, start + pages))
        mine = -(-n // page) - pages
        need.append(have + list(range(count, count + mine)))
        count += mine
    shuffle = torch.randperm(count, generator=torch.Generator().manual_seed(int(seed)))
    width = max(len(p) for p in need)
    table = torch.full((len(rows), width), count, dtype=torch.int32)  # unused cells name the pool's last page, which holds zeros
    for i, p in enumerate(need):
        table[i, :len(p)] = shuffle[p].int()
    new = [r[1] for r in rows]
    start = torch.tensor([0] + new).cumsum(0).int()
    held = torch.tensor([r[0] for r in rows], dtype=torch.int32)
    spread = (0.3 * rand(2, kvh, 1, dim)).exp()                       # channels of unequal size, a few of them large
    spread[0, :, :, ::37] *= 4
    s = {"case": dict(c), "table_host": table, "table": table.to(DEVICE), "start_host": start, "start": start.to(DEVICE),
         "held_host": held, "held": held.to(DEVICE), "slots": torch.arange(len(rows), dtype=torch.int32, device=DEVICE),
         "scale": dim ** -0.5, "tokens": int(start[-1])}
    if c.get("fp8", True):
        kv = torch.zeros(count + 1, 2, kvh, page, dim + 1, dtype=torch.uint8, device=DEVICE)
    else:
        kv = torch.zeros(count + 1, 2, kvh, page, dim, dtype=torch.bfloat16, device=DEVICE)
    for a in range(0, count, 1024):
        b = min(count, a + 1024)
        x = rand(b - a, 2, kvh, page, dim) * spread
        kv[a:b] = _pack(*_quantised(x)) if c.get("fp8", True) else x.bfloat16()
    s["kv"] = kv
    if c["op"] == "write":
        t = s["tokens"]
        row = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(new))
        at = torch.cat([torch.arange(n - k, n) for n, k, *_ in rows])
        rotary = c["rotary"]
        angle = torch.arange(4096 + 704, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, max(rotary, 2), 2, dtype=torch.float64) / max(rotary, 2))
        s |= {"qkv": (rand(t, heads + 2 * kvh, dim) * torch.cat([spread[0, :1, 0].expand(heads, dim), spread[0, :, 0], spread[1, :, 0]])
                      ).bfloat16().view(t, -1),
              "positions": at.int().to(DEVICE), "write": (table[row, at // page].long() * page + at % page).int().to(DEVICE),
              "turn": torch.cat([angle.cos(), angle.sin()], -1).float().to(DEVICE) if rotary else None,
              "q_gain": (1 + 0.1 * rand(dim)).bfloat16() if c["norm"] else None, "k_gain": (1 + 0.1 * rand(dim)).bfloat16() if c["norm"] else None,
              "touched": shuffle.int().to(DEVICE)}
    else:
        s["q"] = (2.0 * rand(s["tokens"], heads, dim) / spread[0, :, 0].repeat_interleave(heads // kvh, 0)).bfloat16()
        s["sinks"] = rand(heads) if c["sink"] else None
    return s


# ---------------------------------------------------------------- the plain forms
def _turned(x, s, gain):
    """Heads [tokens, n, dim] in 32 bits: RMS norm with `gain`, then the rotation of the first `rotary` numbers."""
    if gain is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain.float()
    r = s["case"]["rotary"]
    if r:
        half = r // 2
        cs = s["turn"][s["positions"].long()][:, None]
        a, b, cos, sin = x[..., :half], x[..., half:r], cs[..., :half], cs[..., half:]
        x = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    return x


def _plain_write(s):
    c = s["case"]
    heads, kvh, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].float().view(-1, heads + 2 * kvh, dim)
    q = _turned(x[:, :heads], s, s["q_gain"])
    new = torch.stack([_turned(x[:, heads:heads + kvh], s, s["k_gain"]), x[:, heads + kvh:]], 1)      # [tokens, 2, kv_heads, dim]
    codes, e = _quantised(new)
    new = codes.view(torch.float8_e4m3fn).float() * _power(e)[..., None]
    pages = _values(s["kv"])
    at = s["write"].long()
    pages[at // page, :, :, at % page] = new
    return q.bfloat16(), pages[s["touched"].long()].bfloat16()


def _plain_attention(s):
    """Every row's keys gathered, all scores at once."""
    c = s["case"]
    heads, kvh, dim, window = c["heads"], c["kv_heads"], c["dim"], c.get("window", 0)
    start, held = s["start"].long(), s["held"].long()
    new = start[1:] - start[:-1]
    rows = len(held)
    most, page = int((s["start_host"][1:] - s["start_host"][:-1]).max()), c["page"]
    length = s["table"].shape[1] * page
    outs = torch.empty_like(s["q"])
    cuts = [(0, rows)] if most == 1 else [(0, rows - 1), (rows - 1, rows)]       # rows of one token; the row of a portion
    for a, b in [cut for cut in cuts if cut[1] > cut[0]]:
        kv = _values(s["kv"][s["table"][a:b].long().flatten()]).view(b - a, -1, 2, kvh, page, dim)
        keys, vals = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, b - a, kvh, length, dim)
        here = int(s["start_host"][b]) - int(s["start_host"][a])
        per = here // (b - a)                                         # query tokens of each of these rows
        q = s["q"][int(s["start_host"][a]):int(s["start_host"][b])].float().view(b - a, per, kvh, heads // kvh, dim)
        q = q.permute(0, 2, 3, 1, 4).reshape(b - a, kvh, -1, dim)     # [rows, kv_heads, group * per, dim]
        scores = (q @ keys.transpose(-1, -2)).view(b - a, heads, per, length) * s["scale"]
        pos = (held[a:b] - new[a:b])[:, None] + torch.arange(per, device=DEVICE)
        j = torch.arange(length, device=DEVICE)
        sees = j <= pos[..., None]
        if window:
            sees &= pos[..., None] - j < window
        scores = scores.masked_fill(~sees[:, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            top = torch.maximum(top, s["sinks"][None, :, None, None])
        w = (scores - top).exp()
        total = w.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            total = total + (s["sinks"][None, :, None, None] - top).exp()
        o = (w.view(b - a, kvh, -1, length) @ vals).view(b - a, heads, per, dim) / total
        outs[int(s["start_host"][a]):int(s["start_host"][b])] = o.transpose(1, 2).reshape(here, heads, dim).to(outs.dtype)
    return outs


# ---------------------------------------------------------------- the framework's calls
def _kernels():
    from holon_b200.kernels import load_kernels
    if "kernels" not in _loaded:
        _loaded["kernels"] = load_kernels(DEVICE)
    return _loaded["kernels"]


_loaded: dict = {}


def _step(s):
    """What the step function lays out once for all layers of a step: its rows, and which of them share pages."""
    from holon_b200.engine.batch import Rows, SharedPrefix
    if "rows" not in s:
        starts, held = s["start_host"].numpy(), s["held_host"].numpy()
        new = starts[1:] - starts[:-1]
        ones = int((new == 1).sum())
        s["rows"] = Rows(s["slots"], s["start"], s["held"], len(held), s["tokens"], ones, int(new.max()), int(held.max()), starts, held)
        s["shared"] = SharedPrefix.of(s["table_host"].numpy()[:ones], held[:ones], s["case"]["page"], DEVICE) \
            if s["case"]["op"] == "shared" else None
    return s["rows"], s["shared"]


def _own_write(s):
    k, c = _kernels(), s["case"]
    q = torch.empty(s["tokens"], c["heads"], c["dim"], dtype=torch.bfloat16, device=DEVICE)
    k.qk_norm_rope_kv_write(q, s["qkv"], s["positions"], s["turn"], c["rotary"], s["q_gain"], s["k_gain"], EPS, 0.0, s["kv"],
                            s["write"], c["heads"], c["kv_heads"], c["dim"])
    pages = torch.empty(len(s["touched"]), 2, c["kv_heads"], c["page"], c["dim"], dtype=torch.bfloat16, device=DEVICE)
    k.kv_read(pages, s["kv"], s["touched"])
    return q, pages


def _own_attention(s):
    k, c = _kernels(), s["case"]
    rows, shared = _step(s)
    out = torch.empty_like(s["q"])
    k.paged_attention(out, s["q"], s["kv"], s["table"], rows, s["scale"], c.get("window", 0), s["sinks"], shared=shared)
    return out


def run(s):
    if own:
        return _own_write(s) if s["case"]["op"] == "write" else _own_attention(s)
    return _plain_write(s) if s["case"]["op"] == "write" else _plain_attention(s)


# ---------------------------------------------------------------- from the definition, in 64 bits
def _code_values():
    """The 256 numbers that codes stand for: sign, exponent of 7 less, fraction of eighths; 127 and 255 are no numbers."""
    out = []
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        v = math.ldexp(f / 8, -6) if e == 0 else math.ldexp(1 + f / 8, e - 7)
        out.append(math.nan if b & 127 == 127 else -v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEVICE)


def _exact_pages(kv, pages):
    """[pages, 2, kv_heads, page, dim] in 64 bits."""
    kv = kv[pages.long()]
    if kv.dtype != torch.uint8:
        return kv.double()
    n, two, kvh, page, d1 = kv.shape
    flat = kv.reshape(n, two, kvh, -1).long()
    scale = 2.0 ** (flat[..., page * (d1 - 1):].double() - 127)
    return _code_values()[flat[..., :page * (d1 - 1)]].view(n, two, kvh, page, d1 - 1) * scale[..., None]


def _exact_write(c, s):
    heads, kvh, dim, page, r = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rotary"]
    x = s["qkv"].double().view(-1, heads + 2 * kvh, dim).clone()
    for a, b, gain in ((0, heads, s["q_gain"]), (heads, heads + kvh, s["k_gain"])):
        if gain is not None:
            x[:, a:b] = x[:, a:b] / torch.sqrt(torch.mean(x[:, a:b] ** 2, -1, keepdim=True) + EPS) * gain.double()
    if r:
        cs = s["turn"].double()[s["positions"].long()].view(-1, 1, 2, r // 2)
        z = torch.complex(x[:, :heads + kvh, :r // 2].contiguous(), x[:, :heads + kvh, r // 2:r].contiguous()) * torch.complex(cs[:, :, 0].contiguous(), cs[:, :, 1].contiguous())
        x[:, :heads + kvh, :r // 2], x[:, :heads + kvh, r // 2:r] = z.real, z.imag
    new = x[:, heads:].view(-1, 2, kvh, dim)
    largest = new.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(largest / 448)).clamp(LOW, HIGH)
    e = torch.where(largest / 448 <= 2.0 ** (e - 1), e - 1, e).clamp(LOW, HIGH)          # (a logarithm that was rounded up)
    y = new / 2.0 ** e
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    step = torch.where(y.abs() / step >= 16, step * 2, torch.where((y.abs() / step < 8) & (step > 2.0 ** -9), step / 2, step))
    new = torch.round(y / step) * step * 2.0 ** e
    pages = _exact_pages(s["kv"], torch.arange(s["kv"].shape[0], device=DEVICE))
    at = s["write"].long()
    pages[at // page, :, :, at % page] = new
    return x[:, :heads], pages[s["touched"].long()]


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "write":
        return _exact_write(c, s)
    heads, kvh, dim, page, window = c["heads"], c["kv_heads"], c["dim"], c["page"], c.get("window", 0)
    out = torch.empty(s["tokens"], heads, dim, dtype=torch.float64, device=DEVICE)
    for b, (n, new, *_) in enumerate(_rows(c)):
        a = int(s["start_host"][b])
        kv = _exact_pages(s["kv"], s["table"][b, :-(-n // page)])
        pos = torch.arange(n - new, n, device=DEVICE)[:, None]
        j = torch.arange(n, device=DEVICE)[None]
        hidden = (j > pos) | ((j <= pos - window) if window else torch.zeros_like(j, dtype=torch.bool))
        for h in range(kvh):
            keys, vals = (kv[:, part, h].reshape(-1, dim)[:n] for part in (0, 1))
            for i in range(h * heads // kvh, (h + 1) * heads // kvh) if new > 1 else (slice(h * heads // kvh, (h + 1) * heads // kvh),):
                q = s["q"][a:a + new, i].double().reshape(-1, dim)
                scores = torch.where(hidden, -math.inf, q @ keys.T * s["scale"])
                total = torch.logsumexp(scores, -1)
                if s["sinks"] is not None:
                    total = torch.logaddexp(total, s["sinks"][i].double().expand_as(total))
                out[a:a + new, i] = (torch.exp(scores - total[:, None]) @ vals).view(out[a:a + new, i].shape)
    return out
