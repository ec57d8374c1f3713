"""Operators of the paged 4-bit key/value cache, as cases that can be timed.

Three operators that share one cache (its layout is in include/s2p_b200_ext.h, "paged 4-bit cache"):

  append     norms of queries and keys for each head and the position rotation in one pass over a tick's raw q|k|v rows; queries
             come out in bf16, keys and values go into the sequences' pages in 4 bits.  The rows are then read back.
  attention  causal attention of a batch of ragged sequences over their pages: single tokens, prompt slices, both at once.
  pages      what a scheduler does between ticks: sequences fork from a voice's prefix, give their pages back, grow, and the pool is
             compacted so that its used part is contiguous again.

A position of one kv head is 160 bytes: 128 codes of 4 bits for the key and as many for the value, and for each group of 32
channels a scale s and a smallest value m in f16; a code c stands for s c + m.
"""
import ctypes as C
import importlib
import math

import torch

own = False

DIM = 128                 # width of a head
PAGE = 64                 # positions of a page
BLOCK = 16                # positions that lie together
TOKEN_BYTES = 160
EPS, ROPE_BASE = 1e-6, 1000000.0
ALIGNED = 64              # table columns are rounded up to this


def listed():
    return [
        # one listener's next token, in a layer
        {"name": "append_1row", "kind": "append", "n": 1, "len": 513, "rows": 1, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # the lockstep tick of a server with long contexts
        {"name": "append_batch32", "kind": "append", "n": 32, "len": 8192, "rows": 1, "prompts": 32, "q_heads": 32, "kv_heads": 8},
        # a slice of a long document beside seven listeners' tokens
        {"name": "append_slice2048", "kind": "append", "n": 8, "len": 8100, "rows": 2048, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # one listener at the start of a read
        {"name": "attn_1x512", "kind": "attention", "n": 1, "len": 512, "rows": 1, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # one listener deep in a long read
        {"name": "attn_1x8000", "kind": "attention", "n": 1, "len": 8000, "rows": 1, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # a server with long contexts
        {"name": "attn_32x8192", "kind": "attention", "n": 32, "len": 8192, "rows": 1, "prompts": 32, "q_heads": 32, "kv_heads": 8},
        # a full server with short ones
        {"name": "attn_128x1024", "kind": "attention", "n": 128, "len": 1024, "rows": 1, "prompts": 128, "q_heads": 32, "kv_heads": 8},
        # a short sentence behind a cached voice
        {"name": "attn_slice77", "kind": "attention", "n": 1, "len": 1101, "rows": 77, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # the last slice of a long document
        {"name": "attn_slice2048", "kind": "attention", "n": 1, "len": 8100, "rows": 2048, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # a request's slice in the same tick as fifteen listeners' tokens
        {"name": "attn_mixed", "kind": "attention", "n": 16, "len": 1500, "rows": 512, "prompts": 1, "q_heads": 32, "kv_heads": 8},
        # requests that start from two cached voices, over all layers of the model
        {"name": "pages_fork", "kind": "fork", "n": 24, "len": 1101, "layers": 36, "kv_heads": 8},
        # half of the sequences end, the pool is compacted, as many new ones begin
        {"name": "pages_turnover", "kind": "turnover", "n": 16, "len": 700, "layers": 36, "kv_heads": 8},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "attention", "fork", "turnover"))
    if kind in ("fork", "turnover"):
        n = _spread(rng, 2, 24) if kind == "fork" else 2 * _spread(rng, 1, 8)
        return {"kind": kind, "n": n, "len": _spread(rng, 65, 900 if kind == "fork" else 600), "layers": _spread(rng, 2, 36), "kv_heads": rng.choice((4, 8, 8))}
    q_heads, kv_heads = rng.choice(((32, 8), (32, 8), (32, 8), (16, 8), (8, 8), (64, 8), (32, 2)))
    form = rng.choice(("tokens", "tokens", "slice", "mixed"))
    if form == "tokens":
        n = _spread(rng, 1, 128)
        length = _spread(rng, 1, min(16384, 32 * 8192 * 8 // (n * max(kv_heads, q_heads // 4))))
        return {"kind": kind, "n": n, "len": length, "rows": 1, "prompts": n, "q_heads": q_heads, "kv_heads": kv_heads}
    n = 1 if form == "slice" else _spread(rng, 2, 16)
    rows = _spread(rng, 2, 1024 if form == "slice" else 512)
    length = rows + _spread(rng, 1, 4096 if form == "slice" else 1024)
    return {"kind": kind, "n": n, "len": length, "rows": rows, "prompts": 1, "q_heads": q_heads, "kv_heads": kv_heads}


def _lens(case):
    """Positions that each sequence holds, the rows of this pass among them: ragged, the first the longest."""
    n, top = case["n"], case["len"]
    return [max(1, top - (i * 613) % max(1, top // 3)) for i in range(n)]


def _rows(case):
    """Rows of each sequence in this pass: `prompts` of them bring `rows`, the others one token."""
    return [min(t, case["rows"] if i < case["prompts"] else 1) for i, t in enumerate(_lens(case))]


def _voices(case):
    """Positions of the two voices that requests fork from."""
    return [case["len"], max(3, case["len"] - PAGE // 2)]


def _pages_of(t):
    return -(-t // PAGE)


def work(case):
    """Each input read once and each output written once."""
    lens = _lens(case)
    if case["kind"] in ("fork", "turnover"):
        page = case["layers"] * case["kv_heads"] * PAGE * TOKEN_BYTES
        if case["kind"] == "fork":
            lens = _voices(case)
            moved = sum((lens[i % 2] - (i // 2) % 3) % PAGE > 0 for i in range(case["n"]))
        else:
            moved = min(sum(map(_pages_of, lens[0::2])), sum(map(_pages_of, lens[1::2])))
        return {"bytes": 2 * moved * page + 4 * sum(map(_pages_of, lens)), "flops": 0}
    rows, hq, hk = _rows(case), case["q_heads"], case["kv_heads"]
    r = sum(rows)
    if case["kind"] == "append":
        raw, back = r * (hq + 2 * hk) * DIM * 2, 2 * r * hk * DIM * 2
        return {"bytes": raw + r * hq * DIM * 2 + 2 * r * hk * TOKEN_BYTES + back, "flops": r * (hq + 2 * hk) * DIM * 10}
    seen = sum(q * t - q * (q - 1) // 2 for q, t in zip(rows, lens))
    return {"bytes": sum(lens) * hk * TOKEN_BYTES + 2 * r * hq * DIM * 2, "flops": 4 * seen * hq * DIM}


# ---- the layout of a block of 16 positions --------------------------------------------------------------------------------

def _layout():
    """For each of a block's 2560 bytes, where it stands when the positions' 160 bytes are put one behind the other."""
    at = [0] * (BLOCK * TOKEN_BYTES)
    for tok in range(BLOCK):
        for b in range(64):
            at[tok * 64 + b] = tok * TOKEN_BYTES + b
            g, w = divmod(b, 8)
            at[1024 + (tok >> 3) * 512 + g * 64 + ((tok >> 1) & 3) * 16 + (tok & 1) * 8 + w] = tok * TOKEN_BYTES + 64 + b
        for b in range(16):
            at[2048 + tok * 16 + b] = tok * TOKEN_BYTES + 128 + b
            half, which = divmod(b, 8)
            group, byte = divmod(which, 2)
            at[2304 + half * 128 + (tok >> 1) * 16 + group * 4 + (tok & 1) * 2 + byte] = tok * TOKEN_BYTES + 144 + b
    return at


def _key_channels():
    return [32 * j + 8 * t + i for t in range(4) for j in range(4) for i in range(8)]


def _value_channels():
    return [32 * j + 4 * g + i for g in range(8) for j in range(4) for i in range(4)]


_tables = {}


def _table(name, device):
    """The layout's permutations on the GPU: they are the cache's format, not of any input."""
    if (name, device) not in _tables:
        made = {"block": _layout, "key": _key_channels, "value": _value_channels}[name.split("_")[0]]()
        t = torch.tensor(made, device=device)
        _tables[name, device] = torch.argsort(t) if name.endswith("_back") else t
    return _tables[name, device]


def _quantise(x):
    """Codes, scales and smallest values of groups of 32 channels of x [..., 128] in 32 bits."""
    g = x.clamp(-65504.0, 65504.0).unflatten(-1, (4, 32))
    low = g.amin(-1)
    s = ((g.amax(-1) - low) / 15.0).half()
    m = low.half()
    step = s.float()[..., None]
    c = torch.where(step > 0, ((g - m.float()[..., None]) / step).round().clamp(0, 15), torch.zeros_like(g))
    return c.to(torch.uint8).flatten(-2), s, m


def _token_bytes(k, v):
    """The 160 bytes of each position and head, from keys and values [..., 128] in 32 bits."""
    (kc, ks, km), (vc, vs, vm) = _quantise(k), _quantise(v)
    kc, vc = kc[..., _table("key", k.device)], vc[..., _table("value", k.device)]
    pair = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    return torch.cat([pair(kc), pair(vc)] + [p.contiguous().view(torch.uint8) for p in (ks, km, vs, vm)], -1)


def _token_values(raw):
    """Keys and values [..., 128] in 32 bits from the positions' 160 bytes."""
    part = lambda a, b: raw[..., a:b].contiguous()  # noqa: E731
    codes = lambda p: torch.stack([p & 15, p >> 4], -1).flatten(-2).float()  # noqa: E731
    par = part(128, 160).view(torch.float16).float().unflatten(-1, (4, 4))
    value = lambda c, s, m: (c.unflatten(-1, (4, 32)) * s[..., None] + m[..., None]).flatten(-2)  # noqa: E731
    k = codes(part(0, 64))[..., _table("key_back", raw.device)]
    v = codes(part(64, 128))[..., _table("value_back", raw.device)]
    return value(k, par[..., 0, :], par[..., 1, :]), value(v, par[..., 2, :], par[..., 3, :])


def _blocks(tokens):
    """[..., 16 m, 160] bytes of positions as [..., m, 2560] bytes of blocks."""
    return tokens.unflatten(-2, (-1, BLOCK)).flatten(-2)[..., _table("block", tokens.device)]


def _tokens(blocks):
    """The inverse of _blocks."""
    return blocks[..., _table("block_back", blocks.device)].unflatten(-1, (BLOCK, TOKEN_BYTES)).flatten(-3, -2)


# ---- what a program has in hand ---------------------------------------------------------------------------------------------

def _cache_values(g, n, heads, length):
    """Keys and values as a model caches them: normed keys with a few strong channels, values of unequal heads."""
    shape = (n, heads, length, DIM)
    k = torch.randn(shape, device="cuda", generator=g) * (0.6 + torch.rand(heads, 1, DIM, device="cuda", generator=g))
    v = torch.randn(shape, device="cuda", generator=g) * (0.3 + torch.rand(heads, 1, 1, device="cuda", generator=g))
    return k, v


def _describe(s, layers, kv_heads, q_heads, rows):
    """The library's descriptors of the cache and the batch: pointers and sizes, and a zeroed workspace."""
    capi = importlib.import_module("s2pro-native_b200.capi")
    s["lib"], s["capi"] = capi.load_library(), capi
    p = lambda t: t.data_ptr()  # noqa: E731
    cache = capi.Kv4(p(s["pages"]), p(s["table"]), p(s["lens"]), p(s["refs"]), None, 0, s["refs"].numel(), layers, kv_heads, q_heads, s["table"].shape[0], s["table"].shape[1])
    size = s["lib"].s2p_b200_kv4_work_bytes(C.byref(cache), rows)
    s["work"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
    cache.work, cache.work_bytes = s["work"].data_ptr(), size
    s["cache"] = cache
    if "row0" in s:
        s["batch"] = capi.Kv4Batch(p(s["seqs"]), p(s["row0"]), p(s["pos0"]), s["seqs"].numel(), rows, s["max_rows"])
    s["stream"] = torch.cuda.current_stream().cuda_stream


def _prepare_pages(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, n, width = _lens(case), case["n"], case["layers"] * case["kv_heads"] * PAGE * TOKEN_BYTES
    fork = case["kind"] == "fork"
    if fork:  # two voices at the head of the pool's sequences, the others empty
        lens = _voices(case)
    seqs = n + 2 if fork else n
    held = [_pages_of(t) for t in lens]
    spare = 2 * n + 5 if fork else max(held) + 3
    pages = sum(held) + spare
    stride = -(-max(held) // ALIGNED) * ALIGNED
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    s = {"kind": case["kind"], "turn": 0}
    s["pages"] = torch.randint(-(1 << 62), 1 << 62, (pages, width // 8), device="cuda", generator=g)
    s["table"] = torch.full((seqs, stride), -1, dtype=torch.int32, device="cuda")
    s["lens"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, h in enumerate(held):
        s["table"][i, :h] = order[at:at + h]
        s["lens"][i] = lens[i]
        at += h
    s["refs"][order[:at].long()] = 1
    s["info"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    if fork:  # every request shares all of its voice but a few last tokens of its own choice
        s["parents"], s["children"] = [i % 2 for i in range(n)], [2 + i for i in range(n)]
        s["tokens"] = [lens[i % 2] - (i // 2) % 3 for i in range(n)]
    else:
        s["halves"] = [list(range(h, n, 2)) for h in (0, 1)]
        s["grow"] = []
        for half in s["halves"]:
            row0 = [0]
            for i in half:
                row0.append(row0[-1] + lens[i])
            t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
            s["grow"].append({"seqs": t(half), "row0": t(row0), "pos0": t([0] * len(half)), "rows": row0[-1], "max_rows": max(lens[i] for i in half)})
    if own:
        _describe(s, case["layers"], case["kv_heads"], case["kv_heads"], 1)
        lists = lambda v: (C.c_int32 * len(v))(*v)  # noqa: E731
        if fork:
            s["lists"] = [lists(s[k]) for k in ("parents", "children", "tokens")]
        else:
            s["lists"] = [lists(h) for h in s["halves"]]
            s["batches"] = [s["capi"].Kv4Batch(b["seqs"].data_ptr(), b["row0"].data_ptr(), b["pos0"].data_ptr(), b["seqs"].numel(), b["rows"], b["max_rows"]) for b in s["grow"]]
    return s


def prepare(case, seed):
    if case["kind"] in ("fork", "turnover"):
        return _prepare_pages(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, rows, n, hq, hk = _lens(case), _rows(case), case["n"], case["q_heads"], case["kv_heads"]
    total, r = [_pages_of(t) for t in lens], sum(rows)
    pages = sum(total) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    stride = -(-max(total) // ALIGNED) * ALIGNED
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"kind": case["kind"], "max_len": max(lens), "max_rows": max(rows), "rows": r, "hq": hq, "hk": hk}
    s["row0"] = dev([sum(rows[:i]) for i in range(n + 1)])
    s["pos0"] = dev([t - q for t, q in zip(lens, rows)])
    s["seqs"] = torch.randperm(n, device="cuda", generator=g).to(torch.int32)
    s["table"] = torch.full((n, stride), -1, dtype=torch.int32, device="cuda")
    s["lens"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    s["lens"][s["seqs"].long()] = dev(lens)
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
    s["refs"][order[:pages - 3].long()] = 1
    place = torch.full((n, stride), -1, dtype=torch.int32)
    at = 0
    for i, t in enumerate(total):
        place[i, :t] = torch.arange(at, at + t, dtype=torch.int32)
        at += t
    place = place.cuda()
    s["table"][s["seqs"].long()] = torch.where(place >= 0, order[place.clamp(min=0).long()], place)
    s["pages"] = torch.zeros((pages, hk, PAGE * TOKEN_BYTES), dtype=torch.uint8, device="cuda")
    if case["kind"] == "attention":
        k, v = _cache_values(g, at, hk, PAGE)
        for a in range(0, at, 1024):  # piece by piece: the temporaries are large
            b = min(at, a + 1024)
            s["pages"][order[a:b].long()] = _blocks(_token_bytes(k[a:b], v[a:b])).flatten(-2)
        del k, v
        s["q"] = (torch.randn(r, hq * DIM, device="cuda", generator=g) * 1.5).bfloat16()
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["qkv"] = (torch.randn(r, (hq + 2 * hk) * DIM, device="cuda", generator=g) * (0.5 + torch.rand(1, hq + 2 * hk, 1, device="cuda", generator=g)).expand(1, -1, DIM).reshape(1, -1)).bfloat16()
        s["q_norm"] = (1 + 0.1 * torch.randn(DIM, device="cuda", generator=g)).bfloat16()
        s["k_norm"] = (1 + 0.1 * torch.randn(DIM, device="cuda", generator=g)).bfloat16()
        s["q"] = torch.zeros(r, hq * DIM, dtype=torch.bfloat16, device="cuda")
        s["k"] = torch.zeros(r, hk * DIM, dtype=torch.bfloat16, device="cuda")
        s["v"] = torch.zeros_like(s["k"])
    if own:
        _describe(s, 1, hk, hq, r)
        if case["kind"] == "append":
            s["pointers"] = [s[x].data_ptr() for x in ("qkv", "q_norm", "k_norm", "q", "k", "v")]
        else:
            s["pointers"] = [s[x].data_ptr() for x in ("q", "out")]
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------

def _positions(s):
    """For each row of the batch its entry and its position."""
    count = (s["row0"][1:] - s["row0"][:-1]).long()
    entry = torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count, output_size=s["rows"])
    return entry, torch.arange(s["rows"], device="cuda") - s["row0"][entry].long() + s["pos0"][entry].long()


def _append(s):
    hq, hk = s["hq"], s["hk"]
    entry, pos = _positions(s)
    x = s["qkv"].float().unflatten(-1, (hq + 2 * hk, DIM))
    q, k, v = x.split((hq, hk, hk), 1)
    normed = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w.float()  # noqa: E731
    turn = torch.exp(torch.arange(DIM // 2, device="cuda", dtype=torch.float64) * (-math.log(ROPE_BASE) / (DIM // 2)))
    angle = pos.double()[:, None] * turn
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    rotate = lambda t: torch.stack([t[..., 0::2] * cos - t[..., 1::2] * sin, t[..., 1::2] * cos + t[..., 0::2] * sin], -1).flatten(-2)  # noqa: E731
    s["q"].copy_(rotate(normed(q, s["q_norm"])).flatten(1))
    raw = _token_bytes(rotate(normed(k, s["k_norm"])), v)
    page = s["table"][s["seqs"][entry].long(), pos // PAGE].long()
    where = (_table("block_back", raw.device).unflatten(0, (BLOCK, TOKEN_BYTES))[pos % BLOCK] + (pos % PAGE // BLOCK * (BLOCK * TOKEN_BYTES))[:, None])[:, None]
    flat = where + ((page * hk)[:, None] + torch.arange(hk, device="cuda"))[..., None] * (PAGE * TOKEN_BYTES)
    pool = s["pages"].view(-1)
    pool[flat] = raw
    k, v = _token_values(pool[flat])
    s["k"].copy_(k.flatten(1))
    s["v"].copy_(v.flatten(1))
    return [s["q"], s["k"], s["v"]]


def _attention(s):
    hq, hk, n = s["hq"], s["hk"], s["seqs"].numel()
    top = _pages_of(s["max_len"])
    table = s["table"][s["seqs"].long(), :top].long()
    raw = s["pages"][table.clamp(min=0)].unflatten(-1, (-1, BLOCK * TOKEN_BYTES))
    k, v = _token_values(_tokens(raw).transpose(1, 2).flatten(2, 3))          # [n, hk, top * 64, 128]
    entry, pos = _positions(s)
    row = torch.arange(s["rows"], device="cuda") - s["row0"][entry].long()
    q = torch.zeros((n, s["max_rows"], hq * DIM), device="cuda")
    q[entry, row] = s["q"].float()
    q = q.view(n, s["max_rows"], hk, hq // hk, DIM).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = q @ k.transpose(-1, -2) / math.sqrt(DIM)                          # [n, hk, rows * group, positions]
    last = s["pos0"].long()[:, None] + torch.arange(s["max_rows"], device="cuda")
    seen = (torch.arange(top * PAGE, device="cuda") <= last[..., None]) & (table >= 0).repeat_interleave(PAGE, 1)[:, None]
    score = score.unflatten(2, (s["max_rows"], -1)).masked_fill(~seen[:, None, :, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    out = (p / p.sum(-1, keepdim=True)).flatten(2, 3) @ v
    out = out.view(n, hk, s["max_rows"], hq // hk, DIM).permute(0, 2, 1, 3, 4).flatten(2)
    s["out"].copy_(out[entry, row])
    return s["out"]


def _free_pages(s):
    return (s["refs"] == 0).nonzero().flatten()


def _release(s, seqs):
    held = s["table"][seqs].flatten().long()
    s["refs"].index_add_(0, held.clamp(min=0), -(held >= 0).int())
    s["table"][seqs] = -1
    s["lens"][seqs] = 0


def _fork(s):
    dev = lambda v: torch.tensor(v, device="cuda")  # noqa: E731
    parents, children = dev(s["parents"]), dev(s["children"])
    _release(s, children)
    tokens = torch.minimum(dev(s["tokens"]), s["lens"][parents].long())
    full, rest = tokens // PAGE, tokens % PAGE > 0
    source = s["table"][parents, full.clamp(max=s["table"].shape[1] - 1)].long()
    need, free = rest & (source >= 0), _free_pages(s)
    rank = need.long().cumsum(0)
    given = ~need | (rank <= free.numel())
    take = need & given
    fresh = free[(rank - 1)[take]]
    s["pages"][fresh] = s["pages"][source[take]]
    column = torch.arange(s["table"].shape[1], device="cuda")
    new = torch.where((column < full[:, None]) & given[:, None], s["table"][parents], -1)
    new[take.nonzero().flatten(), full[take]] = fresh.int()
    s["table"][children] = new
    s["refs"].index_add_(0, new.clamp(min=0).flatten().long(), (new >= 0).flatten().int())
    s["lens"][children] = torch.where(given, tokens, 0).int()
    s["info"].copy_(torch.stack([(s["refs"] == 0).sum(), (~given).sum()]))
    return [s["pages"], s["table"], s["lens"], s["refs"], s["info"]]


def _compact(s):
    used = s["refs"] > 0
    count = used.sum()
    number = torch.arange(used.numel(), device="cuda")
    source, to = number[used & (number >= count)], number[~used & (number < count)]
    s["pages"][to] = s["pages"][source]
    s["refs"][to] = s["refs"][source]
    s["refs"][source] = 0
    number[source] = to
    s["table"].copy_(torch.where(s["table"] >= 0, number[s["table"].clamp(min=0).long()], s["table"]))


def _grow(s, b):
    seqs, count = b["seqs"].long(), (b["row0"][1:] - b["row0"][:-1]).long()
    held = s["lens"][seqs].long()
    first, last = -(-held // PAGE), -(-(held + count) // PAGE)
    need, free = last - first, _free_pages(s)
    upto = need.cumsum(0)
    given = (last <= s["table"].shape[1]) & ((need == 0) | (upto <= free.numel()))
    got = torch.where(given, need, 0)
    entry = torch.repeat_interleave(torch.arange(seqs.numel(), device="cuda"), got)
    step = torch.arange(entry.numel(), device="cuda") - (got.cumsum(0) - got)[entry]
    fresh = free[(upto - need)[entry] + step]
    s["table"][seqs[entry], first[entry] + step] = fresh.int()
    s["refs"][fresh] = 1
    b["pos0"].copy_(torch.where(given, held, -1))
    s["lens"][seqs] = torch.where(given, held + count, held).int()
    s["info"].copy_(torch.stack([(s["refs"] == 0).sum(), (~given).sum()]))


def _turnover(s):
    turn = s["turn"]
    _release(s, torch.tensor(s["halves"][turn], device="cuda"))
    _compact(s)
    _grow(s, s["grow"][turn])
    s["turn"] = 1 - turn
    return [s["pages"], s["table"], s["lens"], s["refs"], s["info"], s["grow"][turn]["pos0"]]


# ---- the library's calls ----------------------------------------------------------------------------------------------------

def _own(s):
    lib, check, cache, stream = s["lib"], s["capi"].check, C.byref(s["cache"]), s["stream"]
    if s["kind"] == "attention":
        q, out = s["pointers"]
        check(lib.s2p_b200_kv4_attention(cache, C.byref(s["batch"]), 0, q, out, stream), "attention")
        return s["out"]
    if s["kind"] == "append":
        qkv, q_norm, k_norm, q, k, v = s["pointers"]
        check(lib.s2p_b200_kv4_append(cache, C.byref(s["batch"]), 0, qkv, q_norm, k_norm, EPS, ROPE_BASE, q, stream), "append")
        check(lib.s2p_b200_kv4_read(cache, C.byref(s["batch"]), 0, k, v, stream), "read")
        return [s["q"], s["k"], s["v"]]
    info = s["info"].data_ptr()
    if s["kind"] == "fork":
        parents, children, tokens = s["lists"]
        check(lib.s2p_b200_kv4_fork(cache, parents, children, tokens, len(parents), info, stream), "fork")
        return [s["pages"], s["table"], s["lens"], s["refs"], s["info"]]
    turn = s["turn"]
    half = s["lists"][turn]
    check(lib.s2p_b200_kv4_release(cache, half, len(half), stream), "release")
    check(lib.s2p_b200_kv4_compact(cache, info, stream), "compact")
    check(lib.s2p_b200_kv4_reserve(cache, C.byref(s["batches"][turn]), info, stream), "reserve")
    s["turn"] = 1 - turn
    return [s["pages"], s["table"], s["lens"], s["refs"], s["info"], s["grow"][turn]["pos0"]]


def run(state):
    if own:
        return _own(state)
    return {"attention": _attention, "append": _append, "fork": _fork, "turnover": _turnover}[state["kind"]](state)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------

def _exact_places(which):
    """Where the format keeps channel d of position `tok` of a block's keys (0) or values (1): byte and shift of the code, bytes of s and m."""
    got = []
    for tok in range(BLOCK):
        for d in range(DIM):
            j, e = d // 32, d % 32
            if which == 0:
                byte = tok * 64 + (e // 8) * 16 + j * 4 + (e % 8) // 2
                at = 2048 + tok * 16 + 2 * j
                got.append((byte, 4 * (e % 2), at, at + 8))
            else:
                byte = 1024 + (tok // 8) * 512 + (e // 4) * 64 + (tok // 2 % 4) * 16 + (tok % 2) * 8 + 2 * j + (e % 4) // 2
                at = 2304 + (tok // 2) * 16 + 4 * j + 2 * (tok % 2)
                got.append((byte, 4 * (e % 2), at, at + 128))
    return torch.tensor(got, device="cuda").T


def _exact_value(block, places):
    """Keys or values [..., 16, 128] of blocks [..., 2560] in 64 bits."""
    byte, shift, s, m = places
    code = (block[..., byte].int() >> shift.int()) & 15
    bits = block.contiguous().view(torch.float16)
    return (bits[..., s // 2].double() * code.double() + bits[..., m // 2].double()).unflatten(-1, (BLOCK, DIM))


def _exact_quantised(x):
    """What the cache holds for x [..., 128], both in 64 bits."""
    out = torch.empty_like(x)
    for j in range(4):
        g = x[..., 32 * j:32 * j + 32]
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        s, m = ((high - low) / 15).half().double(), low.half().double()
        out[..., 32 * j:32 * j + 32] = m + s * ((g - m) / s).round().clamp(0, 15)
    return out


def exact(case, seed):
    if case["kind"] not in ("append", "attention"):
        return None  # whole numbers
    s = prepare(case, seed)
    lens, rows, hq, hk = _lens(case), _rows(case), case["q_heads"], case["kv_heads"]
    if case["kind"] == "append":
        pos = torch.cat([torch.arange(t - q, t, device="cuda") for t, q in zip(lens, rows)]).double()
        x = s["qkv"].double().view(len(pos), hq + 2 * hk, DIM)
        outs = []
        for part, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hk], s["k_norm"])):
            y = part / (part.pow(2).sum(-1, keepdim=True) / DIM + EPS).sqrt() * w.double()
            z = torch.empty_like(y)
            for i in range(DIM // 2):
                a = pos * ROPE_BASE ** (-2.0 * i / DIM)
                c, n = torch.cos(a)[:, None], torch.sin(a)[:, None]
                z[..., 2 * i] = y[..., 2 * i] * c - y[..., 2 * i + 1] * n
                z[..., 2 * i + 1] = y[..., 2 * i] * n + y[..., 2 * i + 1] * c
            outs.append(z)
        q, k = outs
        return [q.reshape(len(pos), -1), _exact_quantised(k).reshape(len(pos), -1), _exact_quantised(x[:, hq + hk:]).reshape(len(pos), -1)]
    out = torch.zeros(sum(rows), hq, DIM, dtype=torch.float64, device="cuda")
    at, places = 0, [_exact_places(0), _exact_places(1)]
    for i, (t, r) in enumerate(zip(lens, rows)):
        pages = s["table"][int(s["seqs"][i]), :_pages_of(t)].long()
        blocks = s["pages"][pages].view(len(pages), hk, PAGE // BLOCK, -1)
        k, v = (_exact_value(blocks, w).transpose(0, 1).reshape(hk, -1, DIM)[:, :t] for w in places)
        hidden = torch.arange(t, device="cuda")[None] > torch.arange(t - r, t, device="cuda")[:, None]
        for h in range(hq):
            z = s["q"][at:at + r, h * DIM:(h + 1) * DIM].double() @ k[h // (hq // hk)].T / math.sqrt(DIM)
            out[at:at + r, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[h // (hq // hk)]
        at += r
    return out.reshape(sum(rows), -1)
