"""Plain 64-bit counterparts of the paged 4-bit cache's operators, and the structs to call them with, for its tests.

Everything here is written from the layout that include/s2p_b200_ext.h documents, with no code of the library."""
import ctypes as C
import functools

import torch

PAGE, BLOCK = 64, 2560


def places(which):
    """[16, 128]: byte of the code, its shift, byte of s and of m, for each position of a block and channel (0 keys, 1 values)."""
    byte, shift, s, m = (torch.zeros(16, 128, dtype=torch.long) for _ in range(4))
    for i in range(16):
        for d in range(128):
            j, e = divmod(d, 32)
            if which == 0:
                byte[i, d] = 64 * i + 16 * (e // 8) + 4 * j + (e % 8) // 2
                s[i, d], m[i, d] = 2048 + 16 * i + 2 * j, 2056 + 16 * i + 2 * j
            else:
                byte[i, d] = 1024 + 512 * (i // 8) + 64 * (e // 4) + 16 * (i // 2 % 4) + 8 * (i % 2) + 2 * j + (e % 4) // 2
                s[i, d] = 2304 + 16 * (i // 2) + 4 * j + 2 * (i % 2)
                m[i, d] = s[i, d] + 128
            shift[i, d] = 4 * (d % 2)
    return byte, shift, s, m


def unpack(blocks, which):
    """codes, s, m [..., 16, 128] as doubles, of blocks [..., 2560] (bytes, on the CPU)."""
    byte, shift, s, m = places(which)
    half = blocks.contiguous().view(torch.float16).double()
    return ((blocks[..., byte].long() >> shift) & 15).double(), half[..., s // 2], half[..., m // 2]


def quantise(x):
    """codes, s, m of x [..., 128] (32-bit floats): the documented rule, in IEEE single precision."""
    x = x.float().clamp(-65504, 65504).unflatten(-1, (4, 32))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, m = ((hi - lo) / 15).half(), lo.half()
    c = torch.where(s > 0, ((x - m.float()) / s.float()).round().clamp(0, 15), torch.zeros(()))
    back = lambda t: t.expand_as(x).flatten(-2)  # noqa: E731
    return c.flatten(-2).to(torch.uint8), back(s), back(m)


def pack(blocks, which, i, codes, s, m):
    """Writes one position's codes, s and m [..., 128] into blocks [..., 2560] (CPU), place i."""
    byte, shift, at_s, at_m = (t[i] for t in places(which))
    half = blocks.view(torch.float16)
    half[..., at_s // 2] = s.half()
    half[..., at_m // 2] = m.half()
    for d in range(128):
        b = blocks[..., byte[d]]
        blocks[..., byte[d]] = (b & (0xF0 if shift[d] == 0 else 0x0F)) | (codes[..., d] << int(shift[d]))


class Cache:
    """A cache on the GPU with its descriptor.  `pages` starts as `fill` bytes (0xFF: NaN everywhere)."""

    def __init__(self, lib, capi, n_pages, layers=1, kv_heads=2, q_heads=8, max_seqs=4, stride=8, rows=64, fill=0xFF, device="cuda"):
        self.lib, self.capi = lib, capi
        self.layers, self.kv_heads, self.q_heads, self.n_pages, self.stride = layers, kv_heads, q_heads, n_pages, stride
        self.pages = torch.full((n_pages, layers, kv_heads, 4, BLOCK), fill, dtype=torch.uint8, device=device)
        self.table = torch.full((max_seqs, stride), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=device)
        self.info = torch.full((2,), -7, dtype=torch.int32, device=device)
        self.c = capi.Kv4(self.pages.data_ptr(), self.table.data_ptr(), self.lens.data_ptr(), self.refs.data_ptr(), None, 0,
                          n_pages, layers, kv_heads, q_heads, max_seqs, stride)
        size = lib.s2p_b200_kv4_work_bytes(C.byref(self.c), rows)
        assert size > 0
        self.work = torch.zeros(size, dtype=torch.uint8, device=device)
        self.c.work, self.c.work_bytes = self.work.data_ptr(), size

    def batch(self, seqs, counts, pos0=None, rows=None, max_rows=None):
        """A batch of `counts` rows each; pos0 None: to be filled by reserve."""
        dev = lambda v: torch.tensor(v, dtype=torch.int32, device=self.pages.device)  # noqa: E731
        row0 = [0]
        for n in counts:
            row0.append(row0[-1] + n)
        b = lambda: None  # noqa: E731
        b.seqs, b.row0, b.pos0 = dev(list(seqs)), dev(row0), dev(list(pos0) if pos0 is not None else [-5] * len(counts))
        b.rows = row0[-1] if rows is None else rows
        b.c = self.capi.Kv4Batch(b.seqs.data_ptr(), b.row0.data_ptr(), b.pos0.data_ptr(), len(counts), b.rows,
                                 max(list(counts) + [0]) if max_rows is None else max_rows)
        return b

    def status(self, what, *args):
        return getattr(self.lib, "s2p_b200_kv4_" + what)(C.byref(self.c), *args)

    def call(self, what, *args):
        self.capi.check(self.status(what, *args), what)

    def reserve(self, b, stream=None):
        self.call("reserve", C.byref(b.c), self.info.data_ptr(), stream)

    def append(self, b, qkv, q, layer=0, q_norm=None, k_norm=None, eps=1e-6, base=1e6, stream=None):
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.call("append", C.byref(b.c), layer, p(qkv), p(q_norm), p(k_norm), eps, base, p(q), stream)

    def attention(self, b, q, out, layer=0, stream=None):
        self.call("attention", C.byref(b.c), layer, q.data_ptr(), out.data_ptr(), stream)

    def read(self, b, k, v, layer=0, stream=None):
        self.call("read", C.byref(b.c), layer, k.data_ptr(), v.data_ptr(), stream)

    def lists(self, *v):
        return [(C.c_int32 * max(1, len(x)))(*x) for x in v]

    def fork(self, parents, children, tokens, stream=None):
        self.call("fork", *self.lists(parents, children, tokens), len(parents), self.info.data_ptr(), stream)

    def release(self, seqs, stream=None):
        self.call("release", *self.lists(seqs), len(seqs), stream)

    def compact(self, stream=None):
        self.call("compact", self.info.data_ptr(), stream)

    def values(self, seq, length, layer=0):
        """keys, values, and for values s c and |m|, [kv_heads, length, 128] as doubles; and which positions have a page."""
        n = -(-length // PAGE)
        entries = self.table[seq, :n].cpu().long()
        there = ((entries >= 0) & (entries < self.n_pages))
        blocks = self.pages[entries.clamp(0, self.n_pages - 1).to(self.pages.device), layer].cpu()  # [n, heads, 4, 2560]
        out = []
        for which in (0, 1):
            c, s, m = (t.permute(1, 0, 2, 3, 4).reshape(self.kv_heads, n * PAGE, 128)[:, :length] for t in unpack(blocks, which))
            out += [s * c + m, s * c + m.abs()]
        return out[0], out[2], out[3], there.repeat_interleave(PAGE)[:length]


def fill(cache, seq, length, seed, order=None, scale=1.0, layer=0):
    """Gives a sequence `length` positions of random keys and values in pages of a random order (or `order`)."""
    g = torch.Generator().manual_seed(seed)
    n = -(-length // PAGE)
    if order is None:
        free = (cache.refs == 0).nonzero().flatten().cpu()
        order = free[torch.randperm(len(free), generator=g)[:n]]
        cache.refs[order.to(cache.refs.device)] = 1
    blocks = cache.pages[order.to(cache.pages.device), layer].cpu()
    for which in (0, 1):
        x = torch.randn(n, cache.kv_heads, 4, 16, 128, generator=g) * scale
        codes, s, m = quantise(x)
        fresh = blocks.clone()
        byte, shift, at_s, at_m = places(which)
        half = fresh.view(torch.float16)
        half[..., at_s // 2], half[..., at_m // 2] = s, m
        low = torch.zeros_like(fresh)
        for i in (0, 1):  # even channels, then odd ones
            low[..., byte[:, i::2]] |= codes[..., i::2] << (4 * i)
        fresh[..., byte[:, 0::2]] = low[..., byte[:, 0::2]]
        seen = torch.arange(n * PAGE).view(n, 1, 4, 16) < length  # positions behind the length keep what was there
        touched = torch.zeros(n, 1, 4, BLOCK, dtype=torch.bool)
        for i in range(16):
            for at in (byte[i], at_s[i], at_s[i] + 1, at_m[i], at_m[i] + 1):
                touched[..., at] |= seen[..., i:i + 1]
        blocks = torch.where(touched, fresh, blocks)
    cache.pages[order.to(cache.pages.device), layer] = blocks.to(cache.pages.device)
    cache.table[seq, :n] = order.int().to(cache.table.device)
    cache.lens[seq] = length


def attention(cache, seq, first, q, layer=0):
    """For rows q [rows, q_heads * 128] at positions first, first + 1, ...: the result in 64 bits and a bound on what the kernel may be off.

    The kernel rounds a weight p to f16 (2^-11 of it) and p s to f16 (2^-11 again); the sum of weights is not rounded.  So a value's part
    s c p / sum is off by at most 2^-10 of it, the part m p / sum by 2^-11 (second order: 2^-20); scores and their
    exponentials are in 32 bits (|logit| < 64 here: 2^-24 * 64 * a few, below 2^-15 of a weight).  A weight or a product below f16's normal range is off by 2^-25 at most,
    over 4 for the head room, and the largest weight is at least 1, so the sum is: 2^-25 (15 + |v|) for each position.  And the result is rounded to bf16: 2^-8 of it.

    For prompt slices it is a value s c + m that is rounded to f16 in place of p s, 2^-11 again.  Keys are, too, which moves a logit by 2^-11 sum |q k| / sqrt(128) at the
    worst; the bound leaves no room for that (of 128 channels and many positions, of either sign, little is left): it is narrower than the worst case."""
    rows, group = q.shape[0], cache.q_heads // cache.kv_heads
    k, v, mass, there = cache.values(seq, first + rows, layer)
    x = q.double().cpu().view(rows, cache.kv_heads, group, 128)
    z = torch.einsum("rhgd,htd->rhgt", x, torch.nan_to_num(k)) / 128 ** 0.5
    seen = (torch.arange(first + rows) <= first + torch.arange(rows)[:, None]) & there
    z = z.masked_fill(~seen[:, None, None], -torch.inf)
    p = torch.nan_to_num(torch.softmax(z, -1))  # a row that sees nothing: zeros
    v, mass = (torch.where(there[None, :, None], t, 0.0) for t in (v, mass))
    out = torch.einsum("rhgt,htd->rhgd", p, v)
    bound = torch.einsum("rhgt,htd->rhgd", p, mass) * (2 ** -10 + 2 ** -14) + (first + rows) * 2 ** -25 * (15 + v.abs().max())
    return out.reshape(rows, -1), bound.reshape(rows, -1) + out.abs().reshape(rows, -1) * 2 ** -8


@functools.lru_cache(None)
def places_on(device, which):
    return tuple(t.to(device) for t in places(which))


def store(cache, seq, keys, values, layer=0):
    """Gives a sequence keys and values [kv_heads, length, 128] in free pages of a random order; positions behind the length keep what was there."""
    heads, length, _ = keys.shape
    n, dev = -(-length // PAGE), cache.pages.device
    free = (cache.refs == 0).nonzero().flatten()
    order = free[torch.randperm(len(free), generator=torch.Generator().manual_seed(length)).to(dev)[:n]]
    cache.refs[order], cache.table[seq, :n], cache.lens[seq] = 1, order.int(), length
    pos = torch.arange(length, device=dev)
    page, block, place = order[pos // PAGE], pos % PAGE // 16, pos % 16
    flat, half = cache.pages[:, layer].view(-1), cache.pages[:, layer].view(-1).view(torch.float16)
    assert flat.data_ptr() == cache.pages.data_ptr()  # (caches of one layer)
    for which, x in ((0, keys), (1, values)):
        byte, _, at_s, at_m = (t[place] for t in places_on(dev, which))
        codes, s, m = quantise(x.to(dev).float())
        for h in range(heads):
            base = (((page * heads + h) * 4 + block) * BLOCK)[:, None]
            flat[base + byte[:, 0::2]] = codes[h, :, 0::2] | codes[h, :, 1::2] << 4
            half[(base + at_s) // 2], half[(base + at_m) // 2] = s[h], m[h]


def attention_close(cache, seq, first, q, lift=12, layer=0):
    """The result in 64 bits, and how far roundings that are independent of one another carry it: for sums of many positions this is far narrower than
    the sum of worst cases in `attention`, and a part or a page that is left out shows.

    With weights p_t (sum 1), |delta| <= 1 independent, a kernel returns sum_t p_t v_t + sum_t a_t delta_t, rounded to bf16 (2^-8 of it), where a_t collects
      2^-11 p_t |v_t|             the weight in f16,
      2^-11 p_t (s c + |m|)       the product p s, or the value s c + m, in f16,
      2^-11 p_t |v_t - out| k_t   the keys in f16 for slices, k_t^2 = sum over channels of (q k)^2 / 128, by the softmax's derivative,
      2^-15 p_t |v_t - out|       logits below 64 in 32 bits and their exponentials.
    Hoeffding: |sum a delta| > 8 sqrt(sum a^2) has a probability below 2 e^-32.  Below f16's normal range a rounding is off by 2^-25: of a weight against the
    largest (1 in slices, 2^lift for tokens, where values reach 2^(13 - lift) fifteenths): 2^-25 |v| or 2^-25 2^-lift 15 max(1, s) a position, in the same way."""
    rows, heads, group, length = q.shape[0], cache.kv_heads, cache.q_heads // cache.kv_heads, first + q.shape[0]
    n = -(-length // PAGE)
    dev = cache.pages.device
    entries = cache.table[seq, :n].long()
    there = ((entries >= 0) & (entries < cache.n_pages)).repeat_interleave(PAGE)[:length]
    blocks = cache.pages[entries.clamp(0, cache.n_pages - 1), layer]
    half = blocks.view(torch.float16)
    held = []
    for which in (0, 1):
        byte, shift, s, m = places_on(dev, which)
        parts = [((blocks[..., byte] >> shift.to(torch.uint8)) & 15).double(), half[..., s // 2].double(), half[..., m // 2].double()]
        parts = [t.permute(1, 0, 2, 3, 4).reshape(heads, n * PAGE, 128)[:, :length] for t in parts]
        held += [torch.where(there[None, :, None], t, 0.0) for t in (parts[1] * parts[0] + parts[2], parts[1] * parts[0] + parts[2].abs(), parts[1])]
    k, _, _, v, mass, s = held
    x = q.double().view(rows, heads, group, 128)
    z = torch.einsum("rhgd,htd->rhgt", x, k) / 128 ** 0.5
    kk = torch.einsum("rhgd,htd->rhgt", x.square(), k.square()) / 128
    seen = (torch.arange(length, device=dev) <= first + torch.arange(rows, device=dev)[:, None]) & there
    p = torch.softmax(z.masked_fill(~seen[:, None, None], -torch.inf), -1)
    out = torch.einsum("rhgt,htd->rhgd", p, v)
    p2 = p.square()
    near = p2 * (kk * 2.0 ** -22 + 2.0 ** -30)
    spread = (torch.einsum("rhgt,htd->rhgd", near, v.square()) - 2 * out * torch.einsum("rhgt,htd->rhgd", near, v) + out.square() * near.sum(-1, keepdim=True)).clamp_min(0)
    square = 2.0 ** -22 * torch.einsum("rhgt,htd->rhgd", p2, v.square() + mass.square()) + spread
    small = p.amax(-1, keepdim=True) * (2.0 ** -25 * max(float(v.abs().max()), 15 * 2.0 ** -lift * max(1.0, float(s.max()))) * length ** 0.5)
    bound = 8 * (square.sqrt() + small) * (1 + 2 ** -6) + out.abs() * 2 ** -8
    return out.reshape(rows, -1), bound.reshape(rows, -1)
