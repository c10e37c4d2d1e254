"""The 4-bit key/value cache in 64 bits: its groups, its records, and attention over what they stand for.

A group of 32 channels stands for lo + s * code: lo the minimum rounded down to bfloat16, s the span above lo over 15 rounded
up, code the nearest whole number in 0..15.  A record holds 16 tokens of one head (see ``places``)."""
import torch

GROUP, UNIT = 32, 16
F64 = torch.float64


def floor_bf16(x):
    """The largest number of eight significant bits that is not above x (float64)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.floor(m * 256.0) / 256.0, e)


def held(x):
    return torch.nan_to_num(x.double(), nan=0.0, posinf=2.0 ** 120, neginf=-2.0 ** 120).clamp(-2.0 ** 120, 2.0 ** 120)


def quantise(x):
    """[..., D] -> lo, s [..., D / 32], codes [..., D]."""
    g = held(x).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    lo = floor_bf16(g.amin(-1))
    s = -floor_bf16(-(g.amax(-1) - lo) / 15.0)
    c = torch.round((g - lo[..., None]) / torch.where(s > 0, s, 1.0)[..., None]).clamp(0, 15)
    return lo, s, (c * (s > 0)[..., None]).flatten(-2).long()


def dequantise(lo, s, codes):
    return (lo[..., None] + s[..., None] * codes.double().reshape(*codes.shape[:-1], codes.shape[-1] // GROUP, GROUP)).flatten(-2)


def places(D):
    """Where a record keeps things: the bits of the keys' and values' codes, [16, D], and the byte of each number but the
    kind's own offset, [16, G]; kind n (lo and s of the keys, lo and s of the values) begins at byte 16 D + n D."""
    G = D // GROUP
    t, c = torch.arange(UNIT)[:, None], torch.arange(D)[None]
    g, j, e, r, i = c // 32, c % 32 // 8, c % 8, c % 32 // 4, c % 4
    k = ((t * 4 + j) * G + g) * 32 + 16 * (e % 2) + 4 * (e // 2)
    v = 8 * D * 8 + ((t // 2 * 8 + r) * G + g) * 32 + 16 * (t % 2) + 4 * i
    n = ((t // 2 * G + torch.arange(G)[None]) * 2 + t % 2) * 2
    return k, v, n


def pack(k, v):
    """[tokens, heads, D] keys and values, tokens a multiple of 16 -> records uint8 [tokens / 16, heads, 20 D]."""
    N, KV, D = k.shape
    bits_k, bits_v, at = places(D)
    rec = torch.zeros((N // UNIT, KV, 20 * D), dtype=torch.long)
    for x, bits, kind in ((k, bits_k, 0), (v, bits_v, 2)):
        lo, s, codes = quantise(x)
        codes = codes.reshape(N // UNIT, UNIT, KV, D).transpose(1, 2)
        rec.scatter_add_(2, (bits // 8).flatten().expand(N // UNIT, KV, -1), (codes << (bits % 8)).flatten(2))
        for m, number in enumerate((lo, s)):
            raw = number.bfloat16()
            assert torch.equal(raw.double(), number)                  # eight significant bits
            raw = (raw.view(torch.int16).long() & 0xffff).reshape(N // UNIT, UNIT, KV, D // GROUP).transpose(1, 2)
            where = 16 * D + (kind + m) * D + at
            rec[:, :, where.flatten()] = (raw & 255).flatten(2)
            rec[:, :, (where + 1).flatten()] = (raw >> 8).flatten(2)
    return rec.to(torch.uint8)


def unpack(rec):
    """Records uint8 [..., 20 D] -> keys, values float64 [..., 16, D]."""
    D = rec.shape[-1] // 20
    bits_k, bits_v, at = places(D)
    rec = rec.long()
    out = []
    for bits, kind in ((bits_k, 0), (bits_v, 2)):
        codes = rec[..., bits // 8] >> (bits % 8) & 15
        lo, s = ((rec[..., 16 * D + n * D + at] | rec[..., 16 * D + n * D + at + 1] << 8).to(torch.int32) << 16
                 for n in (kind, kind + 1))
        out.append(dequantise(lo.view(torch.float32).double(), s.view(torch.float32).double(), codes))
    return out


def to_pages(records, table, num_pages, page_tokens, fill=0xff):
    """One request's records [n, heads, 20 D] laid into pages [num_pages, heads, page_tokens, 5 D / 4] at ``table``; what no
    token fills holds ``fill`` (0xff: codes of 15 and numbers that are NaN)."""
    n, KV, w = records.shape
    per = page_tokens // UNIT
    pages = torch.full((num_pages, KV, per, w), fill, dtype=torch.uint8)
    for i in range(n):
        pages[table[i // per], :, i % per] = records[i]
    return pages.reshape(num_pages, KV, page_tokens, w // UNIT)


def attention(q, k, v, scale, window=None):
    """q [n, H, D] the last rows of a request with keys and values [N, KV, D], in 64 bits: outputs [n, H, D], and for the
    tolerances: sum of weight * |value|, and sum of weight * |value - output|, both [n, H, D]; sum |q||k| at most [n, H]."""
    n, H, D = q.shape
    N, KV = k.shape[:2]
    q = q.double().reshape(n, KV, H // KV, D)
    k, v = k.double(), v.double()
    s = torch.einsum("nkgd,tkd->nkgt", q, k) * scale
    pos = torch.arange(N - n, N)[:, None]
    key = torch.arange(N)[None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    seen = seen[:, None, None]
    w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1) if N else s
    w = torch.where(seen.any(-1, keepdim=True), w, 0.0).nan_to_num(0.0)
    o = torch.einsum("nkgt,tkd->nkgd", w, v)
    heavy = torch.einsum("nkgt,tkd->nkgd", w, v.abs())
    spread = torch.stack([torch.einsum("kgt,tkgd->kgd", w[i], (v[:, :, None] - o[i][None]).abs()) for i in range(n)]) \
        if n else o
    reach = (torch.einsum("nkgd,tkd->nkgt", q.abs(), k.abs()).masked_fill(~seen, 0.0).amax(-1) if N else s.sum(-1))
    return (o.reshape(n, H, D), heavy.reshape(n, H, D), spread.reshape(n, H, D), reach.reshape(n, H))
