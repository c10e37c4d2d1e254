"""Cases for timing the 4-bit cache: the maps that say where tokens go, the write, and the attention that reads it.

The kinds, and what each stands for:

maps       a step's row maps and block tables from its requests' lengths and one list of pages
write      a step's fused projection: bias, rotation, queries out, keys and values into 4-bit pages; then the written
           rows read back as the values they stand for
attention  causal attention over 4-bit pages, from one token a request to whole prompts

A key or value of one head is cut into groups of 32 channels; a group holds ``lo`` and ``s`` (bfloat16) and a code of
0..15 a channel, and stands for lo + s * code.  ``lo`` is the group's minimum rounded down, ``s`` the span above it
divided by 15 and rounded up.  A record holds 16 tokens of one head, in this order: the keys' codes, the values' codes,
the keys' lo and s, the values' lo and s (see ``_unpack``).  Head counts and sizes are those of the Qwen2.5 layers that
the repository's benchmarks run.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
THETA = 1e6
GROUP = 32
HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "14b": (40, 8, 128)}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the integers of a decode step of 64 requests
        dict(name="maps_64", kind="maps", step="1/300-8192x64", page=16, spare=0),
        # the integers of a step of long prompt portions beside decoded tokens, padded to a bucket
        dict(name="maps_prompts", kind="maps", step="4096/36864,3001/9000,8192/8192,1/1-65536x61", page=16, spare=35),
        # a decode step at the headline batch
        dict(name="write_8", kind="write", size="7b", step="1/500-2049x8", page=16, dtype="bfloat16", spare=0),
        # a whole prompt at far positions
        dict(name="write_2048", kind="write", size="7b", step="2048/32768", page=16, dtype="bfloat16", spare=0),
        # ragged portions of the 32-bit path, heads of 64
        dict(name="write_f32", kind="write", size="0.5b", step="700/1100,1/5000,76/76", page=32, dtype="float32", spare=3),
        # one user, a short context: the smallest call
        dict(name="decode_1", kind="attention", size="1.5b", step="1/777", page=16, window=0, dtype="bfloat16"),
        # the headline batch
        dict(name="decode_8", kind="attention", size="7b", step="1/2048x8", page=16, window=0, dtype="bfloat16"),
        # many users with ragged contexts
        dict(name="decode_64", kind="attention", size="7b", step="1/300-8192x64", page=16, window=0, dtype="bfloat16"),
        # one user with a very long context
        dict(name="decode_long", kind="attention", size="14b", step="1/131071", page=64, window=0, dtype="bfloat16"),
        # a whole prompt
        dict(name="prompt_4096", kind="attention", size="7b", step="4096/4096", page=16, window=0, dtype="bfloat16"),
        # portions behind contexts beside decoded tokens, heads of 64, a window
        dict(name="mixed", kind="attention", size="0.5b", step="512/8000,37/1001,5/3333,1/200-6000x9", page=32, window=4096,
             dtype="bfloat16"),
        # decoded tokens and a short portion of the 32-bit path
        dict(name="few_f32", kind="attention", size="1.5b", step="1/900-2500x4,29/600", page=16, window=0, dtype="float32"),
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of the range."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["maps", "write", "write", "attention", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 48, 64])
    if kind == "maps":
        n = _spread(rng, 1, 256)
        step = "1/%d-%dx%d" % (_spread(rng, 1, 500), _spread(rng, 500, 16384), n)
        for _ in range(rng.choice([0, 1, 2])):
            rows = _spread(rng, 2, 4096)
            step += ",%d/%d" % (rows, rows + rng.choice([0, _spread(rng, 1, 16384)]))
        return dict(kind=kind, step=step, page=page, spare=rng.choice([0, rng.randrange(1, 40)]))
    size = rng.choice(list(HEADS))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if kind == "write":
        rows = _spread(rng, 1, 2048)
        step = "%d/%d" % (rows, rows + rng.choice([0, _spread(rng, 1, 60000)]))
        if rng.random() < 0.5:
            step += ",1/%d-%dx%d" % (_spread(rng, 1, 500), _spread(rng, 500, 16384), _spread(rng, 1, 64))
        return dict(kind=kind, size=size, step=step, page=page, dtype=dtype, spare=rng.choice([0, rng.randrange(1, 9)]))
    window = rng.choice([0, 0, 0, _spread(rng, 64, 4096)])
    form = rng.choice(["decode", "decode", "long", "portions", "portions"])
    if form == "decode":
        step = "1/%d-%dx%d" % (_spread(rng, 1, 1000), _spread(rng, 1000, 8192), _spread(rng, 1, 64))
    elif form == "long":
        step = "1/%d" % _spread(rng, 16384, 131072)
    else:
        most = 2048 if dtype == "bfloat16" else 128
        step = ",".join("%d/%d" % (r, r + rng.choice([0, _spread(rng, 1, 2000)])) for r in
                        (_spread(rng, 2, most) for _ in range(rng.choice([1, 2, 3]))))
        if rng.random() < 0.4:
            step += ",1/%d-%dx%d" % (_spread(rng, 1, 500), _spread(rng, 500, 3000), _spread(rng, 1, 6))
    return dict(kind=kind, size=size, step=step, page=page, window=window, dtype=dtype)


def _step(case):
    """[(rows, keys)] of the case's requests: "rows/keys", or "rows/low-highxN" for N requests of spread key counts."""
    out = []
    for item in case["step"].split(","):
        rows, keys = item.split("/")
        n = 1
        if "x" in keys:
            keys, n = keys.split("x")
        low, high = (keys.split("-") * 2)[:2]
        low, high, n = int(low), max(int(low), int(high)), int(n)
        order = list(range(n))
        random.Random(n).shuffle(order)
        out += [(int(rows), max(int(rows), high if n == 1 else low + (high - low) * k // (n - 1))) for k in order]
    return out


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    step, page = _step(case), case["page"]
    rows, keys = [r for r, _ in step], [k for _, k in step]
    need = [-(-k // page) for k in keys]
    total = sum(need) + 7                                  # the pool has more pages than the step holds
    pool = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)[:sum(need)].contiguous()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    st = dict(case=case, pages=pool, q_len=ints(rows), seq_len=ints(keys), context=ints([k - r for r, k in step]),
              num_rows=sum(rows) + case.get("spare", 0), width=max(need))
    if case["kind"] == "maps":
        return st
    H, KV, D = HEADS[case["size"]]
    dtype = DTYPES[case["dtype"]]
    at = [0]
    for n in need:
        at.append(at[-1] + n)
    table = torch.full((len(step), max(need)), -1, dtype=torch.int32, device=DEVICE)
    owner = torch.repeat_interleave(torch.arange(len(step), device=DEVICE), torch.tensor(need, device=DEVICE))
    table[owner, torch.arange(sum(need), device=DEVICE) - ints(at)[owner]] = pool
    T = sum(rows)
    who = torch.repeat_interleave(torch.arange(len(step), device=DEVICE), ints(rows))
    starts = torch.cumsum(ints(rows), 0) - ints(rows)
    pos = torch.arange(T, device=DEVICE) - starts[who] + st["context"][who]
    if case["kind"] == "write":
        slots = table[who, pos // page] * page + pos % page
        spare = case["spare"]                              # rows behind the last request: no slot
        st["positions"] = torch.cat([pos, pos.new_zeros(spare)]).to(torch.int32)
        st["slots"] = torch.cat([slots, slots.new_full((spare,), -1)]).to(torch.int32)
        width = (H + 2 * KV) * D
        st["qkv"] = torch.randn((T + spare, width), generator=g, device=DEVICE).to(dtype)
        st["bias"] = torch.randn(width, generator=g, device=DEVICE)      # queries and keys of these models lean far
        st["inv_freq"] = (THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEVICE) / D)).float()
        st["q_out"] = torch.empty((T + spare, H * D), dtype=dtype, device=DEVICE)
        st["cache"] = torch.zeros((total, KV, page, D * 5 // 4), dtype=torch.uint8, device=DEVICE)
        return st
    st["block_table"], st["q_start"] = table, starts.to(torch.int32)
    # Queries that prefer some keys: scores with a deviation of two and more.  Keys with a bias of their channel.
    st["q"] = (2.0 * torch.randn((T, H * D), generator=g, device=DEVICE)).to(dtype)
    st["out"] = torch.zeros((T, H * D), dtype=dtype, device=DEVICE)
    st["cache"] = _random_cache(g, total, KV, page, D)
    st["most_rows"], st["most_keys"] = max(rows), max(keys)
    return st


def _random_cache(g, pages, KV, page, D):
    """Full pages whose codes and groups are as those of normal keys and values: codes near 7.5, spans of about four."""
    n, G = pages * KV * (page // 16), D // GROUP
    codes = torch.randint(0, 256, (n, 16 * D), generator=g, device=DEVICE, dtype=torch.uint8)
    half = torch.randint(0, 256, (n, 16 * D), generator=g, device=DEVICE, dtype=torch.uint8)
    # the mean of two uniform nibbles, so that middle codes are the common ones
    mean = lambda a, b: torch.div(a.int() + b.int(), 2, rounding_mode="floor")  # noqa: E731
    codes = (mean(codes & 15, half & 15) | (mean(codes >> 4, half >> 4) << 4)).to(torch.uint8)
    span = 3.0 + 2.0 * torch.rand((n, 2, 16 * G), generator=g, device=DEVICE)
    lean = 0.3 * torch.randn((n, 2, 16 * G), generator=g, device=DEVICE)
    params = torch.stack([lean - span / 2, span / 15], dim=2).to(torch.bfloat16)       # [n, k/v, lo/s, ...]
    params = params.reshape(n, 64 * G).view(torch.uint8)
    return torch.cat([codes, params], dim=1).reshape(pages, KV, page, D * 5 // 4).contiguous()


# ------------------------------------------------------------------------------------------------ plain forms
def _unpack(records, D):
    """uint8 [..., 20 D] records of 16 tokens -> (keys, values) float32 [..., 16, D]."""
    lead, G = records.shape[:-1], D // GROUP
    nibbles = lambda b: torch.stack([b & 15, b >> 4], dim=-1).float()  # noqa: E731
    # keys: [token][j][group] words; byte b of a word holds channels (0, 2), (4, 6), (1, 3), (5, 7) of 32 group + 8 j
    k = nibbles(records[..., :8 * D].reshape(*lead, 16, 4, G, 2, 2)).reshape(*lead, 16, 4, G, 2, 4)
    k = k.transpose(-1, -2).transpose(-4, -3).reshape(*lead, 16, G, GROUP)
    # values: [pair][r][group] words; two bytes a token of the pair: channels 32 group + 4 r + 0..3
    v = nibbles(records[..., 8 * D:16 * D].reshape(*lead, 8, 8, G, 2, 2)).reshape(*lead, 8, 8, G, 2, 4)
    n = len(lead)
    v = v.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(*lead, 16, G, GROUP)
    # lo and s of the keys, then of the values: [pair][group][token of the pair]
    p = records[..., 16 * D:].contiguous().view(torch.bfloat16).float().reshape(*lead, 4, 8, G, 2)
    p = p.transpose(-1, -2).reshape(*lead, 4, 16, G, 1)
    k = p[..., 0, :, :, :] + p[..., 1, :, :, :] * k
    v = p[..., 2, :, :, :] + p[..., 3, :, :, :] * v
    return k.reshape(*lead, 16, D), v.reshape(*lead, 16, D)


def _plain_maps(st):
    q_len, context, page = st["q_len"].long(), st["context"].long(), st["case"]["page"]
    R, T, W = q_len.numel(), st["num_rows"], st["width"]
    q_end = torch.cumsum(q_len, 0)
    q_start, seq_len = q_end - q_len, context + q_len
    row = torch.arange(T, device=DEVICE)
    who = (row[:, None] >= q_end[None, :]).sum(1)
    live = who < R
    safe = who.clamp(max=R - 1)
    positions = torch.where(live, row - q_start[safe] + context[safe], 0)
    need = (seq_len + page - 1) // page
    first = torch.cumsum(need, 0) - need
    i = torch.arange(W, device=DEVICE)
    at = (first[:, None] + i).clamp(max=st["pages"].numel() - 1)
    table = torch.where(i < need[:, None], st["pages"].long()[at], -1)
    slots = torch.where(live, table[safe, positions // page] * page + positions % page, -1)
    who = torch.where(live, who, -1)
    return dict(q_start=q_start.int(), seq_len=seq_len.int(), positions=positions.int(), request_of_row=who.int(),
                slots=slots.int(), block_table=table.int())


def _down(x):
    """float32 rounded down to a bfloat16's bits."""
    b = x.contiguous().view(torch.int32)
    return (torch.where(x < 0, b + 0xffff, b) & -65536).view(torch.float32)


def _plain_quantised(x):
    x = x.reshape(*x.shape[:-1], -1, GROUP)
    lo = _down(x.amin(-1, keepdim=True))
    s = -_down(-(x.amax(-1, keepdim=True) - lo) / 15.0)
    codes = torch.where(s > 0, torch.round((x - lo) / s), 0.0).clamp(0.0, 15.0)
    return (lo + s * codes).flatten(-2)


def _plain_write(st):
    H, KV, D = HEADS[st["case"]["size"]]
    dtype = st["qkv"].dtype
    x = st["qkv"].float() + st["bias"]
    T = x.shape[0]
    angle = st["positions"].double()[:, None] * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    qk = x[:, :(H + KV) * D].reshape(T, H + KV, D)
    a, b = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    live = (st["slots"] >= 0)[:, None, None]
    k = torch.where(live, _plain_quantised(qk[:, H:]), 0.0)
    v = torch.where(live, _plain_quantised(x[:, (H + KV) * D:].reshape(T, KV, D)), 0.0)
    return dict(q=qk[:, :H].reshape(T, H * D).to(dtype), k=k.bfloat16(), v=v.bfloat16())


def _rows_of_requests(st):
    """Row numbers [R, most rows] (0 where a request has fewer), which of them are rows, and their positions."""
    i = torch.arange(st["most_rows"], device=DEVICE)
    live = i < st["q_len"][:, None]
    row = torch.where(live, st["q_start"][:, None] + i, 0).long()
    return row, live, (st["seq_len"] - st["q_len"])[:, None] + i


def _plain_attention(st):
    case = st["case"]
    H, KV, D = HEADS[case["size"]]
    R, N, page = st["q_len"].numel(), st["most_keys"], case["page"]
    held = st["cache"].reshape(st["cache"].shape[0], KV, page // 16, 20 * D)[st["block_table"].clamp(min=0).long()]
    k, v = (y.permute(0, 2, 1, 3, 4, 5).reshape(R, KV, -1, D)[:, :, :N] for y in _unpack(held, D))
    row, live, pos = _rows_of_requests(st)
    q = st["q"].float()[row].reshape(R, -1, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(R, KV, -1, D)
    key = torch.arange(N, device=DEVICE)
    seen = (key <= pos[..., None]) & (key < st["seq_len"][:, None, None])
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    seen = seen[:, None].expand(R, H // KV, -1, N).reshape(R, 1, -1, N)
    s = torch.where(seen, q @ k.transpose(-1, -2) * D ** -0.5, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.reshape(R, KV, H // KV, -1, D).permute(0, 3, 1, 2, 4).reshape(R, -1, H * D)
    out = st["out"]
    out[row[live]] = o[live].to(out.dtype)
    return out


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"maps": _plain_maps, "write": _plain_write, "attention": _plain_attention}[kind](st)
    from paged_batch_engine_b200.csrc import ops
    case = st["case"]
    page = case["page"]
    if kind == "maps":
        m = ops.page_maps(st["q_len"], st["context"], st["pages"], page, st["num_rows"], st["width"])
        return dict(q_start=m.q_start, seq_len=m.seq_len, positions=m.positions, request_of_row=m.request_of_row,
                    slots=m.slots, block_table=m.block_table)
    H, KV, D = HEADS[case["size"]]
    if kind == "write":
        ops.kv4_write(st["qkv"], st["bias"], st["q_out"], st["cache"], st["positions"], st["slots"], st["inv_freq"], H, KV,
                      D, D, page)
        k, v = ops.kv4_read(st["cache"], st["slots"], torch.bfloat16)
        return dict(q=st["q_out"], k=k, v=v)
    return ops.kv4_attention(st["q"], st["cache"], st["out"], st["q_start"], st["q_len"], st["seq_len"], st["block_table"],
                             H, KV, D, D ** -0.5, case["window"] or None, page, st["most_rows"], st["most_keys"])


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    step, page = _step(case), case["page"]
    T = sum(r for r, _ in step)
    need = [-(-k // page) for _, k in step]
    if case["kind"] == "maps":
        rows = T + case["spare"]
        return {"bytes": 4 * (2 * len(step) + sum(need) + 2 * len(step) + 3 * rows + len(step) * max(need)),
                "flops": 4 * rows + 2 * len(step) * max(need)}
    H, KV, D = HEADS[case["size"]]
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "write":
        rows = T + case["spare"]
        moved = rows * (H + 2 * KV) * D * size + rows * H * D * size + T * KV * D * 5 // 4 + rows * 2 * KV * D * 2
        return {"bytes": moved + 4 * ((H + 2 * KV) * D + D // 2 + 2 * rows), "flops": rows * (H + 2 * KV) * D * 6}
    keys, pairs = 0, 0
    for r, n in step:
        low = max(0, n - r - case["window"] + 1) if case["window"] else 0
        keys += n - low
        seen = (n - i for i in range(r))
        pairs += sum(min(x, case["window"]) if case["window"] else x for x in seen)
    return {"bytes": keys * KV * D * 5 // 4 + 2 * T * H * D * size + 4 * sum(need), "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_floor(x):
    """The largest number of eight significant bits that is not above x."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.floor(m * 256.0) / 256.0, e)


def _exact_group(x):
    lo = _exact_floor(x.min(-1, keepdim=True).values)
    s = -_exact_floor((lo - x.max(-1, keepdim=True).values) / 15.0)
    c = torch.round((x - lo) / torch.where(s > 0, s, 1.0)).clamp(0, 15)
    return lo + s * c


def exact(case, seed):
    if case["kind"] == "maps":
        return None
    st = prepare(case, seed)
    H, KV, D = HEADS[case["size"]]
    if case["kind"] == "write":
        x = st["qkv"].double() + st["bias"].double()
        T, half = x.shape[0], D // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                           st["positions"].double().outer(st["inv_freq"].double()))
        heads = x.view(T, H + 2 * KV, 2, half)
        z = torch.complex(heads[:, :H + KV, 0], heads[:, :H + KV, 1]) * turn[:, None]
        turned = torch.cat([z.real, z.imag], dim=-1)
        live = (st["slots"] >= 0).double()[:, None, None, None]
        groups = torch.cat([turned[:, H:], heads[:, H + KV:].flatten(2)], dim=1).view(T, 2 * KV, D // GROUP, GROUP)
        kept = (_exact_group(groups) * live).view(T, 2 * KV, D)
        return dict(q=turned[:, :H].reshape(T, H * D), k=kept[:, :KV].contiguous(), v=kept[:, KV:].contiguous())
    page, G = case["page"], D // GROUP
    cache = st["cache"].view(-1, KV, page // 16, 20 * D)
    channel = torch.arange(D, device=DEVICE)
    g, e, i = channel // 32, channel % 8, channel % 4
    tok = torch.arange(16, device=DEVICE)[:, None]
    # the bit at which a token's channel begins, within the keys' and within the values' codes
    k_bit = 32 * ((tok * 4 + channel % 32 // 8) * G + g) + 16 * (e % 2) + 4 * (e // 2)
    v_bit = 32 * ((tok // 2 * 8 + channel % 32 // 4) * G + g) + 16 * (tok % 2) + 4 * i
    at = (tok // 2 * G + g) * 2 + tok % 2
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEVICE)
    row0 = 0
    for r, (n, keys) in enumerate(_step(case)):
        records = cache[st["block_table"][r, :-(-keys // page)].long()].transpose(0, 1).reshape(KV, -1, 20 * D)
        codes = records[..., :16 * D].long()
        numbers = records[..., 16 * D:].contiguous().view(torch.bfloat16).double()
        value = lambda bits, base, lo, s: (numbers[..., lo * 16 * G + at] + numbers[..., s * 16 * G + at] * (  # noqa: E731
            codes[..., base + bits // 8] // (1 << (bits % 8)) % 16).double()).flatten(1, 2)[:, :keys]
        k, v = value(k_bit, 0, 0, 1), value(v_bit, 8 * D, 2, 3)
        step = max(1, (1 << 27) // (H * keys))             # rows at a time
        for o in range(0, n, step):
            m = min(step, n - o)
            q = st["q"][row0 + o:row0 + o + m].double().view(m, KV, H // KV, D)
            score = torch.einsum("mkgd,knd->kgmn", q, k) / math.sqrt(D)
            gap = torch.arange(keys - n + o, keys - n + o + m, device=DEVICE)[:, None] - torch.arange(keys, device=DEVICE)
            hidden = (gap < 0) | (gap >= case["window"]) if case["window"] else gap < 0
            w = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
            out[row0 + o:row0 + o + m] = torch.einsum("kgmn,knd->mkgd", w, v).reshape(m, H * D)
        row0 += n
    return out
