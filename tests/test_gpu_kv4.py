"""The 4-bit cache on the GPU against 64 bits: step maps, write and read-back, attention, and a run of them together.

Tolerances.  Half a step of bfloat16 is 2^-8 of a value (eps / 2), of float32 2^-24.
* maps: whole numbers, equal.
* write: a key or value read back in float32 is off the float32 value by at most s / 2, s read from the record, and a few
  float32 roundings of the rotation; lo and s lie within one bfloat16 step of the group's minimum and span.  Queries are off
  by the output's half step and the rotation's roundings: |a| + |b| times 8 * 2^-24.
* attention, weights w, values v, output o = sum w v: rounding the weights (once, and once more with the values' s) moves o by
  at most 2 * 2^-8 * sum w |v_code part|, where the code part is at most |v| + |lo|; the output's own rounding by 2^-8 |o|;
  scores that are off by d move o by at most 2 d * sum w |v - o|.  In float32 the factors are three terms: 2^-22 in their place,
  and sums over N keys, 2^-24 * (N / 16 + 64) of sum w |v|.
"""
import numpy as np
import pytest
import torch

from tests.plain import plain_kv4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def ops():
    from paged_batch_engine_b200.csrc import ops as o
    return o


def ints(x):
    return torch.as_tensor(x, dtype=torch.int32).to(DEV)


# ------------------------------------------------------------------ maps
def plain_maps(q_len, context, pages, P, rows, width, stride):
    R = len(q_len)
    out = dict(q_start=[], seq_len=[], positions=[], request_of_row=[], slots=[], table=np.full((R, width), -1, np.int64))
    first = 0
    for r, (q, c) in enumerate(zip(q_len, context)):
        out["q_start"].append(len(out["positions"]))
        out["seq_len"].append(q + c)
        need = -(-(q + c) // (P * stride))
        at = lambda i: (pages[i] if i < len(pages) else -1) if pages is not None else i  # noqa: E731
        for i in range(min(need, width)):
            out["table"][r, i] = at(first + i)
        for p in range(c, c + q):
            e = p // stride
            page = at(first + e // P)
            out["positions"].append(p)
            out["request_of_row"].append(r)
            out["slots"].append(page * P + e % P if page >= 0 else -1)
        first += need
    pad = rows - len(out["positions"])
    for name, v in (("positions", 0), ("request_of_row", -1), ("slots", -1)):
        out[name] = (out[name] + [v] * max(0, pad))[:rows]
    return out


@pytest.mark.parametrize("q_len,context,P,stride,spare,short", [
    ([1], [0], 16, 1, 0, 0), ([1], [15], 16, 1, 0, 0), ([1], [16], 16, 1, 3, 0), ([0], [0], 16, 1, 2, 0),
    ([5, 0, 1, 33, 7], [0, 40, 16, 15, 1000], 16, 1, 0, 0),
    ([5, 0, 1, 33, 7], [0, 0, 16, 15, 100], 3, 4, 5, 0),
    ([17, 1, 2], [9, 77, 31], 8, 1, 1, 4),                       # a page list that ends early
    ([1] * 700 + [300], list(range(700)) + [77], 16, 1, 9, 0),  # more requests than a block has threads
])
@pytest.mark.parametrize("listed", [True, False])
def test_page_maps(q_len, context, P, stride, spare, short, listed):
    g = torch.Generator().manual_seed(len(q_len) * P + stride)
    need = sum(-(-(q + c) // (P * stride)) for q, c in zip(q_len, context))
    pages = torch.randperm(need + 5, generator=g)[:max(0, need - short)].tolist() if listed else None
    if listed and need > 3:
        pages[1] = -1                                            # a page given back
    rows, width = sum(q_len) + spare, max(1, max(-(-(q + c) // (P * stride)) for q, c in zip(q_len, context))) + 2
    want = plain_maps(q_len, context, pages, P, rows, width, stride)
    got = ops().page_maps(ints(q_len), ints(context), ints(pages) if listed else None, P, rows, width, stride)
    for name in ("q_start", "seq_len", "positions", "request_of_row", "slots"):
        assert getattr(got, name).tolist() == want[name], name
    assert torch.equal(got.block_table.cpu().long(), torch.from_numpy(want["table"]))


def test_page_maps_sums_beyond_32_bits():
    """Contexts whose pages together pass 2^31: pages behind the list's end, slots beyond int32, are -1."""
    n, c = 40, 2 ** 30
    got = ops().page_maps(ints([1] * n), ints([c] * n), None, 1, n, 2)
    first = [i * (c + 1) for i in range(n)]
    assert got.positions.tolist() == [c] * n
    assert got.slots.tolist() == [f + c if f + c < 2 ** 31 else -1 for f in first]
    assert got.block_table[:, 0].tolist() == [f if f < 2 ** 31 else -1 for f in first]
    got = ops().page_maps(ints([1]), ints([2 ** 20]), ints([2 ** 30] * 2 ** 16 + [2 ** 30]), 16, 1, 1)
    assert got.slots.tolist() == [-1]


# ------------------------------------------------------------------ write and read
def raw_numbers(pages, slots, P, D):
    """lo and s as the pages hold them: float64 [T, KV, 4, G]."""
    n, KV = pages.shape[:2]
    rec = pages.cpu().reshape(n, KV, P // 16, 20 * D)
    _, _, at = plain.places(D)
    out = torch.empty(len(slots), KV, 4, D // 32, dtype=torch.float64)
    for i, s in enumerate(slots):
        held = rec[s // P, :, s % P // 16].long()
        for kind in range(4):
            where = 16 * D + kind * D + at[s % 16]
            b = (held[:, where] | held[:, where + 1] << 8).to(torch.int32) << 16
            out[i, :, kind] = b.view(torch.float32).double()
    return out


def plain_turned(qkv, bias, positions, inv_freq, H, KV, D, rot, interleaved):
    x = qkv.double() + (bias.double() if bias is not None else 0.0)
    x = x.reshape(x.shape[0], H + 2 * KV, D)
    t = x.clone()
    if inv_freq is not None and rot:
        a = positions.double()[:, None] * inv_freq.double()
        c, s = a.cos()[:, None], a.sin()[:, None]
        i0 = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
        i1 = i0 + 1 if interleaved else i0 + rot // 2
        u, v = x[:, :H + KV, i0], x[:, :H + KV, i1]
        t[:, :H + KV, i0] = u * c - v * s
        t[:, :H + KV, i1] = v * c + u * s
    return t, x.abs()


WRITES = [
    # H, KV, D, P, rotary, interleaved, bias, rows
    (28, 4, 128, 16, 128, False, True, 1), (28, 4, 128, 16, 128, False, True, 9), (14, 2, 64, 32, 64, False, True, 33),
    (12, 2, 128, 48, 64, False, False, 17), (3, 3, 64, 16, 64, True, True, 5), (8, 1, 128, 16, 0, False, True, 6),
    (40, 8, 128, 64, 128, True, False, 70), (6, 1, 64, 16, 34, False, True, 40), (48, 16, 128, 16, 128, False, True, 3),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", WRITES, ids=str)
def test_write_and_read(shape, dtype):
    H, KV, D, P, rot, interleaved, with_bias, T = shape
    o, g = ops(), torch.Generator().manual_seed(sum(shape))
    n = -(-T // P) + 3
    qkv = torch.randn(T, (H + 2 * KV) * D, generator=g) * torch.logspace(-2, 2, T)[:, None]
    qkv = qkv.to(dtype)
    bias = torch.randn((H + 2 * KV) * D, generator=g) if with_bias else None
    positions = torch.randint(0, 200000, (T,), generator=g)
    slots = torch.randperm(n * P, generator=g)[:T]
    live = torch.ones(T, dtype=torch.bool)
    if T > 4:
        slots[2], slots[3], live[2:4] = -1, n * P, False          # no slot, and one behind the last page
    inv = (10000.0 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))).float() if rot else None
    pages = torch.full((n, KV, P, o.kv4_width(D)), 0xa5, dtype=torch.uint8, device=DEV)
    q = torch.empty(T, H * D, dtype=dtype, device=DEV)
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    o.kv4_write(dev(qkv), dev(bias), q, pages, ints(positions), ints(slots), dev(inv), H, KV, D, rot, P, interleaved)
    want, size = plain_turned(qkv, bias, positions, inv, H, KV, D, rot, interleaved)
    near = 8 * 2 ** -24 * size.amax(-1, keepdim=True) * 2          # the rotation's and the bias's float32 roundings
    err = (q.cpu().double().reshape(T, H, D) - want[:, :H]).abs()
    assert (err <= near[:, :H] + want[:, :H].abs() * (2 ** -8 if dtype == BF else 2 ** -24)).all()
    got = torch.stack(o.kv4_read(pages, ints(slots), F32), 1).cpu().double()       # [T, 2, KV, D]
    kept = want[:, H:].reshape(T, 2, KV, D)
    num = raw_numbers(pages, slots[live].tolist(), P, D)                           # [live, KV, 4, G]
    lo, s = (torch.stack([num[:, :, k], num[:, :, k + 2]], 1) for k in (0, 1))     # [live, 2, KV, G]
    groups = kept[live].reshape(-1, 2, KV, D // 32, 32)
    slack = near[live, H:].reshape(-1, 2, KV, 1)
    mn, mx = groups.amin(-1), groups.amax(-1)
    assert (lo <= mn + slack).all() and (lo >= mn - mn.abs() * 2 ** -7 - slack * 1.01).all()
    span = (mx - lo) / 15
    assert (s >= span - slack).all() and (s <= (span + slack) * (1 + 2 ** -7)).all()
    err = (got[live].reshape(groups.shape) - groups).abs()
    assert (err <= (s * (0.5 + 2 ** -16) + slack + 2 ** -23 * (lo.abs() + 16 * s))[..., None]).all()
    assert (got[~live] == 0).all()
    same = torch.stack(o.kv4_read(pages, ints(slots), BF), 1).cpu()
    assert torch.equal(same, got.float().to(BF))
    # nothing but the rows' own bytes was written
    again = torch.full_like(pages, 0x5a)
    o.kv4_write(dev(qkv), dev(bias), q, again, ints(positions), ints(slots), dev(inv), H, KV, D, rot, P, interleaved)
    untouched = ((pages == 0xa5) & (again == 0x5a)).sum().item()
    assert untouched == (n * P - int(live.sum())) * KV * o.kv4_width(D)


@pytest.mark.parametrize("D,P,KV", [(64, 16, 3), (128, 32, 2)])
def test_write_is_the_oracle_where_nothing_rounds(D, P, KV):
    """No rotation, no bias, bfloat16 rows: the records are the oracle's, byte for byte, NaN and infinities too."""
    o, g = ops(), torch.Generator().manual_seed(D)
    T = 4 * P
    x = torch.randn(T, (1 + 2 * KV) * D, generator=g) * torch.logspace(-30, 30, T)[:, None]
    x[3] = 0.0
    x[5, D:] = 7.3
    x[7, D + 5], x[9, D + 40], x[11, D + 33] = float("nan"), float("inf"), float("-inf")
    x = x.to(BF)
    table = torch.randperm(6, generator=g)[:4].tolist()
    pages = torch.full((6, KV, P, o.kv4_width(D)), 0xff, dtype=torch.uint8, device=DEV)
    slots = ints([table[t // P] * P + t % P for t in range(T)])
    q = torch.empty(T, D, dtype=BF, device=DEV)
    o.kv4_write(x.to(DEV), None, q, pages, ints(range(T)), slots, None, 1, KV, D, 0, P)
    k, v = (x[:, D + i * KV * D:D + (i + 1) * KV * D].double().reshape(T, KV, D) for i in (0, 1))
    want = plain.to_pages(plain.pack(k, v), table, 6, P)
    assert torch.equal(pages.cpu(), want)
    assert torch.equal(q.cpu().view(torch.int16), x[:, :D].contiguous().view(torch.int16))


def test_write_nothing():
    o = ops()
    q = torch.empty(0, 4 * 64, dtype=BF, device=DEV)
    pages = torch.zeros(2, 2, 16, 80, dtype=torch.uint8, device=DEV)
    o.kv4_write(torch.empty(0, 8 * 64, dtype=BF, device=DEV), None, q, pages, ints([]), ints([]), None, 4, 2, 64, 0, 16)
    k, v = o.kv4_read(pages, ints([]))
    assert k.shape == v.shape == (0, 2, 64)
    x = torch.randn(3, 8 * 64, device=DEV).to(BF)                      # a layer that reads another layer's pages
    q = torch.empty(3, 4 * 64, dtype=BF, device=DEV)
    o.kv4_write(x, None, q, None, ints([0, 1, 2]), None, None, 4, 2, 64, 0, 16)
    assert torch.equal(q, x[:, :256])


# ------------------------------------------------------------------ attention
class Case:
    """Requests [(rows, keys)] with random pages; what no token fills holds NaN."""

    def __init__(self, H, KV, D, P, window, step, dtype, seed=0, q_scale=2.0, edit=None):
        o, g = ops(), torch.Generator().manual_seed(seed + D + P)
        self.H, self.KV, self.D, self.P, self.window, self.step, self.dtype = H, KV, D, P, window, step, dtype
        self.scale = D ** -0.5
        need = [-(-n // P) for _, n in step]
        order = torch.randperm(sum(need) + 3, generator=g).tolist()
        pages = torch.full((sum(need) + 3, KV, P, o.kv4_width(D)), 0xff, dtype=torch.uint8)
        self.tables, self.kv, at = [], [], 0
        for (_, n), m in zip(step, need):
            table, at = order[at:at + m], at + m
            self.tables.append(table)
            k = torch.randn(n, KV, D, generator=g) + 0.5 * torch.randn(KV, D, generator=g)
            v = torch.randn(n, KV, D, generator=g) + 0.5 * torch.randn(KV, D, generator=g)
            if edit:
                edit(k, v)
            fill = -n % 16
            rec = plain.pack(torch.cat([k, k.new_zeros(fill, KV, D)]), torch.cat([v, v.new_zeros(fill, KV, D)]))
            if n:
                held = [x.transpose(1, 2).reshape(n + fill, KV, D)[:n] for x in plain.unpack(rec)]
            else:
                held = [torch.zeros(0, KV, D, dtype=torch.float64)] * 2
            self.kv.append(held)
            for t in range(n, n + fill):                            # places behind the last token
                _, _, where = plain.places(D)
                for kind in range(4):
                    w = 16 * D + kind * D + where[t % 16]
                    rec[-1, :, w] = 0xff
                    rec[-1, :, w + 1] = 0xff
            per = P // 16
            for i in range(rec.shape[0]):
                pages.view(-1, KV, per, 20 * D)[table[i // per], :, i % per] = rec[i]
        self.pages = pages.to(DEV)
        self.T = sum(max(0, r) for r, _ in step)
        self.q = (q_scale * torch.randn(self.T, H * D, generator=g)).to(dtype)
        width = max(need + [1]) + 2
        self.table = torch.full((len(step), width), -1, dtype=torch.int32)
        for r, t in enumerate(self.tables):
            self.table[r, :len(t)] = torch.tensor(t, dtype=torch.int32)

    def args(self, spare=0):
        rows = [r for r, _ in self.step]
        starts = np.cumsum([0] + rows[:-1])
        self.out = torch.full((self.T + spare, self.H * self.D), 7.0, dtype=self.dtype, device=DEV)
        q = torch.cat([self.q, torch.full((spare, self.H * self.D), float("nan"), dtype=self.dtype)]).to(DEV)
        return [q, self.pages, self.out, ints(starts), ints(rows), ints([n for _, n in self.step]), self.table.to(DEV), self.H,
                self.KV, self.D, self.scale, self.window, self.P, max(rows), max(n for _, n in self.step)]

    def check(self, out):
        at = 0
        for (rows, n), (k, v) in zip(self.step, self.kv):
            if rows == 0:
                continue
            got = out[at:at + rows].cpu().double().reshape(rows, self.H, self.D)
            seen = min(rows, n)                                     # rows before the first key see none
            assert (got[:rows - seen] == 0).all()
            q = self.q[at + rows - seen:at + rows].reshape(seen, self.H, self.D)
            at += rows
            o, heavy, spread, reach = plain.attention(q, k, v, self.scale, self.window)
            lean = 2 * v.abs().max() if n else 0.0                  # |code part| and |lo| of a value, at most
            step = 2 ** -8 if self.dtype == BF else 2 ** -22
            most = 2 ** -24 * (n / 16 + 64)
            # scores: rounding keys to bfloat16 in the form for prompts, float32 sums in both
            d = (self.scale * reach * (2 ** -8 if self.dtype == BF else 2 ** -18))[..., None]
            tol = 2 * step * (heavy + lean) + most * (heavy + lean) + step * o.abs() + 2 * d * spread + 2 ** -20
            err = (got[rows - seen:] - o).abs()
            assert torch.isfinite(got).all() and (err <= tol).all(), (rows, n, float((err / tol).max()))
            # and in the mean far nearer than at worst
            rel = float(err.norm() / o.norm()) if n else 0.0
            assert rel <= (2 ** -7 if self.dtype == BF else 2 ** -17), (rows, n, rel)


STEPS = {
    "one": [(1, 1)], "few": [(1, 5), (1, 16), (1, 17), (1, 31)], "long": [(1, 3001)], "many": [(1, 40 * i + 1) for i in range(20)],
    "short_portions": [(2, 2), (3, 40), (2, 17), (1, 100), (5, 5)],
    "portions": [(70, 70), (1, 300), (33, 500), (130, 131), (17, 17)],
    "prompt": [(300, 300)], "none": [(0, 0), (1, 50), (0, 20), (3, 2), (2, 0), (40, 33)],
}
HEADS = [(28, 4, 128, 16), (14, 2, 64, 32), (12, 2, 128, 48), (4, 4, 64, 16), (24, 1, 64, 16), (40, 8, 128, 64), (20, 1, 128, 16)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("step", STEPS, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("window", [None, 37])
def test_attention(heads, step, window, dtype):
    c = Case(*heads, window, STEPS[step], dtype, seed=len(step))
    out = ops().kv4_attention(*c.args(spare=3))
    c.check(out)
    assert (out[c.T:] == 7.0).all()                                # rows of no request stay


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("at", [0, 15, 16, 255, 256, 1000, 1029])
def test_attention_one_key_stands_out(at, dtype):
    """The row's output is that key's value, wherever it lies."""
    def edit(k, v):
        k.mul_(0.05)
        k[at] = 0.0
        k[at, :, 0] = 15.0
    c = Case(4, 2, 64, 16, None, [(1, 1030)], dtype, seed=at, edit=edit)
    c.q.zero_()
    c.q.view(-1, 4, 64)[:, :, 0] = 40.0
    out = ops().kv4_attention(*c.args())
    v = c.kv[0][1][at].repeat_interleave(2, 0)
    assert (out[0].cpu().double().reshape(4, 64) - v).abs().max() <= (2 ** -8 if dtype == BF else 2 ** -18) * 3 * v.abs().max()


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_far_scores_and_sizes(rows):
    """Scores of hundreds, keys and values of 2^30 and 2^-30 beside each other: finite, and right to the values' size."""
    def edit(k, v):
        v[::2] *= 2.0 ** 30
        v[1::2] *= 2.0 ** -30
    c = Case(14, 2, 64, 16, None, [(rows, 200)], BF, q_scale=60.0, edit=edit)
    c.check(ops().kv4_attention(*c.args()))


def test_attention_pages_that_are_none():
    """Keys at a table entry that is no page are not seen; the table may end before the keys do."""
    for rows in (1, 70):
        c = Case(14, 2, 64, 16, None, [(rows, 160), (rows, 90)], BF)
        args = c.args()
        c.table[0, 2], c.table[0, 5] = -1, 1 << 20
        args[6] = c.table[:, :5].to(DEV).contiguous() if rows == 1 else c.table.to(DEV)
        out = ops().kv4_attention(*args)
        seen = torch.ones(160, dtype=torch.bool)
        seen[32:48] = False
        seen[80:96] = False
        if rows == 1:
            seen[80:] = False
            k, v = (x[seen] for x in c.kv[0])
            o, *_ = plain.attention(c.q[:1].reshape(1, 14, 64), k, v, c.scale)
            assert (out[:1].cpu().double().reshape(1, 14, 64) - o).abs().max() <= 2 ** -5
        else:
            assert torch.isfinite(out).all()


def test_attention_strided_table_and_hints():
    """The table may be a slice; the hints choose the launch, not the result."""
    c = Case(28, 4, 128, 16, None, [(1, 700), (20, 300), (1, 3), (90, 90)], BF)
    args = c.args()
    want = ops().kv4_attention(*args).clone()
    wide = torch.full((4, args[6].shape[1] + 9), -5, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + args[6].shape[1]] = args[6]
    args[6] = wide[:, 4:4 + args[6].shape[1]]
    assert torch.equal(ops().kv4_attention(*args), want)
    for most_rows, most_keys in ((1, 1), (90, 1 << 20), (4096, 700)):
        args[13:] = [most_rows, most_keys]
        args[2].fill_(7.0)
        c.check(ops().kv4_attention(*args))


def test_attention_same_bits_twice():
    for step in ([(1, 5000), (1, 30)], [(200, 200), (3, 900)]):
        c = Case(28, 4, 128, 16, None, step, BF)
        args = c.args()
        first = ops().kv4_attention(*args).clone()
        for _ in range(3):
            args[2].fill_(7.0)
            assert torch.equal(ops().kv4_attention(*args), first)


def test_attention_captured_and_on_two_streams():
    """Two captured graphs, replayed on two streams at once with inputs that change, beside eager calls."""
    cases = [Case(28, 4, 128, 16, None, [(1, 900)] * 6, BF, seed=1), Case(14, 2, 64, 32, 300, [(60, 2000), (1, 400)], BF, seed=2)]
    args = [c.args() for c in cases]
    want, graphs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for a, s in zip(args, streams):
        want.append(ops().kv4_attention(*a).clone())
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            ops().kv4_attention(*a)
        graphs.append(graph)
    for round_ in range(4):
        for a, s, graph in zip(args, streams, graphs):
            with torch.cuda.stream(s):
                a[2].fill_(7.0)
                graph.replay()
        torch.cuda.synchronize()
        for a, w, c in zip(args, want, cases):
            assert torch.equal(a[2], w)
    args[0][0].neg_()                                             # other queries, the same graph
    graphs[0].replay()
    torch.cuda.synchronize()
    cases[0].q.neg_()
    cases[0].check(args[0][2])


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_steps_of_a_cache(dtype):
    """Prompts, a portion behind its context and decoded tokens, step by step: maps, write, attention over what the steps
    before wrote; against attention over the read-back keys and values."""
    o, g = ops(), torch.Generator().manual_seed(3)
    H, KV, D, P = 12, 2, 128, 16
    lens, held = [0, 0, 0], [[], [], []]
    pages = torch.full((64, KV, P, o.kv4_width(D)), 0xff, dtype=torch.uint8, device=DEV)
    pool = torch.randperm(64, generator=g).tolist()
    inv = (1e4 ** (-torch.arange(0, D, 2).double() / D)).float().to(DEV)
    for step in ([40, 7, 0], [1, 60, 16], [1, 1, 1], [1, 1, 1], [20, 1, 2]):
        for r, n in enumerate(step):
            while len(held[r]) * P < lens[r] + n:
                held[r].append(pool.pop())
        T = sum(step)
        m = o.page_maps(ints(step), ints(lens), ints(sum(held, [])), P, T, 8)
        qkv = torch.randn(T, (H + 2 * KV) * D, generator=g).to(dtype).to(DEV)
        q, out = (torch.empty(T, H * D, dtype=dtype, device=DEV) for _ in range(2))
        o.kv4_write(qkv, None, q, pages, m.positions, m.slots, inv, H, KV, D, D, P)
        o.kv4_attention(q, pages, out, m.q_start, ints(step), m.seq_len, m.block_table, H, KV, D, D ** -0.5, None, P,
                        max(step), max(a + b for a, b in zip(step, lens)))
        at = 0
        for r, n in enumerate(step):
            lens[r] += n
            if not n:
                continue
            slots = ints([held[r][p // P] * P + p % P for p in range(lens[r])])
            k, v = (x.cpu().double() for x in o.kv4_read(pages, slots, F32))
            want, *_ = plain.attention(q[at:at + n].cpu().reshape(n, H, D), k, v, D ** -0.5)
            got = out[at:at + n].cpu().double().reshape(n, H, D)
            assert float((got - want).norm() / want.norm()) <= (2 ** -7 if dtype == BF else 2 ** -17)
            at += n


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cluster", [0, 1, 2, 4, 8, 16])
def test_attention_every_shape_of_launch(cluster, dtype, monkeypatch):
    """Clusters of every size, fewer of them than items, and tiles shared evenly: right, and the same rows left alone."""
    o = ops()
    for heads, step in (((28, 4, 128, 16), [(1, 700), (2, 300), (1, 3), (0, 9), (1, 1100)]), ((14, 2, 64, 32), [(9, 1000), (1, 40)]),
                        ((5, 5, 128, 16), [(1, 1), (1, 15), (1, 16), (1, 17)])):
        rows = 16 if dtype == BF and cluster % 3 == 1 else 8
        monkeypatch.setattr(o, "_kv4_shape", lambda *a: (rows, 3 * max(cluster, 1), cluster))
        c = Case(*heads, None, step, dtype, seed=cluster)
        out = o.kv4_attention(*c.args(spare=2))
        c.check(out)
        assert (out[c.T:] == 7.0).all()
        assert torch.equal(o.kv4_attention(*c.args(spare=2)), out)


# ------------------------------------------------------------------ small portions with the tcgen05 kernel too
PORTIONS = {**{k: STEPS[k] for k in ("short_portions", "portions", "prompt", "none")}, "alone": [(3, 40)], "tail": [(129, 2000), (9, 9)]}


@pytest.mark.parametrize("step", PORTIONS, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("window", [None, 37])
def test_attention_of_portions_by_tcgen05(heads, step, window, monkeypatch):
    """Portions too small for that kernel to be chosen: it takes them all the same."""
    o = ops()
    monkeypatch.setattr(o, "KV4_LITTLE_WORK", 0)
    monkeypatch.setattr(o, "KV4_FEW_PACKED", 16)
    c = Case(*heads, window, PORTIONS[step], BF, seed=len(step) + 1)
    out = o.kv4_attention(*c.args(spare=3))
    c.check(out)
    assert (out[c.T:] == 7.0).all()
    for splits in (1, 2, 5):                                       # shared along the keys, more splits than tiles too
        monkeypatch.setattr(o, "multiprocessors", lambda device: 1 << 20)
        monkeypatch.setattr(o, "KV4_SPLIT_KEYS", 1)
        monkeypatch.setattr(o, "KV4_MOST_SPLITS", splits)
        c.check(o.kv4_attention(*c.args(spare=3)))


@pytest.mark.parametrize("test", [lambda: test_attention_far_scores_and_sizes(40), test_attention_pages_that_are_none,
                                  test_attention_strided_table_and_hints, test_attention_same_bits_twice,
                                  test_attention_captured_and_on_two_streams, lambda: test_steps_of_a_cache(BF)],
                         ids=["sizes", "pages", "hints", "bits", "captured", "steps"])
def test_tcgen05_again(test, monkeypatch):
    monkeypatch.setattr(ops(), "KV4_LITTLE_WORK", 0)
    monkeypatch.setattr(ops(), "KV4_FEW_PACKED", 1)
    test()


def test_little_work_goes_to_one_kernel(monkeypatch):
    """Which kernels a call launches, by its hints."""
    o = ops()
    calls = []
    real = o._kv4_prompt_fn()
    monkeypatch.setattr(o, "_kv4_prompt_fn", lambda: lambda *a: calls.append(a[2:4]) or real(*a))
    for step, rows, keys, there in (([(37, 300)], 37, 300, 0), ([(600, 600)], 600, 600, 1), ([(37, 300)] * 9, 37, 300, 1),
                                    ([(37, 300)], 37, 1 << 17, 1), ([(1, 300)], 1, 1 << 17, 0)):
        calls.clear()
        c = Case(28, 4, 128, 16, None, step, BF, seed=7)
        args = c.args()
        args[13:] = [rows, keys]
        c.check(o.kv4_attention(*args))
        assert len(calls) == there, (step, rows, keys)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lens", [[0], [5, 15, 16, 17, 31, 32], [700] * 3, [4000, 3, 100], [300 + 16 * i for i in range(40)]], ids=len)
@pytest.mark.parametrize("captured", [False, True])
def test_attention_beside_the_write(lens, dtype, captured):
    """``settled``: lists and older keys may be read beside the write of the step's own keys, which are waited for.  The same bits
    as a call that waits for everything, token after token, as a record fills and the next begins."""
    o, g = ops(), torch.Generator().manual_seed(len(lens))
    H, KV, D, P, R = 12, 2, 128, 16, len(lens)
    width = (max(lens) + 24) // P + 1
    table = torch.randperm(R * width, generator=g).to(torch.int32).reshape(R, width)
    pages = torch.full((R * width, KV, P, o.kv4_width(D)), 0xff, dtype=torch.uint8, device=DEV)
    for r, n in enumerate(lens):
        if n:
            x = torch.randn(n, (H + 2 * KV) * D, generator=g).to(dtype).to(DEV)
            slots = ints([int(table[r, p // P]) * P + p % P for p in range(n)])
            o.kv4_write(x, None, torch.empty(n, H * D, dtype=dtype, device=DEV), pages, ints(range(n)), slots, None, H, KV, D, 0, P)
    qkv = torch.empty(R, (H + 2 * KV) * D, dtype=dtype, device=DEV)
    positions, slots, seq, starts, ones = (ints([0] * R) for _ in range(5))
    starts.copy_(torch.arange(R)), ones.fill_(1)
    q, out, want = (torch.empty(R, H * D, dtype=dtype, device=DEV) for _ in range(3))
    bt = table.to(DEV)

    def step(into, settled):
        o.kv4_write(qkv, None, q, pages, positions, slots, None, H, KV, D, 0, P)
        o.kv4_attention(q, pages, into, starts, ones, seq, bt, H, KV, D, D ** -0.5, None, P, 1, max(lens) + 24, settled)

    graph = torch.cuda.CUDAGraph()
    if captured:
        slots.fill_(-1), seq.fill_(0)
        step(out, True)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step(out, True)
    for t in range(20):
        at = [n + t for n in lens]
        qkv.copy_(torch.randn(R, (H + 2 * KV) * D, generator=g))
        positions.copy_(torch.tensor(at)), seq.copy_(torch.tensor(at) + 1)
        slots.copy_(torch.tensor([int(table[r, p // P]) * P + p % P for r, p in enumerate(at)]))
        graph.replay() if captured else step(out, True)
        torch.cuda.synchronize()
        o.kv4_attention(q, pages, want, starts, ones, seq, bt, H, KV, D, D ** -0.5, None, P, 1, max(lens) + 24)
        assert torch.isfinite(out).all() and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(28, 4, 128, 128, False), (14, 2, 64, 64, False), (40, 8, 128, 128, True), (1, 1, 64, 0, False),
                                   (6, 2, 128, 96, False)], ids=str)
def test_write_many_rows(shape, dtype):
    """More rows than blocks: the same bytes and queries as row by row in calls of 50, also where rows in between write nothing."""
    H, KV, D, rot, interleaved = shape
    o, g = ops(), torch.Generator().manual_seed(H)
    T, P = 1901, 32
    qkv = (torch.randn(T, (H + 2 * KV) * D, generator=g) * torch.logspace(-3, 3, T)[:, None]).to(dtype).to(DEV)
    bias = torch.randn((H + 2 * KV) * D, generator=g).to(DEV)
    positions, order = ints(torch.randint(0, 100000, (T,), generator=g).tolist()), torch.randperm(64 * P, generator=g)[:T]
    order[::7] = -1
    slots = ints(order.tolist())
    inv = (1e4 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))).float().to(DEV) if rot else None
    made = []
    for portion in (T, 50):
        pages = torch.full((64, KV, P, o.kv4_width(D)), 0xa5, dtype=torch.uint8, device=DEV)
        q = torch.empty(T, H * D, dtype=dtype, device=DEV)
        for at in range(0, T, portion):
            some = slice(at, at + portion)
            o.kv4_write(qkv[some], bias, q[some], pages, positions[some].clone(), slots[some].clone(), inv, H, KV, D, rot, P,
                        interleaved)
        made.append((pages, q))
    assert torch.equal(made[0][0], made[1][0])
    assert torch.equal(made[0][1], made[1][1])


@pytest.mark.parametrize("rows", [1, 460])
def test_pages_beyond_4_gigabytes(rows):
    """Write, read and attention (either kernel) at pages whose bytes lie behind 2^32."""
    o, g = ops(), torch.Generator().manual_seed(rows)
    H, KV, D, P, n = 14, 2, 128, 16, 460
    count = (1 << 32) // (KV * P * o.kv4_width(D)) + 200
    pages = torch.empty((count, KV, P, o.kv4_width(D)), dtype=torch.uint8, device=DEV)
    pages[:64].fill_(0xff)
    far = count - 1 - torch.randperm(100, generator=g)[:-(-n // P)]
    slots = ints([int(far[p // P]) * P + p % P for p in range(n)])
    x = torch.randn(n, (H + 2 * KV) * D, generator=g).to(BF)
    q = torch.empty(n, H * D, dtype=BF, device=DEV)
    o.kv4_write(x.to(DEV), None, q, pages, ints(range(n)), slots, None, H, KV, D, 0, P)
    k, v = (y.cpu() for y in o.kv4_read(pages, slots, F32))
    for have, want in ((k, x[:, H * D:(H + KV) * D]), (v, x[:, (H + KV) * D:])):
        assert torch.equal(have.double(), plain.dequantise(*plain.quantise(want.double().reshape(n, KV, D))).float().double())
    own = q[n - rows:].contiguous()
    out = o.kv4_attention(own, pages, torch.empty_like(own), ints([0]), ints([rows]), ints([n]), far.to(torch.int32)[None].to(DEV), H,
                          KV, D, D ** -0.5, None, P, rows, n)
    want, *_ = plain.attention(own.cpu().reshape(rows, H, D), k, v, D ** -0.5)
    err = (out.cpu().double().reshape(rows, H, D) - want).norm() / want.norm()
    assert float(err) <= 2 ** -7                                   # as Case.check bounds the mean error
