"""Attention over 4-bit pages where it can go wrong at its edges: row tiles without a key, queries that are NaN, pages that are
none, tokens that a row does not see.

Tolerances are those of ``test_gpu_kv4.Case.check`` unless a test says otherwise; outputs of rows without a key are zero exactly.
"""
import pytest
import torch

from tests.plain import plain_kv4 as plain
from tests import test_gpu_kv4
from tests.test_gpu_kv4 import BF, DEV, F32, Case, ops

pytestmark = pytest.mark.gpu


def by_tcgen05(monkeypatch, splits=None):
    """Every request goes to the tcgen05 kernel; with ``splits``, its keys are shared by as many blocks."""
    o = ops()
    monkeypatch.setattr(o, "KV4_LITTLE_WORK", 0)
    monkeypatch.setattr(o, "KV4_FEW_PACKED", 1)
    if splits is not None:
        monkeypatch.setattr(o, "multiprocessors", lambda device: 1 << 20)
        monkeypatch.setattr(o, "KV4_SPLIT_KEYS", 1)
        monkeypatch.setattr(o, "KV4_MOST_SPLITS", splits)


# ------------------------------------------------------------------ row tiles without a key
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("step", [[(300, 0)], [(300, 20)], [(700, 100), (130, 0), (64, 64)]], ids=str)
@pytest.mark.parametrize("heads", [(28, 4, 128, 16), (14, 2, 64, 32), (4, 4, 64, 16), (4, 4, 128, 16)], ids=str)
def test_row_tiles_without_a_key(heads, step, splits, monkeypatch):
    """Requests of more rows than keys by whole row tiles: zeros there, whatever the queries."""
    by_tcgen05(monkeypatch, splits)
    c = Case(*heads, None, step, BF, seed=len(step), q_scale=50.0)
    out = ops().kv4_attention(*c.args(spare=3))
    c.check(out)                                                   # zero exactly before a request's first key
    assert (out[c.T:] == 7.0).all()


# ------------------------------------------------------------------ queries that are no numbers
@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("splits", [None, 1, 5])
@pytest.mark.parametrize("step", [[(300, 320)], [(300, 20), (40, 700)], [(1, 900), (3, 40)]], ids=str)
def test_a_query_that_is_no_number_spoils_its_own_row_alone(step, splits, bad, monkeypatch):
    if splits is not None:
        by_tcgen05(monkeypatch, splits)
    c = Case(14, 2, 64, 16, None, step, BF, seed=5)
    clean = ops().kv4_attention(*c.args()).clone()
    c.check(clean)
    args = c.args()
    places = [(r, h) for r, h in ((0, 3), (c.T // 2, 0), (c.T // 2, 13), (c.T - 1, 6))]
    for r, h in places:
        args[0][r, h * 64 + 7] = bad
    out = ops().kv4_attention(*args)
    at = 0
    for rows, n in step:
        for r, h in places:
            if at <= r < at + rows and r - at >= rows - n:         # a row that sees a key
                assert torch.isnan(out[r, h * 64:h * 64 + 64]).all()
        at += rows
    for r, h in places:
        out[r, h * 64:h * 64 + 64] = clean[r, h * 64:h * 64 + 64]
    c.check(out)


# ------------------------------------------------------------------ pages that are none
@pytest.mark.parametrize("dtype,splits", [(F32, None), (BF, None), (BF, 1), (BF, 3)], ids=["f32", "bf16", "tcgen05", "tcgen05-3"])
@pytest.mark.parametrize("short", [False, True])
def test_portions_see_no_key_of_a_page_that_is_none(short, splits, dtype, monkeypatch):
    """Portions of 70 rows: keys at entries that are no page, and behind the table's end, take no part, in either kernel."""
    if splits is not None:
        by_tcgen05(monkeypatch, splits)
    step = [(70, 160), (70, 90)]
    c = Case(14, 2, 64, 16, None, step, dtype)
    args = c.args()
    gone = [{2, 5}, {0}]
    c.table[0, 2], c.table[0, 5], c.table[1, 0] = -1, 1 << 20, -7
    width = 8 if short else c.table.shape[1]
    args[6] = c.table[:, :width].to(DEV).contiguous()
    out = ops().kv4_attention(*args)
    at = 0
    for r, (rows, n) in enumerate(step):
        k, v = c.kv[r]
        seen = torch.tensor([t // 16 not in gone[r] and t // 16 < width for t in range(n)])
        q = c.q[at:at + rows].double().reshape(rows, 2, 7, 64)
        s = torch.einsum("nkgd,tkd->nkgt", q, k) * c.scale
        see = seen[None] & (torch.arange(n)[None] <= torch.arange(n - rows, n)[:, None])
        w = torch.softmax(s.masked_fill(~see[:, None, None], float("-inf")), -1).nan_to_num(0.0)
        o = torch.einsum("nkgt,tkd->nkgd", w, v).reshape(rows, 14, 64)
        got = out[at:at + rows].cpu().double().reshape(rows, 14, 64)
        at += rows
        # as Case.check bounds the mean error; a key that is counted all the same moves a row by a sixtieth or more
        assert torch.isfinite(got).all()
        assert float((got - o).norm() / o.norm()) <= (2 ** -7 if dtype == BF else 2 ** -17)
        blind = ~see.any(-1)
        assert (got[blind] == 0).all()
        err = (got - o).norm(dim=(1, 2)) / o.norm(dim=(1, 2)).clamp_min(2 ** -10)
        assert float(err.max()) <= (2 ** -6 if dtype == BF else 2 ** -16)


# ------------------------------------------------------------------ what a row does not see
def check_rows(c, out):
    """``Case.check`` row by row: nothing but the keys that a row sees enters its tolerance."""
    at = 0
    for (rows, n), (k, v) in zip(c.step, c.kv):
        q = c.q[at:at + rows].reshape(rows, c.H, c.D)
        got = out[at:at + rows].cpu().double().reshape(rows, c.H, c.D)
        at += rows
        o, heavy, spread, reach = plain.attention(q, k, v, c.scale, c.window)
        pos, key = torch.arange(n - rows, n)[:, None], torch.arange(n)[None]
        see = (key <= pos) & (key > pos - (c.window or n))
        lean = 2 * torch.where(see, v.abs().amax((1, 2))[None], 0.0).amax(1)[:, None, None]
        step, d = 2 ** -8 if c.dtype == BF else 2 ** -22, 2 ** -8 if c.dtype == BF else 2 ** -18
        tol = 2 * step * (heavy + lean) + 2 ** -24 * (n / 16 + 64) * (heavy + lean) + step * o.abs() \
            + 2 * d * c.scale * reach[..., None] * spread
        err = (got - o).abs()
        assert torch.isfinite(got).all() and (err <= tol).all(), (rows, n, float((err / tol).max()))
        # and in a row's mean far nearer, but for rows whose scores a large key decides
        calm = ~(see & (k.abs().amax((1, 2)) > 50)[None]).any(1)
        rel = (err.norm(dim=(1, 2)) / o.norm(dim=(1, 2)))[calm]
        assert (rel <= (2 ** -6 if c.dtype == BF else 2 ** -16)).all(), (rows, n, rel)


def large_token(place, size, which):
    def edit(k, v):
        for x in which:
            if place < len(k):
                (k if x == "k" else v)[place] *= 2.0 ** size
    return edit


FORMS = [(BF, False), (F32, False), (BF, True)]


@pytest.mark.parametrize("dtype,prompt", FORMS, ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64, 16), (4, 4, 128, 32)], ids=str)
@pytest.mark.parametrize("window", [None, 3])
@pytest.mark.parametrize("which", ["v", "k"])
@pytest.mark.parametrize("size", [7, 12, 20, 30, 50])
@pytest.mark.parametrize("place", [71, 72, 79, 80])
def test_a_token_that_a_row_does_not_see_leaves_it_alone(place, size, which, window, heads, dtype, prompt, monkeypatch):
    """A token of 2^size times the others' keys or values, in the record of the rows' own keys and behind it: rows before it are as
    near as without it, and so are rows whose window has left it behind."""
    if "k" in which and size > 30:
        size = 30                                                  # scores of such keys leave float32 sooner than values
    if prompt:
        by_tcgen05(monkeypatch)
    c = Case(*heads, window, [(9, 76), (9, 84)], dtype, seed=place, edit=large_token(place, size, which))
    check_rows(c, ops().kv4_attention(*c.args()))


# ------------------------------------------------------------------ scores far from zero
FAR = [(BF, False), (F32, False), (BF, True)]


@pytest.mark.parametrize("dtype,prompt", FAR, ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64, 16), (4, 4, 128, 32)], ids=str)
@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("size", [10, 20, 23, 25, 30, 45])
def test_scores_far_from_zero(size, rows, heads, dtype, prompt, monkeypatch):
    """Queries of 2^size: one key has all of a row's weight, and the output is its value, where no other key's score comes near.

    A score is off by at most 2^-8 of its reach (as in ``Case.check``): rows whose second score is within twice that of the
    first are not looked at, but for being finite."""
    if prompt:
        by_tcgen05(monkeypatch)
    step = [(rows, 500), (rows, 77)]
    c = Case(*heads, None, step, dtype, seed=size, q_scale=2.0 ** size)
    out = ops().kv4_attention(*c.args()).cpu().double().reshape(c.T, c.H, c.D)
    assert torch.isfinite(out).all()
    at, looked = 0, 0
    for (n, keys), (k, v) in zip(step, c.kv):
        q = c.q[at:at + n].double().reshape(n, c.KV, -1, c.D)
        s = torch.einsum("nkgd,tkd->nkgt", q, k) * c.scale
        reach = torch.einsum("nkgd,tkd->nkgt", q.abs(), k.abs()).amax(-1) * c.scale
        see = torch.arange(keys)[None] <= torch.arange(keys - n, keys)[:, None]
        two = s.masked_fill(~see[:, None, None], float("-inf")).topk(2, -1)
        clear = two.values[..., 0] - two.values[..., 1] > 2 * 2 ** -8 * reach + 60.0
        want = torch.gather(v.permute(1, 0, 2)[None, :, None].expand(n, -1, q.shape[2], -1, -1), 3,
                            two.indices[..., :1, None].expand(-1, -1, -1, -1, c.D))[..., 0, :]
        err = (out[at:at + n].reshape(want.shape) - want).abs()[clear]
        assert (err <= (2 ** -7 if dtype == BF else 2 ** -17) * 3 * v.abs().max()).all()
        looked += int(clear.sum())
        at += n
    assert looked > c.T * c.H // 2


@pytest.mark.parametrize("dtype,prompt", FAR, ids=str)
@pytest.mark.parametrize("size", [20, 30, 50])
@pytest.mark.parametrize("place", [71, 72, 79, 80])
def test_a_token_of_large_key_and_value(place, size, dtype, prompt, monkeypatch):
    """Its score decides the rows that see it, whatever its size; the rows that do not stay as near as without it."""
    if prompt:
        by_tcgen05(monkeypatch)
    for heads in ((14, 2, 64, 16), (4, 4, 128, 32)):
        c = Case(*heads, None, [(9, 76), (9, 84)], dtype, seed=place, edit=large_token(place, size, "kv"))
        check_rows(c, ops().kv4_attention(*c.args()))


# ------------------------------------------------------------------ windows that hold every key, scales that leave nothing
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5], ids=str)
@pytest.mark.parametrize("step", [[(3, 2), (5, 40), (1, 0)], [(300, 20), (2, 0), (40, 40)]], ids=str)
def test_windows_longer_than_any_request(step, window, prompt, monkeypatch):
    """The same bits as without a window, for rows before the first key too."""
    if prompt:
        by_tcgen05(monkeypatch)
    c = Case(14, 2, 64, 16, None, step, BF, seed=3)
    want = ops().kv4_attention(*c.args()).clone()
    c.check(want)
    args = c.args()
    args[11] = window
    assert torch.equal(ops().kv4_attention(*args), want)


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("scale", [1e-10, 1e-30])
def test_scores_that_are_nothing(scale, prompt, monkeypatch):
    """Queries, or queries and keys, of zero under a scale that brings their units out of float32's range: plain means of the values."""
    if prompt:
        by_tcgen05(monkeypatch)
    for edit in (None, lambda k, v: k.zero_()):
        c = Case(14, 2, 64, 16, 37, [(40, 90), (1, 70)], BF, seed=4, edit=edit)
        c.q.zero_()
        c.scale = scale
        c.check(ops().kv4_attention(*c.args()))


# ------------------------------------------------------------------ many key/value heads
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(64, 64, 128, 16, 128, False, True, 5), (128, 64, 128, 16, 0, False, True, 3),
                                   (96, 96, 64, 32, 32, True, True, 7)], ids=str)
def test_write_of_many_key_value_heads(shape, dtype):
    """Rotations that keep rows in registers have no limit on heads."""
    test_gpu_kv4.test_write_and_read(shape, dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_attention_of_many_key_value_heads(dtype):
    for step in ([(1, 70), (1, 3)], [(40, 90)]):
        c = Case(64, 64, 128, 16, None, step, dtype, seed=6)
        c.check(ops().kv4_attention(*c.args()))


# ------------------------------------------------------------------ lists that a kernel makes
def test_maps_made_on_the_device_are_complete_before_the_steps_kernels(monkeypatch):
    """Attention kernels read block tables before they wait for the kernel before them: behind the launches that make the
    tables comes one that no kernel begins beside."""
    from paged_batch_engine_b200.cache import CacheManager, KVGroupSpec
    from paged_batch_engine_b200.engine import batch
    seen = []
    maps, fence = batch.ops.page_maps, batch.complete_before_what_follows
    monkeypatch.setattr(batch.ops, "page_maps", lambda *a: seen.append("maps") or maps(*a))
    monkeypatch.setattr(batch, "complete_before_what_follows", lambda device: seen.append("fence") or fence(device))
    groups = [KVGroupSpec((0,), 2, 64, None), KVGroupSpec((1,), 2, 64, 20)]
    for limit, want in ((1 << 30, []), (1, ["maps", "maps", "fence"])):
        monkeypatch.setattr(batch, "MAPS_ROWS", limit)
        seen.clear()
        m, entries = CacheManager(groups, 16, [40, 40], max_requests=4), []
        for rows in (40, 1):
            h = m.add_request()
            assert m.reserve(h, rows)
            entries.append(batch.StepEntry(h, [1] * rows, [0]))
        batch.StepContext(m, entries, torch.device(DEV), [])
        assert seen == want


# ------------------------------------------------------------------ attention beside the write, as a step calls the two
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("window", [None, 37])
@pytest.mark.parametrize("heads", [(28, 4, 128, 16), (14, 2, 64, 32), (24, 1, 64, 16), (40, 8, 128, 64)], ids=str)
@pytest.mark.parametrize("step", [[(1, 0), (1, 15), (1, 700)], [(5, 0), (3, 16), (1, 300), (40, 100)], [(2, 3001)], [(130, 40), (1, 64)]],
                         ids=str)
def test_attention_beside_the_write_of_portions(step, heads, window, prompt, monkeypatch):
    """``settled`` with portions: rows of ``step`` (rows, tokens before them) follow a projection and their own write, and have the
    bits of a call that waits for everything."""
    if prompt:
        by_tcgen05(monkeypatch)
    o, g = ops(), torch.Generator().manual_seed(len(step))
    H, KV, D, P = heads
    lens = [b + r for r, b in step]
    width = max(-(-n // P) for n in lens) + 1
    table = torch.randperm(len(step) * width, generator=g).to(torch.int32).reshape(len(step), width)
    pages = torch.full((len(step) * width, KV, P, o.kv4_width(D)), 0xff, dtype=torch.uint8, device=DEV)
    every = lambda first: [int(table[r, p // P]) * P + p % P for r, (n, b) in enumerate(step) for p in first(n, b)]  # noqa: E731
    old = test_gpu_kv4.ints(every(lambda n, b: range(b)))
    if len(old):
        x = torch.randn(len(old), (H + 2 * KV) * D, generator=g).to(BF).to(DEV)
        o.kv4_write(x, None, torch.empty(len(old), H * D, dtype=BF, device=DEV), pages, torch.zeros_like(old), old, None, H, KV, D, 0, P)
    T = sum(r for r, _ in step)
    slots = test_gpu_kv4.ints(every(lambda n, b: range(b, b + n)))
    rows, at = test_gpu_kv4.ints([r for r, _ in step]), test_gpu_kv4.ints([0] + [r for r, _ in step][:-1]).cumsum(0, dtype=torch.int32)
    seq, bt = test_gpu_kv4.ints(lens), table.to(DEV)
    weight = (torch.randn((H + 2 * KV) * D, 256, generator=g) / 16).to(BF).to(DEV)
    hidden = torch.randn(4, T, 256, generator=g).to(BF).to(DEV)
    torch.cuda.synchronize()
    for x in hidden:
        q, out, want = (torch.empty(T, H * D, dtype=BF, device=DEV) for _ in range(3))
        for into, settled in ((out, True), (want, False)):
            pages.view(-1)[:1].add_(0)                             # the call before it is behind a launch of its own
            qkv = o.linear(x, weight, None, out_dtype=BF, kind=1)
            o.kv4_write(qkv, None, q, pages, torch.zeros_like(slots), slots, None, H, KV, D, 0, P)
            o.kv4_attention(q, pages, into, at, rows, seq, bt, H, KV, D, D ** -0.5, window, P, max(r for r, _ in step), max(lens), settled)
        assert torch.isfinite(out).all() and torch.equal(out, want)


# ------------------------------------------------------------------ keys and values that lean
@pytest.mark.parametrize("dtype,prompt", FORMS, ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64, 16), (28, 4, 128, 16)], ids=str)
def test_keys_and_values_that_lean_by_many_spans(heads, dtype, prompt, monkeypatch):
    """Channels that lie far from zero in every token, as a bias on the projection makes them: groups' lo many times their s."""
    if prompt:
        by_tcgen05(monkeypatch)

    def edit(k, v):
        k[:, :, ::7] += 40.0
        k[:, :, 32:48] += 25.0
        v[:, :, 5::9] -= 60.0
    c = Case(*heads, None, [(40, 200), (1, 333), (3, 3)], dtype, seed=8, q_scale=0.25, edit=edit)
    check_rows(c, ops().kv4_attention(*c.args()))


def test_as_many_requests_as_a_call_takes():
    """Their lists fill the block's shared memory; the last request is as right as the first."""
    n = ops().KV4_MAX_REQUESTS
    c = Case(2, 1, 64, 16, None, [(1, 3 + i % 5) if i % 1000 == 0 or i == n - 1 else (0, 0) for i in range(n)], BF, seed=9)
    c.check(ops().kv4_attention(*c.args()))
    c = Case(2, 1, 64, 16, None, [(70, 75) if i == n - 1 else (0, 0) for i in range(n)], BF, seed=9)
    for few in (64, 1):
        args = c.args()
        ops().KV4_FEW_PACKED, kept = few, ops().KV4_FEW_PACKED
        try:
            c.check(ops().kv4_attention(*args))
        finally:
            ops().KV4_FEW_PACKED = kept


@pytest.mark.parametrize("dtype,prompt", FORMS, ids=str)
@pytest.mark.parametrize("place", [0, 33, 64, 90])
def test_large_values_that_weigh_nothing(place, dtype, prompt, monkeypatch):
    """A row that sees a value 2^16 times the others', at a score far below theirs: the others' mean, as near as without it (weights
    keep their eleven bits down to 2^-20 of the largest value that a row sees)."""
    if prompt:
        by_tcgen05(monkeypatch)

    def edit(k, v):
        k.zero_()
        k[place, :, 0] = -15.0
        v[place] *= 2.0 ** 16
    c = Case(4, 2, 64, 16, None, [(9, 110)], dtype, seed=place, edit=edit)
    c.q.zero_()
    c.q.view(-1, 4, 64)[:, :, 0] = 60.0                            # a score of -112: a weight of 2^-162
    out = ops().kv4_attention(*c.args()).cpu().double().reshape(9, 4, 64)
    v = c.kv[0][1].repeat_interleave(2, 1)
    for i in range(9):
        n = 110 - 8 + i
        seen = [t for t in range(n) if t != place]
        # weights are equal: rounded once with s (2^-11, to float32 nothing), and the output once
        tol = (2 ** -8 + 2 ** -11 if dtype == BF else 2 ** -17) * 3 * v[seen].abs().amax()
        assert ((out[i] - v[seen].mean(0)).abs() <= tol).all()


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("heads", [(28, 4, 128, 16), (14, 2, 64, 32)], ids=str)
def test_records_of_tokens_far_apart(heads, window, splits, monkeypatch):
    """Tokens 2^-12 and 2^-14 of the others' size, constant ones and zero ones, all over a prompt."""
    by_tcgen05(monkeypatch, splits)

    def edit(k, v):
        v[::7] *= 2.0 ** -12
        k[::5] *= 2.0 ** -14
        v[3::50], k[4::50], v[9::90] = 0.0, 0.0, 0.75
        k[100:140], v[100:140] = 0.0, 0.0
    c = Case(*heads, window, [(300, 700), (45, 45)], BF, seed=11, edit=edit)
    out = ops().kv4_attention(*c.args(spare=2))
    c.check(out)
    assert (out[c.T:] == 7.0).all()
