"""Attention over 4-bit pages where it can go wrong at its edges: row tiles without a key, queries that are NaN, pages that are none.

Tolerances are those of ``test_gpu_kv4.Case.check`` unless a test says otherwise; outputs of rows without a key are zero exactly.
"""
import pytest
import torch

from tests.plain import plain_kv4 as plain
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
