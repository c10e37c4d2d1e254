"""Steps whose row maps and block tables the device makes give every model's logits bit for bit as the host's do."""
import pytest
import torch

from tests import helpers

pytestmark = pytest.mark.gpu
MODELS = dict(TINY_B=helpers.TINY_B, TINY_D=helpers.TINY_D, GEB_A=helpers.GEB_A, GEB_C=helpers.GEB_C, BAV_A=helpers.BAV_A,
              BAV_B=helpers.BAV_B, GUS_A=helpers.GUS_A, MOB_A=helpers.MOB_A, TUT_A=helpers.TUT_A, MAL_A=helpers.MAL_A)


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", MODELS)
def test_logits_do_not_depend_on_who_makes_the_maps(name, dtype, bits, monkeypatch):
    from paged_batch_engine_b200.config.specs import ConfigError
    from paged_batch_engine_b200.engine import batch
    from paged_batch_engine_b200.engine.runner import ModelRunner
    config, made = MODELS[name], []
    for limit in (1 << 30, 1):
        monkeypatch.setattr(batch, "MAPS_ROWS", limit)
        try:
            runner = ModelRunner.from_random(config, seed=3, dtype=dtype, cache_bits=bits, page_tokens=16, num_pages=40, max_requests=4)
        except ConfigError:
            return                                                 # this model keeps no cache in four bits
        g = torch.Generator().manual_seed(7)
        handles = [runner.cache.add_request() for _ in range(3)]
        rows = []
        for step in ((70, 1, 20), (1, 33, 1), (1, 1, 1), (5, 0, 40)):
            entries = []
            for h, n in zip(handles, step):
                if n:
                    assert runner.cache.reserve(h, n)
                    tokens = torch.randint(0, runner.model.spec.vocab_size - 8, (n,), generator=g).tolist()
                    entries.append(batch.StepEntry(h, tokens, list(range(n))))
            rows.append(runner.step(entries).float().cpu())
        made.append(rows)
    for a, b in zip(*made):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_what_int32_does_not_hold_is_minus_one():
    """Positions and lengths beyond 2^31 - 1, and starts behind so many rows."""
    from paged_batch_engine_b200.csrc import ops
    top = 2 ** 31 - 1
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:0")  # noqa: E731
    m = ops.page_maps(ints([5, 2]), ints([top - 2, top - 2]), None, 16, 8, 0)
    assert m.positions.tolist() == [top - 2, top - 1, top, -1, -1, top - 2, top - 1, 0]
    assert m.request_of_row.tolist() == [0] * 5 + [1] * 2 + [-1]
    assert m.seq_len.tolist() == [-1, top] and m.q_start.tolist() == [0, 5]
    m = ops.page_maps(ints([top, top, 1]), ints([0, 0, 0]), None, 16, 1, 0)
    assert m.q_start.tolist() == [0, top, -1] and m.positions.tolist() == [0]
