"""The engine with its keys and values in four bits, against the plain implementation over what the engine's pages stand for.

A value next to the border of two codes may fall either way by the last bit of a float32 sum, so the plain implementation
takes the keys and values that the pages hold (read back by ``kv4_read``) and checks that each lies within half a step of its
own.  Logits then differ as they do over a cache in the run dtype: in bfloat16 by activations of 8 bits (2 % of the largest
logit), in float32 by the sums' order (2e-5) and by the weights' and queries' terms of three bfloat16, which come to the same
again."""
import os
import subprocess
import sys

import pytest
import torch

from tests import replay_util as ru
from tests.helpers import TINY_D, load_plain, make_model_folder
from tests.plain import plain_kv4, plain_qwen2 as plain

pytestmark = pytest.mark.gpu
TOL_F32 = 5e-5
TOL_BF16_REL = 0.02
ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))

# heads of 64, three on one; heads of 128, two key/value heads; the first with a window on its second layer
MODELS = {
    "h64": dict(TINY_D, use_sliding_window=False),
    "h128": dict(TINY_D, use_sliding_window=False, hidden_size=160, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                 vocab_size=397, eos_token_id=396),
    "window": dict(TINY_D, sliding_window=70),
}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {n: make_model_folder(tmp_path_factory.mktemp(n), cfg, seed=5, sharpen=5.0) for n, cfg in MODELS.items()}


def runner(folder, dtype, pool=2048, **kw):
    from paged_batch_engine_b200.engine.runner import ModelRunner
    return ModelRunner.from_folder(folder, dtype=dtype, device="cuda:0", page_tokens=16, max_cache_tokens=pool, max_requests=8,
                                   poison=True, cache_bits=4, **kw)


def requests(cfg, lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {f"r{i}": torch.randint(0, cfg["vocab_size"] - 8, (n,), generator=g).tolist() for i, n in enumerate(lens)}


def watch(run):
    """{handle: [layer][keys or values]: rows}: what the pages stand for, read when a step's tokens are marked computed (a
    window gives pages back after that)."""
    from paged_batch_engine_b200.csrc import ops
    kept, real = {}, run.cache.commit
    layers = range(len(run.model.blocks))

    def commit(handle, n):
        first = run.cache.context_len(handle)
        if first == 0:
            kept[handle] = [([], []) for _ in layers]
        for layer in layers:
            lc = run.storage.layer(layer)
            slots = [run.cache.slot_of_token(handle, lc.group, p) for p in range(first, first + n)]
            got = ops.kv4_read(lc.tensors["kv4"], torch.tensor(slots, dtype=torch.int32, device="cuda:0"), torch.float32)
            for x, held in zip(got, kept[handle][layer]):
                held.append(x.cpu())
        real(handle, n)

    run.cache.commit = commit
    return kept


def plain_over(monkeypatch, cfg, w, tokens, pages, exact):
    layer = iter(pages)
    real = plain.causal_attention

    def attention(q, k, v, scale, window=None):
        held = [torch.cat(x) for x in next(layer)]
        for x, have in zip((k, v), held):
            _, s, _ = plain_kv4.quantise(x)
            if exact:
                # half a step, the step one place of its eight bits larger, and the float32 sums' own difference
                assert ((have - x).abs() <= s.repeat_interleave(32, -1) * 0.504 + 1e-4 * x.abs().max()).all()
        return real(q, *held, scale, window)

    monkeypatch.setattr(plain, "causal_attention", attention)
    try:
        return plain.forward_logits(cfg, w, tokens)
    finally:
        monkeypatch.setattr(plain, "causal_attention", real)


SCHEDULES = {"whole": lambda r: ru.whole(r), "tail": lambda r: ru.tail_decoded(r, 20), "portions": lambda r: ru.portions(r),
             "mixed": lambda r: ru.mixed(r, seed=3)}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("schedule", SCHEDULES, ids=str)
@pytest.mark.parametrize("name", MODELS, ids=str)
def test_schedules_agree_with_plain(folders, monkeypatch, name, schedule, dtype):
    from paged_batch_engine_b200.engine.replay import TraceReplayer
    cfg, w = load_plain(folders[name])
    reqs = requests(cfg, [1, 17, 45, 130])
    records = SCHEDULES[schedule](reqs)
    run = runner(folders[name], dtype)
    pages, names, kept = watch(run), {}, {}
    replayer = TraceReplayer(run, decode_graphs=True)
    real = run.cache.add_request

    def add_request(rid):
        handle = real(rid)
        names[rid] = handle
        pages.pop(handle, None)
        return handle

    run.cache.add_request = add_request
    free = run.cache.free

    def give_back(handle):
        kept.update({rid: pages[handle] for rid, h in names.items() if h == handle and rid not in kept})
        free(handle)

    run.cache.free = give_back
    got = ru.run_records(run, records, replayer)
    if schedule == "tail":
        assert replayer.graph_steps > 0
    for rid, tokens in reqs.items():
        want = plain_over(monkeypatch, cfg, w, tokens, kept[rid], dtype == "float32")
        assert len(got[rid]) == len(tokens)
        worst = max(float((got[rid][p] - want[p]).abs().max()) for p in got[rid])
        assert worst <= (TOL_F32 if dtype == "float32" else TOL_BF16_REL * float(want.abs().max())), (rid, worst)


@pytest.mark.parametrize("name", MODELS, ids=str)
def test_generation(folders, name):
    """Greedy tokens with and without captured graphs and in a pool so small that requests are preempted: each is the largest of
    the logits that its sequence has when it is replayed, up to the few codes that sums of another order turn over (far less than
    activations of 8 bits move: 2 % of the largest logit)."""
    from paged_batch_engine_b200 import Engine, SamplingParams
    prompts = list(requests(MODELS[name], [5, 33, 90, 150], seed=1).values())
    params = SamplingParams(max_new_tokens=24, ignore_eos=True)
    run = runner(folders[name], "float32")
    kw = dict(dtype="float32", page_size=16, max_num_batched_tokens=64, prefill_chunk_cap=48, kv_cache_bits=4)
    for more in (dict(num_pages=64), dict(num_pages=64, use_cuda_graphs=False), dict(num_pages=17)):
        got = Engine(folders[name], **kw, **more).generate(prompts, params)
        assert [len(r.output_tokens) for r in got] == [24] * 4
        assert (sum(r.preemptions for r in got) > 0) == (more["num_pages"] == 17)
        for prompt, result in zip(prompts, got):
            tokens = prompt + result.output_tokens
            logits = ru.run_records(run, ru.portions({"r": tokens}))["r"]
            for i, token in enumerate(result.output_tokens):
                row = logits[len(prompt) + i - 1]
                assert float(row.max() - row[token]) <= TOL_BF16_REL * float(row.abs().max()), (more, i)
    wide = Engine(folders[name], num_pages=64, **{**kw, "dtype": "bfloat16"}).generate(prompts, params)
    assert [len(r.output_tokens) for r in wide] == [24] * 4


def test_a_pool_holds_more_tokens(folders):
    from paged_batch_engine_b200.engine.runner import ModelRunner
    four = runner(folders["h128"], "bfloat16")
    sixteen = ModelRunner.from_folder(folders["h128"], dtype="bfloat16", page_tokens=16, max_cache_tokens=64)
    assert sixteen.storage.bytes_per_token() * 10 == four.storage.bytes_per_token() * 32
    assert four.storage.paged[0]["kv4"].dtype == torch.uint8


def test_commands(folders, tmp_path):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "pbe-qwen"), folders["h64"], "--prompt-ids", "1,2,3,4",
                          "--max-new-tokens=6", "--ignore-eos", "--kv-cache-bits=4", "--kv-cache-blocks-per-layer=16"],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "steps:6" in out.stdout, out.stderr[-2000:]
    trace = '{"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [2]}], "end": ["a"]}\n'
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "trace_run"), "--model", folders["h64"], "--dtype", "float32",
                          "--out", str(tmp_path), "--max-tokens", "64", "--kv-cache-bits", "4"], input=trace, capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0 and "done 0" in out.stdout, out.stderr[-2000:]
    assert os.path.getsize(tmp_path / "0.f32") == 4 * MODELS["h64"]["vocab_size"]


@pytest.mark.parametrize("window", [None, 60])
def test_step_maps_made_on_the_device(monkeypatch, window):
    """The row maps and block tables of a step are the same integers whether the host makes them or the device."""
    from paged_batch_engine_b200.cache import CacheManager, KVGroupSpec
    from paged_batch_engine_b200.engine import batch
    groups = [KVGroupSpec((0,), 2, 64, None)] + ([KVGroupSpec((1,), 2, 64, window)] if window else [])
    m = CacheManager(groups, 16, [400] * len(groups), max_requests=16)
    entries = []
    for before, rows in ((0, 33), (100, 1), (250, 40), (16, 16), (7, 2)):
        h = m.add_request()
        for done in range(0, before, 50):
            n = min(50, before - done)
            assert m.reserve(h, n)
            m.commit(h, n)
        assert m.reserve(h, rows + 20)                             # pages beyond the step are held too
        entries.append(batch.StepEntry(h, [1] * rows, [0]))
    made = {}
    for limit in (1 << 30, 1):
        monkeypatch.setattr(batch, "MAPS_ROWS", limit)
        made[limit] = batch.StepContext(m, entries, torch.device("cuda:0"), [(0, 2, 16, None)])
    a, b = made[1 << 30], made[1]
    for x, y in ((a.positions, b.positions), (a.request_of_row, b.request_of_row), (a.q_start, b.q_start), (a.seq_len, b.seq_len)):
        assert torch.equal(x, y)
    for g in range(len(groups)):
        x, y = a.group(g), b.group(g)
        assert torch.equal(x.slots, y.slots) and x.bt_stride == y.bt_stride and x.block_table.shape == y.block_table.shape
        for r, n in enumerate(a.seq_len_host):
            pages = -(-int(n) // 16)
            assert torch.equal(x.block_table[r, :pages], y.block_table[r, :pages])
            assert (y.block_table[r, pages:] == -1).all()
    assert a.most_rows == b.most_rows == 40 and a.longest_keys == 290


@pytest.mark.parametrize("schedule", ["whole", "mixed"])
@pytest.mark.parametrize("name", MODELS, ids=str)
def test_portions_by_tcgen05(folders, monkeypatch, name, schedule):
    """The same where the tcgen05 kernel takes the portions, which it does for larger ones."""
    from paged_batch_engine_b200.csrc import ops
    monkeypatch.setattr(ops, "KV4_LITTLE_WORK", 0)
    monkeypatch.setattr(ops, "KV4_FEW_PACKED", 8)
    test_schedules_agree_with_plain(folders, monkeypatch, name, schedule, "bfloat16")
