"""The 4-bit cache without a GPU: the oracle's records, and what the entry points refuse."""
import pytest
import torch

from paged_batch_engine_b200.csrc import ops
from tests.plain import plain_kv4 as plain


@pytest.mark.parametrize("D", [64, 128])
def test_oracle_records_hold_every_code_once(D):
    k_bits, v_bits, at = plain.places(D)
    bits = torch.cat([k_bits.flatten(), v_bits.flatten()])
    assert torch.equal(bits.sort().values, torch.arange(2 * 16 * D) * 4)
    assert torch.equal(at.flatten().sort().values, torch.arange(16 * D // 32) * 2)
    assert 16 * D + 3 * D + int(at.max()) + 2 == 20 * D == 16 * ops.kv4_width(D)


@pytest.mark.parametrize("D", [64, 128])
def test_oracle_quantisation(D):
    g = torch.Generator().manual_seed(D)
    x = torch.randn(32, 3, D, generator=g, dtype=torch.float64) * torch.logspace(-3, 3, 32)[:, None, None]
    x[0, 0] = 0.0
    x[1, 0, :32] = 7.3
    lo, s, c = plain.quantise(x)
    back = plain.dequantise(lo, s, c)
    step = s.repeat_interleave(32, -1)
    assert ((back - x).abs() <= step / 2 * (1 + 2 ** -40)).all()
    rec = plain.pack(x, -x)
    k, v = plain.unpack(rec)
    k2 = k.transpose(1, 2).reshape(32, 3, D)
    assert torch.equal(k2, back)
    assert torch.equal(v.transpose(1, 2).reshape(32, 3, D), plain.dequantise(*plain.quantise(-x)))


def _write_args(**change):
    H, KV, D, P, T = 4, 2, 64, 16, 3
    a = dict(qkv=torch.zeros(T, (H + 2 * KV) * D, dtype=torch.bfloat16), bias=torch.zeros((H + 2 * KV) * D),
             q_out=torch.zeros(T, H * D, dtype=torch.bfloat16), pages=torch.zeros(5, KV, P, 80, dtype=torch.uint8),
             positions=torch.zeros(T, dtype=torch.int32), slots=torch.zeros(T, dtype=torch.int32),
             inv_freq=torch.zeros(D // 2), num_heads=H, num_kv_heads=KV, head_dim=D, rotary_dim=D, page_tokens=P)
    a.update(change)
    return a


def _attn_args(**change):
    H, KV, D, P, T, R = 4, 2, 64, 16, 3, 2
    a = dict(q=torch.zeros(T, H * D, dtype=torch.bfloat16), pages=torch.zeros(5, KV, P, 80, dtype=torch.uint8),
             out=torch.zeros(T, H * D, dtype=torch.bfloat16), q_start=torch.zeros(R, dtype=torch.int32),
             q_len=torch.ones(R, dtype=torch.int32), seq_len=torch.ones(R, dtype=torch.int32),
             block_table=torch.zeros(R, 4, dtype=torch.int32), num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1,
             window=None, page_tokens=P, most_rows=1, most_keys=1)
    a.update(change)
    return a


def _ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


REFUSALS = [
    (ops.kv4_write, _write_args, dict(head_dim=96), "head sizes"),
    (ops.kv4_write, _write_args, dict(page_tokens=8), "multiple of 16"),
    (ops.kv4_write, _write_args, dict(pages=torch.zeros(5, 2, 16, 64, dtype=torch.uint8)), "pages must be"),
    (ops.kv4_write, _write_args, dict(pages=torch.zeros(5, 2, 16, 80, dtype=torch.int8)), "pages must be"),
    (ops.kv4_write, _write_args, dict(pages=torch.zeros(5, 2, 16, 160, dtype=torch.uint8)[..., :80]), "contiguous"),
    (ops.kv4_write, _write_args, dict(pages=torch.zeros(5 * 2 * 16 * 80 + 8, dtype=torch.uint8)[8:].view(5, 2, 16, 80)),
     "16-byte"),
    (ops.kv4_write, _write_args, dict(q_out=torch.zeros(3, 256)), "do not agree"),
    (ops.kv4_write, _write_args, dict(qkv=torch.zeros(3, 512, dtype=torch.float16),
                                      q_out=torch.zeros(3, 256, dtype=torch.float16)), "float32 or bfloat16"),
    (ops.kv4_write, _write_args, dict(bias=torch.zeros(512, dtype=torch.bfloat16)), "bias"),
    (ops.kv4_write, _write_args, dict(positions=_ints(2)), "positions"),
    (ops.kv4_write, _write_args, dict(slots=None), "slots"),
    (ops.kv4_write, _write_args, dict(slots=torch.zeros(3, dtype=torch.int64)), "slots"),
    (ops.kv4_write, _write_args, dict(rotary_dim=63), "inv_freq"),
    (ops.kv4_write, _write_args, dict(rotary_dim=32), "inv_freq"),
    (ops.kv4_attention, _attn_args, dict(num_heads=5), "multiple"),
    (ops.kv4_attention, _attn_args, dict(head_dim=32), "head sizes"),
    (ops.kv4_attention, _attn_args, dict(page_tokens=24), "multiple of 16"),
    (ops.kv4_attention, _attn_args, dict(out=torch.zeros(3, 256)), "one dtype"),
    (ops.kv4_attention, _attn_args, dict(q=torch.zeros(3, 512, dtype=torch.bfloat16)[:, ::2]), "contiguous"),
    (ops.kv4_attention, _attn_args, dict(q_len=torch.ones(2, dtype=torch.int64)), "int32"),
    (ops.kv4_attention, _attn_args, dict(seq_len=_ints(3)), "int32"),
    (ops.kv4_attention, _attn_args, dict(block_table=_ints(3, 4)), "block_table"),
    (ops.kv4_attention, _attn_args, dict(block_table=_ints(2, 8)[:, ::2]), "block_table"),
    (ops.kv4_attention, _attn_args, dict(window=-1), "window"),
    (ops.kv4_attention, _attn_args, {}, "CUDA devices only"),
    (ops.kv4_write, _write_args, {}, "CUDA devices only"),
]


@pytest.mark.parametrize("entry,args,change,words", REFUSALS, ids=lambda x: getattr(x, "__name__", None))
def test_refusals(entry, args, change, words):
    with pytest.raises(ops.KernelError, match=words):
        entry(**args(**change))


def test_read_refusals():
    pages = torch.zeros(5, 2, 16, 80, dtype=torch.uint8)
    with pytest.raises(ops.KernelError, match="int32"):
        ops.kv4_read(pages, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ops.KernelError, match="head sizes"):
        ops.kv4_read(torch.zeros(5, 2, 16, 64, dtype=torch.uint8), _ints(3))
    with pytest.raises(ops.KernelError, match="multiple of 16"):
        ops.kv4_read(torch.zeros(5, 2, 8, 80, dtype=torch.uint8), _ints(3))
    with pytest.raises(ops.KernelError, match="CUDA devices only"):
        ops.kv4_read(pages, _ints(3))


@pytest.mark.parametrize("change,words", [
    (dict(q_len=torch.zeros(2, dtype=torch.int64)), "int32"), (dict(context=_ints(3)), "int32"),
    (dict(pages=_ints(2, 2)), "one int32 list"), (dict(page_tokens=0), "at least 1"), (dict(stride=0), "at least 1"),
    (dict(rows=-1), "not negative"), (dict(q_len=_ints(0), context=_ints(0)), "requests"),
    (dict(q_len=_ints(8193), context=_ints(8193)), "requests"), (dict(rows=1 << 30, width=1 << 29), "int32 counts"),
    ({}, "CUDA devices only")])
def test_map_refusals(change, words):
    a = dict(q_len=_ints(2), context=_ints(2), pages=_ints(4), page_tokens=16, rows=2, width=2)
    a.update(change)
    with pytest.raises(ops.KernelError, match=words):
        ops.page_maps(**a)


def _model(cfg, bits=4, dtype=torch.bfloat16):
    from paged_batch_engine_b200.config import load_config
    from paged_batch_engine_b200.engine.runner import build_model
    return build_model(load_config(cfg)[1] if isinstance(cfg, dict) else cfg, dtype, "cpu", cache_bits=bits)


def test_a_model_with_a_4_bit_cache():
    from paged_batch_engine_b200.cache.storage import CacheStorage
    from tests.helpers import TINY_D
    model = _model(TINY_D)
    assert ("kv4_attention", None) in model.kernel_libraries() and not any(b.mixer.work_keys() for b in model.blocks)
    assert model.shaped_by_keys() and model.decode_capturable()
    st = CacheStorage(model.cache_needs, 16, 8, 4, torch.bfloat16, "cpu", poison=True)
    pages = st.layer(0).tensors["kv4"]
    assert pages.dtype == torch.uint8 and tuple(pages.shape) == (8, 1, 16, 80) and bool((pages == 0xff).all())
    assert st.layer(0).k is None and len(st.groups) == 2          # a layer with a window has a pool of its own
    plain_model = _model(TINY_D, bits=None)
    wide = CacheStorage(plain_model.cache_needs, 16, 8, 4, torch.bfloat16, "cpu")
    assert wide.bytes_per_token() * 10 == st.bytes_per_token() * 32
    assert not plain_model.shaped_by_keys()


def test_models_that_keep_no_4_bit_cache():
    from paged_batch_engine_b200.config.specs import ConfigError
    from paged_batch_engine_b200.engine.runner import ModelRunner
    from tests import helpers
    with pytest.raises(ConfigError, match="head sizes"):
        _model(helpers.TINY_C)
    with pytest.raises(ConfigError, match="8 bits"):
        _model(helpers.TINY_D, bits=8)
    with pytest.raises(ConfigError, match="keeps no cache in 4 bits"):
        _model(helpers.GUS_A)
    with pytest.raises(ValueError, match="multiple of 16"):
        ModelRunner(_model(helpers.TINY_D), page_tokens=8, num_pages=4)


def test_shapes_of_the_direct_kernel():
    """Blocks of clusters are whole clusters, at most what the GPU holds; what clusters do not take is shared out evenly."""
    for requests in (1, 2, 7, 64, 500):
        for kv, group in ((1, 1), (2, 6), (4, 7), (8, 5)):
            for rows in (1, 3, 9):
                for keys in (0, 1, 16, 17, 200, 777, 4096, 8192, 100000):
                    for d, wide in ((64, True), (128, True), (128, False)):
                        tile, blocks, cluster = ops._kv4_shape(requests, kv * group, kv, d, rows, keys, wide, 148)
                        assert tile in (8, 16) and 1 <= blocks <= 592 and cluster in (0, 1, 2, 4, 8, 16)
                        if cluster:
                            assert blocks == cluster * requests * kv * -(-rows * group // tile)
                            assert -(-keys // 16) <= cluster * ops.KV4_CLUSTER_UNITS
