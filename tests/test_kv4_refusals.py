"""More of what the 4-bit cache's entry points refuse, and what they do not, without a GPU."""
import pytest
import torch

from paged_batch_engine_b200.csrc import ops
from tests.test_kv4 import _attn_args, _ints, _write_args


def test_no_heads():
    """Refused before a launch shape is worked out from them."""
    none = torch.zeros(5, 0, 16, 80, dtype=torch.uint8)
    with pytest.raises(ops.KernelError, match="at least one"):
        ops.kv4_read(none, _ints(3))
    wide = torch.zeros(3, 0, dtype=torch.bfloat16)
    for change in (dict(num_heads=0, num_kv_heads=0, qkv=wide, q_out=wide, bias=None, pages=none),
                   dict(num_heads=0, num_kv_heads=0, qkv=wide, q_out=wide, bias=None, pages=None),
                   dict(num_kv_heads=0, qkv=torch.zeros(3, 256, dtype=torch.bfloat16), bias=None, pages=none),
                   dict(num_heads=0, qkv=torch.zeros(3, 256, dtype=torch.bfloat16), q_out=wide, bias=None)):
        with pytest.raises(ops.KernelError, match="at least one"):
            ops.kv4_write(**_write_args(**change))
    with pytest.raises(ops.KernelError, match="multiple"):
        ops.kv4_attention(**_attn_args(num_heads=0, num_kv_heads=0, q=wide, out=wide, pages=none))


def test_queries_beyond_the_prompt_kernels_counting(monkeypatch):
    """The tcgen05 kernel counts rows of queries by eight numbers in 32 bits: calls with more go to the other kernel."""
    calls = []

    def library(name):
        return lambda *a: calls.append(name) or 0
    monkeypatch.setattr(ops, "_ready", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    monkeypatch.setattr(ops, "multiprocessors", lambda device: 148)
    monkeypatch.setattr(ops, "tc5_attention_error_buffer", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(ops, "_kv4_prompt_fn", lambda: library("prompt"))
    monkeypatch.setattr(ops, "_kv4_fns", lambda: ops.Kv4Fns(None, None, library("few")))
    for rows, there in ((1 << 20, ["prompt"]), (1 << 25, ["few"])):
        calls.clear()
        q = torch.empty(rows, 16 * 64, dtype=torch.bfloat16, device="meta")
        one = torch.zeros(1, dtype=torch.int32, device="meta")
        ops.kv4_attention(q, torch.empty(5, 2, 16, 80, dtype=torch.uint8, device="meta"), torch.empty_like(q), one, one, one,
                          torch.zeros(1, 4, dtype=torch.int32, device="meta"), 16, 2, 64, 0.1, None, 16, rows, rows)
        assert calls == there


FITS = [(64, 128, 128, False, True), (64, 128, 0, False, True), (64, 128, 64, True, True), (47, 128, 64, False, True),
        (48, 128, 64, False, False), (95, 64, 32, False, True), (96, 64, 32, False, False)]


@pytest.mark.parametrize("KV,D,rot,interleaved,fits", FITS)
def test_many_key_value_heads(KV, D, rot, interleaved, fits):
    """Only a rotation by halves of a part of the channels has a limit, which a model meets when it is built."""
    from paged_batch_engine_b200.config.specs import ConfigError, PartSpec
    from paged_batch_engine_b200.parts.attention import GQAttention
    qkv = torch.zeros(3, 3 * KV * D, dtype=torch.bfloat16)
    args = _write_args(qkv=qkv, bias=None, q_out=torch.zeros(3, KV * D, dtype=torch.bfloat16),
                       pages=torch.zeros(2, KV, 16, D * 5 // 4, dtype=torch.uint8), inv_freq=torch.zeros(rot // 2),
                       num_heads=KV, num_kv_heads=KV, head_dim=D, rotary_dim=rot)
    with pytest.raises(ops.KernelError, match="CUDA devices only" if fits else "shared memory"):
        ops.kv4_write(**args, interleaved=interleaved)
    position = PartSpec("rope", dict(theta=1e4, head_dim=D, rotary_dim=rot, pairing="interleaved" if interleaved else "half")) \
        if rot else None
    mixer = GQAttention(hidden_size=64, num_heads=KV, num_kv_heads=KV, head_dim=D, position=position, dtype=torch.bfloat16,
                        device="cpu")
    if fits:
        mixer.use_cache_bits(4)
        assert mixer.cache_bits == 4
    else:
        with pytest.raises(ConfigError, match="key/value heads"):
            mixer.use_cache_bits(4)
        assert mixer.cache_bits is None


def test_more_requests_than_a_call_takes():
    with pytest.raises(ops.KernelError, match="at most 8192 requests"):
        ops.kv4_attention(**_attn_args(q_start=_ints(8193), q_len=_ints(8193), seq_len=_ints(8193), block_table=_ints(8193, 4)))
