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
