"""The operators of a bounded cache at their limits, on the host."""
import pytest
import torch

from kinetics_b200 import EvictingKVManager, ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv_heads, heads", [(8, 32), (4, 32), (2, 4), (1, 8)])
@pytest.mark.parametrize("keep", [1024, 2048, 4096])
def test_a_managers_workspace_serves_every_number_of_active_slots(keep, kv_heads, heads, dtype):
    class Cfg:
        hidden_size, num_attention_heads, num_key_value_heads, head_dim, num_hidden_layers = 128 * heads, heads, kv_heads, 128, 1

    need = None
    for slots in (1, 8, 16, 24, 32, 64):
        kv = EvictingKVManager(Cfg, slots, 8192, "meta", dtype, keep=keep)
        need = need or [ops.decode_mass_workspace_bytes(n, kv_heads, heads // kv_heads, kv.pages_per_slot, dtype) for n in range(1, 65)]
        assert kv._decode_workspace().nbytes == max(need[:slots])


def test_a_size_for_fewer_sequences():
    size = lambda n, **kw: ops.decode_mass_workspace_bytes(n, 8, 4, 192, torch.bfloat16, **kw)
    assert size(16) == 0 < size(10)                                     # a cluster each; balanced
    assert size(16, fewer=True) == size(10) == size(10, fewer=True) and size(9, fewer=True) == 0
    assert size(0) == size(0, fewer=True) == 0
