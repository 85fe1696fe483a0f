"""What the 8-bit layer refuses, on any host."""
import pytest
import torch

from dsl_tool_amd import layer8 as L


def test_refusals():
    wq, wo, n = torch.zeros(512, 128), torch.zeros(128, 256), torch.ones(128)
    with pytest.raises(ValueError, match="multiple"):
        L.Int8AttentionLayer(wq, wo, n, q_heads=4, kv_heads=3, dim=64)
    with pytest.raises(ValueError, match="w_qkv"):
        L.Int8AttentionLayer(wq, wo, n, q_heads=4, kv_heads=1, dim=64)
    with pytest.raises(ValueError, match="GPU"):
        L.Int8AttentionLayer(wq, wo, n, q_heads=4, kv_heads=2, dim=64)
