"""What a product on 4-bit weights allocates beside its result."""

import pytest
import torch

import gpu_ragged_dot_amd as rd

pytestmark = pytest.mark.gpu


def _call_bytes(m, k, n, dtype, scale_dtype):
    """Bytes that a call had allocated at its peak, beside its operands and its result."""
    w = rd.pack_int4(torch.randint(0, 16, (1, k, n), dtype=torch.uint8, device="cuda"), torch.ones((1, k // 128, n), device="cuda").to(scale_dtype))
    x, gs = torch.randn(m, k, device="cuda").to(dtype), torch.tensor([m], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = rd.ragged_dot_int4(x, w, gs)
    result = -(-y.numel() * y.element_size() // 512) * 512  # the allocator's granularity
    return torch.cuda.max_memory_allocated() - before - result


def test_a_workspace_where_tiles_may_be_cut_and_none_where_there_are_none():
    size = (4096, 2048, 4096)
    assert _call_bytes(*size, torch.bfloat16, torch.bfloat16) >= 64 << 20
    assert _call_bytes(*size, torch.float16, torch.float16) >= 64 << 20
    assert _call_bytes(*size, torch.float16, torch.bfloat16) == 0  # the streaming kernel only
    assert _call_bytes(8, 2048, 4096, torch.bfloat16, torch.bfloat16) == 0
