"""A batch without sequences: every packed row is one that no sequence owns."""

from __future__ import annotations

import pytest

from helpers import host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("width", [0, 3])
@pytest.mark.parametrize("tokens", [0, 37])
def test_a_batch_without_sequences(quant, width, tokens, cuda_device):
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    bf16 = torch.bfloat16
    store = torch.float8_e4m3fn if quant else bf16
    kc, vc = (torch.ones((4, 16, 2, 128), device=cuda_device).to(store) for _ in range(2))
    ks, vs = (torch.full((4, 2, 16), 127, device=cuda_device, dtype=torch.uint8).view(torch.float8_e8m0fnu)
              for _ in range(2)) if quant else (None, None)
    kw = dict(k_scales=ks, v_scales=vs)
    cu = torch.zeros((1,), device=cuda_device, dtype=torch.int32)
    lens = torch.zeros((0,), device=cuda_device, dtype=torch.int32)
    table = torch.zeros((0, width), device=cuda_device, dtype=torch.int32)
    _lib.read_error_flags()
    # what the allocator hands out next holds other numbers
    torch.full((4 * max(tokens, 1), 2, 128), 5.0, device=cuda_device, dtype=bf16)
    for got in fa.kvcache_gather_varlen(kc, vc, cu, lens, table, tokens, **kw):
        assert got.shape == (tokens, 2, 128) and not host(got).any()
    x = torch.ones((tokens, 2, 128), device=cuda_device, dtype=bf16)
    before = kc.view(torch.uint8).clone()
    fa.kvcache_append_varlen(2 * x, x, kc, vc, cu, lens, table, **kw)
    assert torch.equal(kc.view(torch.uint8), before)
    q = torch.ones((tokens, 8, 128), device=cuda_device, dtype=bf16)
    for max_q in (0, 1, 5):
        out = torch.full_like(q, 7.0)
        plan = fa.kvcache_chunk_plan(cu, lens, tokens, max_q, q_heads=8, kv_heads=2, causal=True)
        for p in (None, plan):
            fa.flash_attn_varlen_with_kvcache(q, kc, vc, cu, lens, table, max_q, causal=True, plan=p, out=out, **kw)
            assert (host(out) == 7.0).all()
    assert _lib.read_error_flags() == 0
