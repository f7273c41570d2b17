"""Offsets that a decode step cannot take raise the error flag (their rows stay unwritten)."""

from __future__ import annotations

import pytest

from helpers import host
from varlen_oracle import make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("cu", [[0, 2, 3], [1, 0, 2], [0, 1, 9], [-1, 0, 1]])
def test_bad_offsets_of_a_decode_step_are_flagged(quant, cu, cuda_device):
    """More rows than max_seqlen_q, decreasing, past the packed rows, negative."""
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    b = make_batch(1800, [1, 2], [40, 30], quant=quant)
    t = b.device(cuda_device)
    _lib.read_error_flags()
    out = torch.full_like(t["q"], 7.0)
    fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], torch.tensor(cu, device=cuda_device), t["lens"],
                                      t["table"], 1, causal=True, k_scales=t["ks"], v_scales=t["vs"], out=out)
    torch.cuda.synchronize()
    assert _lib.read_error_flags() == _lib.FLAG_BAD_ORDER
    ok = [i for i in range(2) if cu[i + 1] - cu[i] == 1 and 0 <= cu[i] and cu[i + 1] <= 3]
    rows = [cu[i] for i in ok]
    assert (host(out)[[r for r in range(3) if r not in rows]] == 7.0).all()
    assert not (host(out)[rows] == 7.0).any()


@pytest.mark.parametrize("quant", [True, False])
def test_idle_sequences_and_padding_rows_raise_nothing(quant, cuda_device):
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    b = make_batch(1810, [1, 0, 1], [40, 30, 700], quant=quant)
    t = b.device(cuda_device)
    _lib.read_error_flags()
    fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 1, causal=True,
                                      k_scales=t["ks"], v_scales=t["vs"])
    torch.cuda.synchronize()
    assert _lib.read_error_flags() == 0


@pytest.mark.parametrize("cu", [[0, 60, 50, 64], [0, 4, 30, 65], [-1, 4, 30, 64]])
def test_a_plan_of_bad_offsets_is_empty_and_flagged(cu, cuda_device):
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    _lib.read_error_flags()
    lens = torch.full((3,), 100, dtype=torch.int32, device=cuda_device)
    plan = fa.kvcache_chunk_plan(torch.tensor(cu, device=cuda_device), lens, 64, 60, q_heads=8, kv_heads=2, causal=True)
    assert int(plan.table[0]) == 0
    assert _lib.read_error_flags() == _lib.FLAG_BAD_ORDER
    fa.kvcache_chunk_plan(torch.tensor([3, 4, 30, 60], device=cuda_device), lens, 64, 60, q_heads=8, kv_heads=2, causal=True)
    torch.cuda.synchronize()
    assert _lib.read_error_flags() == 0  # rows before the first offset and past the last are padding
