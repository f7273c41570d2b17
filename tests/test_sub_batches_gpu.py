"""Offsets that start past zero: rows before cu_seqlens[0] belong to no sequence, in every entry."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host
from mxflashattn_b200 import synthetic as syn
from varlen_oracle import assert_attention, make_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _flags_stay_clear(cuda_device):
    import torch

    from mxflashattn_b200 import _lib

    _lib.read_error_flags()
    yield
    torch.cuda.synchronize()
    assert _lib.read_error_flags() == 0


def _shifted(seed, first, new, total, dev, **kw):
    """A batch whose packed tensors hold ``first`` rows of other sequences before its own."""
    import torch

    b = make_batch(seed, new, total, **kw)
    t = b.device(dev)
    T = int(b.cu[-1])
    t["cu"] = t["cu"] + first
    q = torch.full((first + T, b.hq, b.d), 3.0, device=dev, dtype=t["q"].dtype)
    q[first:] = t["q"]
    t["q"] = q
    return b, t, T


@pytest.mark.parametrize("quant", [True, False])
def test_append_writes_no_row_before_the_first_offset(quant, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    first, new, total = 6, [3, 0, 20], [90, 5, 20]
    b, t, T = _shifted(1700, first, new, total, cuda_device, quant=quant)
    rng = np.random.default_rng(1)
    x = torch.from_numpy(syn.round_dtype(rng.standard_normal((2, first + T, b.hkv, b.d), dtype=np.float32), "bf16"))
    x = x.to(cuda_device, torch.bfloat16)
    before = {n: t[n].view(torch.uint8).clone() for n in ("kc", "vc", "ks", "vs") if t[n] is not None}
    fa.kvcache_append_varlen(x[0], x[1], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], k_scales=t["ks"],
                             v_scales=t["vs"])
    k, v = fa.kvcache_gather_varlen(t["kc"], t["vc"], t["cu"] - first, t["lens"], t["table"], T, k_scales=t["ks"],
                                    v_scales=t["vs"])
    if not quant:
        assert torch.equal(k, x[0, first:]) and torch.equal(v, x[1, first:])
    rows = np.concatenate([b.slots(i, n - m, n) for i, (m, n) in enumerate(zip(new, total))])
    own = np.zeros(b.k.shape[0] * b.page, bool)
    own[rows] = True
    for n in ("kc", "vc"):
        changed = (t[n].view(torch.uint8) != before[n]).flatten(2).any(dim=-1).flatten().cpu().numpy()
        assert not changed[~own].any()
    for n in ("ks", "vs") if quant else ():
        changed = (t[n].view(torch.uint8) != before[n]).any(dim=1).flatten().cpu().numpy()
        assert not changed[~own].any()


@pytest.mark.parametrize("quant", [True, False])
def test_gather_returns_zeros_before_the_first_offset(quant, cuda_device):
    import mxflashattn_b200 as fa

    first, new, total = 6, [3, 0, 20], [90, 5, 20]
    b, t, T = _shifted(1710, first, new, total, cuda_device, quant=quant)
    for got, want in zip(fa.kvcache_gather_varlen(t["kc"], t["vc"], t["cu"], t["lens"], t["table"], first + T + 2,
                                                  k_scales=t["ks"], v_scales=t["vs"]), (b.k, b.v)):
        rows = np.concatenate([b.slots(i, n - m, n) for i, (m, n) in enumerate(zip(new, total))])
        got = host(got).astype(np.float64)
        assert not got[:first].any() and not got[first + T:].any()
        assert np.array_equal(got[first:first + T], want.reshape(-1, b.hkv, b.d)[rows])


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("page,new,total", [(16, [3, 0, 20], [90, 5, 20]), (5, [3, 0, 20], [90, 5, 20]),
                                            (16, [1, 0, 1], [90, 5, 400])])
def test_attention_leaves_rows_before_the_first_offset_alone(quant, page, new, total, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    first = 6
    b, t, T = _shifted(1720, first, new, total, cuda_device, quant=quant, page=page)
    out = torch.full((first + T, b.hq, b.d), 7.0, device=cuda_device, dtype=torch.bfloat16)
    _, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], max(new),
                                               causal=True, k_scales=t["ks"], v_scales=t["vs"], out=out,
                                               return_softmax_lse=True)
    assert (host(out)[:first] == 7.0).all()
    assert_attention(host(out)[first:], host(lse)[first:], b, b.d ** -0.5, True, f"page {page}")
