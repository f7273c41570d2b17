"""An e8m0 byte of 255 is NaN: a key's makes the rows that see it NaN, a value's their outputs only."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host
from varlen_oracle import attention64, make_batch

pytestmark = pytest.mark.gpu


def _nan_byte(t, b, name, places):
    """Byte 255 for head 0 of the given (sequence, position) tokens."""
    import torch

    scales = t[name].view(torch.uint8)
    for s, pos in places:
        slot = int(b.slots(s, pos, pos + 1)[0])
        scales[slot // b.page, 0, slot % b.page] = 255


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("which", ["ks", "vs"])
@pytest.mark.parametrize("new", [1, 3, 130])
def test_a_nan_scale_reaches_every_row_that_sees_it(new, which, sign, cuda_device):
    """Decode step, converted tiles and unpacked rows; the raw score of the key is positive or negative."""
    import torch

    import mxflashattn_b200 as fa

    b = make_batch(1600, [new] * 3, [new, 5000, 700], hq=8, hkv=2, quant=True)
    places = ((0, 0), (1, 3000), (2, 700 - new))
    group = b.hq // b.hkv
    for s, pos in places:  # every query of head 0 points along the key's codes, or against them
        slot = int(b.slots(s, pos, pos + 1)[0])
        b.q[int(b.cu[s]):int(b.cu[s + 1]), :group] = sign * b.k_codes.reshape(-1, b.hkv, b.d)[slot, 0] / 512.0
    t = b.device(cuda_device)
    _nan_byte(t, b, which, places)
    out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], new, 5000,
                                                 causal=True, k_scales=t["ks"], v_scales=t["vs"],
                                                 return_softmax_lse=True)
    out, lse = host(out), host(lse)
    want, want_lse, _, _ = attention64(b, b.d ** -0.5, True)
    assert np.isnan(out[:, :group]).all()
    assert np.isfinite(out[:, group:]).all() and np.abs(out[:, group:] - want[:, group:]).max() < 3e-2
    if which == "ks":
        assert np.isnan(lse[:, :group]).all()
        lse, want_lse = lse[:, group:], want_lse[:, group:]
    assert np.abs(lse - want_lse).max() < 1e-3  # (a value takes no part in the LSE)


@pytest.mark.parametrize("which", ["ks", "vs"])
def test_a_nan_scale_of_a_later_token_reaches_no_earlier_query(which, cuda_device):
    """Also in a decode step of several queries, which the C entry takes."""
    import torch

    from mxflashattn_b200 import _lib

    b = make_batch(1610, [2, 2], [40, 2], hq=8, hkv=2, quant=True)
    t = b.device(cuda_device)
    _nan_byte(t, b, which, ((0, 39), (1, 1)))
    out = torch.empty_like(t["q"])
    lse = torch.empty((4, b.hq), device=cuda_device, dtype=torch.float32)
    counters = torch.zeros((1024,), device=cuda_device, dtype=torch.int32)
    lib = _lib.load()
    rc = lib.mxfa_kvcache_step_attention_launch(
        t["q"].data_ptr(), t["kc"].data_ptr(), t["vc"].data_ptr(), t["ks"].data_ptr(), t["vs"].data_ptr(),
        t["cu"].data_ptr(), t["lens"].data_ptr(), t["table"].data_ptr(), None, out.data_ptr(), lse.data_ptr(), None, 0,
        counters.data_ptr(), 4, 2, 2, b.hq, b.hkv, b.d, b.page, t["table"].shape[1], t["kc"].shape[0], 1, 64, 1, 1,
        b.d ** -0.5, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.MXFA_OK
    out, lse = host(out), host(lse)
    want, want_lse, _, _ = attention64(b, b.d ** -0.5, True)
    group = b.hq // b.hkv
    for s in (0, 1):
        first, second = 2 * s, 2 * s + 1
        assert np.abs(out[first] - want[first]).max() < 3e-2 and np.abs(lse[first] - want_lse[first]).max() < 1e-3
        assert np.isnan(out[second, :group]).all()
        assert np.abs(out[second, group:] - want[second, group:]).max() < 3e-2
        assert np.isnan(lse[second, :group]).all() if which == "ks" else np.abs(lse - want_lse).max() < 1e-3
