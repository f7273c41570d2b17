"""V rows under 2^-60, the smallest that the row sum's exponents take: they count as what they are."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import HALF_ULP_REL, host
from varlen_oracle import attention64, make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 3, 130])
@pytest.mark.parametrize("low,high", [(-66, -60), (-64, -50), (-60, -58), (-66, 0)])
def test_values_under_the_smallest_exponent(low, high, new, cuda_device):
    """Scales 2^low .. 2^high times the usual ones: decode step, converted tiles, unpacked rows."""
    import mxflashattn_b200 as fa

    b = make_batch(2100, [new, new], [max(new, 300), 900], hq=4, hkv=2, quant=True)
    rng = np.random.default_rng(6)
    b.v_scale *= np.exp2(rng.integers(low, high + 1, size=b.v_scale.shape).astype(np.float64))
    b.v = b.v_codes * b.v_scale[..., None]
    t = b.device(cuda_device)
    out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], new, 900,
                                                 causal=True, k_scales=t["ks"], v_scales=t["vs"],
                                                 return_softmax_lse=True)
    want, want_lse, absv, reach = attention64(b, b.d ** -0.5, True)
    score = reach * b.d * 2.0 ** -23
    tol = 1.001 * HALF_ULP_REL["bf16"] * np.abs(want) + (1.01 * 2.0 ** -8 + 2 * score[..., None]) * absv
    # P's smallest step at exponent -60, for up to 900 keys
    tol = tol + 900 * 2.0 ** -25 * 448 * 2.0 ** -60
    err = np.abs(host(out).astype(np.float64) - want)
    assert (err <= tol).all(), f"{np.max(err / tol):.1f} times the bound"
    assert (np.abs(host(lse) - want_lse) <= 2e-5 + score + 2.0 ** -22 * np.abs(want_lse)).all()


def test_rows_at_the_smallest_scale_vanish(cuda_device):
    """Byte 1: values under 2^-117, alone in their tiles and among others."""
    import mxflashattn_b200 as fa

    for new in (1, 3, 130):
        for every in (1, 2):
            b = make_batch(2110, [new, new], [300, 900], hq=4, hkv=2, quant=True)
            b.v_scale[:, ::every] = 2.0 ** -126
            b.v = b.v_codes * b.v_scale[..., None]
            t = b.device(cuda_device)
            out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], new, 900,
                                                         causal=True, k_scales=t["ks"], v_scales=t["vs"],
                                                         return_softmax_lse=True)
            want, want_lse, absv, reach = attention64(b, b.d ** -0.5, True)
            tol = 1.001 * HALF_ULP_REL["bf16"] * np.abs(want) + (1.01 * 2.0 ** -8 + reach[..., None] * b.d * 2.0 ** -22) * absv
            assert (np.abs(host(out).astype(np.float64) - want) <= tol + 2.0 ** -75).all()
            assert np.abs(host(lse) - want_lse).max() < 1e-3
