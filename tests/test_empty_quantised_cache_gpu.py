"""Long pieces whose sequences have nothing cached: every row is empty."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host
from varlen_oracle import make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("new", [1, 20, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_empty_caches_are_zero(quant, new, causal, cuda_device):
    import mxflashattn_b200 as fa

    b = make_batch(1900, [new, new], [0, 0], hq=8, hkv=2, quant=quant)
    t = b.device(cuda_device)
    for max_k in (0, None):
        out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], new, max_k,
                                                     causal=causal, k_scales=t["ks"], v_scales=t["vs"],
                                                     return_softmax_lse=True)
        assert not host(out).any() and np.isneginf(host(lse)).all()
