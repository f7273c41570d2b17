"""Steps of more tiles than one grid dimension of 65,535."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", [True, False])
def test_more_than_65535_tiles(quant, cuda_device):
    """128 query heads on one KV head: a tile is one token."""
    import torch

    import mxflashattn_b200 as fa

    T, hq, d = 70000, 128, 64
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(3)
    x = torch.randn((2, 4, 16, 1, d), generator=gen, device=cuda_device, dtype=torch.float16)
    q = torch.randn((T, hq, d), generator=gen, device=cuda_device, dtype=torch.float16)
    kc, vc, kw, values = x[0], x[1], {}, x.float()
    if quant:
        kc, vc = (c.to(torch.float8_e4m3fn) for c in x)
        one = torch.full((4, 1, 16), 127, device=cuda_device, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        kw = dict(k_scales=one, v_scales=one)
        values = torch.stack([kc.float(), vc.float()])
    cu = torch.tensor([0, T], device=cuda_device, dtype=torch.int32)
    lens = torch.tensor([50], device=cuda_device, dtype=torch.int32)
    table = torch.tensor([[2, 0, 3, 1]], device=cuda_device, dtype=torch.int32)
    out, lse = fa.flash_attn_varlen_with_kvcache(q, kc, vc, cu, lens, table, T, 50, return_softmax_lse=True, **kw)
    k, v = (c[table[0].long()].reshape(64, d)[:50].double() for c in values)
    for lo in (0, 65500, T - 40):
        s = q[lo:lo + 40].double() @ k.T / d ** 0.5
        want = torch.softmax(s, dim=-1) @ v
        bound = 2.0 ** -11 * want.abs() + 2.0 ** -10 * (torch.softmax(s, dim=-1) @ v.abs()) + 1e-6
        assert (np.abs(host(out[lo:lo + 40]) - want.cpu().numpy()) <= bound.cpu().numpy()).all()
        assert np.abs(host(lse[lo:lo + 40]) - torch.logsumexp(s, dim=-1).cpu().numpy()).max() < 1e-3
