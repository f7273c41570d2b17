"""A decode step of more sequences than the split-KV kernel's grid holds runs on the tiled kernel."""

from __future__ import annotations

import contextlib

import pytest


@pytest.mark.parametrize("batch,name", [(65535, "mxfa_kvcache_step_attention_launch"),
                                        (65536, "mxfa_kvcache_varlen_attention_launch")])
def test_the_step_kernel_gets_what_its_grid_holds(batch, name, monkeypatch):
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib, backend
    from test_backend_marshalling import STREAM, _Recorder

    rec = _Recorder(_lib.load())
    monkeypatch.setattr(backend, "_LIB", [rec])
    monkeypatch.setattr(backend, "_on", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(backend, "_stream", lambda t: STREAM)
    monkeypatch.setattr(backend, "_chunk_sizes", lambda kv_heads, head_dim: (5000, 256))
    q = torch.zeros(batch, 1, 64, dtype=torch.float16)
    cache = torch.zeros(3, 16, 1, 64, dtype=torch.float16)
    cu, lens = torch.arange(batch + 1, dtype=torch.int32), torch.ones(batch, dtype=torch.int32)
    table = torch.zeros(batch, 1, dtype=torch.int32)
    plan = fa.KvChunkPlan(batch, batch, 1, 1, 1, True, torch.zeros(64, dtype=torch.int32), None, torch.device("cpu"))
    backend.flash_attn_varlen_with_kvcache(q, cache, cache, cu, lens, table, 1, 16, 0.1, True, None, None, plan)
    assert rec.calls[-1][0] == name


@pytest.mark.gpu
def test_seventy_thousand_single_tokens(cuda_device):
    import torch

    import mxflashattn_b200 as fa

    batch = 70000
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(5)
    kc, vc = torch.randn((2, 40, 16, 1, 64), generator=gen, device=cuda_device, dtype=torch.float16)
    q = torch.randn((batch, 2, 64), generator=gen, device=cuda_device, dtype=torch.float16)
    lens = torch.randint(0, 17, (batch,), generator=gen, device=cuda_device, dtype=torch.int32)
    table = torch.randint(0, 40, (batch, 1), generator=gen, device=cuda_device, dtype=torch.int32)
    cu = torch.arange(batch + 1, device=cuda_device, dtype=torch.int32)
    out, lse = fa.flash_attn_varlen_with_kvcache(q, kc, vc, cu, lens, table, 1, 16, causal=True, return_softmax_lse=True)
    k, v = (c[table[:, 0].long()][:, :, 0].double() for c in (kc, vc))
    s = torch.einsum("bhd,bkd->bhk", q.double(), k) / 8.0
    s = s.masked_fill((torch.arange(16, device=cuda_device) >= lens[:, None])[:, None], -float("inf"))
    want_lse = torch.logsumexp(s, dim=-1)
    p = torch.exp(s - want_lse[..., None].clamp(min=-1e30))
    want, absv = torch.einsum("bhk,bkd->bhd", p, v), torch.einsum("bhk,bkd->bhd", p, v.abs())
    # the output's one rounding, P's, and 64 products of each score in 32 bits
    bound = 2.0 ** -11 * want.abs() + (1.01 * 2.0 ** -11 + 2.0 ** -14) * absv + 2.0 ** -24
    assert ((out.double() - want).abs() <= bound).all()
    empty = lens == 0
    assert not out[empty].any() and torch.isneginf(lse[empty]).all()
    assert (lse[~empty].double() - want_lse[~empty]).abs().max() < 1e-4
