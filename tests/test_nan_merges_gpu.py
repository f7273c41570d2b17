"""A NaN state of one rank reaches the merged output of a context-parallel group."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host
from mxflashattn_b200 import synthetic as syn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("bad", [0, 1, 2])
def test_a_rank_of_nan_makes_the_merged_row_nan(head_dim, bad, cuda_device):
    import torch

    from mxflashattn_b200 import backend

    rows = 5
    rec = torch.randn((3, rows, head_dim + 1), device=cuda_device)
    rec[:, 4, head_dim] = -float("inf")      # a row that no rank has keys for
    rec[1, 1, head_dim] = -float("inf")      # one rank without keys: whatever its O holds
    rec[1, 1, :head_dim] = float("nan")
    rec[bad, 2] = float("nan")               # scores of NaN
    rec[bad, 3, 7] = float("nan")            # one value of NaN
    out, lse = backend.lse_merge(rec, rows, head_dim, torch.bfloat16, lse=True)
    out, lse = host(out), host(lse)
    assert np.isnan(out[2]).all() and np.isnan(lse[2])
    assert np.isnan(out[3, 7]) and np.isfinite(np.delete(out[3], 7)).all() and np.isfinite(lse[3])
    assert np.isfinite(out[:2]).all() and np.isfinite(lse[:2]).all()
    assert not out[4].any() and np.isneginf(lse[4])


@pytest.mark.parametrize("splits", [1, 3])
def test_a_nan_key_reaches_the_packed_record(splits, cuda_device):
    import torch

    from mxflashattn_b200 import backend

    case = syn.paged_case(1950, batch=2, q_heads=8, kv_heads=2, head_dim=128, dtype="bf16", page_size=16,
                          lengths=[700, 300])
    q = torch.from_numpy(case.q).to(cuda_device, torch.bfloat16)
    kc = torch.from_numpy(case.k_cache).to(cuda_device, torch.bfloat16)
    vc = torch.from_numpy(case.v_cache).to(cuda_device, torch.bfloat16)
    table = torch.from_numpy(case.block_table).to(cuda_device)
    lens = torch.from_numpy(case.cache_seqlens).to(cuda_device)
    kc[int(case.block_table[0, 600 // 16]), 600 % 16, 0, 5] = float("nan")
    cap = 16 * case.block_table.shape[1]
    packed = backend.kvcache_attention_packed(q, kc, vc, lens, table, case.softmax_scale, num_splits=splits,
                                              chunk_len=-(-cap // splits // 16) * 16)
    rec = host(packed).reshape(2, 8, 129)
    assert np.isnan(rec[0, :4]).all()
    assert np.isfinite(rec[0, 4:]).all() and np.isfinite(rec[1]).all()


@pytest.mark.parametrize("one_launch", [True, False])
def test_a_nan_key_reaches_the_exchanged_output(one_launch, cuda_device):
    import datetime
    import socket

    import torch
    import torch.distributed as dist

    from mxflashattn_b200 import _lib
    from mxflashattn_b200 import context_split as cs

    _lib.read_error_flags()
    case = syn.paged_case(1960, batch=2, q_heads=8, kv_heads=2, head_dim=128, dtype="bf16", page_size=16,
                          lengths=[3000, 300])
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1,
                            timeout=datetime.timedelta(seconds=60))
    fused = None
    try:
        ll, table = cs.local_view(case.cache_seqlens, case.block_table, 1, 0, 16)
        q = torch.from_numpy(case.q).to(cuda_device, torch.bfloat16)
        kc = torch.from_numpy(case.k_cache).to(cuda_device, torch.bfloat16)
        vc = torch.from_numpy(case.v_cache).to(cuda_device, torch.bfloat16)
        kc[int(case.block_table[0, 2000 // 16]), 2000 % 16, 0, 5] = float("nan")
        sl, bt = torch.from_numpy(ll).to(cuda_device), torch.from_numpy(table).to(cuda_device)
        fused = cs.FusedContextParallelDecode(2, 8, 2, 128, device=cuda_device)
        fused.one_launch = one_launch
        for _ in range(2):  # both halves of the exchange buffer
            out, lse = fused(q, kc, vc, sl, bt, case.softmax_scale, return_lse=True)
            out, lse = host(out).reshape(2, 8, 128), host(lse).reshape(2, 8)
            assert np.isnan(out[0, :4]).all() and np.isnan(lse[0, :4]).all()
            assert np.isfinite(out[0, 4:]).all() and np.isfinite(out[1]).all()
            assert np.isfinite(lse[0, 4:]).all() and np.isfinite(lse[1]).all()
    finally:
        if fused is not None:
            fused.close()
        dist.destroy_process_group()
    assert _lib.read_error_flags() == 0
