"""GPU parity of the ragged paged-cache operators (append, read-back, attention) against 64-bit definitions."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import host
from mxflashattn_b200 import synthetic as syn
from varlen_oracle import assert_attention, make_batch, quantise64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _flags_stay_clear(cuda_device):
    import torch

    from mxflashattn_b200 import _lib

    _lib.read_error_flags()
    yield
    torch.cuda.synchronize()
    assert _lib.read_error_flags() == 0


# ------------------------------------------------------------------------------------------------- append, read-back

def _append_inputs(seed, T, hkv, d, dtype, layout, dev):
    import torch

    rng = np.random.default_rng(seed)
    k = rng.standard_normal((T, hkv, d), dtype=np.float32) * np.exp(rng.standard_normal((T, hkv, 1))).astype(np.float32)
    v = rng.standard_normal((T, hkv, d), dtype=np.float32)
    if T > 2:
        k[1, 0] = 0.0                       # an all-zero row
        k[2, 0] *= 1e-30 if dtype == "bf16" else 1e-7
        v[1, 0, :] = 7.0                    # max / 448 is an exact power of two
        v[2, 0, 0] = 448.0
    k, v = syn.round_dtype(k, dtype), syn.round_dtype(v, dtype)
    tdt = syn.torch_dtype(dtype)
    kt, vt = torch.from_numpy(k).to(dev, tdt), torch.from_numpy(v).to(dev, tdt)
    if layout == "fused":    # slices of one projection
        qkv = torch.zeros((T, 3 + 2 * hkv, d), device=dev, dtype=tdt)
        qkv[:, 3:3 + hkv], qkv[:, 3 + hkv:] = kt, vt
        kt, vt = qkv[:, 3:3 + hkv], qkv[:, 3 + hkv:]
    elif layout == "odd":    # rows that start two bytes past a 16-byte boundary
        pad = torch.zeros((T, hkv, 2 * d + 3), device=dev, dtype=tdt)
        pad[:, :, 1:1 + d], pad[:, :, 2 + d:2 + 2 * d] = kt, vt
        kt, vt = pad[:, :, 1:1 + d], pad[:, :, 2 + d:2 + 2 * d]
    elif layout == "heads_first":
        kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (kt, vt))
    elif layout == "d_strided":
        kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kt, vt))
    return k, v, kt, vt


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("layout", ["packed", "fused", "odd", "heads_first", "d_strided"])
def test_append_writes_the_defined_codes_and_only_them(quant, dtype, d, layout, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    new, total, page, hkv = [1, 0, 37, 16, 5], [1, 9, 300, 16, 40], 16, 3
    b = make_batch(11, new, total, hkv=hkv, hq=hkv, d=d, page=page, dtype=dtype)
    T = int(b.cu[-1])
    k, v, kt, vt = _append_inputs(12, T, hkv, d, dtype, layout, cuda_device)
    pages = b.k.shape[0]
    tdt = syn.torch_dtype(dtype)
    store = torch.float8_e4m3fn if quant else tdt
    caches = [torch.full((pages, page, hkv, d), 1.5, device=cuda_device).to(store) for _ in range(2)]
    scales = [torch.full((pages, hkv, page), 3, device=cuda_device, dtype=torch.uint8).view(torch.float8_e8m0fnu)
              for _ in range(2)] if quant else [None, None]
    cu, lens, table = (torch.from_numpy(np.asarray(x)).to(cuda_device) for x in (b.cu, np.array(total), b.table))
    fa.kvcache_append_varlen(kt, vt, caches[0], caches[1], cu, lens, table, k_scales=scales[0], v_scales=scales[1])
    torch.cuda.synchronize()
    rows = np.concatenate([b.slots(i, t - n, t) for i, (n, t) in enumerate(zip(new, total))])
    for x, cache, scale in ((k, caches[0], scales[0]), (v, caches[1], scales[1])):
        want = np.full((pages * page, hkv, d), 1.5)
        if quant:
            codes, s = quantise64(x)
            want[rows] = codes
            want_s = np.full((pages * page, hkv), 2.0 ** (3 - 127))
            want_s[rows] = s
            got_s = scale.float().cpu().numpy().astype(np.float64).transpose(0, 2, 1).reshape(-1, hkv)
            assert np.array_equal(got_s, want_s)
        else:
            want[rows] = x
        assert np.array_equal(host(cache).reshape(-1, hkv, d).astype(np.float64), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_keeps_nan_saturates_infinity_and_their_row_stays_usable(dtype, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    x = syn.round_dtype(np.random.default_rng(3).standard_normal((4, 1, 128), dtype=np.float32), dtype)
    x[0, 0, 5], x[1, 0, 7], x[2, 0, 9], x[3, 0, :] = np.nan, np.inf, -np.inf, np.inf
    xt = torch.from_numpy(x).to(cuda_device, syn.torch_dtype(dtype))
    kc, vc = (torch.zeros((1, 16, 1, 128), device=cuda_device).to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros((1, 1, 16), device=cuda_device, dtype=torch.uint8).view(torch.float8_e8m0fnu)
              for _ in range(2))
    fa.kvcache_append_varlen(xt, xt, kc, vc, torch.tensor([0, 4], device=cuda_device),
                             torch.tensor([4], device=cuda_device),
                             torch.zeros((1, 1), device=cuda_device, dtype=torch.int32), k_scales=ks, v_scales=vs)
    codes, scale = quantise64(x)
    got = host(kc)[0, :4].astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(x.astype(np.float64)))
    assert np.array_equal(got[~np.isnan(got)], codes[~np.isnan(codes)])
    assert np.array_equal(ks.float().cpu().numpy()[0, :, :4].T.astype(np.float64), scale)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("dtype,d,page", [("bf16", 128, 16), ("fp16", 64, 8), ("bf16", 64, 5), ("fp16", 128, 24)])
def test_gather_returns_the_cached_values(quant, dtype, d, page, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    new, total = [0, 1, 100, 7, 33], [20, 1, 100, 64, 57]
    b = make_batch(21, new, total, d=d, page=page, dtype=dtype, quant=quant, poison=np.nan)
    t = b.device(cuda_device)
    T = int(b.cu[-1])
    k, v = fa.kvcache_gather_varlen(t["kc"], t["vc"], t["cu"], t["lens"], t["table"], T + 3, k_scales=t["ks"],
                                    v_scales=t["vs"], dtype=syn.torch_dtype(dtype))
    rows = np.concatenate([b.slots(i, x - n, x) for i, (n, x) in enumerate(zip(new, total))])
    for got, want in ((k, b.k), (v, b.v)):
        want = want.reshape(-1, b.hkv, d)[rows]
        want = want.astype(np.float16).astype(np.float64) if dtype == "fp16" else want  # e4m3 * 2^k is exact in bf16
        assert np.array_equal(host(got)[:T].astype(np.float64), want)
        assert not host(got)[T:].any()


def test_append_then_gather_returns_the_quantised_values(cuda_device):
    import torch

    import mxflashattn_b200 as fa

    new, total = [5, 129, 1], [5, 200, 33]
    b = make_batch(31, new, total, quant=True)
    t = b.device(cuda_device)
    T = int(b.cu[-1])
    rng = np.random.default_rng(5)
    x = syn.round_dtype(rng.standard_normal((2, T, b.hkv, b.d), dtype=np.float32), "bf16")
    kt, vt = torch.from_numpy(x).to(cuda_device, torch.bfloat16)
    fa.kvcache_append_varlen(kt, vt, t["kc"], t["vc"], t["cu"], t["lens"], t["table"], k_scales=t["ks"],
                             v_scales=t["vs"])
    k, v = fa.kvcache_gather_varlen(t["kc"], t["vc"], t["cu"], t["lens"], t["table"], T, k_scales=t["ks"],
                                    v_scales=t["vs"])
    for got, src in ((k, x[0]), (v, x[1])):
        codes, scale = quantise64(src)
        assert np.array_equal(host(got).astype(np.float64), codes * scale[..., None])


# ------------------------------------------------------------------------------------------------------- attention

def _attend(b, dev, causal, scale=None, index_dtype=None, plan=False, **kw):
    import torch

    import mxflashattn_b200 as fa

    t = b.device(dev, index_dtype)
    scale = b.d ** -0.5 if scale is None else scale
    if plan:
        kw["plan"] = fa.kvcache_chunk_plan(t["cu"], t["lens"], t["q"].shape[0], max(b.new), q_heads=b.hq,
                                           kv_heads=b.hkv, causal=causal)
    out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], max(b.new),
                                                 max(b.total), softmax_scale=scale, causal=causal, k_scales=t["ks"],
                                                 v_scales=t["vs"], return_softmax_lse=True, **kw)
    torch.cuda.synchronize()
    return host(out), host(lse), scale


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (6, 2), (8, 2), (8, 1), (5, 1), (32, 2)])
def test_ragged_pieces_match_the_definition(quant, dtype, d, hq, hkv, cuda_device):
    b = make_batch(100 + hq + d, [1, 0, 37, 130, 3, 64], [1, 50, 37, 300, 257, 128], hq=hq, hkv=hkv, d=d, dtype=dtype,
                   quant=quant, poison=np.nan)
    out, lse, scale = _attend(b, cuda_device, True, plan=hq == 8)
    assert_attention(out, lse, b, scale, True, f"hq{hq} hkv{hkv} d{d} {dtype} quant{quant}")


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("page", [1, 5, 8, 16, 24, 48, 64, 128, 256])
def test_pages_that_end_inside_a_tile(quant, page, cuda_device):
    b = make_batch(200 + page, [3, 70, 1], [131, 70, 257], page=page, quant=quant, poison=np.nan)
    out, lse, scale = _attend(b, cuda_device, True)
    assert_attention(out, lse, b, scale, True, f"page{page}")


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,total", [([1], [1]), ([1], [0]), ([5], [3]), ([0, 2], [4, 0]), ([128], [128]), ([129], [129]),
                                       ([127], [255]), ([200, 5], [100, 2]), ([32], [1000]), ([33], [1024]),
                                       ([2], [4097]), ([1, 1, 1], [1, 5000, 128])])
def test_lengths_that_leave_rows_empty_and_edges_of_tiles(quant, causal, new, total, cuda_device):
    b = make_batch(300 + len(new) + total[0], new, total, quant=quant, poison=np.nan)
    out, lse, scale = _attend(b, cuda_device, causal)
    assert_attention(out, lse, b, scale, causal, f"new{new} total{total} causal{causal}")


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "fp16")])
def test_single_tokens_of_many_sequences(quant, d, dtype, cuda_device):
    rng = np.random.default_rng(7)
    total = [int(x) for x in rng.integers(1, 700, size=40)]
    b = make_batch(400, [1] * 40, total, d=d, dtype=dtype, quant=quant, poison=np.nan)
    for plan in (False, True):
        out, lse, scale = _attend(b, cuda_device, True, plan=plan)
        assert_attention(out, lse, b, scale, True, f"singles plan{plan}")


@pytest.mark.parametrize("quant", [True, False])
def test_prompt_piece_mixed_with_decodes(quant, cuda_device):
    new = [200] + [1] * 9 + [0] + [17]
    total = [900, 1, 2, 127, 128, 129, 500, 16, 17, 1300, 40, 17]
    b = make_batch(500, new, total, hq=16, hkv=4, quant=quant, poison=np.nan)
    for plan in (False, True):
        out, lse, scale = _attend(b, cuda_device, True, plan=plan)
        assert_attention(out, lse, b, scale, True, f"mixed plan{plan}")


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("scale", [0.0, -0.05, 1.5])
def test_scales_zero_negative_and_sharp(quant, scale, cuda_device):
    b = make_batch(600, [40, 3], [300, 260], quant=quant, spread=0.1)
    out, lse, _ = _attend(b, cuda_device, True, scale=scale)
    assert_attention(out, lse, b, scale, True, f"scale {scale}")


@pytest.mark.parametrize("quant", [True, False])
def test_rescales_when_late_keys_tower_over_early_ones(quant, cuda_device):
    b = make_batch(610, [40, 1], [700, 900], spread=0.0)
    flat = b.k.reshape(-1, b.hkv, b.d)
    for s, t in enumerate(b.total):
        for lo in range(0, t, 130):
            flat[b.slots(s, lo, min(lo + 3, t))] *= 1.0 + lo / 40.0
    b.k = syn.round_dtype(b.k.astype(np.float32), "bf16").astype(np.float64)
    if quant:
        b.quant = True
        b.k_codes, b.k_scale = quantise64(b.k)
        b.v_codes, b.v_scale = quantise64(b.v)
        b.k, b.v = b.k_codes * b.k_scale[..., None], b.v_codes * b.v_scale[..., None]
    out, lse, scale = _attend(b, cuda_device, True)
    assert_attention(out, lse, b, scale, True, "late large keys")


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_later_tokens_bad_values_reach_no_earlier_query(quant, value, cuda_device):
    """A non-finite K or V row of token j is seen by queries at positions >= j only."""
    if quant and not np.isnan(value):
        pytest.skip("e4m3 codes have no infinity")
    b = make_batch(700, [60, 5], [200, 5], quant=quant)
    for s, bad in ((0, 170), (1, 2)):
        slot = int(b.slots(s, bad, bad + 1)[0])
        for x in (b.v.reshape(-1, b.hkv, b.d),) + ((b.v_codes.reshape(-1, b.hkv, b.d),) if quant else ()):
            x[slot, :, 3] = value
        for x in (b.k.reshape(-1, b.hkv, b.d),) + ((b.k_codes.reshape(-1, b.hkv, b.d),) if quant else ()):
            x[slot, :, 3] = np.nan
    out, lse, scale = _attend(b, cuda_device, True)
    clean = [i for s, (n, t, bad) in enumerate(zip(b.new, b.total, (170, 2)))
             for i in range(int(b.cu[s]), int(b.cu[s]) + n) if t - n + i - int(b.cu[s]) < bad]
    dirty = sorted(set(range(int(b.cu[-1]))) - set(clean))
    good = make_batch(700, [60, 5], [200, 5], quant=quant)
    from varlen_oracle import attention64

    want, want_lse, _, _ = attention64(good, scale, True)
    assert np.isfinite(out[clean]).all() and np.isfinite(lse[clean]).all()
    assert np.abs(out[clean] - want[clean]).max() < 3e-2 and np.abs(lse[clean] - want_lse[clean]).max() < 1e-3
    assert np.isnan(out[dirty]).all() and np.isnan(lse[dirty]).all()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_bad_value_in_v_reaches_its_column_of_the_queries_that_see_it(value, cuda_device):
    b = make_batch(710, [60, 5], [200, 5])
    for s, bad in ((0, 170), (1, 2)):
        b.v.reshape(-1, b.hkv, b.d)[int(b.slots(s, bad, bad + 1)[0]), :, 3] = value
    out, lse, scale = _attend(b, cuda_device, True)
    assert np.isfinite(lse).all()
    for s, (n, t, bad) in enumerate(zip(b.new, b.total, (170, 2))):
        for i in range(n):
            row = out[int(b.cu[s]) + i]
            assert np.isfinite(np.delete(row, 3, axis=1)).all()
            seen = t - n + i >= bad
            got = row[:, 3]
            assert np.isfinite(got).all() if not seen else np.isnan(got).all() if np.isnan(value) else (got == value).all()


@pytest.mark.parametrize("quant", [True, False])
def test_padding_rows_strided_queries_int64_indices_and_out(quant, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    b = make_batch(800, [9, 40], [100, 41], quant=quant)
    t = b.device(cuda_device, torch.int64)
    T = int(b.cu[-1])
    fused = torch.zeros((T + 5, b.hq + 4, b.d), device=cuda_device, dtype=torch.bfloat16)
    fused[:T, 2:2 + b.hq] = t["q"]
    q = fused[:, 2:2 + b.hq]
    out = torch.full((T + 5, b.hq, b.d), 9.0, device=cuda_device, dtype=torch.bfloat16)
    scale = b.d ** -0.5
    got, lse = fa.flash_attn_varlen_with_kvcache(q, t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 40, causal=True,
                                                 k_scales=t["ks"], v_scales=t["vs"], out=out, return_softmax_lse=True)
    assert got is out
    assert (host(out)[T:] == 9.0).all()
    assert_attention(host(out)[:T], host(lse)[:T], b, scale, True, "strided")
    odd = torch.zeros((T, b.hq, b.d + 1), device=cuda_device, dtype=torch.bfloat16)[:, :, 1:]
    odd.copy_(t["q"])
    again = fa.flash_attn_varlen_with_kvcache(odd, t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 40, causal=True,
                                              k_scales=t["ks"], v_scales=t["vs"])
    assert torch.equal(again, out[:T])


def test_results_do_not_change_from_call_to_call_nor_on_another_stream(cuda_device):
    import torch

    import mxflashattn_b200 as fa

    b = make_batch(900, [1, 64, 1, 2], [3000, 700, 129, 2500], quant=True)
    t = b.device(cuda_device)
    args = (t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 64)
    kw = dict(causal=True, k_scales=t["ks"], v_scales=t["vs"])
    first = fa.flash_attn_varlen_with_kvcache(*args, **kw)
    for _ in range(3):
        assert torch.equal(fa.flash_attn_varlen_with_kvcache(*args, **kw), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = fa.flash_attn_varlen_with_kvcache(*args, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)


def test_replay_in_a_cuda_graph_follows_the_lengths(cuda_device):
    import torch

    import mxflashattn_b200 as fa

    b = make_batch(910, [1, 1, 1], [200, 33, 150], quant=True)
    t = b.device(cuda_device)
    run = lambda: fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 1,  # noqa: E731
                                                    causal=True, k_scales=t["ks"], v_scales=t["vs"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    t["lens"].copy_(torch.tensor([100, 5, 150], dtype=torch.int32))
    graph.replay()
    b.total = [100, 5, 150]
    assert_attention(host(out), None, b, b.d ** -0.5, True, "replay")


def test_bad_pages_and_short_tables_are_flagged_not_read(cuda_device):
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    b = make_batch(920, [4], [200], quant=True)
    t = b.device(cuda_device)
    kw = dict(k_scales=t["ks"], v_scales=t["vs"])
    bad = t["table"].clone()
    bad[0, 3] = 10_000
    for table, lens, flag in ((bad, t["lens"], _lib.FLAG_PAGE_OUT_OF_RANGE),
                              (t["table"][:, :5].contiguous(), t["lens"], _lib.FLAG_TABLE_TOO_NARROW)):
        fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], lens, table, 4, causal=True, **kw)
        torch.cuda.synchronize()
        assert _lib.read_error_flags() & flag
    x = torch.zeros((4, b.hkv, b.d), device=cuda_device, dtype=torch.bfloat16)
    before = t["kc"].view(torch.uint8).clone()
    fa.kvcache_append_varlen(x, x, t["kc"], t["vc"], t["cu"], torch.tensor([2], device=cuda_device), t["table"], **kw)
    torch.cuda.synchronize()
    assert _lib.read_error_flags() & _lib.FLAG_TABLE_TOO_NARROW
    changed = (t["kc"].view(torch.uint8) != before).any(dim=-1).any(dim=-1).sum().item()
    assert changed <= 2


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("max_k", [None, 100])
def test_decode_step_with_idle_sequences_padding_rows_and_an_understated_length(quant, max_k, cuda_device):
    import torch

    import mxflashattn_b200 as fa

    new, total = [1, 0, 1, 1, 0, 1], [3000, 50, 1, 777, 0, 16]
    b = make_batch(930, new, total, hq=8, hkv=2, quant=quant, poison=np.nan)
    t = b.device(cuda_device)
    q = torch.zeros((6, b.hq, b.d), device=cuda_device, dtype=torch.bfloat16)
    q[:4] = t["q"]
    out = torch.full_like(q, 7.0)
    plan = fa.kvcache_chunk_plan(t["cu"], t["lens"], 6, 1, q_heads=8, kv_heads=2, causal=True)
    for p in (None, plan):
        _, lse = fa.flash_attn_varlen_with_kvcache(q, t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 1, max_k,
                                                   causal=True, k_scales=t["ks"], v_scales=t["vs"], plan=p, out=out,
                                                   return_softmax_lse=True)
        assert (host(out)[4:] == 7.0).all()
        assert_attention(host(out)[:4], host(lse)[:4], b, b.d ** -0.5, True, f"step max_k {max_k}")


@pytest.mark.parametrize("new,total", [([1, 1], [700, 300]), ([40, 3], [700, 300])])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("low,high", [(-30, 8), (-24, -20), (0, 0)])
def test_values_whose_scales_differ_widely(new, total, dtype, d, low, high, cuda_device):
    """V rows between 2^low and 2^high: the error stays relative to the attention over |V|, whatever the scales."""
    from varlen_oracle import attention64

    b = make_batch(940, new, total, hq=4, hkv=2, d=d, dtype=dtype, quant=True)
    rng = np.random.default_rng(1)
    lo = max(low, -14) if dtype == "fp16" else low
    size = np.exp2(rng.integers(lo, max(high, lo) + 1, size=b.v.shape[:3]).astype(np.float64))
    b.v_codes, b.v_scale = quantise64(syn.round_dtype((b.v * size[..., None]).astype(np.float32), dtype))
    b.v = b.v_codes * b.v_scale[..., None]
    out, lse, scale = _attend(b, cuda_device, True)
    want, want_lse, absv, reach = attention64(b, scale, True)
    storage = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -10}[dtype]
    tol = 1.01 * storage * np.abs(want) + (2.0 ** -10 + 4 * d * 2.0 ** -23 * reach[..., None]) * absv
    tol += 2.0 ** -24 if dtype == "fp16" else 0.0
    assert (np.abs(out - want) <= tol).all(), f"worst {np.max(np.abs(out - want) / np.maximum(tol, 1e-300)):.2f} of the bound"
    assert np.abs(lse - want_lse).max() <= 2e-5 + d * 2.0 ** -23 * reach.max()


@pytest.mark.parametrize("new,total", [([1, 1], [700, 300]), ([40, 3], [700, 300])])
def test_keys_and_queries_of_any_size(new, total, cuda_device):
    """K rows between 2^-40 and 2^20 with queries scaled to match, beyond f16's range on both sides."""
    from varlen_oracle import attention64

    b = make_batch(950, new, total, hq=4, hkv=2, quant=True)
    rng = np.random.default_rng(2)
    size = np.exp2(rng.integers(-40, 21, size=b.k.shape[:3]).astype(np.float64))
    b.k_codes, b.k_scale = quantise64(syn.round_dtype((b.k * size[..., None]).astype(np.float32), "bf16"))
    b.k = b.k_codes * b.k_scale[..., None]
    for q_size in (2.0 ** -20, 2.0 ** 20):
        b.q = syn.round_dtype(b.q * np.float32(q_size / np.abs(b.q).max()), "bf16")
        scale = 2.0 ** -20 / q_size
        out, lse, _ = _attend(b, cuda_device, True, scale=scale)
        want, want_lse, absv, reach = attention64(b, scale, True)
        tol = np.maximum(1e-2, 2.0 ** -8 * np.abs(want)) + (2.0 ** -10 + 4 * b.d * 2.0 ** -23 * reach[..., None]) * absv
        assert (np.abs(out - want) <= tol).all()
        assert np.abs(lse - want_lse).max() <= 2e-5 + b.d * 2.0 ** -23 * reach.max()


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("new", [1, 3])
def test_a_nan_in_a_visible_key_reaches_the_output(quant, new, cuda_device):
    """Whatever split of the keys holds it, and also when no other key is visible."""
    total = [new, 20000, 3000, 40]
    b = make_batch(960, [new] * 4, total, hq=8, hkv=2, quant=quant)
    for s, at in ((0, 0), (1, 13000), (2, 2990)):
        slot = int(b.slots(s, at, at + 1)[0])
        for x in (b.k.reshape(-1, b.hkv, b.d),) + ((b.k_codes.reshape(-1, b.hkv, b.d),) if quant else ()):
            x[slot, :, 7] = np.nan
    out, lse, scale = _attend(b, cuda_device, True)
    dirty = 3 * new
    assert np.isnan(out[:dirty]).all() and np.isnan(lse[:dirty]).all()
    assert np.isfinite(out[dirty:]).all() and np.isfinite(lse[dirty:]).all()


@pytest.mark.parametrize("unpack", [True, False])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
def test_quantised_pieces_unpacked_or_converted_in_the_kernel(unpack, dtype, d, cuda_device, monkeypatch):
    """Both ways through a quantised cache, on the same batch, whatever the rule would choose."""
    from mxflashattn_b200 import backend

    monkeypatch.setattr(backend, "unpack_pays", lambda *a: unpack)
    b = make_batch(970, [130, 1, 40, 0], [700, 300, 40, 129], hq=8, hkv=2, d=d, dtype=dtype, quant=True, poison=np.nan)
    out, lse, scale = _attend(b, cuda_device, True)
    assert_attention(out, lse, b, scale, True, f"unpack {unpack}")


def test_the_unpacking_rule_takes_long_pieces_and_bounded_memory():
    from mxflashattn_b200.backend import unpack_pays

    assert unpack_pays(1024, 1, 4, 8, 128, 16384)            # 32 tiles of one sequence
    assert not unpack_pays(64, 1, 4, 8, 128, 16384)          # two tiles
    assert not unpack_pays(543, 32, 4, 8, 128, 4608)         # one piece among decodes
    assert not unpack_pays(1 << 17, 64, 4, 8, 128, 1 << 17)  # scratch of 34 GB


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("new,total,hq,hkv", [
    ([600] * 5, [600] * 5, 4, 4),                    # whole waves and a split remainder
    ([33] * 40, [200] * 40, 8, 2),                   # many tiles of a few keys
    ([5, 1, 1], [6000, 30, 700], 16, 1),             # one long sequence among short ones
    ([1] * 30 + [2], [3] * 30 + [9000], 2, 1),
])
def test_plans_that_split_tiles(quant, new, total, hq, hkv, cuda_device):
    b = make_batch(980 + len(new), new, total, hq=hq, hkv=hkv, d=64, dtype="fp16", quant=quant)
    out, lse, scale = _attend(b, cuda_device, True, plan=True)
    assert_attention(out, lse, b, scale, True, "split plan")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch,hq,hkv", [(1, 8, 2), (40, 32, 8), (1500, 4, 4), (3000, 16, 1)])
def test_a_plan_covers_every_tile_once(causal, batch, hq, hkv, cuda_device):
    """Items of each tile: the parts 0 .. nsplit-1 cover its key tiles without gap or overlap."""
    import torch

    import mxflashattn_b200 as fa

    rng = np.random.default_rng(batch)
    new = rng.integers(0, 3 if batch > 100 else 400, size=batch)
    new[0] += 1
    total = np.where(rng.random(batch) < 0.1, new // 2, new + rng.integers(0, 3000, size=batch))
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    plan = fa.kvcache_chunk_plan(torch.from_numpy(cu).to(cuda_device), torch.from_numpy(total).to(cuda_device),
                                 int(cu[-1]), int(new.max()), q_heads=hq, kv_heads=hkv, causal=causal)
    table = plan.table.cpu().numpy()
    items = table[16:16 + 12 * table[0]].reshape(-1, 12)
    tok = 128 // (hq // hkv)
    seen = {}
    for b, row0, ntok, pos0, length, kt0, kt1, nsplit, split, part0, group, _ in items.tolist():
        seen.setdefault((b, row0), []).append((split, kt0, kt1, nsplit, ntok, pos0, length, part0, group))
    want = [(b, int(cu[b]) + t, min(tok, int(new[b]) - t)) for b in range(batch) for t in range(0, int(new[b]), tok)]
    assert sorted(seen) == [(b, r) for b, r, _ in want]
    used = []
    for b, row0, ntok in want:
        parts = sorted(seen[(b, row0)])
        pos = int(total[b]) - int(new[b]) + row0 - int(cu[b])
        end = max(min(pos + ntok, int(total[b])), 0) if causal else int(total[b])
        tiles = max(1, -(-end // 128))
        assert [p[0] for p in parts] == list(range(parts[0][3])) and len(parts) == parts[0][3]
        edges = [0] + [p[2] for p in parts]
        assert [p[1] for p in parts] == edges[:-1] and edges[-1] == tiles
        assert all(p[4:7] == (ntok, pos, int(total[b])) for p in parts)
        if len(parts) > 1:
            assert len({p[7:] for p in parts}) == 1
            used += range(parts[0][7], parts[0][7] + len(parts))
    assert len(used) == len(set(used))


def test_query_offsets_that_decrease_make_an_empty_plan(cuda_device):
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    cu = torch.tensor([0, 60, 0, 60, 0, 60], dtype=torch.int32, device=cuda_device)
    lens = torch.full((5,), 100, dtype=torch.int32, device=cuda_device)
    plan = fa.kvcache_chunk_plan(cu, lens, 60, 60, q_heads=128, kv_heads=1, causal=True)
    assert int(plan.table[0]) == 0
    assert _lib.read_error_flags() == _lib.FLAG_BAD_ORDER


def test_a_plan_of_another_batch_of_the_same_counts_stays_in_bounds(cuda_device):
    """A stale plan gives wrong numbers, but nothing outside the tensors is touched and no tile is waited for."""
    import torch

    import mxflashattn_b200 as fa
    from mxflashattn_b200 import _lib

    b = make_batch(990, [60, 4], [300, 400], quant=True)
    t = b.device(cuda_device)
    stale = fa.kvcache_chunk_plan(torch.tensor([0, 4, 64], device=cuda_device), torch.tensor([9000, 70], device=cuda_device),
                                  64, 60, q_heads=b.hq, kv_heads=b.hkv, causal=True)
    kw = dict(causal=True, k_scales=t["ks"], v_scales=t["vs"])
    args = (t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 60)
    good = fa.flash_attn_varlen_with_kvcache(*args, **kw)
    fa.flash_attn_varlen_with_kvcache(*args, plan=stale, **kw)
    torch.cuda.synchronize()
    assert _lib.read_error_flags() & ~(_lib.FLAG_TABLE_TOO_NARROW | _lib.FLAG_PAGE_OUT_OF_RANGE) == 0
    assert torch.equal(fa.flash_attn_varlen_with_kvcache(*args, **kw), good)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("new", [1, 20])
def test_offsets_past_32_bits(quant, new, cuda_device):
    """A cache of more than 2^31 elements, the sequence in its last pages."""
    import torch

    import mxflashattn_b200 as fa

    b = make_batch(1000, [new], [150], hq=8, hkv=8, quant=quant, spare_pages=0)
    t = b.device(cuda_device)
    pages = (1 << 31) // (16 * 8 * 128) + 40
    shift = pages - b.k.shape[0]
    big = {}
    for n in ("kc", "vc", "ks", "vs"):
        if t[n] is not None:
            x = torch.zeros((pages,) + t[n].shape[1:], device=cuda_device, dtype=torch.uint8 if quant else t[n].dtype)
            x[shift:] = t[n].view(torch.uint8) if quant else t[n]
            big[n] = x.view(t[n].dtype)
    table = torch.where(t["table"] >= 0, t["table"] + shift, t["table"])
    kw = dict(k_scales=big.get("ks"), v_scales=big.get("vs"))
    out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], big["kc"], big["vc"], t["cu"], t["lens"], table, new, 150,
                                                 causal=True, return_softmax_lse=True, **kw)
    assert_attention(host(out), host(lse), b, b.d ** -0.5, True, "large cache")
    x = torch.randn((new, 8, 128), device=cuda_device, dtype=torch.bfloat16)
    fa.kvcache_append_varlen(x, 2 * x, big["kc"], big["vc"], t["cu"], t["lens"], table, **kw)
    k, v = fa.kvcache_gather_varlen(big["kc"], big["vc"], t["cu"], t["lens"], table, new, **kw)
    for got, src in ((k, x), (v, 2 * x)):
        codes, scale = quantise64(host(src))
        assert np.array_equal(host(got).astype(np.float64), codes * scale[..., None] if quant else host(src))


def test_two_streams_at_once_keep_their_workspaces_apart(cuda_device):
    import torch

    import mxflashattn_b200 as fa

    b = make_batch(1010, [1, 3], [6000, 5000], hq=4, hkv=1, d=64, dtype="fp16", quant=True)
    t = b.device(cuda_device)
    run = lambda: fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"], 3,  # noqa: E731
                                                    causal=True, k_scales=t["ks"], v_scales=t["vs"])
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
