"""Refusals and argument slots of the ragged paged-cache operators (CPU, no device)."""

from __future__ import annotations

import contextlib

import pytest
import torch

import mxflashattn_b200 as fa
from mxflashattn_b200 import _lib, backend
from test_backend_marshalling import NAMES, STREAM, _Recorder

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _args(quant=False, T=6, B=2, HQ=8, HKV=2, D=128, pages=7, PS=16, dtype=torch.bfloat16):
    store = E4M3 if quant else dtype
    a = {"q": torch.zeros(T, HQ, D, dtype=dtype), "k": torch.zeros(T, HKV, D, dtype=dtype),
         "v": torch.zeros(T, HKV, D, dtype=dtype), "k_cache": torch.zeros(pages, PS, HKV, D, dtype=store),
         "v_cache": torch.zeros(pages, PS, HKV, D, dtype=store), "cu": torch.tensor([0, 2, 6], dtype=torch.int32),
         "lens": torch.tensor([2, 20], dtype=torch.int32), "table": torch.zeros(B, 3, dtype=torch.int32),
         "k_scales": None, "v_scales": None}
    if quant:
        a["k_scales"] = torch.zeros(pages, HKV, PS, dtype=torch.uint8).view(E8M0)
        a["v_scales"] = torch.zeros(pages, HKV, PS, dtype=torch.uint8).view(E8M0)
    return a


def _append(a, **kw):
    return fa.kvcache_append_varlen(a["k"], a["v"], a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"],
                                    k_scales=a["k_scales"], v_scales=a["v_scales"], **kw)


def _gather(a, total=6, **kw):
    return fa.kvcache_gather_varlen(a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"], total,
                                    k_scales=a["k_scales"], v_scales=a["v_scales"], **kw)


def _attend(a, max_q=4, **kw):
    return fa.flash_attn_varlen_with_kvcache(a["q"], a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"], max_q,
                                             k_scales=a["k_scales"], v_scales=a["v_scales"], **kw)


CACHE_FAULTS = [
    ("k_cache", lambda a: a["k_cache"][0], ValueError, "rank 4"),
    ("k_cache", lambda a: None, TypeError, "torch.Tensor"),
    ("v_cache", lambda a: a["v_cache"][:, :8], ValueError, "identical shapes"),
    ("v_cache", lambda a: a["v_cache"].float().to(torch.float16), ValueError, "same dtype"),
    ("k_cache", lambda a: a["k_cache"].transpose(0, 1).contiguous().transpose(0, 1), ValueError, "contiguous"),
    ("cu", lambda a: a["cu"][:2], ValueError, "one entry more"),
    ("cu", lambda a: a["cu"].float(), TypeError, "int32 or int64"),
    ("lens", lambda a: a["lens"][None], ValueError, "rank 1"),
    ("lens", lambda a: [2, 20], TypeError, "torch.Tensor"),
    ("table", lambda a: a["table"][:1], ValueError, "one row per sequence"),
    ("table", lambda a: a["table"][:, :0], ValueError, "at least one column"),
    ("table", lambda a: None, ValueError, "block_table is required"),
]


@pytest.mark.parametrize("call", [_append, _gather, _attend])
@pytest.mark.parametrize("name,fault,error,message", CACHE_FAULTS)
def test_shared_refusals(call, name, fault, error, message):
    a = _args()
    a[name] = fault(a)
    with pytest.raises(error, match=message):
        call(a)


@pytest.mark.parametrize("call", [_append, _gather, _attend])
def test_scales_go_with_quantised_caches_only(call):
    a = _args(quant=True)
    a["v_scales"] = None
    with pytest.raises(ValueError, match="either both"):
        call(a)
    a["k_scales"] = None
    with pytest.raises(ValueError, match="needs k_scales"):
        call(a)
    b = _args()
    b["k_scales"] = b["v_scales"] = _args(quant=True)["k_scales"]
    with pytest.raises(ValueError, match="float8_e4m3fn caches only"):
        call(b)
    c = _args(quant=True)
    c["k_scales"] = c["k_scales"].view(torch.uint8)
    with pytest.raises(TypeError, match="float8_e8m0fnu"):
        call(c)
    d = _args(quant=True)
    d["v_scales"] = d["v_scales"].view(torch.uint8).transpose(1, 2).contiguous().view(E8M0)
    with pytest.raises(ValueError, match="kv_heads, page_size"):
        call(d)
    e = _args(dtype=torch.float32)
    with pytest.raises(TypeError, match="float16, bfloat16 or float8_e4m3fn"):
        call(e)
    f = _args(D=96)
    with pytest.raises(ValueError, match="64 or 128"):
        call(f)


def test_append_refusals():
    a = _args()
    a["k"] = a["k"][:, :1]
    with pytest.raises(ValueError, match="matching the cache"):
        _append(a)
    a = _args()
    a["v"] = a["v"][:5]
    with pytest.raises(ValueError, match="identical shapes"):
        _append(a)
    a = _args()
    a["k"] = a["v"] = a["k"].half()
    with pytest.raises(ValueError, match="cache's dtype"):
        _append(a)
    a = _args(quant=True)
    a["k"] = a["v"] = a["k"].float()
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        _append(a)


def test_rows_that_are_already_codes_are_refused():
    a = _args(quant=True)
    a["k"] = a["v"] = a["k"].to(E4M3)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        _append(a)
    b = _args(quant=True)
    b["q"] = b["q"].to(E4M3)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        _attend(b)


def test_gather_refusals():
    with pytest.raises(ValueError, match="non-negative"):
        _gather(_args(), total=-1)
    with pytest.raises(ValueError, match="own dtype"):
        _gather(_args(), dtype=torch.float16)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        _gather(_args(quant=True), dtype=torch.float32)


def test_attention_refusals():
    a = _args()
    a["q"] = a["q"][None]
    with pytest.raises(ValueError, match="rank 3"):
        _attend(a)
    a = _args(HQ=7)
    with pytest.raises(ValueError, match="multiple of kv heads"):
        _attend(a)
    a = _args()
    a["q"] = a["q"].half()
    with pytest.raises(ValueError, match="cache's dtype"):
        _attend(a)
    a = _args(quant=True)
    a["q"] = a["q"].float()
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        _attend(a)
    a = _args()
    a["q"] = a["q"][:, :, :64]
    with pytest.raises(ValueError, match="same head dimension"):
        _attend(a)
    a = _args()
    with pytest.raises(ValueError, match="max_seqlen_q"):
        _attend(a, max_q=-1)
    with pytest.raises(ValueError, match="max_seqlen_k"):
        _attend(a, max_seqlen_k=-1)
    with pytest.raises(ValueError, match="softmax_scale"):
        _attend(a, softmax_scale=float("nan"))
    other = fa.KvChunkPlan(6, 2, 4, 16, 2, False, None)
    with pytest.raises(ValueError, match="another batch"):
        _attend(a, plan=other)
    with pytest.raises(ValueError, match="out must be"):
        _attend(a, out=torch.zeros(6, 8, 64, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="kvcache_chunk_plan"):
        _attend(a, plan=3)


def test_strict_validation_reads_the_lengths(monkeypatch):
    monkeypatch.setenv("MXFLASHATTN_STRICT_VALIDATION", "1")
    a = _args()
    a["lens"] = torch.tensor([2, 49], dtype=torch.int32)
    for call in (_append, _gather, _attend):
        with pytest.raises(ValueError, match="enough pages"):
            call(a)
    a["lens"] = torch.tensor([1, 20], dtype=torch.int32)
    for call in (_append, _gather):
        with pytest.raises(ValueError, match="own tokens"):
            call(a)
    a = _args()
    a["table"][1, 1] = 7
    with pytest.raises(ValueError, match="out-of-range page"):
        _attend(a)
    a = _args()
    a["cu"] = torch.tensor([0, 4, 2], dtype=torch.int32)
    with pytest.raises(ValueError, match="must start at zero"):
        _attend(a)


@pytest.mark.parametrize("call", [_append, _gather, _attend])
def test_tensors_on_the_cpu_are_refused_by_the_dispatcher(call):
    with pytest.raises(fa.BackendUnavailableError, match="accelerator_tensor"):
        call(_args())


# -------------------------------------------------------------------------------- argument slots of the C ABI

@pytest.fixture
def rec(monkeypatch):
    recorder = _Recorder(_lib.load())
    monkeypatch.setattr(backend, "_LIB", [recorder])
    monkeypatch.setattr(backend, "_on", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(backend, "_stream", lambda t: STREAM)
    return recorder


def test_append_and_gather_pass_each_argument_in_its_slot(rec):
    a = _args(quant=True)
    qkv = torch.zeros(6, 12, 128, dtype=torch.bfloat16)
    k, v = qkv[:, 8:10], qkv[:, 10:12]
    backend.kvcache_append_varlen(k, v, a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"], a["k_scales"],
                                  a["v_scales"])
    name, c = rec.calls[-1]
    assert name == "mxfa_kvcache_append_varlen_launch" and set(c) == set(NAMES[name])
    want = dict(k=k.data_ptr(), v=v.data_ptr(), k_cache=a["k_cache"].data_ptr(), v_cache=a["v_cache"].data_ptr(),
                k_scales=a["k_scales"].data_ptr(), v_scales=a["v_scales"].data_ptr(), cu_seqlens=a["cu"].data_ptr(),
                seqlens=a["lens"].data_ptr(), block_table=a["table"].data_ptr(), total=6, B=2, HKV=2, D=128, PS=16,
                BTW=3, num_pages=7, k_token_stride=1536, k_head_stride=128, v_token_stride=1536, v_head_stride=128,
                bf16=1, stream=STREAM)
    assert c == want
    ko, vo = torch.zeros(6, 2, 128, dtype=torch.float16), torch.zeros(6, 2, 128, dtype=torch.float16)
    backend.kvcache_gather_varlen(a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"], a["k_scales"],
                                  a["v_scales"], ko, vo)
    name, c = rec.calls[-1]
    want = {n: want[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales", "cu_seqlens", "seqlens", "block_table",
                                 "total", "B", "HKV", "D", "PS", "BTW", "num_pages", "stream")}
    assert name == "mxfa_kvcache_gather_varlen_launch"
    assert c == dict(want, k_out=ko.data_ptr(), v_out=vo.data_ptr(), bf16=0)


def _attend_call(rec, a, max_q, plan, **kw):
    backend.flash_attn_varlen_with_kvcache(a["q"], a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"], max_q, 48,
                                           0.5, True, a["k_scales"], a["v_scales"], plan, None, True, **kw)
    return rec.calls[-1]


def _common(a, **over):
    want = dict(q=a["q"].data_ptr(), k_cache=a["k_cache"].data_ptr(), v_cache=a["v_cache"].data_ptr(),
                k_scales=a["k_scales"].data_ptr(), v_scales=a["v_scales"].data_ptr(), cu_seqlens_q=a["cu"].data_ptr(),
                seqlens=a["lens"].data_ptr(), block_table=a["table"].data_ptr(), total_q=6, B=2, HQ=8, HKV=2, D=128,
                PS=16, BTW=3, num_pages=7, causal=1, bf16=1, scale=0.5, stream=STREAM)
    want.update(over)
    return want


def test_attention_passes_each_argument_in_its_slot(rec):
    a = _args(quant=True)
    table = torch.zeros(4096, dtype=torch.int32)
    plan = fa.KvChunkPlan(6, 2, 4, 8, 2, True, table, None, torch.device("cpu"))
    name, c = _attend_call(rec, a, 4, plan)
    assert name == "mxfa_kvcache_varlen_attention_launch" and set(c) == set(NAMES[name])
    want = _common(a, plan=table.data_ptr(), plan_bytes=4096 * 4, q_token_stride=1024, q_head_stride=128,
                   workspace_bytes=5000)
    assert {k: c[k] for k in want} == want
    assert len({c["out"], c["lse"], c["workspace"], c["counters"]} - {None}) == 4


def test_a_decode_step_passes_each_argument_in_its_slot(rec):
    a = _args(quant=True)
    order = torch.zeros(2, dtype=torch.int32)
    plan = fa.KvChunkPlan(6, 2, 1, 8, 2, True, None, order, torch.device("cpu"))
    name, c = _attend_call(rec, a, 1, plan)
    assert name == "mxfa_kvcache_step_attention_launch" and set(c) == set(NAMES[name])
    want = _common(a, length_order=order.data_ptr(), max_q=1, num_splits=1, chunk_len=48)
    assert {k: c[k] for k in want} == want


def test_unpacking_hands_the_attention_its_scratch_as_a_cache(rec, monkeypatch):
    monkeypatch.setattr(backend, "unpack_pays", lambda *a: True)
    a = _args(quant=True)
    plan = fa.KvChunkPlan(6, 2, 4, 8, 2, True, torch.zeros(4096, dtype=torch.int32), None, torch.device("cpu"))
    name, c = _attend_call(rec, a, 4, plan)
    unpack, u = rec.calls[-2]
    assert unpack == "mxfa_kvcache_unpack_launch" and set(u) == set(NAMES[unpack])
    want = {k: v for k, v in _common(a, rows=128).items() if k in NAMES[unpack]}
    assert {k: u[k] for k in want} == want
    assert c["k_scales"] is None and c["v_scales"] is None and c["PS"] == 128 and c["num_pages"] == 2 and c["BTW"] == 1
    assert (c["k_cache"], c["v_cache"], c["block_table"]) == (u["k_out"], u["v_out"], u["table_out"])
    assert u["v_out"] - u["k_out"] == 2 * 128 * 2 * 128 * 2


@pytest.fixture(autouse=True)
def _fixed_chunk_sizes(monkeypatch):
    monkeypatch.setattr(backend, "_chunk_sizes", lambda kv_heads, head_dim: (5000, 256))


# ------------------------------------------------------------------------------------------- host guards of the C ABI

@pytest.fixture(scope="module")
def lib():
    from mxflashattn_b200 import build

    build.build()
    return _lib.load()


def _guard_args(name, **over):
    base = dict(k=4096, v=4096, q=4096, k_cache=4096, v_cache=4096, k_scales=None, v_scales=None, cu_seqlens=4096,
                cu_seqlens_q=4096, seqlens=4096, block_table=4096, k_out=4096, v_out=4096, out=4096, lse=None, total=4,
                total_q=4, B=2, HQ=8, HKV=2, D=128, PS=16, BTW=4, num_pages=8, k_token_stride=256, k_head_stride=128,
                v_token_stride=256, v_head_stride=128, q_token_stride=1024, q_head_stride=128, causal=1, bf16=1,
                scale=0.1, stream=None, plan=4096, plan_bytes=1 << 20, workspace=4096,
                workspace_bytes=1 << 30, counters=4096, length_order=None, max_q=1, num_splits=1, chunk_len=64)
    base.update(over)
    return [base[n] for n in NAMES[name]]


ENTRIES = ("mxfa_kvcache_append_varlen_launch", "mxfa_kvcache_gather_varlen_launch",
           "mxfa_kvcache_varlen_attention_launch", "mxfa_kvcache_step_attention_launch")


@pytest.mark.parametrize("name", ENTRIES)
@pytest.mark.parametrize("over,status", [
    (dict(D=96), _lib.MXFA_ERR_UNSUPPORTED), (dict(HKV=0), _lib.MXFA_ERR_INVALID), (dict(PS=0), _lib.MXFA_ERR_INVALID),
    (dict(num_pages=0), _lib.MXFA_ERR_INVALID), (dict(BTW=0), _lib.MXFA_ERR_INVALID),
    (dict(total=-1, total_q=-1), _lib.MXFA_ERR_INVALID), (dict(k_cache=None), _lib.MXFA_ERR_INVALID),
    (dict(block_table=None), _lib.MXFA_ERR_INVALID), (dict(seqlens=None), _lib.MXFA_ERR_INVALID),
    (dict(k_scales=4096), _lib.MXFA_ERR_INVALID), (dict(v_cache=4100), _lib.MXFA_ERR_INVALID),
    (dict(BTW=2 ** 30), _lib.MXFA_ERR_UNSUPPORTED), (dict(total=0, total_q=0, k_cache=None), _lib.MXFA_OK),
])
def test_entries_refuse_before_any_device_work(lib, name, over, status):
    assert getattr(lib, name)(*_guard_args(name, **over)) == status


def test_attention_entry_refuses_bad_queries(lib):
    name = "mxfa_kvcache_varlen_attention_launch"
    for over in (dict(q=None), dict(out=None), dict(q=4104), dict(q_token_stride=1025), dict(HQ=7), dict(plan=None),
                 dict(plan_bytes=64), dict(workspace=None), dict(workspace_bytes=64), dict(counters=None)):
        assert getattr(lib, name)(*_guard_args(name, **over)) == _lib.MXFA_ERR_INVALID, over


def test_step_entry_refuses_what_the_decode_kernel_does_not_take(lib):
    name = "mxfa_kvcache_step_attention_launch"
    call = lambda **over: getattr(lib, name)(*_guard_args(name, **over))  # noqa: E731
    quant = dict(k_scales=4096, v_scales=4096)
    assert call(D=64, **quant) == _lib.MXFA_ERR_UNSUPPORTED
    assert call(PS=24, **quant) == _lib.MXFA_ERR_UNSUPPORTED
    assert call(k_scales=4104, v_scales=4096) == _lib.MXFA_ERR_INVALID
    for over in (dict(counters=None), dict(max_q=-1), dict(q=None), dict(HQ=7), dict(q=4104),
                 dict(num_splits=3, workspace=None)):
        assert call(**over) == _lib.MXFA_ERR_INVALID, over
    assert call(max_q=0, q=None) == _lib.MXFA_OK


def test_unpack_entry_refuses(lib):
    name = "mxfa_kvcache_unpack_launch"
    base = dict(k_scales=4096, v_scales=4096, rows=128, table_out=4096)
    call = lambda **over: getattr(lib, name)(*_guard_args(name, **{**base, **over}))  # noqa: E731
    assert call(D=96) == _lib.MXFA_ERR_UNSUPPORTED
    assert call(B=70000) == _lib.MXFA_ERR_UNSUPPORTED
    for over in (dict(k_scales=None, v_scales=None), dict(k_out=None), dict(table_out=None), dict(v_out=4104),
                 dict(seqlens=None), dict(rows=-1), dict(k_scales=4098, v_scales=4096)):
        assert call(**over) == _lib.MXFA_ERR_INVALID, over
    assert call(rows=0, k_out=None) == _lib.MXFA_OK


def test_plan_entry_refuses_and_sizes_are_host_only(lib):
    name = "mxfa_kvcache_chunk_plan_launch"
    assert getattr(lib, name)(*_guard_args(name, HQ=7)) == _lib.MXFA_ERR_INVALID
    assert getattr(lib, name)(*_guard_args(name, seqlens=None)) == _lib.MXFA_ERR_INVALID
    assert getattr(lib, name)(*_guard_args(name, plan_bytes=32)) == _lib.MXFA_ERR_INVALID
    assert getattr(lib, name)(*_guard_args(name, HQ=258)) == _lib.MXFA_ERR_UNSUPPORTED
    assert getattr(lib, name)(*_guard_args(name, total_q=0, plan=None)) == _lib.MXFA_OK
    small, large = lib.mxfa_chunk_plan_bytes(1, 1, 32, 8), lib.mxfa_chunk_plan_bytes(4096, 64, 32, 8)
    assert 0 < small < large and lib.mxfa_chunk_plan_bytes(0, 1, 32, 8) == 0
    assert lib.mxfa_chunk_workspace_bytes(8, 128) > lib.mxfa_chunk_workspace_bytes(8, 64) > 0
    assert lib.mxfa_chunk_counter_bytes(8) > 0


def test_plan_refuses_tensors_that_are_not_on_a_device():
    a = _args()
    with pytest.raises(ValueError, match="CUDA device"):
        fa.kvcache_chunk_plan(a["cu"], a["lens"], 6, 4, q_heads=8, kv_heads=2)
    with pytest.raises(TypeError, match="torch.Tensor"):
        fa.kvcache_chunk_plan(a["cu"], [1, 2], 6, 4, q_heads=8, kv_heads=2)
