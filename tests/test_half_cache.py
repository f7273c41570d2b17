"""fp16 queries over a quantised cache by way of unpacked rows: arguments and refusals of the C entry (CPU)."""

from __future__ import annotations

import contextlib

import pytest
import torch

import mxflashattn_b200 as fa
from mxflashattn_b200 import _lib, backend
from test_backend_marshalling import NAMES, STREAM, _Recorder
from test_varlen_cache import _args, _common, _guard_args

NAME = "mxfa_kvcache_varlen_attention_half_launch"


def test_the_entry_gets_the_cache_the_scratch_and_the_flags(monkeypatch):
    rec = _Recorder(_lib.load())
    monkeypatch.setattr(backend, "_LIB", [rec])
    monkeypatch.setattr(backend, "_on", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(backend, "_stream", lambda t: STREAM)
    monkeypatch.setattr(backend, "_chunk_sizes", lambda kv_heads, head_dim: (5000, 256))
    monkeypatch.setattr(backend, "unpack_pays", lambda *a: True)
    a = _args(quant=True, dtype=torch.float16)
    table = torch.zeros(4096, dtype=torch.int32)
    plan = fa.KvChunkPlan(6, 2, 4, 8, 2, True, table, None, torch.device("cpu"))
    backend.flash_attn_varlen_with_kvcache(a["q"], a["k_cache"], a["v_cache"], a["cu"], a["lens"], a["table"], 4, 48, 0.5,
                                           True, a["k_scales"], a["v_scales"], plan, None, True)
    name, c = rec.calls[-1]
    assert name == NAME and set(c) == set(NAMES[name])
    want = _common(a, plan=table.data_ptr(), plan_bytes=4096 * 4, q_token_stride=1024, q_head_stride=128,
                   workspace_bytes=5000, rows=128)
    del want["bf16"]
    assert {k: c[k] for k in want} == want
    assert c["v_rows"] - c["k_rows"] == 2 * 128 * 2 * 128 * 2
    assert len({c[n] for n in ("out", "lse", "workspace", "counters", "k_rows", "table_out", "inexact")} - {None}) == 7


def test_the_entry_refuses_before_any_device_work():
    lib = _lib.load()

    def call(**over):
        base = dict(k_scales=4096, v_scales=4096, k_rows=4096, v_rows=4096, table_out=4096, inexact=4096, rows=128)
        base.update(over)
        rest = {k: v for k, v in base.items() if k not in ("k_rows", "v_rows", "table_out", "inexact", "rows")}
        values = dict(zip([n for n in NAMES[NAME] if n not in ("k_rows", "v_rows", "table_out", "inexact", "rows")],
                          _guard_values(rest)))
        return getattr(lib, NAME)(*[base[n] if n in base else values[n] for n in NAMES[NAME]])

    def _guard_values(rest):
        known = dict(zip(NAMES["mxfa_kvcache_varlen_attention_launch"],
                         _guard_args("mxfa_kvcache_varlen_attention_launch", **rest)))
        return [known[n] for n in NAMES[NAME] if n not in ("k_rows", "v_rows", "table_out", "inexact", "rows")]

    for over in (dict(inexact=None), dict(rows=0), dict(k_scales=None, v_scales=None), dict(k_rows=None),
                 dict(v_rows=4104), dict(table_out=None), dict(q=4104), dict(HQ=7), dict(BTW=0), dict(seqlens=None)):
        assert call(**over) == _lib.MXFA_ERR_INVALID, over
    for over in (dict(D=96), dict(PS=12), dict(HQ=258), dict(B=70000)):
        assert call(**over) == _lib.MXFA_ERR_UNSUPPORTED, over
    assert call(total_q=0, q=None) == _lib.MXFA_OK
    assert lib.mxfa_unpack_flag_bytes(3, 130) == 3 * 9 * 4 and lib.mxfa_unpack_flag_bytes(0, 130) == 0
