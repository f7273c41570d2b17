"""The unpacking rule leaves batches to the converting kernel that the unpacking launch does not take."""

from __future__ import annotations


def test_the_rule_knows_the_launch_limit():
    from mxflashattn_b200 import _lib
    from mxflashattn_b200.backend import unpack_pays
    from test_varlen_cache import _guard_args

    assert not unpack_pays(70000 * 4, 70000, 128, 1, 64, 32)
    assert unpack_pays(60000 * 4, 60000, 128, 1, 64, 32)
    name = "mxfa_kvcache_unpack_launch"
    args = _guard_args(name, k_scales=4096, v_scales=4096, rows=128, table_out=4096, B=65536)
    assert getattr(_lib.load(), name)(*args) == _lib.MXFA_ERR_UNSUPPORTED
    assert not unpack_pays(65536 * 4, 65536, 128, 1, 64, 32)
