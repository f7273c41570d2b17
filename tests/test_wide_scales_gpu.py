"""Row scales far apart within one tile: what a query does not see, or weighs with almost nothing, costs it no bits.

Bounds: half an ulp of the stored output, the rounding of P (2^-11 in f16, 2^-8 where a bf16 call runs on unpacked
rows) and of the scores (2^-23 per product) against the attention over |V|, and P's smallest step: 2^-25 of the largest
contribution for each key.
"""

from __future__ import annotations

import numpy as np
import pytest

from helpers import HALF_ULP_REL, host
from varlen_oracle import attention64, make_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["converted", "unpacked", "by the rule"])
def path(request, monkeypatch):
    """Sets the way that the quantised calls go, and tells it for a batch: True where its rows are unpacked first."""
    from mxflashattn_b200 import backend

    rule = backend.unpack_pays

    def chosen(total_q, *rest):
        if request.param == "converted":
            return False
        return rule(1 << 20 if request.param == "unpacked" else total_q, *rest)  # (as if the call were long enough)

    monkeypatch.setattr(backend, "unpack_pays", chosen)
    return lambda b: chosen(*_rule_arguments(b))


def _rule_arguments(b):
    return int(b.cu[-1]), len(b.new), b.hq // b.hkv, b.hkv, b.d, max(b.total)


def _attend(b, dev, scale, max_q=None):
    import mxflashattn_b200 as fa

    t = b.device(dev)
    out, lse = fa.flash_attn_varlen_with_kvcache(t["q"], t["kc"], t["vc"], t["cu"], t["lens"], t["table"],
                                                 max_q or max(b.new), max(b.total), softmax_scale=scale, causal=True,
                                                 k_scales=t["ks"], v_scales=t["vs"], return_softmax_lse=True)
    return host(out).astype(np.float64), host(lse).astype(np.float64)


def _refresh(b):
    b.k, b.v = b.k_codes * b.k_scale[..., None], b.v_codes * b.v_scale[..., None]


def _check(out, lse, b, scale, rows, unpacked, what):
    want, want_lse, absv, reach = attention64(b, scale, True)
    p_round = HALF_ULP_REL["bf16"] if unpacked and b.dtype == "bf16" else 2.0 ** -11
    score = reach * b.d * 2.0 ** -23
    top = np.zeros_like(lse)  # the largest p |v| of each row
    k, v = b.k.reshape(-1, b.hkv, b.d), b.v.reshape(-1, b.hkv, b.d)
    for s, (n, t) in enumerate(zip(b.new, b.total)):
        at = b.slots(s, 0, t)
        for i in range(n):
            r, end = int(b.cu[s]) + i, t - n + i + 1
            for h in range(b.hq):
                hk = h // (b.hq // b.hkv)
                p = np.exp(k[at[:end], hk] @ b.q[r, h].astype(np.float64) * scale - want_lse[r, h])
                top[r, h] = (p * np.abs(v[at[:end], hk]).max(axis=1)).max()
    tol = 1.001 * HALF_ULP_REL[b.dtype] * np.abs(want) + (1.01 * p_round + 2 * score[..., None]) * absv
    tol = tol + (max(b.total) * 2.0 ** -24 * top)[..., None] + (2.0 ** -24 if b.dtype == "fp16" else 0.0)
    err = np.abs(out - want)[rows]
    assert (err <= tol[rows]).all(), f"{what}: {np.max(err / np.maximum(tol[rows], 1e-300)):.1f} times the bound"
    bound = 2e-5 + score + 2.0 ** -22 * np.abs(want_lse)
    assert (np.abs(lse - want_lse)[rows] <= bound[rows]).all(), f"{what}: LSE"


@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("gap", [3, 7, 8, 14, 22, 23, 34, 50])
def test_later_tokens_of_large_scale_cost_earlier_queries_nothing(gap, dtype, d, which, path, cuda_device):
    new, total, large = [40, 24], [300, 210], 20
    b = make_batch(2000, new, total, hq=4, hkv=2, d=d, dtype=dtype, quant=True)
    for s, t in enumerate(total):
        at = b.slots(s, t - large, t)
        for name in which:
            getattr(b, name + "_scale").reshape(-1, b.hkv)[at] *= 2.0 ** gap
    _refresh(b)
    out, lse = _attend(b, cuda_device, d ** -0.5)
    rows = [int(b.cu[s]) + i for s, n in enumerate(new) for i in range(n - large)]
    _check(out, lse, b, d ** -0.5, rows, path(b), f"gap {gap}")


@pytest.mark.parametrize("new", [2, 260])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 128), ("fp16", 64)])
@pytest.mark.parametrize("low,gap", [(2.5, 10), (2.5, 22), (2.5, 30), (0.75, 18)])
def test_a_large_value_of_little_weight(low, gap, dtype, d, new, path, cuda_device):
    """Key 140's score is far under the others and its V up to 2^30 larger: its part is small, the others' exact."""
    b = make_batch(2010, [new], [400], hq=4, hkv=2, d=d, dtype=dtype, quant=True)
    b.q[:] = 1.0
    slot = int(b.slots(0, 140, 141)[0])
    b.k_codes.reshape(-1, b.hkv, d)[slot] = -low
    b.k_scale.reshape(-1, b.hkv)[slot] = 1.0
    b.v_scale.reshape(-1, b.hkv)[slot] *= 2.0 ** gap
    _refresh(b)
    out, lse = _attend(b, cuda_device, d ** -0.5)
    _check(out, lse, b, d ** -0.5, slice(None), path(b), f"gap {gap}")


@pytest.mark.parametrize("new", [2, 260])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rows_of_zeros_among_others(dtype, new, path, cuda_device):
    """Their scale is the smallest there is."""
    b = make_batch(2020, [new, 1], [400, 200], hq=4, hkv=2, dtype=dtype, quant=True)
    for codes, scale in ((b.k_codes, b.k_scale), (b.v_codes, b.v_scale)):
        codes[:, ::3], scale[:, ::3] = 0.0, 2.0 ** -126
    b.v_codes[:, ::5], b.v_scale[:, ::5] = 0.0, 2.0 ** -126
    _refresh(b)
    out, lse = _attend(b, cuda_device, b.d ** -0.5)
    _check(out, lse, b, b.d ** -0.5, slice(None), path(b), "zeros")


@pytest.mark.parametrize("new", [3, 270])
@pytest.mark.parametrize("low,high", [(5, 17), (12, 20), (-4, 4)])
def test_keys_past_the_largest_half(low, high, new, path, cuda_device):
    """fp16 queries over keys between 2^low and 2^high times their size."""
    b = make_batch(2030, [new, 2], [400, 200], hq=4, hkv=2, dtype="fp16", quant=True)
    rng = np.random.default_rng(4)
    b.k_scale *= np.exp2(rng.integers(low, high + 1, size=b.k_scale.shape).astype(np.float64))
    b.q = (b.q * 2.0 ** -6).astype(np.float32)
    _refresh(b)
    scale = 2.0 ** (6 - high) * b.d ** -0.5
    out, lse = _attend(b, cuda_device, scale)
    _check(out, lse, b, scale, slice(None), False, f"keys 2^{low} .. 2^{high}")
