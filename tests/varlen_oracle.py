"""A ragged batch over a paged cache in 64 bits, sequence by sequence: inputs, quantisation, attention, tolerances."""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from helpers import HALF_ULP_REL, OUT_ATOL, P_ROUND_REL
from mxflashattn_b200 import synthetic as syn


def quantise64(x: np.ndarray):
    """(e4m3 values, scale) of each row of x by the definition, in 64 bits."""
    x = np.asarray(x, np.float64)
    mag = np.where(np.isfinite(x), np.abs(x), 0.0).max(axis=-1)
    scale = np.full(mag.shape, 2.0 ** -126)
    while (over := mag > 448.0 * scale).any():
        scale = np.where(over, 2.0 * scale, scale)
    with np.errstate(invalid="ignore"):
        y = x / scale[..., None]
        a = np.minimum(np.abs(y), 448.0)  # NaN stays NaN
        _, expo = np.frexp(np.where(np.isnan(a), 1.0, a))  # a = m * 2^expo, m in [0.5, 1)
        step = np.exp2(np.maximum(expo - 1, -6) - 3.0)
        codes = np.copysign(np.round(a / step) * step, y)  # np.round: ties to even
    return np.where(np.abs(codes) > 448.0, np.copysign(448.0, codes), codes), scale


def e4m3_tensor(values: np.ndarray):
    import torch

    return torch.from_numpy(np.asarray(values, np.float32)).to(torch.float8_e4m3fn)


def e8m0_tensor(scale: np.ndarray):
    """Scales [pages, page size, heads] as the cache's [pages, heads, page size] e8m0 tensor."""
    import torch

    byte = (np.round(np.log2(np.asarray(scale, np.float64))) + 127).astype(np.uint8)
    return torch.from_numpy(np.ascontiguousarray(byte.transpose(0, 2, 1))).view(torch.float8_e8m0fnu)


@dataclass
class Batch:
    """Host side of a ragged batch: ``new[b]`` packed tokens, ``total[b]`` cached ones that include them."""

    new: list
    total: list
    hq: int
    hkv: int
    d: int
    page: int
    dtype: str
    quant: bool
    q: np.ndarray        # [T, HQ, D]
    k: np.ndarray        # cache values [P, PS, HKV, D], dequantised, float64
    v: np.ndarray
    k_codes: np.ndarray | None
    v_codes: np.ndarray | None
    k_scale: np.ndarray | None  # [P, PS, HKV]
    v_scale: np.ndarray | None
    table: np.ndarray
    cu: np.ndarray

    def slots(self, b, lo, hi):
        pos = np.arange(lo, hi)
        return self.table[b, pos // self.page] * self.page + pos % self.page

    def device(self, dev, index_dtype=None):
        import torch

        tdt = syn.torch_dtype(self.dtype)
        idt = index_dtype or torch.int32
        t = {"q": torch.from_numpy(self.q).to(dev, tdt),
             "cu": torch.from_numpy(self.cu).to(dev, idt),
             "lens": torch.tensor(self.total, dtype=idt, device=dev),
             "table": torch.from_numpy(self.table).to(dev, idt), "ks": None, "vs": None}
        if self.quant:
            t["kc"], t["vc"] = e4m3_tensor(self.k_codes).to(dev), e4m3_tensor(self.v_codes).to(dev)
            t["ks"], t["vs"] = e8m0_tensor(self.k_scale).to(dev), e8m0_tensor(self.v_scale).to(dev)
        else:
            t["kc"] = torch.from_numpy(self.k.astype(np.float32)).to(dev, tdt)
            t["vc"] = torch.from_numpy(self.v.astype(np.float32)).to(dev, tdt)
        return t


def make_batch(seed, new, total, *, hq=8, hkv=2, d=128, page=16, dtype="bf16", quant=False, poison=None, spare_pages=2,
               extra_cols=1, spread=0.5):
    """Seeded batch; unused table entries are -1, unowned cache slots hold ``poison`` (e.g. NaN) when given."""
    rng = np.random.default_rng(seed)
    need = [-(-t // page) for t in total]
    pages = sum(need) + spare_pages
    perm = rng.permutation(pages)
    width = max(max(need, default=0), 1) + extra_cols
    table = np.full((len(new), width), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = syn.round_dtype(rng.standard_normal((int(cu[-1]), hq, d), dtype=np.float32), dtype)
    chan = np.exp(spread * rng.standard_normal((hkv, d))).astype(np.float32)
    k = syn.round_dtype(rng.standard_normal((pages, page, hkv, d), dtype=np.float32) * chan, dtype).astype(np.float64)
    v = syn.round_dtype(rng.standard_normal((pages, page, hkv, d), dtype=np.float32), dtype).astype(np.float64)
    kc = vc = ks = vs = None
    owned = np.zeros((pages * page,), bool)
    batch = Batch(list(new), list(total), hq, hkv, d, page, dtype, quant, q, k, v, kc, vc, ks, vs, table, cu)
    for b, t in enumerate(total):
        owned[batch.slots(b, 0, t)] = True
    owned = owned.reshape(pages, page)
    if quant:
        kc, ks = quantise64(k)
        vc, vs = quantise64(v)
        batch.k, batch.v = kc * ks[..., None], vc * vs[..., None]
        batch.k_codes, batch.v_codes, batch.k_scale, batch.v_scale = kc, vc, ks, vs
    if poison is not None:
        for x in (batch.k, batch.v) + ((kc, vc) if quant else ()):
            x[~owned] = poison
    return batch


def attention64(batch: Batch, scale, causal):
    """(out, lse, attention over |V|, largest sum |q k| scale) of every packed row; masked keys take no part at all."""
    T = int(batch.cu[-1])
    out = np.zeros((T, batch.hq, batch.d))
    lse = np.full((T, batch.hq), -np.inf)
    absv = np.zeros((T, batch.hq, batch.d))
    reach = np.zeros((T, batch.hq))
    k, v = batch.k.reshape(-1, batch.hkv, batch.d), batch.v.reshape(-1, batch.hkv, batch.d)
    for b, (n, t) in enumerate(zip(batch.new, batch.total)):
        at = batch.slots(b, 0, t)
        for i in range(n):
            row = int(batch.cu[b]) + i
            end = min(t, t - n + i + 1) if causal else t
            if end <= 0:
                continue
            for h in range(batch.hq):
                hk = h // (batch.hq // batch.hkv)
                kk, vv = k[at[:end], hk], v[at[:end], hk]
                qq = batch.q[row, h].astype(np.float64)
                s = kk @ qq * scale
                m = s.max()
                p = np.exp(s - m)
                out[row, h] = p @ vv / p.sum()
                lse[row, h] = m + np.log(p.sum())
                absv[row, h] = p @ np.abs(vv) / p.sum()
                reach[row, h] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
    return out, lse, absv, reach


def assert_attention(got_out, got_lse, batch, scale, causal, what=""):
    """Output: half an ulp of storage (or the framework's absolute bound) plus P rounded once to 16 bits; LSE: 32-bit
    accumulation of D products of each score (at most 2^-23 of their absolute sum a step) and of the exponentials."""
    out, lse, absv, reach = attention64(batch, scale, causal)
    g = np.asarray(got_out, np.float64)
    assert np.isfinite(g).all(), f"{what}: non-finite output"
    score = reach * batch.d * 2.0 ** -23  # error of a score, natural-log units; moves P by as much, relatively
    tol = np.maximum(OUT_ATOL[batch.dtype], 1.001 * HALF_ULP_REL[batch.dtype] * np.abs(out))
    tol = tol + (1.01 * P_ROUND_REL[batch.dtype] + 2 * score[..., None]) * absv + 1e-6
    bad = np.abs(g - out) > tol
    assert not bad.any(), f"{what}: {bad.sum()} outputs off, worst {np.abs(g - out)[bad].max():.3e}"
    if got_lse is not None:
        gl = np.asarray(got_lse, np.float64)
        empty = np.isneginf(lse)
        assert (np.isneginf(gl) == empty).all(), f"{what}: LSE of empty rows"
        err = np.abs(np.where(empty, 0.0, gl) - np.where(empty, 0.0, lse))
        assert (err <= 2e-5 + score + 2.0 ** -22 * np.abs(np.where(empty, 0.0, lse))).all(), f"{what}: LSE off {err.max():.3e}"
