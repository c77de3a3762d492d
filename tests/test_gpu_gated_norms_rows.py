"""GPU: gated norms of widths whose rows one wave or four waves hold, by the number of rows: the same bits either way, and the
formula in 64 bits (bounds as in test_gpu_gated_norms.py: 2^-17 of the magnitudes for the fp32 sums)."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from _serving import LEAST, UNIT, norms

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [64, 512, 520, 768, 1016, 1024, 1032])
@pytest.mark.parametrize("post", [True, False])
def test_rows_do_not_depend_on_how_many_there_are(pkg, dtype, k, post):
    mod = importlib.import_module(f"{pkg.__name__}.opt.gated_norms")
    m = 1101
    gen = torch.Generator().manual_seed(k)
    x, y = (2 * torch.randn(m, k, generator=gen)).to(dtype), (0.7 * torch.randn(m, k, generator=gen)).to(dtype)
    gate = (0.5 + 0.3 * torch.randn(m, k, generator=gen)).to(dtype)
    weights = [(1 + 0.1 * torch.randn(k, generator=gen)).to(dtype) for _ in range(2)]
    ins = [x, y, gate, weights[0] if post else None, weights[1]]
    dev = [None if t is None else t.to(DEV) for t in ins]
    h, n = mod.gated_norms(*dev, 0.5, 1e-6)
    hq, q, s = mod.gated_norms_quant(*dev, 0.5, 1e-6)
    assert torch.equal(h, hq)
    for rows in (1, 600, 1023, 1024):
        part = [t[:rows] if t is not None and t.ndim == 2 else t for t in dev]
        assert all(torch.equal(a, b[:rows]) for a, b in zip(mod.gated_norms(*part, 0.5, 1e-6), (h, n))), rows
        assert all(torch.equal(a, b[:rows]) for a, b in zip(mod.gated_norms_quant(*part, 0.5, 1e-6), (h, q, s))), rows
    rh, rn, size = norms(*ins, 0.5, 1e-6)
    slack = 2.0 ** -17 * size
    inv = 1 / np.sqrt((rh * rh).mean(1, keepdims=True) + 1e-6)
    bn = slack * inv * np.abs(weights[1].double().numpy()) + 2.0 ** -17 * np.abs(rn)
    s64 = s.double().cpu().numpy()
    for got, want, bound in ((h, rh, UNIT[dtype] * np.abs(rh) + slack + LEAST[dtype]), (n, rn, bn + UNIT[dtype] * np.abs(rn) + LEAST[dtype]),
                             (q.double() * s.double(), rn, bn + s64 * (0.5 + 127 * 2.0 ** -22))):
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= bound).all(), f"{(err / bound).max():.3f} of the bound"
