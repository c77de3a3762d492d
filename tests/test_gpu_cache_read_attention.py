"""GPU: what the INT8 cache gives back, taken by the package's dense attention, against 64 bits.

A bound per row: half an fp16 step of every softmax weight (in its sum and in the product) and of the output, fp32 scores; over
the cache's codes the read's own rounding besides, half an fp16 step of every key and value.
"""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from _serving import LEAST, UNIT, Cache, f32, starts_of, tables

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
FP16 = torch.float16


def _int32(*arrays):
    return [torch.from_numpy(np.array(a, dtype=np.int32, order="C")).to(DEV) for a in arrays]


def _dense(q, k, v, scale, rounded):
    """q, k, v [tokens, dim] in 64 bits -> (out, bound); rounded: k and v may be off by half an fp16 step each."""
    s = (q @ k.T) * scale
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    out, size = w @ v, np.abs(q) @ np.abs(k).T * scale
    slip = (q.shape[1] + 8) * 2.0 ** -24 * size.max(1, keepdims=True)
    if rounded:                                           # a key's rounding moves its score, by as much at most
        slip = slip + 2.0 ** -11 * size.max(1, keepdims=True)
    spread = w @ np.abs(v)
    bound = (2 * (2.0 ** -11 + slip) + 2.0 ** -20) * spread + 2 * 2.0 ** -25 * np.abs(v).sum(0) * w.max(1, keepdims=True)
    if rounded:
        bound = bound + 2.0 ** -11 * spread
    return out, bound + UNIT[FP16] * np.abs(out) + LEAST[FP16]


@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("n", [64, 200])
def test_dense_attention_over_a_cache_read_back(ops, pkg, page, n):
    """A prompt written and read back, attended by ``attention_d64`` without a mask: each head against the values read back,
    and against the cache's codes; the cache's own attention beside it.  Another head's output is past these bounds."""
    kv = importlib.import_module(f"{pkg.__name__}.opt.int8_kv_cache")
    heads, dim, batch = 3, 64, 2
    table, pool = tables([n] * batch, page, -(-n // page), seed=page)
    ref = Cache(pool, heads, dim, page)
    cache = ref.handle(kv, DEV)
    gen = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(batch * n, heads, dim, generator=gen).half() for _ in range(3))
    starts, lens = starts_of([n] * batch), [n] * batch
    ints = _int32(starts, lens, table)
    cache.write(k.to(DEV), v.to(DEV), *ints)
    ref.write(f32(k), f32(v), starts, lens, table)
    kk, vv = cache.read(*_int32([0] * batch), *ints[1:], n)
    dense = ops.decoder_fused_qk_rope.attention_d64(q.view(batch, n, heads, dim).to(DEV), kk, vv, 0.125)
    own = cache.attend(q.to(DEV), *ints, 0.125, causal=False).view(batch, n, heads, dim)
    for b in range(batch):
        for h in range(heads):
            x = f32(q)[b * n:(b + 1) * n, h].astype(np.float64)
            codes = [a[:n] for a in ref.keys_of(table, b, h, range(-(-n // page)))[:2]]
            read = [f32(t[b, :, h]).astype(np.float64) for t in (kk, vv)]
            for what, got, (kx, vx), rounded in (("values read", dense, read, False), ("codes", dense, codes, True),
                                                 ("own attention", own, codes, False)):
                want, bound = _dense(x, kx, vx, 0.125, rounded)
                err = np.abs(got[b, :, h].double().cpu().numpy() - want)
                assert (err <= bound).all(), f"{what}, item {b}, head {h}: {(err / bound).max():.2f} of the bound"
                # an output that is not this head's is past the bound nearly everywhere
                other = np.abs(got[b, :, (h + 1) % heads].double().cpu().numpy() - want)
                assert (other > bound).mean() > 0.8
