"""GPU: calls of attention over the INT8 cache that reach its kernels' less common paths, against 64 bits."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from _serving import Cache, f32, starts_of, tables

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
FP16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def mod(pkg):
    return importlib.import_module(f"{pkg.__name__}.opt.int8_kv_cache")


def _int32(*arrays):
    return [torch.from_numpy(np.array(a, dtype=np.int32, order="C")).to(DEV) for a in arrays]


def _queries(tokens, heads, dim, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (1.5 * torch.randn(tokens, heads, dim, generator=gen)).to(dtype)


def _within(got, want, bound, what=""):
    err = np.abs(got.double().cpu().numpy() - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} past the bound, first at {np.argwhere(bad)[0].tolist()}, " \
                          f"largest {np.nanmax(err / bound):.3g} of it"


@pytest.mark.parametrize("dtype,dim,page", [(FP16, 64, 32), (BF16, 64, 64), (FP16, 64, 128), (FP16, 128, 32), (BF16, 128, 128)])
@pytest.mark.parametrize("kv", [1, 64])
def test_long_tiles_of_few_steps(mod, dtype, dim, page, kv):
    """Long row tiles over so few keys that the two halves of a workgroup's waves meet once, twice or a few times, sequences
    without a key among them; with 64 kv heads enough tiles for 512 rows at dim 64."""
    heads, new = 8 * kv, [80, 80, 70, 80, 80, 80]
    lens = [0, 1, 64, 65, 129, 200]
    table, pool = tables(lens, page, 8, seed=page)
    ref = Cache(pool, kv, dim, page, seed=dim)
    cache = ref.handle(mod, DEV)
    starts = starts_of(new)
    q = _queries(sum(new), heads, dim, dtype, seed=91)
    h = kv - 1
    one = Cache(pool, 1, dim, page)
    one.k, one.v, one.ks, one.vs = ref.k[:, h:], ref.v[:, h:], ref.ks[:, h:], ref.vs[:, h:]
    for causal in (True, False):
        want, bound = one.attend(f32(q[:, 8 * h:]), starts, lens, table, dim ** -0.5, causal, dtype)
        for hint in (None, 78):                           # both kernels; the long tiles alone
            out = cache.attend(q.to(DEV), *_int32(starts, lens, table), dim ** -0.5, causal=causal, max_new=hint)
            _within(out[:, 8 * h:], want, bound, f"causal {causal}, max_new {hint}")
