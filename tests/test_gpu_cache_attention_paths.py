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


def _shared(pool, kv, dim, page, batch, width, seed):
    """A cache of few pages, and tables that name them over and over: long sequences of little memory."""
    ref = Cache(pool, kv, dim, page, seed=seed)
    return ref, np.random.default_rng(seed).integers(0, pool, (batch, width)).astype(np.int32)


@pytest.mark.parametrize("dtype,dim,page", [(FP16, 64, 32), (BF16, 128, 32), (FP16, 64, 128)])
def test_more_pages_of_a_split_than_a_wave_looks_up_at_once(mod, dtype, dim, page):
    """512 (sequence, head) pairs, so that the keys are not split, over up to 600 pages: each wave looks its pages up in three
    rounds; some pages are not there."""
    kv, batch, width = 2, 256, 600
    ref, table = _shared(40, kv, dim, page, batch, width, seed=page)
    table[:, 255:258] = -1
    table[7, 64:] = 10 ** 6
    lens = [width * page - 37 * b for b in range(batch)]
    cache = ref.handle(mod, DEV)
    q = _queries(batch, 2 * kv, dim, dtype, seed=94)
    out = cache.attend(q.to(DEV), *_int32(starts_of([1] * batch), lens, table), dim ** -0.5, max_new=1)
    for b in (0, 7, 100, 255):
        want, bound = ref.attend(f32(q[b:b + 1]), [0, 1], lens[b:b + 1], table[b:b + 1], dim ** -0.5, True, dtype)
        _within(out[b:b + 1], want, bound, f"sequence {b}")


@pytest.mark.parametrize("dtype,dim,page,group", [(FP16, 64, 32, 1), (BF16, 128, 64, 4), (FP16, 64, 128, 16)])
def test_lists_longer_than_a_wave_looks_up_at_once(mod, dtype, dim, page, group):
    """Lists of 700 entries for single tokens of 128 sequences (one split): entries past the sequence, a page named twice, and
    runs of no page among them."""
    kv, batch, width, blocks = 2, 128, 720, 700
    ref, table = _shared(30, kv, dim, page, batch, width, seed=page + 1)
    lens = [width * page - 5 * page * b - 3 for b in range(batch)]
    rng = np.random.default_rng(95)
    lists = np.stack([np.stack([rng.permutation(width)[:blocks] for _ in range(kv)]) for _ in range(batch)]).astype(np.int32)
    lists[:, :, 300:330] = -1
    lists[:, 1, 5] = lists[:, 1, 650] = 2
    cache = ref.handle(mod, DEV)
    q = _queries(batch, kv * group, dim, dtype, seed=96)
    out = cache.attend_selected(q.to(DEV), *_int32(lists), *_int32(starts_of([1] * batch), lens, table), dim ** -0.5)
    for b in (0, 77, 127):
        want, bound = ref.attend(f32(q[b:b + 1]), [0, 1], lens[b:b + 1], table[b:b + 1], dim ** -0.5, True, dtype, lists[b:b + 1])
        _within(out[b:b + 1], want, bound, f"sequence {b}")


@pytest.mark.parametrize("repeat", [False, True])
@pytest.mark.parametrize("dtype,dim,page,group,blocks", [(FP16, 64, 32, 1, 60), (BF16, 128, 64, 4, 200), (FP16, 64, 32, 7, 900),
                                                         (FP16, 128, 128, 2, 330)])
def test_unions_of_many_pages(mod, repeat, dtype, dim, page, group, blocks):
    """Chunks over 1000 pages whose tokens' lists together have more than 256: a thread lists several pages, a wave looks its
    entries up in several rounds; with a list that names a page twice, each token's own list."""
    kv, new, width = 2, [21, 3], 1001
    ref, table = _shared(30, kv, dim, page, 2, width, seed=page + 2)
    lens = [width * page - 5, 700 * page + 1]
    rng = np.random.default_rng(97)
    lists = np.stack([np.stack([np.sort(rng.permutation(width)[:blocks]) for _ in range(kv)]) for _ in range(24)]).astype(np.int32)
    lists[3:6, 0] = -1
    if repeat:
        lists[2, 1, 0] = lists[2, 1, blocks - 1]
    starts = starts_of(new)
    cache = ref.handle(mod, DEV)
    q = _queries(24, kv * group, dim, dtype, seed=98)
    out = cache.attend_selected(q.to(DEV), *_int32(lists), *_int32(starts, lens, table), dim ** -0.5)
    for t in (0, 2, 3, 13, 20, 21, 23):
        b = 0 if t < 21 else 1
        end = lens[b] - new[b] + t - starts[b] + 1        # the token's own length
        want, bound = ref.attend(f32(q[t:t + 1]), [0, 1], [end], table[b:b + 1], dim ** -0.5, True, dtype, lists[t:t + 1])
        _within(out[t:t + 1], want, bound, f"token {t}")
    assert (out[3:6, :group] == 0).all()


@pytest.mark.parametrize("dtype,dim,group,width,blocks", [(FP16, 64, 1, 257, 256), (BF16, 128, 4, 1000, 33), (FP16, 128, 16, 2100, 700),
                                                          (BF16, 64, 7, 5000, 4096), (FP16, 64, 2, 32768, 48)])
def test_selection_of_single_tokens_over_many_pages(mod, dtype, dim, group, width, blocks):
    """A token of each sequence over more than 256 pages, up to the widest table: equal scores in numbers (few pages named
    over and over), NaN scales, pages that are not there, a sequence shorter than its list."""
    kv, page = (1, 32) if width > 2100 else (2, 64)
    ref, table = _shared(50, kv, dim, page, 3, width, seed=width)
    ref.ks[7] = np.nan
    table[:, 11] = -1
    lens = [width * page, (width - 1) * page - 3, min(blocks, 300) * page - 1]
    cache = ref.handle(mod, DEV)
    q = _queries(3, kv * group, dim, dtype, seed=99)
    ints = _int32(starts_of([1] * 3), lens, table)
    there = table.copy()
    there[there == 7] = -1                                # for the restatement: a page without a score comes last too
    for sink, local in ((1, 1), (0, 3)):
        picked = cache.select(q.to(DEV), *ints, blocks, sink=sink, local=local)
        assert np.array_equal(picked.cpu().numpy(), ref.select(f32(q), [0, 1, 2, 3], lens, there, blocks, sink, local))
