"""GPU: attention over pages of the INT8 cache whose value scales are apart by far, or as large as the type holds.

The bound of an output counts each key's own error alone: half an fp16 step of its softmax weight, or half the smallest step
of fp16 where the weight is small, times that key's value; a weight that is below every step of fp16 is zero.  So a large
value that a row hardly weighs buys no slack for the others.
"""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from _serving import LEAST, UNIT, Cache, f32, starts_of, tables

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
FP16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def mod(pkg):
    return importlib.import_module(f"{pkg.__name__}.opt.int8_kv_cache")


def _int32(*arrays):
    return [torch.from_numpy(np.array(a, dtype=np.int32, order="C")).to(DEV) for a in arrays]


def _attend(ref, h, q, starts, lens, table, scale, causal, dtype):
    """Head h of the cache for queries [tokens, dim], 64 bits -> (out, bound)."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(len(lens)):
        n, length = starts[b + 1] - starts[b], int(lens[b])
        every = ref.keys_of(table, b, h, range(-(-length // ref.page)))
        for i in range(n):
            t = starts[b] + i
            seen = length - n + i + 1 if causal else length
            k, v = every[0][every[2] < seen], every[1][every[2] < seen]
            x = q[t].astype(np.float64)
            s = (k @ x) * scale
            w = np.exp(s - s.max())
            top = 1 / w.sum()                             # the largest weight
            w *= top
            out[t] = w @ v
            # Weights are fp16 numbers of at least 2^6 (2^7 times the fraction of the value scale) and less than 2^15 for the
            # largest weight: half a step is 2^-11 of a weight or 2^-25, and 2^-25 / 2^6 = 2^-31 of the largest; what is below
            # 2^-25 / 2^15 = 2^-40 of it is less than half the smallest step and becomes zero (2^-42 here, for scores that are a little off).
            # In the sum and in the product; scores and exp2 as in Cache.attend.
            step = np.where(w < 2.0 ** -42 * top, w, np.maximum(2.0 ** -11 * w, 2.0 ** -31 * top))
            slip = 2 * (ref.dim + 8) * 2.0 ** -24 * scale * float((np.abs(k) @ np.abs(x)).max()) + 2.0 ** -20
            bound[t] = step @ np.abs(v) + step.sum() * np.abs(out[t]) + slip * (w @ np.abs(v))
    return out, bound + UNIT[dtype] * np.abs(out) + LEAST[dtype]


def _within(got, want, bound, what):
    err = np.abs(got.double().cpu().numpy() - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} past the bound, first at {np.argwhere(bad)[0].tolist()}, " \
                          f"largest {np.nanmax(err / bound):.3g} of it"


# exponents of the pages' value scales, the largest 0: codes that are exact next to those of the largest end at -24
STEPS = (0, -24, -25, -26, -30, -35, -36, -2)
FAR = (-60, 0, -31, -90, -47, -20, -70, -88)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,exponents,largest", [(FP16, STEPS, 8), (BF16, STEPS, 0), (BF16, FAR, 30)])
@pytest.mark.parametrize("dim,page,kv", [(64, 32, 2), (64, 64, 2), (64, 128, 2), (128, 32, 1), (128, 64, 1), (128, 128, 1),
                                         (64, 32, 96), (64, 64, 96), (64, 128, 96)])
def test_rows_keep_the_values_of_their_own_page(mod, dtype, exponents, largest, dim, page, kv, causal):
    """Every row's weight sits on one page, the pages' value scales are apart by up to 2^-90: rows of the small pages hold
    those pages' values, in the long tiles (256 rows, and 512 with 96 kv heads) and in the 16-row tiles."""
    pages = len(exponents)
    new, lens = [200, 170], [pages * page, pages * page - 5]
    table, pool = tables(lens, page, pages, seed=page + dim)
    ref = Cache(pool, kv, dim, page, seed=dim)
    rng = np.random.default_rng(90)
    ref.k[:] = rng.integers(-2, 3, ref.k.shape)
    ref.ks[:] = 1.0
    for b in range(2):
        for j, e in enumerate(exponents):
            ref.k[table[b, j], :, :, j] = 100
            ref.vs[table[b, j]] = 1.7 * 2.0 ** (largest + e) * (1 + 0.1 * (b + j % 3))
    q = 0.3 * rng.standard_normal((sum(new), kv, dim))
    for t in range(sum(new)):
        q[t, :, :pages] = 0
        q[t, :, t % pages] = 16.0                         # 100 x 16 x 1/8: 200 above the other pages' scores
    q = torch.from_numpy(q).to(dtype)
    starts = starts_of(new)
    cache = ref.handle(mod, DEV)
    ints = _int32(starts, lens, table)
    h = kv - 1
    want, bound = _attend(ref, h, f32(q[:, h]), starts, lens, table, 0.125, causal, dtype)
    for hint in (1, None, 170):                           # 16-row tiles; both kernels; the long tiles alone
        out = cache.attend(q.to(DEV), *ints, 0.125, causal=causal, max_new=hint)
        _within(out[:, h], want, bound, f"max_new {hint}")


@pytest.mark.parametrize("codes", ["largest", "random"])
@pytest.mark.parametrize("dim,page,kv,group,new,held,width", [
    (64, 64, 2, 2, 1, 500, 8), (128, 32, 1, 4, 1, 5000, 157), (128, 128, 2, 1, 3, 300, 4),     # 16-row tiles, one split and several
    (64, 64, 1, 4, 100, 300, 8), (128, 32, 1, 2, 120, 2000, 70), (64, 64, 64, 1, 300, 3, 6)])  # long tiles likewise
def test_values_near_the_largest_of_bf16(mod, codes, dim, page, kv, group, new, held, width):
    """Outputs are averages of values, finite where the values are: sums of up to thousands of the largest that bf16 holds, over
    all keys and over selected pages (a token to a workgroup, and several)."""
    lens = [new + held]
    pages = -(-lens[0] // page)
    table, pool = tables(lens, page, width, seed=page + dim)
    ref = Cache(pool, kv, dim, page, seed=dim)
    if codes == "largest":
        ref.v[:] = 127
    ref.vs[:] = 3.38e38 / 127
    rng = np.random.default_rng(92)
    q = torch.from_numpy(rng.standard_normal((new, kv * group, dim))).to(BF16)
    cache = ref.handle(mod, DEV)
    starts = starts_of([new])
    ints = _int32(starts, lens, table)
    lists = np.broadcast_to(np.arange(pages, dtype=np.int32), (new, kv, pages))
    outs = {"all": cache.attend(q.to(DEV), *ints, dim ** -0.5),
            "selected": cache.attend_selected(q.to(DEV), *_int32(lists), *ints, dim ** -0.5)}
    for what, out in outs.items():
        for h in {0, kv * group - 1}:
            want, bound = _attend(ref, h // group, f32(q[:, h]), starts, lens, table, dim ** -0.5, True, BF16)
            _within(out[:, h], want, bound, what)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,dim,page,kv,group,new,held,width", [
    (FP16, 64, 64, 2, 2, 1, 500, 8), (BF16, 128, 32, 1, 4, 1, 5000, 157), (FP16, 128, 128, 2, 1, 3, 300, 4),   # 16-row tiles
    (FP16, 64, 64, 1, 4, 100, 300, 8), (BF16, 128, 32, 1, 2, 120, 2000, 70), (FP16, 64, 32, 64, 1, 300, 3, 10)])  # long tiles
def test_scores_of_many_millions(mod, sign, dtype, dim, page, kv, group, new, held, width):
    """Scores of 1e7 to 1e11, where a step of fp32 is many times the softmax's unit, all positive or all negative: the key that
    stands out has the whole weight; rows of common size beside them keep their accuracy."""
    lens = [new + held]
    pages = -(-lens[0] // page)
    table, pool = tables(lens, page, width, seed=page + dim)
    ref = Cache(pool, kv, dim, page, seed=dim)
    rng = np.random.default_rng(93)
    ref.k[:] = rng.integers(30, 128, ref.k.shape)
    ref.ks[:] = (400 + 100 * rng.random(ref.ks.shape)).astype(np.float32)
    sizes = np.exp(rng.uniform(np.log(30), np.log(6e4), (new, kv * group, 1)))
    small = rng.random((new, kv * group, 1)) < 0.3
    sizes[small] = 1e-6 / dim
    q = torch.from_numpy(sign * sizes * (0.5 + 0.5 * rng.random((new, kv * group, dim)))).to(dtype)
    cache = ref.handle(mod, DEV)
    starts = starts_of([new])
    ints = _int32(starts, lens, table)
    lists = np.broadcast_to(np.arange(pages, dtype=np.int32), (new, kv, pages))
    outs = {"all": cache.attend(q.to(DEV), *ints, 0.125),
            "selected": cache.attend_selected(q.to(DEV), *_int32(lists), *ints, 0.125)}
    for h in {0, kv * group - 1}:
        want, bound = _attend(ref, h // group, f32(q[:, h]), starts, lens, table, 0.125, True, dtype)
        clear = np.ones(new, bool)
        k, v, pos = ref.keys_of(table, 0, h // group, range(pages))
        for t in range(new):
            if small[t, h, 0]:
                continue
            s = np.sort((k[pos <= held + t] @ f32(q[t, h]).astype(np.float64)) * 0.125)
            # fp32 sums of dim exact products are within (dim + 8) 2^-24 of the largest: a key further ahead than
            # twice that and 200 has every other's weight at zero
            clear[t] = len(s) < 2 or s[-1] - s[-2] > 2 * (dim + 8) * 2.0 ** -24 * np.abs(s).max() + 200
            bound[t] = (2.0 ** -10 + UNIT[dtype]) * np.abs(want[t]) + LEAST[dtype]
        assert new == 1 or clear.sum() > new / 2
        for what, out in outs.items():
            _within(out[:, h][torch.from_numpy(clear).to(DEV)], want[clear], bound[clear], what)
            assert torch.isfinite(out[:, h]).all(), what


@pytest.mark.parametrize("hint", [None, 1])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_an_infinite_query_changes_no_bit_of_the_rows_beside_it(mod, dtype, hint):
    """Its row is NaN; the others' weights are made as without it, in the long tiles and in tiles of 16 rows."""
    heads, dim, page, new, held = 2, 64, 64, 192, 900
    table, pool = tables([held + new], page, 18, seed=4)
    ref = Cache(pool, heads, dim, page, seed=5)
    ref.k[..., 0], ref.ks[:] = 127, 0.5
    cache = ref.handle(mod, DEV)
    # scores of 5e5, all nearly alike: a step of fp32 there is a sixteenth, which other roundings would show
    q = torch.randn(new, heads, dim, generator=torch.Generator().manual_seed(6)).to(dtype)
    q[..., 0] = 6e4
    q[::16] = 0
    ints = _int32([0, new], [held + new], table)
    want = cache.attend(q.to(DEV), *ints, 0.125, max_new=hint)
    bad = q.clone()
    bad[::16, :, 0] = float("inf")                        # an infinite score of every key
    out = cache.attend(bad.to(DEV), *ints, 0.125, max_new=hint)
    rows = [t for t in range(new) if t % 16]
    assert torch.isnan(out[::16]).all()
    assert torch.equal(out[rows], want[rows])
