"""GPU: reads of every size; and the key means that a write leaves, of pages that one wave writes and that several do, against those of
the codes that it left."""
from __future__ import annotations

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 32), (64, 64), (128, 32), (64, 128), (128, 64), (128, 128)])
def test_key_means_are_those_of_the_codes(pkg, dtype, dim, page):
    """64 sequences of 8 heads: prompts that end inside a page, then a few tokens appended to each."""
    kv = importlib.import_module(f"{pkg.__name__}.opt.int8_kv_cache")
    heads, batch, width = 8, 64, 4
    gen = torch.Generator().manual_seed(dim + page)
    cache = kv.Int8KVCache.empty(batch * width, heads, dim, page, DEV)
    table = torch.randperm(batch * width, generator=gen).int().view(batch, width).to(DEV)
    lens = torch.zeros(batch, dtype=torch.int32)
    for new in (torch.randint(1, 3 * page, (batch,), generator=gen), torch.randint(0, 4, (batch,), generator=gen)):
        lens = lens + new.int()
        starts = torch.cat([torch.zeros(1), new.cumsum(0)]).int()
        # a mean of its own for every dim, so that a sum that ends up at another dim shows
        k = (torch.randn(int(new.sum()), heads, dim, generator=gen) + torch.linspace(-3, 3, dim)).to(dtype).to(DEV)
        cache.write(k, k, starts.to(DEV), lens.to(DEV), table)
        codes, means = cache.k.cpu(), cache.k_mean.cpu()
        for b in range(batch):
            for j in range(-(-int(lens[b]) // page)):
                held = min(page, int(lens[b]) - j * page)
                p = int(table[b, j])
                total = codes[p, :, :held].sum(1, dtype=torch.int32)
                assert torch.equal(means[p], (total.float() / held).round().to(torch.int8)), (b, j)


@pytest.mark.parametrize("length", [3700, 5300, 70000])
def test_reads_of_every_size_are_the_codes_times_the_scale(pkg, length):
    """Outputs that are stored past the caches (15 and 287 MB) and that are left in them (22 MB): one batch of shared pages, bit for bit."""
    kv = importlib.import_module(f"{pkg.__name__}.opt.int8_kv_cache")
    heads, dim, page, pool = 8, 128, 64, 50
    gen = torch.Generator().manual_seed(length)
    k = torch.randint(-127, 128, (pool, heads, page, dim), generator=gen, dtype=torch.int8).to(DEV)
    v = torch.randint(-127, 128, (pool, heads, dim, page), generator=gen, dtype=torch.int8).to(DEV)
    ks, vs = (torch.rand(pool, heads, generator=gen).to(DEV) for _ in range(2))
    cache = kv.Int8KVCache(k, v, ks, vs, torch.zeros((pool, heads, dim), dtype=torch.int8, device=DEV))
    table = torch.randint(0, pool, (1, -(-length // page)), generator=gen).int().to(DEV)
    ints = [torch.tensor([n], dtype=torch.int32, device=DEV) for n in (0, length)]
    got = cache.read(*ints, table, length)
    ids = table[0].long()
    for out, codes, scale in ((got[0], k, ks), (got[1], v.transpose(2, 3), vs)):
        want = (codes[ids].float() * scale[ids][..., None, None]).half().transpose(1, 2).reshape(-1, heads, dim)[:length]
        assert torch.equal(out[0], want)
