"""QuantizedKVCache.status() over scratch buffers of several streams."""
import pytest
import torch

from test_gpu_kv8 import fill, make, queries

pytestmark = pytest.mark.gpu


def test_status_waits_for_every_stream(lib):
    """An error of a launch that another stream has still ahead is found, and the scratch is sound for that stream's next call"""
    cache, table, rng = make([9000, 100], 2, "e4m3", 12)
    fill(cache, "e4m3", rng)
    q = queries(rng, 2, 8).cuda()
    good = cache.decode(q, num_heads=8)
    broken = cache.page_table.clone()
    broken[1, 3] = cache.num_pages
    side = torch.cuda.Stream()
    a = torch.randn((8192, 8192), device="cuda")
    with torch.cuda.stream(side):
        cache.decode(q, num_heads=8)
    cache.status()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):                                   # some tens of milliseconds
            a @ a
        cache.decode(q, num_heads=8, page_table=broken)
    with pytest.raises(RuntimeError, match="outside the pool"):
        cache.status()
    with torch.cuda.stream(side):
        again = cache.decode(q, num_heads=8)
    cache.status()
    assert torch.equal(again, good)
