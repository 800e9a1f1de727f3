"""The operators' handles and streams that do not wait for the default one."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu


def test_a_new_cache_is_cleared_when_it_is_handed_out(pkg):
    """Its counters and flag are zero then and there, not once the default stream comes to it."""
    sampler = pkg.GpuSampler(0)
    k, v = (torch.zeros((40, 2, 64, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    torch.cuda._sleep(int(2e8))  # (about a tenth of a second)
    cache = pkg.GpuKvCache(sampler, k, v)
    assert torch.cuda.default_stream().query()
    # a context cut into pieces and joined, on a stream of its own
    gen = torch.Generator(device="cuda").manual_seed(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in (k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
        q = torch.randn((1, 4, 64), generator=gen, device="cuda").to(torch.bfloat16)
        n = torch.tensor([2500], dtype=torch.int32, device="cuda")
        out, lse = cache.attend(q, None, n, table, max_kv=2560, scale=0.125, lse=True)
    side.synchronize()
    R.check_attend(out, lse, R.attend(q, [0, 1], [2500], table, k.double(), v.double(), 64, 0.125, 0, 0))
    cache.close()
    sampler.close()


def test_an_error_right_after_a_check_is_kept(pkg, sampler):
    cache = pkg.GpuKvCache.allocate(sampler, 2, 2, 16, 64, "bf16")
    x = torch.zeros((1, 2, 64), device="cuda")
    bad = torch.tensor([32], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(50):
        with torch.cuda.stream(side):
            cache.write(x, x, bad)
        with pytest.raises(ValueError, match="slot"):
            cache.check()
    cache.check()
