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


class Pending:
    """Memory that was freed while the current stream has still to write to it."""

    def __init__(self, *shapes_and_types):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        held = [torch.empty(s, dtype=t, device="cuda") for s, t in shapes_and_types]
        torch.cuda._sleep(int(1e8))
        for t in held:
            t.view(torch.uint8).fill_(0x7f)


def test_outputs_of_another_stream_are_its_own(pkg, sampler):
    gen = torch.Generator(device="cuda").manual_seed(0)
    side = torch.cuda.Stream()
    x = torch.randn((64, 1024), generator=gen, device="cuda").to(torch.bfloat16)
    norm = pkg.GpuRmsNorm(sampler, hidden=1024, out="e4m3", group=128)
    want = norm(x, x)
    Pending(((64, 1024), torch.uint8), ((64, 8), torch.float32), ((64, 1024), torch.bfloat16))
    got = norm(x, x, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(got.out.view(torch.uint8), want.out.view(torch.uint8))
    assert torch.equal(got.scale, want.scale) and torch.equal(got.residual, want.residual)

    cache = pkg.GpuKvCache.allocate(sampler, 32, 4, 16, 128, "bf16")
    kv = torch.randn((500, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    slots = torch.arange(500, dtype=torch.int32, device="cuda")
    cache.write(kv[:, :4], kv[:, 4:], slots)
    Pending(((500, 4, 128), torch.bfloat16), ((500, 4, 128), torch.bfloat16))
    k, v = cache.read(slots, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(k, kv[:, :4]) and torch.equal(v, kv[:, 4:])

    q = torch.randn((40, 8, 128), generator=gen, device="cuda").to(torch.bfloat16)
    starts, n = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 40], [500]))
    table = torch.arange(32, dtype=torch.int32, device="cuda")[None]
    call = dict(max_q=40, max_kv=512, scale=0.1, lse=True)
    want = cache.attend(q, starts, n, table, **call)
    Pending(((40, 8, 128), torch.bfloat16), ((40, 8), torch.float32))
    got = cache.attend(q, starts, n, table, stream=side.cuda_stream, **call)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # given outputs are used as they are, and the default stream has a handle too
    out = torch.empty_like(q)
    assert cache.attend(q, starts, n, table, stream=0, out=out, **call)[0] is out
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    cache.check()


def test_closed_handles_are_refused(pkg):
    sampler = pkg.GpuSampler(0)
    cache, other = (pkg.GpuKvCache.allocate(sampler, 4, 2, 16, 64, "bf16") for _ in range(2))
    norm = pkg.GpuRmsNorm(sampler, hidden=64)
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots, n = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")

    def calls(c):
        return (lambda: c.write(x, x, slots), lambda: c.read(slots), c.check,
                lambda: c.attend(x, None, n, table, max_kv=16, scale=0.1))
    for f in calls(cache):
        f()
    other.close()
    for f in calls(other):
        with pytest.raises(ValueError, match="closed"):
            f()
    for f in calls(cache):
        f()
    torch.cuda.synchronize()
    sampler.close()
    for f in calls(cache) + (lambda: norm(x[0]), lambda: pkg.GpuKvCache.allocate(sampler, 4, 2, 16, 64, "bf16")):
        with pytest.raises(ValueError, match="closed"):
            f()
    cache.close()
    other.close()
