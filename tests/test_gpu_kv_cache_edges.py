"""GpuKvCache.read where its outputs are views."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_that_overlap_are_refused(pkg, sampler):
    cache = pkg.GpuKvCache.allocate(sampler, 4, 2, 16, 64, "bf16")
    x = torch.randn((9, 2, 64), device="cuda").to(torch.bfloat16)
    slots = torch.arange(9, dtype=torch.int32, device="cuda")
    cache.write(x, -x, slots)
    buf = torch.zeros(9 * 4 * 64 + 64, dtype=torch.bfloat16, device="cuda")
    rows = buf[:9 * 256].view(9, 4, 64)
    diagonal = torch.as_strided(buf, (9, 2, 64), (64, 64, 1))
    for out in ((rows[:, :2], rows[:, 1:3]), (diagonal, torch.empty_like(x)), (torch.empty_like(x), diagonal)):
        with pytest.raises(ValueError, match="overlap"):
            cache.read(slots, out=out)
    k, v = cache.read(slots, out=(rows[:, :2], rows[:, 2:]))
    assert torch.equal(k, x) and torch.equal(v, -x)
    k, v = cache.read(slots[:1], out=(rows[:1, :2], rows[:1, 2:]))
    assert torch.equal(k, x[:1]) and torch.equal(v, -x[:1])
