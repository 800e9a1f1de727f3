"""GpuRmsNorm at values and arguments out of the ordinary."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [256, 77, 1536])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_srq_keeps_a_nan(pkg, sampler, hidden, value):
    """A row that is no number leaves as none: in its grid values and in the sum that the LM head adds to every logit."""
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    x = torch.randn((5, hidden), generator=gen, device="cuda")
    norm = pkg.GpuRmsNorm(sampler, hidden=hidden, out="srq", srq_scale=0.03125)
    want = norm(x)
    y = x.clone()
    y[3, 40] = value
    got = norm(y)
    rest = [0, 1, 2, 4]
    assert torch.equal(got.out[rest], want.out[rest]) and torch.equal(got.row_sum[rest], want.row_sum[rest])
    assert got.row_sum[3].isnan() and got.out[3, 40].isnan()
    if value != value:
        assert got.out[3].isnan().all()


def test_a_nan_row_reaches_the_sampler(pkg, sampler):
    import numpy as np
    g = np.random.default_rng(0)
    head = pkg.GpuLmHead(sampler, g.integers(0, 1 << 32, size=(4096, 256 // 16), dtype=np.uint64).astype(np.uint32),
                         np.full(4096, 0.01, np.float32), 0.03125)
    norm = pkg.GpuRmsNorm(sampler, hidden=256, out="srq", srq_scale=0.03125)
    x = torch.randn((3, 256), device="cuda")
    x[1, 7] = float("nan")
    r = norm(x)
    logits = head.logits(r.out, r.row_sum)
    assert logits[1].isnan().all() and logits[[0, 2]].isfinite().all()
    res = head.sample(r.out, r.row_sum, pkg.params_from_config(dict(pkg.DEFAULT_DECODING_CONFIG, temperature=0)))
    flags = res.flags.tolist()
    assert flags[1] & pkg._lib.FLAG_ERR_NONFINITE and not (flags[0] | flags[2]) & pkg._lib.FLAG_ERRORS


def test_numbers_out_of_range_are_refused(pkg, sampler):
    x = torch.ones((2, 64), device="cuda")
    for bad in (dict(eps=1e300), dict(weight_offset=-1e300), dict(group=2 ** 40, out="e4m3")):
        with pytest.raises(ValueError):
            pkg.GpuRmsNorm(sampler, hidden=64, **bad)(x)
