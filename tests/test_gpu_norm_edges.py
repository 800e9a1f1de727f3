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


@pytest.mark.parametrize("rows,hidden", [(3, 64), (700, 1536), (5, 77), (400, 1111), (300, 8192)])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_codes_and_scales_are_the_quotients(pkg, sampler, rows, hidden, group):
    """scale = a / 448 and code = round(y · (448 / a)), each quotient rounded once, on the y that the same norm
    gives as float32; a from 2^-64 up."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, hidden), generator=gen, device="cuda") * torch.exp2(torch.randint(-30, 30, (1, hidden), generator=gen, device="cuda").float())
    w = torch.randn(hidden, generator=gen, device="cuda") * torch.exp2(torch.randint(-90, 60, (hidden,), generator=gen, device="cuda").float())
    y = pkg.GpuRmsNorm(sampler, w, out="f32")(x).out
    got = pkg.GpuRmsNorm(sampler, w, out="e4m3", group=group)(x)
    g = group or hidden
    for i in range(0, hidden, g):
        part = y[:, i:i + g]
        a = part.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -64)
        most = torch.full_like(a, 448.0)  # (a quotient of tensors: torch turns one by a number into a product)
        assert torch.equal(got.scale[:, i // g:i // g + 1], a / most)
        assert torch.equal(got.out[:, i:i + g].view(torch.uint8), (part * (most / a)).to(torch.float8_e4m3fn).view(torch.uint8))
