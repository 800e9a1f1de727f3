"""GpuRmsNorm against the formula in float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def reference(x, r, w, offset, eps):
    h = x.double() + (r.double() if r is not None else 0.0)
    y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps)
    return h, y if w is None else y * (offset + w.double())


def check(res, x, r, w, offset, eps, out, group, srq):
    h, y = reference(x, r, w, offset, eps)
    n = x.shape[1]
    # sum of squares: at most 8 · 4 or 32 adds a thread, 5 shuffles, 32 warps (under 80 roundings
    # of 2^-24, half of it in the root), then the quotient, root, two products and the sum h
    rel = 50 * 2.0 ** -24
    if r is not None:
        assert torch.equal(res.residual, (x.float() + r.float()).to(x.dtype))
    if out in ("f32", "bf16"):
        half = 2.0 ** -8 if out == "bf16" else 0.0
        assert ((res.out.double() - y).abs() <= (rel + half) * y.abs() + 1e-38).all()
    elif out == "srq":
        q = torch.round(res.out.double() / srq)
        assert torch.equal((q.float() * torch.tensor(srq, device=q.device, dtype=torch.float32)), res.out)
        want = (y / srq).clamp(-128, 127)
        assert ((q - want).abs() <= 0.5 + 2 * rel * want.abs() + 1e-6).all()
        assert torch.equal(res.row_sum, q.sum(dim=1).float() * torch.tensor(srq, device=q.device, dtype=torch.float32))
    else:
        g = group or n
        assert res.scale.shape == (x.shape[0], -(-n // g))
        for i in range(0, n, g):
            yy = y[:, i:i + g]
            a = yy.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -64)
            s = res.scale[:, i // g:i // g + 1].double()
            assert ((s - a / 448).abs() <= 2 * rel * a / 448).all()
            back = res.out[:, i:i + g].float().double() * s
            # half a code step: 2^-4 of a normal code, 2^-10 of the scale below
            assert ((back - yy).abs() <= (2.0 ** -4 + 4 * rel) * yy.abs() + (2.0 ** -10 + 448 * 2 * rel) * s).all()


@pytest.mark.parametrize("out,group", [("f32", 0), ("bf16", 0), ("e4m3", 0), ("e4m3", 128), ("e4m3", 64), ("e4m3", 32),
                                       ("srq", 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,hidden,residual", [(1, 1536, True), (3, 1, True), (5, 33, False), (2, 1000, True),
                                                  (300, 256, True), (7, 1111, True), (4, 8192, True), (2, 32768, False),
                                                  (2, 32761, True), (600, 640, False)])
def test_norm_matches_formula(pkg, sampler, rows, hidden, residual, dtype, out, group):
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + hidden)
    x = torch.randn((rows, hidden), generator=gen, device="cuda").to(DT[dtype])
    r = (3 * torch.randn((rows, hidden), generator=gen, device="cuda")).to(DT[dtype]) if residual else None
    w = torch.randn(hidden, generator=gen, device="cuda").to(DT["f32" if dtype == "bf16" else "bf16"])
    norm = pkg.GpuRmsNorm(sampler, w, eps=1e-6, weight_offset=1.0, out=out, group=group,
                          srq_scale=0.03125 if out == "srq" else 0.0)
    check(norm(x, r), x, r, w, 1.0, 1e-6, out, group, 0.03125)


def test_rows_of_zeros_and_tiny_values(pkg, sampler):
    x = torch.zeros((3, 256), device="cuda")
    x[1] = 1e-30
    x[2, 5] = 1.0
    norm = pkg.GpuRmsNorm(sampler, hidden=256, eps=1e-6, out="e4m3", group=64)
    res = norm(x)
    check(res, x, None, None, 0.0, 1e-6, "e4m3", 64, 0)
    assert torch.equal(res.out[0].float(), torch.zeros(256, device="cuda"))
    assert (res.scale[0] == 2.0 ** -64 / 448).all()


@pytest.mark.parametrize("hidden", [512, 77])
def test_nan_and_infinity_stay_in_their_rows(pkg, sampler, hidden):
    x = torch.randn((4, hidden), device="cuda")
    x[1, 3], x[2, 6] = float("nan"), float("inf")
    for out in ("f32", "e4m3"):
        res = pkg.GpuRmsNorm(sampler, hidden=hidden, out=out)(x)
        v = res.out.float()
        assert v[[0, 3]].isfinite().all()
        assert v[1].isnan().all()
        assert v[2, 6].isnan()
        if out == "f32":
            assert (v[2, :6] == 0).all()
        else:
            assert res.scale[1:3].isnan().all() and res.scale[[0, 3]].isfinite().all()


def test_strided_inputs_in_place_residual_and_reused_result(pkg, sampler):
    big = torch.randn((9, 700), device="cuda").to(torch.bfloat16)
    for off, hidden in ((0, 256), (3, 250), (8, 640)):  # aligned, odd start, aligned again
        x = big[:, off:off + hidden]
        r = torch.randn((9, hidden), device="cuda").to(torch.bfloat16)
        w = torch.randn(hidden, device="cuda")
        norm = pkg.GpuRmsNorm(sampler, w, out="bf16")
        want = norm(x, r)
        check(want, x, r, w, 0.0, 1e-6, "bf16", 0, 0)
        r2 = r.clone()
        keep = pkg.RmsNormResult(torch.empty_like(want.out), residual=r2)
        got = norm(x, r2, out=keep)  # the residual stream updated where it is
        assert got is keep and torch.equal(got.out, want.out) and torch.equal(r2, want.residual)


def test_other_stream_and_graph(pkg, sampler):
    x = torch.randn((64, 1536), device="cuda").to(torch.bfloat16)
    norm = pkg.GpuRmsNorm(sampler, hidden=1536, out="e4m3")
    want = norm(x)
    keep = norm(x)
    torch.cuda.synchronize()
    keep.out.view(torch.uint8).zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        norm(x, out=keep)
    s.synchronize()
    assert torch.equal(keep.out.view(torch.uint8), want.out.view(torch.uint8))
    with torch.cuda.graph(graph):
        norm(x, out=keep)
    keep.out.view(torch.uint8).zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(keep.out.view(torch.uint8), want.out.view(torch.uint8))


def test_refusals(pkg, sampler):
    w = torch.ones(64, device="cuda")
    for bad in (dict(out="fp4"), dict(out="srq"), dict(out="bf16", srq_scale=0.5)):
        with pytest.raises(ValueError):
            pkg.GpuRmsNorm(sampler, w, **bad)
    with pytest.raises(ValueError):
        pkg.GpuRmsNorm(sampler)
    with pytest.raises(ValueError):
        pkg.GpuRmsNorm(sampler, w.half())
    x = torch.ones((2, 64), device="cuda")
    norm = pkg.GpuRmsNorm(sampler, w)
    with pytest.raises(ValueError):
        norm(x.half())
    with pytest.raises(ValueError):
        norm(x[:, :63])
    with pytest.raises(ValueError):
        norm(x, x.bfloat16())
    with pytest.raises(ValueError):
        norm(x.cpu())
    with pytest.raises(ValueError):
        norm(torch.ones((64, 2), device="cuda").T)
    with pytest.raises(ValueError):
        pkg.GpuRmsNorm(sampler, w, out="e4m3", group=48)(x)
    with pytest.raises(ValueError):
        pkg.GpuRmsNorm(sampler, w, eps=-1.0)(x)
    with pytest.raises(pkg.SamplerError):
        pkg.GpuRmsNorm(sampler, hidden=32769)(torch.ones((1, 32769), device="cuda"))
    assert norm(x[:0]).out.shape == (0, 64)
