"""GpuKvCache.write / read against the definition (the same float32 operations: equal bits)."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32)


@pytest.mark.parametrize("form", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads,page,dtype", [(1, 1, 16, "bf16"), (37, 3, 16, "f32"), (64, 4, 256, "bf16"),
                                                     (513, 5, 32, "bf16")])
def test_write_then_read(pkg, sampler, form, dim, tokens, heads, page, dtype):
    gen = torch.Generator(device="cuda").manual_seed(tokens + dim)
    pages = -(-tokens // page) + 2
    k, v, ks, vs = R.make_pool(gen, pages, heads, page, dim, form, "cuda")
    want = [t.clone() if t is not None else None for t in (k, v, ks, vs)]
    qkv = torch.randn((tokens, 3 * heads, dim), generator=gen, device="cuda")
    qkv[tokens // 2] *= 1e-3
    qkv[0, heads] = 0.0  # a row of zeros
    qkv = qkv.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    nk, nv = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].to(torch.int32)
    if tokens > 4:
        slots[3] = -1  # padding
    live = slots >= 0
    pg, at = slots[live].long() // page, slots[live].long() % page
    for pool, scale, x in ((want[0], want[2], nk), (want[1], want[3], nv)):
        if form == "bf16":
            pool[pg, :, at] = x[live].to(torch.bfloat16)
        else:
            c, s = R.quantise(x[live], form)
            bits(pool)[pg, :, at] = bits(c)
            scale[pg, :, at] = s
    cache = pkg.GpuKvCache(sampler, k, v, ks, vs)
    cache.write(nk, nv, slots)
    for got, ref in zip((k, v, ks, vs), want):
        if ref is not None:
            assert torch.equal(bits(got), bits(ref))
    for t in (torch.bfloat16, torch.float32):
        rk, rv = cache.read(slots, dtype=t)
        for got, pool, scale in ((rk, k, ks), (rv, v, vs)):
            val = pool.float() if scale is None else pool.float() * scale[..., None]
            ref = torch.zeros_like(got)
            ref[live] = val[pg, :, at].to(t)
            assert torch.equal(got, ref)
    cache.check()


@pytest.mark.parametrize("form", ["bf16", "e4m3", "int8"])
def test_strided_pools_and_unaligned_rows(pkg, sampler, form):
    """Token-major pools, keys and values interleaved in one allocation; new rows at odd offsets."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    pages, page, heads, dim, n = 5, 16, 3, 64, 40
    both = torch.zeros((pages, page, 2, heads, dim), device="cuda").to(R.TYPES[form])
    k, v = both[:, :, 0].permute(0, 2, 1, 3), both[:, :, 1].permute(0, 2, 1, 3)
    ks, vs = (torch.zeros((pages, heads, page), device="cuda") if form != "bf16" else None for _ in range(2))
    cache = pkg.GpuKvCache(sampler, k, v, ks, vs)
    raw = torch.randn((n, heads, dim + 3), generator=gen, device="cuda").to(torch.bfloat16)
    nk, nv = raw[:, :, 1:dim + 1], raw[:, :, 3:]
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n].to(torch.int32)
    cache.write(nk, nv, slots)
    out = torch.empty((n, heads, 2 * dim + 1), device="cuda")
    gk, gv = cache.read(slots, out=(out[:, :, :dim], out[:, :, dim + 1:]))
    for got, x in ((gk, nk), (gv, nv)):
        if form == "bf16":
            ref = x.float()
        else:
            c, s = R.quantise(x, form)
            ref = c.float() * s[..., None]
        assert torch.equal(got, ref)


def test_nan_rows_and_bad_slots(pkg, sampler):
    cache = pkg.GpuKvCache.allocate(sampler, 2, 2, 16, 64, "e4m3")
    x = torch.randn((4, 2, 64), device="cuda")
    x[1, 0, 5] = float("nan")
    slots = torch.tensor([0, 5, 32, -7], dtype=torch.int32, device="cuda")  # 32: past the cache
    cache.write(x, x, slots)
    with pytest.raises(ValueError, match="slot"):
        cache.check()
    cache.check()  # (cleared)
    k, _ = cache.read(slots[:2])
    assert k[0].isfinite().all() and k[1, 0].isnan().all() and k[1, 1].isfinite().all()
    assert cache.k_scale[:, :, 6:].abs().sum() == 0
    z, _ = cache.read(slots[2:])
    assert (z == 0).all()
    with pytest.raises(ValueError, match="slot"):
        cache.check()


def test_refusals(pkg, sampler):
    def pool(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, device="cuda").to(dtype)
    k = pool(2, 1, 16, 64)
    with pytest.raises(ValueError):
        pkg.GpuKvCache(sampler, k, k.float())
    with pytest.raises(ValueError):
        pkg.GpuKvCache(sampler, k, pool(2, 1, 16, 128))
    with pytest.raises(ValueError):
        pkg.GpuKvCache(sampler, k.to(torch.int8), k.to(torch.int8))
    with pytest.raises(ValueError):
        pkg.GpuKvCache(sampler, k, k, torch.zeros((2, 1, 16), device="cuda"), torch.zeros((2, 1, 16), device="cuda"))
    with pytest.raises(ValueError):
        pkg.GpuKvCache(sampler, k.cpu(), k.cpu())
    with pytest.raises(pkg.SamplerError):
        pkg.GpuKvCache(sampler, pool(2, 1, 16, 96), pool(2, 1, 16, 96))
    with pytest.raises(pkg.SamplerError):
        pkg.GpuKvCache(sampler, pool(2, 1, 24, 64), pool(2, 1, 24, 64))
    with pytest.raises(ValueError):  # rows not 16-byte aligned
        wide = pool(2, 1, 16, 68)
        pkg.GpuKvCache(sampler, wide[..., :64], wide[..., 4:])
    with pytest.raises(ValueError):
        pkg.GpuKvCache.allocate(sampler, 2, 1, 16, 64, "int4")
    c = pkg.GpuKvCache(sampler, k, k.clone())
    x = pool(3, 1, 64)
    s = torch.zeros(3, dtype=torch.int32, device="cuda")
    for a in ((x, x.float(), s), (x, x, s.long()), (x[:2], x[:2], s), (x, x, s.cpu()), (x.half(), x.half(), s)):
        with pytest.raises(ValueError):
            c.write(*a)
    with pytest.raises(ValueError):  # outputs that overlap
        c.read(s, out=(x[:1].expand(3, 1, 64), x))
    c.write(x[:0], x[:0], s[:0])
