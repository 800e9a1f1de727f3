"""GpuKvCache.attend against the formula in float64, over masks, layouts and lengths."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, sampler, pkg, lens, heads, group, dim, page, form, seed=0, poison=None, layout="hnd", window=0,
                 sinks=0):
        """lens: (new tokens, cached tokens) per sequence.  poison: every cached value and scale
        that no row of its sequence may read."""
        gen = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for _, n in lens]
        pages = max(1, sum(need)) + 1
        k, v, ks, vs = R.make_pool(gen, pages, heads, page, dim, form, "cuda")
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        cols = max(1, max(need)) + 1
        self.table = torch.full((len(lens), cols), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.max_kv = max(1, max(n for _, n in lens))
        if poison is not None:
            seen = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
            for b, (nq, n) in enumerate(lens):
                lo = max(0, n - nq - window + 1) if window else 0
                for j in range(n):
                    if (j >= lo or j < sinks) and nq > 0:
                        seen[self.table[b, j // page].long(), j % page] = True
            hide = ~seen[:, None, :, None].expand_as(k)
            if form == "bf16":
                k.masked_fill_(hide, poison)
                v.masked_fill_(hide, poison)
            else:
                code = 0x7f if form == "e4m3" else 0x80
                k.view(torch.uint8).masked_fill_(hide, code)
                v.view(torch.uint8).masked_fill_(hide, code)
                ks.masked_fill_(hide[..., 0], poison)
                vs.masked_fill_(hide[..., 0], poison)
        if layout == "nhd":  # token-major pages
            k, v = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (k, v))
        self.kd, self.vd = R.pool_values(k, ks), R.pool_values(v, vs)
        self.cache = pkg.GpuKvCache(sampler, k, v, ks, vs)
        starts = [0]
        for nq, _ in lens:
            starts.append(starts[-1] + nq)
        self.starts, self.lens, self.page = starts, lens, page
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda")
        self.q = (1.5 * torch.randn((starts[-1], heads * group, dim), generator=gen, device="cuda")).to(torch.bfloat16)
        self.scale = dim ** -0.5
        self.window, self.sinks = window, sinks
        self.max_q = max(1, max(nq for nq, _ in lens))

    def run(self, **kw):
        a = dict(max_q=self.max_q, max_kv=self.max_kv, scale=self.scale, window=self.window, sinks=self.sinks, lse=True)
        a.update(kw)
        out, lse = self.cache.attend(self.q, self.q_start, self.kv_len, self.table, **a)
        torch.cuda.synchronize()
        self.cache.check()
        return out, lse

    def reference(self):
        return R.attend(self.q, self.starts, [n for _, n in self.lens], self.table, self.kd, self.vd, self.page,
                        self.scale, self.window, self.sinks)

    def check(self, what="", **kw):
        out, lse = self.run(**kw)
        R.check_attend(out, lse, self.reference(), what)
        return out, lse


FORMS = ["bf16", "e4m3", "int8"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 8, 16])
def test_single_tokens(pkg, sampler, form, dim, group):
    lens = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 65), (1, 200)]
    Case(sampler, pkg, lens, 2, group, dim, 16, form, seed=dim + group, poison=float("nan")).check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(5, 5), (2, 70), (1, 33), (7, 129)], [(40, 40), (33, 300)], [(130, 131), (1, 400)],
                                  [(257, 600)]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (1, 0)])
def test_chunks(pkg, sampler, form, dim, lens, window, sinks):
    Case(sampler, pkg, lens, 2, 3, dim, 32, form, seed=dim, poison=float("nan"), window=window, sinks=sinks).check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("lens", [[(1, 300), (1, 257)], [(100, 300), (30, 257)]])
def test_pages_and_layouts(pkg, sampler, page, layout, lens):
    for form in ("bf16", "int8"):
        Case(sampler, pkg, lens, 3, 2, 128, page, form, layout=layout, poison=float("inf"), window=90, sinks=5).check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("many", [False, True])
def test_rows_that_see_nothing(pkg, sampler, form, many):
    """No cached tokens; more new tokens than cached ones (the first rows stand before position 0);
    no new tokens."""
    n = 60 if many else 4
    lens = [(1, 0), (n, 0), (n, 2), (0, 20), (n, n + 1)]
    c = Case(sampler, pkg, lens, 2, 4, 64, 16, form, poison=float("nan"))
    out, lse = c.check()
    assert (out[:1 + n] == 0).all() and torch.isinf(lse[:1 + n]).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lens,window,sinks", [([(1, 5000)], 0, 0), ([(1, 4100), (1, 3)], 0, 0), ([(3, 5000)], 3000, 4),
                                               ([(20, 2500)], 0, 0)])
def test_split_context(pkg, sampler, form, lens, window, sinks):
    """Few rows and a long context: the context is split over blocks and joined."""
    Case(sampler, pkg, lens, 1, 2, 128, 64, form, poison=float("nan"), window=window, sinks=sinks).check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lens,dim", [([(1, 500), (3, 300)], 128), ([(40, 700)], 64), ([(40, 700)], 128), ([(40, 700)], 256)])
def test_large_scores_and_spread_scales(pkg, sampler, form, lens, dim):
    """Scores far apart (one token takes nearly all the weight, late in the context), and cached
    rows whose scales differ by orders of magnitude."""
    c = Case(sampler, pkg, lens, 2, 4, dim, 16, form, seed=3)
    c.scale = 1.0
    if form != "bf16":
        gen = torch.Generator(device="cuda").manual_seed(11)
        f = torch.exp2(torch.randint(-12, 5, c.cache.v_scale.shape, generator=gen, device="cuda").float())
        c.cache.v_scale.mul_(f)
        c.vd = R.pool_values(c.cache.v, c.cache.v_scale)
    c.check()


@pytest.mark.parametrize("lens", [[(1, 40), (1, 7)], [(70, 140), (9, 9)]])
def test_strided_query_and_output(pkg, sampler, lens):
    c = Case(sampler, pkg, lens, 2, 2, 64, 16, "bf16")
    want, _ = c.check()
    tokens = c.q.shape[0]
    wide = torch.zeros((tokens, 9, 64), dtype=torch.bfloat16, device="cuda")
    wide[:, 1:8:2][:, :4] = c.q
    c.q = wide[:, 1:8:2]
    buf = torch.full((tokens, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    out, _ = c.run(out=buf[:, :, 64:])
    assert torch.equal(out, want) and (buf[:, :, :64] == 7).all()


def test_decode_form_without_starts(pkg, sampler):
    c = Case(sampler, pkg, [(1, 90), (1, 20), (1, 0)], 2, 4, 128, 16, "e4m3")
    want, want_lse = c.check()
    out, lse = c.cache.attend(c.q, None, c.kv_len, c.table, max_kv=c.max_kv, scale=c.scale, lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("lens", [[(1, 700), (1, 33)], [(90, 700), (33, 33)]])
def test_same_bits_every_time_on_another_stream_and_in_a_graph(pkg, sampler, lens):
    c = Case(sampler, pkg, lens, 2, 4, 128, 16, "bf16")
    want, want_lse = c.run()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out, lse = c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_q=c.max_q, max_kv=c.max_kv, scale=c.scale, lse=True)
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    graph = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(graph):
        c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_q=c.max_q, max_kv=c.max_kv, scale=c.scale, out=out, lse_out=lse)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_gradient_of_lse_is_the_attention_output(pkg, sampler):
    """d lse / d q = scale · Σ p k: with values equal to the keys the output is that gradient
    over scale; checked against central differences of the kernel's own lse."""
    c = Case(sampler, pkg, [(1, 50)], 1, 1, 64, 16, "bf16", seed=9)
    c.cache.v.copy_(c.cache.k)
    out, _ = c.run()
    base = c.q.clone()
    step = 0.25  # exact in bf16 next to the rounded q below
    base = (base * 4).round() / 4
    c.q = base
    out, _ = c.run()
    grad = []
    for i in range(0, 64, 7):
        f = []
        for sgn in (1, -1):
            c.q = base.clone()
            c.q[0, 0, i] += sgn * step
            f.append(c.run()[1].double().item())
        grad.append((f[0] - f[1]) / (2 * step))
    got = out.double()[0, 0, ::7] * c.scale
    # third derivative of lse along one axis <= scale^3 · max|k|^3 · 2, times step^2 / 6
    kmax = c.kd.abs().max().item()
    tol = 2 * (c.scale * kmax) ** 3 * step ** 2 / 6 + 1e-4 / step + 2.0 ** -8 * c.scale * kmax
    assert (got - torch.tensor(grad, device="cuda", dtype=torch.float64)).abs().max().item() <= tol


def test_bad_table_and_lengths_are_reported(pkg, sampler):
    c = Case(sampler, pkg, [(1, 100), (1, 40)], 1, 2, 64, 16, "bf16")
    good, _ = c.run()
    kept = c.table.clone()
    c.table[1, 1] = 10 ** 6
    out, _ = c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_kv=c.max_kv, scale=c.scale)
    with pytest.raises(ValueError, match="page"):
        c.cache.check()
    assert torch.equal(out[0], good[0])
    c.cache.check()
    c.table.copy_(kept)
    c.kv_len[0] = 5000
    c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_kv=c.max_kv, scale=c.scale)
    with pytest.raises(ValueError, match="longer"):
        c.cache.check()


def test_refusals(pkg, sampler):
    c = Case(sampler, pkg, [(1, 30), (1, 30)], 2, 2, 64, 16, "bf16")
    ok = dict(q=c.q, q_start=c.q_start, kv_len=c.kv_len, page_table=c.table, max_kv=30, scale=0.1)
    bad = [dict(q=c.q.float()), dict(q=c.q[..., :32]), dict(q=c.q[:, :3]), dict(q_start=c.q_start[:2]),
           dict(kv_len=c.kv_len.long()), dict(page_table=c.table[:1]), dict(max_kv=10 ** 6), dict(max_kv=-1),
           dict(window=-1), dict(sinks=3), dict(scale=float("nan")), dict(max_q=0), dict(q=c.q[:1], q_start=None),
           dict(out=c.q.float()), dict(lse_out=torch.zeros((2, 3), device="cuda")),
           dict(q=c.q.cpu()), dict(kv_len=c.kv_len.cpu())]
    for change in bad:
        with pytest.raises(ValueError):
            c.cache.attend(**{**ok, **change})
    c.cache.attend(**ok)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,heads,window", [([(300, 900), (70, 2000), (513, 513)], 4, 0), ([(1000, 1500)], 8, 200)])
def test_many_rows_repeated(pkg, sampler, form, dim, lens, heads, window):
    """Whole grids of the many-row kernel, many times over: the same bits, and no wait that runs out."""
    c = Case(sampler, pkg, lens, heads, 2, dim, 32, form, seed=dim, window=window, sinks=2 if window else 0)
    want, want_lse = c.check()
    outs = []
    for _ in range(40):
        outs.append(c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_q=c.max_q, max_kv=c.max_kv, scale=c.scale,
                                   window=c.window, sinks=c.sinks, lse=True))
    torch.cuda.synchronize()
    c.cache.check()
    for out, lse in outs:
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,group", [([(700, 3000), (1, 1), (0, 5), (40, 0), (300, 1200)], 16, 4),
                                              ([(64, 2500)] * 9 + [(3, 2)], 16, 8), ([(512, 2049)], 20, 4),
                                              ([(64, 2500), (20, 2400)] * 5, 16, 4)])
@pytest.mark.parametrize("form", FORMS)
def test_balanced_over_items(pkg, sampler, dim, lens, heads, group, form):
    """More items than SMs: the blocks' stretches begin and end inside items, which are then joined."""
    c = Case(sampler, pkg, lens, heads, group, dim, 64, form, seed=dim, poison=float("nan"))
    out, lse = c.run()
    again, lse2 = c.run()
    # the float64 form token by token takes long at these sizes: every 37th token
    tokens = list(range(0, c.q.shape[0], 37))
    keep, starts = [], []
    for b, (nq, n) in enumerate(c.lens):
        for t in range(c.starts[b], c.starts[b + 1]):
            if t in tokens:
                keep.append((t, b, n - nq + (t - c.starts[b])))
    ref = [R.attend(c.q[t:t + 1], [0, 1], [max(p + 1, 0)], c.table[b:b + 1], c.kd, c.vd, c.page, c.scale, 0, 0) for t, b, p in keep]
    ref = [torch.cat(x) for x in zip(*ref)]
    idx = [t for t, _, _ in keep]
    R.check_attend(out[idx], lse[idx], ref)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
@pytest.mark.parametrize("dim,lens,group", [(64, [(20, 300), (3, 130), (1, 65)], 2), (128, [(9, 700), (9, 9)], 6),
                                            (256, [(7, 2100)], 2), (64, [(60, 300), (200, 260), (1, 65)], 4),
                                            (128, [(300, 900), (5, 5)], 2), (256, [(200, 500), (40, 333)], 3)])
@pytest.mark.parametrize("form", FORMS)
def test_values_that_only_some_rows_see(pkg, sampler, form, dim, lens, group, window, sinks, value):
    """An infinity or a NaN in the cached values of one new token and of one at the windows' edge: the rows that do not
    see it give the formula's finite result, the others none."""
    c = Case(sampler, pkg, lens, 2, group, dim, 16, form, seed=dim, window=window, sinks=sinks)
    bad = set()
    for b, (nq, n) in enumerate(lens):
        # from a quarter before the last new token on; up to a quarter after the first
        for j in [n - 1 - nq // 4] + ([max(sinks, n - nq + nq // 4 - window + 1)] if window else []):
            bad.add((b, j))
            pg, off = int(c.table[b, j // 16]), j % 16
            if form == "bf16":
                c.cache.v[pg, :, off, 3] = value
                c.vd[pg, :, off, 3] = value
            else:
                c.cache.v_scale[pg, :, off] = value
                c.vd[pg, :, off] = value
    out, lse = c.run()
    ref = list(c.reference())
    clean = torch.ones(out.shape[0], dtype=torch.bool, device="cuda")
    for b, (nq, n) in enumerate(lens):
        for t in range(nq):
            p = n - nq + t
            for b2, j in bad:
                if b2 == b and j <= p and (not window or j > p - window or j < sinks):
                    clean[c.starts[b] + t] = False
    assert clean.any() and not clean.all()
    R.check_attend(out[clean], lse[clean], [x[clean] for x in ref])
    assert not out[~clean][..., 3].isfinite().any()
    rest = [x[~clean].clone() for x in ref]
    if form == "bf16":  # (the token's other values are finite)
        got = out[~clean].clone()
        got[..., 3] = 0
        rest[0][..., 3] = 0
        rest[2][..., 3] = 0
        R.check_attend(got, lse[~clean], rest)
    again, lse2 = c.run()
    assert torch.equal(out[clean], again[clean]) and torch.equal(lse[clean], lse2[clean])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_balanced_join_has_one_order(pkg, sampler, dim, form):
    """Which piece of a shared item comes last changes no bit."""
    c = Case(sampler, pkg, [(64, 2500)] * 9 + [(3, 2)], 16, 8, dim, 64, form, seed=dim)
    out, lse = c.run()
    for _ in range(20):
        again, lse2 = c.run()
        assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_result_in_place_of_the_query_is_refused(pkg, sampler):
    c = Case(sampler, pkg, [(1, 30)], 2, 2, 64, 16, "bf16")
    with pytest.raises(ValueError, match="out must not be q"):
        c.run(out=c.q)


@pytest.mark.parametrize("scale", [0.0, -0.11, 2.0 ** -40])
@pytest.mark.parametrize("dim,lens", [(64, [(2, 200), (1, 3)]), (128, [(50, 300), (2, 2)]), (256, [(40, 150)])])
@pytest.mark.parametrize("form", FORMS)
def test_scales_of_any_sign(pkg, sampler, form, dim, lens, scale):
    c = Case(sampler, pkg, lens, 2, 4, dim, 16, form, seed=dim, window=90, sinks=2)
    c.scale = scale
    c.check()


@pytest.mark.parametrize("group,heads", [(1, 5), (7, 3), (33, 1), (71, 1)])
@pytest.mark.parametrize("form,dim", [("bf16", 128), ("e4m3", 64), ("int8", 256)])
def test_odd_groups(pkg, sampler, form, dim, group, heads):
    """Row blocks that begin and end inside a token's heads."""
    Case(sampler, pkg, [(1, 333), (3, 64), (11, 200)], heads, group, dim, 32, form, seed=group).check()


@pytest.mark.parametrize("lens", [[(1, 200), (1, 150), (2, 170)], [(40, 200), (33, 180)]])
def test_shared_pages(pkg, sampler, lens):
    """Sequences whose first pages are the same ones."""
    c = Case(sampler, pkg, lens, 2, 4, 128, 32, "bf16", seed=4)
    c.table[1:, :4] = c.table[0, :4]
    c.check()


@pytest.mark.parametrize("form,dim", [("bf16", 128), ("e4m3", 256)])
def test_pools_past_32_bit_offsets(pkg, sampler, form, dim):
    """Pages whose byte offsets pass 2^32 and 2^33: written, read back and attended over."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    typ = R.TYPES[form]
    page, heads = 64, 2
    per_page = heads * page * dim * torch.empty((), dtype=typ).element_size()
    pages = 2 ** 33 // per_page + 8
    k, v = (torch.empty((pages, heads, page, dim), dtype=typ, device="cuda") for _ in range(2))
    scales = [None, None] if form == "bf16" else [torch.zeros((pages, heads, page), device="cuda") for _ in range(2)]
    cache = pkg.GpuKvCache(sampler, k, v, *scales)
    low = 2 ** 32 // per_page
    table = torch.tensor([[pages - 1, 0, low, pages - 2], [low + 1, pages - 3, 1, 2]], dtype=torch.int32, device="cuda")
    lens = [(60, 250), (1, 130)]
    x = [torch.randn((256 + 256, heads, dim), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)]
    slots = (table.reshape(-1).long()[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
    cache.write(x[0], x[1], slots.to(torch.int32))
    want = x if form == "bf16" else [R.pool_values(*R.quantise(t, form)).to(torch.bfloat16) for t in x]
    for got, w in zip(cache.read(slots.to(torch.int32)), want):
        assert torch.equal(got, w)
    q = torch.randn((61, 4, dim), generator=gen, device="cuda").to(torch.bfloat16)
    for starts, rows, q_ in (([0, 60, 61], lens, q), ([0, 1, 2], [(1, 250), (1, 130)], q[:2])):
        out, lse = cache.attend(q_, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda"), table,
                                max_q=rows[0][0], max_kv=256, scale=dim ** -0.5, lse=True)
        small = table.clone()  # the same tokens in a small pool: page i of it is entry i of the table
        small[:] = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
        vals = [(t if form == "bf16" else R.pool_values(*R.quantise(t, form))).double().view(8, page, heads, dim).transpose(1, 2) for t in x]
        ref = R.attend(q_, starts, [n for _, n in rows], small, vals[0], vals[1], page, dim ** -0.5, 0, 0)
        R.check_attend(out, lse, ref)
    cache.check()
