"""GpuKvCache.attend where its masks, pools and lengths are unusual: signs of the scales, pages that are gone, values
that are not finite, contexts of few tiles, offsets out of order."""
import pytest
import torch

import operator_refs as R
from test_gpu_attention import FORMS, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,heads,group", [([(64, 2500)] * 9 + [(3, 2)], 16, 8), ([(20, 1500)] * 40, 8, 4)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_shared_items_beside_another_context(pkg, sampler, form, dim, lens, heads, group):
    """Blocks that walk several items, started late and at odd times because another context's calls hold
    their SMs: a block's warps leave an item far apart, and none may touch what another still needs of it."""
    c = Case(sampler, pkg, lens, heads, group, dim, 64, form, seed=dim)
    want, want_lse = c.run()
    assert torch.equal(c.run()[0], want)
    other = pkg.GpuSampler(0)
    beside = Case(other, pkg, [(30, 700), (1, 900), (90, 500)], 8, 4, dim, 32, form, seed=1)
    side = torch.cuda.Stream()
    outs = []
    for i in range(30):
        with torch.cuda.stream(side):
            for _ in range(1 + i % 3):
                beside.cache.attend(beside.q, beside.q_start, beside.kv_len, beside.table, max_q=beside.max_q,
                                    max_kv=beside.max_kv, scale=beside.scale)
        outs.append(c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_q=c.max_q, max_kv=c.max_kv, scale=c.scale, lse=True))
    torch.cuda.synchronize()
    c.cache.check()
    beside.cache.check()
    for out, lse in outs:
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    tokens = list(range(0, c.q.shape[0], 97))
    seq = [next(b for b in range(len(lens)) if t < c.starts[b + 1]) for t in tokens]
    ref = [R.attend(c.q[t:t + 1], [0, 1], [lens[b][1] - lens[b][0] + t - c.starts[b] + 1], c.table[b:b + 1], c.kd, c.vd,
                    c.page, c.scale, 0, 0) for t, b in zip(tokens, seq) if lens[b][1] >= lens[b][0]]
    keep = [t for t, b in zip(tokens, seq) if lens[b][1] >= lens[b][0]]
    R.check_attend(want[keep], want_lse[keep], [torch.cat(x) for x in zip(*ref)])
    beside.cache.close()
    other.close()


@pytest.mark.parametrize("lens,heads,group,bound", [([(20, 2500)] + [(20, 100)] * 79, 1, 4, 0),
                                                    ([(20, 100), (17, 250), (20, 30), (5, 5), (20, 200)], 16, 4, 16384),
                                                    ([(20, 0)] * 6, 16, 4, 16384)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_fewer_tiles_than_blocks(pkg, sampler, form, dim, lens, heads, group, bound):
    """Many items of few tokens, by their lengths or under a max_kv far above them, on the path that divides all
    items' tiles over the SMs: every row is written, and the counters of the context's workspace are zero again."""
    c = Case(sampler, pkg, lens, heads, group, dim, 64, form, seed=dim, poison=float("nan"))
    if bound:
        c.table = torch.nn.functional.pad(c.table, (0, bound // 64 - c.table.shape[1]), value=-1)
        c.max_kv = bound
    out = torch.full_like(c.q, 7.0)
    c.check(out=out)
    again, _ = c.run()
    assert torch.equal(out, again)
    # contexts cut into pieces right after, in both kernels
    Case(sampler, pkg, [(1, 9000)], 1, 2, dim, 64, form, poison=float("nan")).check()
    c.check()


@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_of_no_sequence_stay_as_they_are(pkg, sampler, dim):
    c = Case(sampler, pkg, [(20, 100)] * 5, 16, 4, dim, 64, "bf16")
    c.table = torch.nn.functional.pad(c.table, (0, 254), value=-1)
    c.q_start.zero_()
    out = torch.full_like(c.q, 7.0)
    c.run(out=out, max_kv=16384)
    assert (out == 7).all()


FEW, MANY = [(1, 300), (2, 130), (1, 17)], [(70, 300), (40, 130), (1, 17)]


@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("signs", ["negative", "mixed"])
def test_cache_scales_of_any_sign(pkg, sampler, form, dim, lens, signs):
    """The pools are the caller's: a value is code times scale, whatever the scale's sign."""
    c = Case(sampler, pkg, lens, 2, 3, dim, 16, form, seed=dim)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for pool, scale, name in ((c.cache.k, c.cache.k_scale, "kd"), (c.cache.v, c.cache.v_scale, "vd")):
        if signs == "negative":
            scale.neg_()
        else:
            scale.mul_(torch.randint(0, 2, scale.shape, generator=gen, device="cuda").float() * 2 - 1)
        setattr(c, name, R.pool_values(pool, scale))
    c.check()


def free_hidden_pages(c):
    """-1 in the table for every page of which no row of the sequence sees a token; how many there are."""
    gone = 0
    for b, (nq, n) in enumerate(c.lens):
        lo = max(0, n - nq - c.window + 1)
        for i in range(-(-n // c.page)):
            if not any(j >= lo or j < c.sinks for j in range(i * c.page, min((i + 1) * c.page, n))):
                c.table[b, i] = -1
                gone += 1
    return gone


@pytest.mark.parametrize("lens", [[(1, 700), (3, 500)], [(40, 900), (90, 700)]])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("form", FORMS)
def test_pages_behind_the_window_may_be_gone(pkg, sampler, form, page, dim, lens):
    """A server frees what no token can see any more: neither kernel looks there."""
    c = Case(sampler, pkg, lens, 2, 3, dim, page, form, seed=dim, poison=float("nan"), window=100, sinks=4)
    want, want_lse = c.run()
    assert free_hidden_pages(c) > 0
    out, lse = c.check()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("form,dim", [("bf16", 64), ("bf16", 128), ("e4m3", 64)])
def test_pages_behind_the_window_may_be_gone_from_shared_items(pkg, sampler, form, dim):
    c = Case(sampler, pkg, [(40, 2500), (30, 1900)] * 5, 16, 4, dim, 16, form, seed=dim, poison=float("nan"), window=1700, sinks=4)
    want, want_lse = c.run()
    assert free_hidden_pages(c) > 0
    out, lse = c.run()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def milliseconds(f, reps=3):
    f()
    t = []
    for _ in range(reps):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        t.append(a.elapsed_time(b))
    return min(t)


@pytest.mark.parametrize("lens,token,most", [([(1, 60000)], 0, 4), ([(300, 8000)], 0, 4), ([(6, 20000)], -1, 8),
                                             ([(300, 8000)], -1, 8)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_cost_of_a_value_that_is_not_finite(pkg, sampler, form, dim, lens, token, most):
    """An infinite value that every row sees, or only the last one: no such call takes many times the usual one's time."""
    c = Case(sampler, pkg, lens, 2, 4, dim, 64, form, seed=dim)
    call = dict(max_q=c.max_q, max_kv=c.max_kv, scale=c.scale)

    def run():
        return c.cache.attend(c.q, c.q_start, c.kv_len, c.table, **call)[0]
    want = run()
    plain = milliseconds(run)
    j = token % lens[0][1]
    pg, off = int(c.table[0, j // 64]), j % 64
    if form == "bf16":
        c.cache.v[pg, :, off, 5] = float("inf")
    else:
        c.cache.v_scale[pg, :, off] = float("inf")
    out = run()
    seen = out if token == 0 else out[-1:]
    assert not seen[..., 5].isfinite().any()
    if form == "bf16":
        seen[..., 5] = want[-seen.shape[0]:][..., 5]
        assert torch.equal(seen, want[-seen.shape[0]:])
    if token != 0:
        assert out[:-1].isfinite().all()
        err = (out[:-1].float() - want[:-1].float()).abs()
        assert (err <= 2.0 ** -7 * want[:-1].float().abs() + 2.0 ** -7 * c.vd.abs().nan_to_num(posinf=0.0).max().item()).all()
    slow = milliseconds(run)
    assert slow < most * plain, f"{plain * 1e3:.0f} -> {slow * 1e3:.0f} us"


@pytest.mark.parametrize("dim,lens,group", [(64, [(6, 130), (3, 65)], 2), (128, [(9, 300)], 5), (256, [(7, 210)], 2),
                                            (64, [(200, 260), (40, 65)], 4), (128, [(300, 500), (5, 5)], 1), (256, [(200, 300)], 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 8)])
@pytest.mark.parametrize("form", ["bf16", "e4m3"])
def test_single_elements_that_only_some_rows_see(pkg, sampler, form, dim, lens, group, window, sinks):
    """NaN elements in new tokens, at the windows' edge and in a sink that not every row has reached: they are in the
    results of the rows that see them, column by column, and in no other."""
    c = Case(sampler, pkg, lens, 2, group, dim, 16, form, seed=dim, window=window, sinks=sinks)
    clean = c.reference()
    bad = {}
    for b, (nq, n) in enumerate(lens):
        at = [n - 1, n - 1 - nq // 2] + ([max(sinks, n - nq + nq // 3 - window + 1)] if window else [])
        if nq == n:
            at.append(2)
        for i, j in enumerate(at):
            pg, off, col = int(c.table[b, j // 16]), j % 16, (7 * i + 3 * b) % dim
            c.cache.v.view(torch.int16 if form == "bf16" else torch.uint8)[pg, :, off, col] = 0x7fc0 if form == "bf16" else 0x7f
            bad.setdefault((b, j), set()).add(col)
    out, lse = c.run()
    hit = torch.zeros_like(out, dtype=torch.bool)
    for b, (nq, n) in enumerate(lens):
        for t in range(nq):
            p = n - nq + t
            for (b2, j), cols in bad.items():
                if b2 == b and j <= p and (not window or j > p - window or j < sinks):
                    hit[c.starts[b] + t, :, list(cols)] = True
    assert hit.any() and out[hit].isnan().all()
    # (the other columns are the untouched cache's, since only the elements named were changed)
    got = torch.where(hit, clean[0].to(out.dtype), out)
    R.check_attend(got, lse, clean)


@pytest.mark.parametrize("lens", [[(2, 40), (3, 50), (1, 60)], [(40, 90), (50, 200), (30, 60)],
                                  [(40, 90), (50, 2000), (30, 60)] * 20])
def test_starts_that_descend_are_reported(pkg, sampler, lens):
    c = Case(sampler, pkg, lens, 8, 2, 64, 16, "bf16")
    good, _ = c.run()
    n = c.starts[-2]
    c.q_start[-1] = n - 1  # (the last sequence: less than no tokens)
    out = torch.full_like(good, 7.0)
    c.cache.attend(c.q, c.q_start, c.kv_len, c.table, max_q=c.max_q, max_kv=c.max_kv, scale=c.scale, out=out)
    with pytest.raises(ValueError, match="outside"):
        c.cache.check()
    c.cache.check()
    assert (out[n:] == 7).all()
    tol = 2.0 ** -6 * c.vd.abs().max().item()  # (the shares of a divided call change with its tiles, and with them a bit here and there)
    assert (out[:n].float() - good[:n].float()).abs().max().item() <= tol


@pytest.mark.parametrize("lens", [[(1, 30), (2, 40)], [(70, 140), (9, 9)]])
def test_results_that_overlap_the_query_or_themselves_are_refused(pkg, sampler, lens):
    c = Case(sampler, pkg, lens, 2, 2, 64, 16, "bf16")
    want, _ = c.run()
    n = c.q.shape[0]
    buf = torch.zeros((n + 4, 12, 64), dtype=torch.bfloat16, device="cuda")
    buf[:n, :4] = c.q
    c.q = buf[:n, :4]
    flat = buf.view(-1)
    lone = torch.zeros(n * 768, dtype=torch.bfloat16, device="cuda")
    for out in (buf[1:n + 1, :4], buf[:n, 2:6], buf[:n, 0:8:2], flat[:n * 256].view(n, 4, 64),  # q's
                torch.as_strided(lone, (n, 4, 64), (64, 64, 1)), torch.as_strided(lone, (n, 4, 64), (128, 64, 1))):  # their own
        with pytest.raises(ValueError, match="must not"):
            c.run(out=out)
    for out in (buf[:n, 4:8], buf[:n, 4:12:2]):  # beside the query in its own buffer
        got, _ = c.run(out=out)
        assert torch.equal(got, want)
    by_head = torch.empty((4, n, 64), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(c.run(out=by_head)[0], want)


@pytest.mark.parametrize("lens", [FEW, MANY])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("factor", [0.0, 2.0 ** -30, 2.0 ** -126, 2.0 ** 55])
def test_cache_scales_of_any_size(pkg, sampler, form, dim, lens, factor):
    """Down to scales whose reciprocal is no float32: the result is finite, and small where the values are."""
    c = Case(sampler, pkg, lens, 2, 3, dim, 16, form, seed=dim)
    c.cache.v_scale.mul_(factor)
    c.vd = R.pool_values(c.cache.v, c.cache.v_scale)
    out, lse = c.run()
    ref = c.reference()
    assert out.isfinite().all()
    if 2.0 ** -60 < c.cache.v_scale.max().item():
        scaled = [ref[0] / factor, ref[1], ref[2] / factor, ref[3]]
        R.check_attend((out.double() / factor), lse, scaled)
    else:
        assert (out.double() - ref[0]).abs().max().item() <= 2.0 ** -80
