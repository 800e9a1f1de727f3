"""Plain float64 forms of the norm, the key/value cache and its attention, and the bounds
their float32 / bf16 / 8-bit results are held to."""
import math

import torch

TINY = 2.0 ** -64
MOST = {"e4m3": 448.0, "int8": 127.0}
TYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def quantise(x, form):
    """Codes and scales over the last axis with the float32 operations of the definition."""
    x = x.float()
    a = x.abs().amax(dim=-1, keepdim=True)
    a = torch.where(a < TINY, torch.full_like(a, TINY), a)  # (keeps a NaN)
    most = torch.full_like(a, MOST[form])  # (a quotient of tensors: torch turns one by a number into a product)
    z = x * (most / a)
    codes = z.to(torch.float8_e4m3fn) if form == "e4m3" else z.round().to(torch.int8)
    return codes, (a / most).squeeze(-1)


def make_pool(gen, pages, heads, page, dim, form, dev, fill=None):
    """(k, v, k_scale, v_scale) of random contents; ``fill``: start from this value instead."""
    out, scales = [], []
    for _ in range(2):
        x = torch.randn((pages, heads, page, dim), generator=gen, device=dev, dtype=torch.float32)
        if form == "bf16":
            out.append(x.to(torch.bfloat16))
            scales.append(None)
        else:
            c, s = quantise(x * (0.2 + torch.rand((pages, heads, page, 1), generator=gen, device=dev)), form)
            out.append(c)
            scales.append(s.contiguous())
    return out[0], out[1], scales[0], scales[1]


def pool_values(pool, scale):
    x = pool.double() if pool.dtype != torch.float8_e4m3fn else pool.float().double()
    return x if scale is None else x * scale.double()[..., None]


def attend(q, q_start, kv_len, table, k, v, page, scale, window, sinks):
    """float64 (out, lse, sum of weights times |v|, largest sum of |q k| products per row).
    k, v: pool values [pages, heads, page, dim] float64; hidden tokens are left out of every sum."""
    tokens, hq, dim = q.shape
    heads = k.shape[1]
    group = hq // heads
    dev = q.device
    out = torch.zeros((tokens, hq, dim), dtype=torch.float64, device=dev)
    absum = torch.zeros_like(out)
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64, device=dev)
    mag = torch.zeros((tokens, hq), dtype=torch.float64, device=dev)
    for b in range(len(kv_len)):
        n, t0, t1 = kv_len[b], q_start[b], q_start[b + 1]
        for t in range(t0, t1):
            p = n - (t1 - t0) + (t - t0)
            js = [j for j in range(n) if j <= p and (not window or j > p - window or j < sinks)]
            if not js:
                continue
            j = torch.tensor(js, device=dev)
            pg = table[b].to(torch.int64)[j // page]
            for h in range(heads):
                kk, vv = k[pg, h, j % page], v[pg, h, j % page]
                qq = q[t, h * group:(h + 1) * group].double()
                s = qq @ kk.T * scale
                w = torch.softmax(s, dim=1)
                sl = slice(h * group, (h + 1) * group)
                out[t, sl] = w @ vv
                absum[t, sl] = w @ vv.abs()
                lse[t, sl] = torch.logsumexp(s, dim=1)
                mag[t, sl] = (qq.abs() @ kk.abs().T * abs(scale)).amax(dim=1)
    return out, lse, absum, mag


def check_attend(got, got_lse, ref, what=""):
    """out: the weights and the result are each rounded once to bf16 (8 significand bits: 2^-8), and the
    float32 scores' error moves a weight by less than 2^-13; lse: float32 accumulation of at most
    dim + 8 products (2^-24 of their magnitudes each), the approximate 2^x and log (2^-21)."""
    out, lse, absum, mag = ref
    dim = out.shape[-1]
    err = (got.double() - out).abs()
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -13) * absum + 2.0 ** -20
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: out off by {(err / tol).max().item():.3g} of its bound at {bad.nonzero()[0].tolist()}"
    if got_lse is not None:
        empty = torch.isinf(lse)
        assert torch.equal(empty, torch.isinf(got_lse) & (got_lse < 0)), f"{what}: rows that see nothing"
        tol = 2.0 ** -21 + (dim + 8) * 2.0 ** -24 * mag + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)
        err = (got_lse.double() - lse).abs()
        bad = ~((err <= tol) | empty)
        assert not bad.any(), f"{what}: lse off by {err[bad].max().item():.3g}"
