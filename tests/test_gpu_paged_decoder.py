"""The example that runs norm, cache, attention and LM head together, against the same layers in plain torch."""
import importlib.util
import os

import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decoder.py")
    spec = importlib.util.spec_from_file_location("paged_decoder", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def norm64(x, w, eps=1e-6):
    x = x.double()
    return x * (x.square().mean(dim=1, keepdim=True) + eps).rsqrt() * w.double()


def plain(model, ids, form):
    """The stream of one sequence's tokens, all at once: norm and attention in float64, rounded to bf16 where the
    operators round, the cached rows through the cache's format."""
    h = model.embed[ids].double()
    n, qh, kh, d = len(ids), model.q_heads, model.kv_heads, model.head_dim
    i, j = torch.arange(n, device=h.device)[:, None], torch.arange(n, device=h.device)[None]
    for layer in model.layers:
        qkv = (norm64(h, layer["weights"][0]).bfloat16() @ layer["qkv"]).view(n, qh + 2 * kh, d)
        q, k, v = qkv[:, :qh].double(), qkv[:, qh:qh + kh], qkv[:, qh + kh:]
        if form != "bf16":
            k, v = (R.pool_values(*R.quantise(x, form)) for x in (k, v))
        k, v = (x.double().repeat_interleave(qh // kh, dim=1) for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
        seen = j <= i
        if layer["window"]:
            seen = seen & ((j > i - layer["window"]) | (j < layer["sinks"]))
        a = torch.einsum("hij,jhd->ihd", s.masked_fill(~seen, float("-inf")).softmax(dim=2), v).bfloat16()
        h = h + (a.reshape(n, qh * d) @ layer["out"]).double()
        gate, up = (norm64(h, layer["weights"][1]).bfloat16() @ layer["up"]).chunk(2, dim=1)
        h = h + ((torch.nn.functional.silu(gate) * up) @ layer["down"]).double()
    return h


@pytest.mark.parametrize("form", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("head_dim,q_heads,kv_heads", [(64, 8, 2), (128, 4, 1), (256, 4, 2)])
def test_decoder(example, pkg, sampler, form, head_dim, q_heads, kv_heads):
    layers = 3
    model = example.PagedDecoder(sampler, layers=layers, hidden=256, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                                 inner=512, vocab=512, format=form, pages=64, window=40, sinks=3, seed=head_dim)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 512, (n,), generator=gen).tolist() for n in (150, 1, 71, 64)]
    params = pkg.params_from_config(dict(pkg.DEFAULT_DECODING_CONFIG, temperature=0))
    streams = []
    forward = model.forward

    def record(*a):
        h, branch = forward(*a)
        streams.append((a[2], h + branch))
        return h, branch

    model.forward = record
    new = 6
    ids = example.generate(model, prompts, new, params, chunk=64)
    assert ids.shape == (len(prompts), new)
    got = [[] for _ in prompts]
    for k, (starts, h) in enumerate(streams):
        alive = [b for b, p in enumerate(prompts) if starts is None or len(p) > 64 * k]
        at = list(range(len(alive) + 1)) if starts is None else starts.tolist()
        for x, b in enumerate(alive):
            got[b].append(h[at[x]:at[x + 1]])
    for b, p in enumerate(prompts):
        h = torch.cat(got[b]).double()
        want = plain(model, p + ids[b, :new - 1].tolist(), form)
        assert h.shape == want.shape
        # per layer about eight roundings (2^-8 of a value each) differ at most: the two norms' results, q k v,
        # weights, attention, the two gates and their product; each moves its branch, which is no larger than the stream,
        # by that share, and an 8-bit code that falls the other way its value by 2^-4 (e4m3), 2^-6 (int8 of a
        # row's largest), as the root of head_dim independent errors
        flip = {"bf16": 0.0, "e4m3": 2.0 ** -4, "int8": 2.0 ** -6}[form] * head_dim ** -0.5 * 2
        tol = layers * (8 * 2.0 ** -8 + flip)
        err = (h - want).norm(dim=1) / want.norm(dim=1)
        assert err.max() <= tol, f"sequence {b}: {err.max().item():.3g} against {tol:.3g}"
        # the token that follows each is the head's best for that stream
        r = model.norm(h[len(p) - 1:].float())
        logits = model.head.logits(r.out, r.row_sum)
        assert torch.equal(logits.gather(1, ids[b].long()[:, None])[:, 0], logits.amax(dim=1))


def test_example_refuses(example, pkg, sampler):
    model = example.PagedDecoder(sampler, layers=1, hidden=256, q_heads=2, kv_heads=1, head_dim=64, inner=64, vocab=512, pages=2)
    params = pkg.params_from_config(dict(pkg.DEFAULT_DECODING_CONFIG, temperature=0))
    with pytest.raises(ValueError, match="pages"):
        example.generate(model, [[1] * 40], 2, params)
