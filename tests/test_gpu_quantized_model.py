"""The dual-stream model with its feed-forwards in 8 bits and its timestep linears
in 4, through the model's own calls."""
import copy

import pytest
import torch

from taomate_amd import dit as D
from taomate_amd import kernels, quant

from .helpers import cosine, gen, randn
from .test_gpu_dit import B, CFG, GH, GW, LA, LT, NF, _inputs, _pes, _small_arena_caches

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("L", [1, 7, 75, 300])
def test_feed_forward(dev, L):
    ff = D.FeedForward(256, 256).to(dev, BF)
    x = randn((2, L, 256), gen(L), BF).to(dev)
    with torch.no_grad():
        plain = ff(x)
        ff.quantize_()
        assert ff.quantized()
        got = ff(x)
        # e4m3 rounds a value by at most 2^-4, in the mean square under 2^-5: the rows, both
        # weights and the activation add up to less than 2 * 2^-5 of the result
        assert (got.float() - plain.float()).norm() <= 2.0 ** -4 * plain.float().norm()
        rows = kernels.adaln_mx(x, eps=None)
        assert torch.equal(ff.forward_rows(rows), got)
        odd = torch.empty(2 * L * 256 + 1, dtype=BF, device=dev)[1:].view(2, L, 256)   # 2 bytes off alignment
        odd.copy_(x)
        assert torch.equal(ff(odd), got)
        strided = torch.empty(2, L, 512, dtype=BF, device=dev)[..., ::2]
        strided.copy_(x)
        assert torch.equal(ff(strided), got) and ff(x[0, 0]).shape == (256,)
    y = ff(x.requires_grad_())             # something else would see the call: the modules run
    y.sum().backward()
    assert torch.equal(y.detach(), ff.net(x).detach()) and x.grad is not None
    with torch.no_grad():
        ff.net[2].weight.mul_(2.0)         # a changed weight: the modules run, on the new values
        z = ff(x)
        assert torch.equal(z, ff.net(x)) and not ff.quantized()


def test_hooks_are_seen(dev):
    ff = D.FeedForward(128, 128).to(dev, BF).quantize_()
    x = randn((1, 4, 128), gen(1), BF).to(dev)
    seen = []
    with torch.no_grad():
        h = ff.net[0].register_forward_hook(lambda *_: seen.append(1))
        assert torch.equal(ff(x), ff.net(x)) and len(seen) == 2
        h.remove()
        assert ff.quantized()


@pytest.mark.parametrize("rows", [1, 2, 16, 17])
def test_timestep_linears(dev, rows):
    m = D.AdaLayerNormSingle(256, 6).to(dev, BF)
    D.init_random_(m, 5)
    t = torch.rand(rows, generator=gen(rows)).to(dev) * 1000
    plain = copy.deepcopy(m)
    lins = [m.emb.timestep_embedder.linear_1, m.emb.timestep_embedder.linear_2, m.linear]
    for lin in lins:
        D._pack_group4(lin, 64)
    with torch.no_grad():
        y, e = m(t, BF)
        # the same linears on the weights that the codes stand for; 17 rows run in bf16
        if rows <= 16:
            for lin, own in zip([plain.emb.timestep_embedder.linear_1, plain.emb.timestep_embedder.linear_2, plain.linear],
                                lins):
                lin.weight.copy_(own._group4.rows.dequantize())
        py, pe = plain(t, BF)
    # the codes' values rounded to bf16 in the plain model (2^-8), the linears' results and the
    # SiLUs in both (2^-8 each), three in a row, over sums whose terms have no common sign
    assert (y.float() - py.float()).norm() <= 6 * 2.0 ** -8 * py.float().norm()
    assert (e.float() - pe.float()).norm() <= 4 * 2.0 ** -8 * pe.float().norm()


def _forward(m, dev, x, caches=None, commit=False):
    to = lambda t: t.to(dev, BF) if t.is_floating_point() else t.to(dev)  # noqa: E731
    vpe, ape, vcpe, acpe = _pes(dev)
    return m.forward_chunk(to(x["video"]), to(x["audio"]), x["sigma"].to(dev), to(x["vctx"]), to(x["actx"]),
                           x["mask"].to(dev), x["mask"].to(dev), vpe, ape, vcpe, acpe,
                           caches or m.init_kv_cache().layers, commit=commit)


@pytest.mark.parametrize("overlap", [False, True], ids=["one stream", "two streams"])
def test_model_step(dev, overlap):
    """A denoising step: quantised linears against the same weights' values in
    bf16, and against the unquantised model."""
    m = D.build_model(CFG, dev, seed=3).overlap_audio_(overlap)
    x = _inputs()
    same = copy.deepcopy(m)
    with torch.no_grad():
        base = _forward(m, dev, x)
        m.quantize_linears_(timestep=True)
        for a, b in zip(m.modules(), same.modules()):
            if isinstance(a, D.FeedForward):
                assert a.quantized()
                b.net[0].proj.weight.copy_(a._mx[0].rows.dequantize())
                b.net[2].weight.copy_(a._mx[1].rows.dequantize())
            elif isinstance(a, torch.nn.Linear) and "_group4" in a.__dict__:
                b.weight.copy_(a._group4.rows.dequantize())
        got, again, want = _forward(m, dev, x), _forward(m, dev, x), _forward(same, dev, x)
        m.quantize_linears_(False)
        back = _forward(m, dev, x)
    for i in range(2):
        assert got[i].isfinite().all() and torch.equal(got[i], again[i]) and torch.equal(back[i], base[i])
        # the same weights: the feed-forwards' activations, 2^-5 in the mean square each
        # of two roundings per feed-forward, are what differs
        assert (got[i].float() - want[i].float()).norm() <= 2.0 ** -4 * want[i].float().norm()
        assert cosine(got[i], base[i]) > 0.99


def test_model_step_runs_the_quantised_kernels(dev, monkeypatch):
    m = D.build_model(CFG, dev, seed=3).quantize_linears_(timestep=True)
    calls = []
    for name in ("adaln_mx", "mx_linear", "group4_linear"):
        fn = getattr(kernels, name)
        monkeypatch.setattr(kernels, name, lambda *a, _f=fn, _n=name, **k: (calls.append(_n), _f(*a, **k))[1])
    with torch.no_grad():
        _forward(m, dev, _inputs())
    n = CFG.num_layers
    assert calls.count("adaln_mx") == 2 * n and calls.count("mx_linear") == 4 * n and calls.count("group4_linear") == 18


def test_model_step_over_arena_caches(dev):
    """The clean commit and a step over its caches, as the streaming loop calls them."""
    m = D.build_model(CFG, dev, seed=3).fuse_qkv_().quantize_linears_(timestep=True)
    x = _inputs()
    with torch.no_grad():
        caches = _small_arena_caches(dev, CFG, x)
        _, _, caches = _forward(m, dev, x, caches, commit=True)
        v, a, _ = _forward(m, dev, x, caches)
    assert v.shape == (B, NF * GH * GW, CFG.out_channels) and a.shape == (B, LA, CFG.out_channels)
    assert v.isfinite().all() and a.isfinite().all() and LT > 0


def test_a_captured_feed_forward_follows_packing_again(dev):
    """Replays read the packed weights: the old ones after a change, the new ones once packed
    again, whatever eager calls in between allocate."""
    ff = D.FeedForward(128, 128).to(dev, BF).quantize_()
    x = randn((1, 16, 128), gen(3), BF).to(dev)
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ff(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = ff(x)
        first = ff(x).clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, first)
        ff.net[2].weight.mul_(-2.0)
        assert not ff.quantized() and torch.equal(ff(x), ff.net(x))
        junk = [torch.full((1 << n,), 255, dtype=torch.uint8, device=dev) for n in range(6, 20)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, first)
        ff.quantize_()
        second = ff(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, second) and not torch.equal(second, first) and len(junk) == 14


def test_captured_timestep_linears_follow_packing_again(dev):
    """``quantize_linears_()`` as documented after new weights: replays read the new 4-bit rows,
    whatever has been allocated since."""
    m = D.build_model(CFG, dev, seed=3).quantize_linears_(timestep=True, group=64)
    emb = m.adaln_single.emb.timestep_embedder
    x = randn((2, 256), gen(5), BF).to(dev)
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            emb(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = emb(x)
        first = emb(x).clone()
        for factor in (-2.0, 0.5):
            emb.linear_2.weight.mul_(factor)
            m.quantize_linears_()
            junk = [torch.full((1 << n,), 255, dtype=torch.uint8, device=dev) for n in range(6, 20)]
            now = emb(x)
            assert emb.linear_2._group4.holds(emb.linear_2) and not torch.equal(now, first) and len(junk) == 14
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, now)
        with pytest.raises(ValueError, match="another layout"):
            m.quantize_linears_(timestep=True, group=32)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, now)
        assert m.quantize_linears_(timestep=False).quantize_linears_(timestep=True, group=32) is m


def test_a_moved_feed_forward_frees_its_weights(dev):
    ff = D.FeedForward(512, 512).to(dev, BF)
    weights = sum(m.weight.untyped_storage().nbytes() for m in (ff.net[0].proj, ff.net[2]))
    torch.cuda.synchronize()
    ff.quantize_()
    before = torch.cuda.memory_allocated()
    ff.to("cpu")
    assert before - torch.cuda.memory_allocated() >= weights
    before = torch.cuda.memory_allocated()
    ff.quantize_(False)
    assert before - torch.cuda.memory_allocated() >= weights // 2   # the 8-bit rows


def test_more_rows_than_a_call_takes(dev):
    """2^23 rows and more run in bf16 instead of being refused; one row fewer in 8 bits."""
    ff = D.FeedForward(32, 32).to(dev, BF).quantize_()
    few = randn((16, 32), gen(9), BF).to(dev)
    rows = 1 << 23
    x = few.repeat(rows // 16, 1)
    with torch.no_grad():
        y = ff(x)
        assert y.shape == x.shape and torch.equal(y, ff.net(x))
        y = ff(x[:rows - 1])
        assert torch.equal(y[:16], ff(few)) and torch.equal(y[-15:], y[:15]) and not torch.equal(y[:16], ff.net(few))
