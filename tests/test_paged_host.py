"""What the paged cache's operators refuse, without a GPU.  Device tensors without storage stand for the operands:
the checks come before any data pointer is read, and a call that passes them ends at its missing pointer."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from taomate_amd import PagedKVCache, _native, kernels

BF = torch.bfloat16


def dev(*shape, dtype=BF):
    with FakeTensorMode():
        return torch.empty(*shape, dtype=dtype, device="cuda")


def i32(*shape):
    return dev(*shape, dtype=torch.int32)


def grow(**kw):
    a = dict(tables=i32(3, 4), lens=i32(3), new=i32(3), free=i32(9), top=i32(1), status=i32(1), block_size=16, tokens=5)
    a.update(kw)
    return kernels.kv_block_grow(**a)


def release(**kw):
    a = dict(tables=i32(3, 4), lens=i32(3), done=dev(3, dtype=torch.bool), free=i32(9), top=i32(1), status=i32(1),
             block_size=16)
    a.update(kw)
    return kernels.kv_block_release(**a)


def append(**kw):
    a = dict(k=dev(5, 2, 64), v=dev(5, 2, 64), k_pool=dev(3, 16, 2, 64), v_pool=dev(3, 16, 2, 64),
             slots=dev(5, dtype=torch.int64))
    a.update(kw)
    return kernels.kv_paged_append(**a)


def token(**kw):
    a = dict(q=dev(3, 4, 64), k_pool=dev(9, 16, 2, 64), v_pool=dev(9, 16, 2, 64), tables=i32(3, 4), lens=i32(3))
    a.update(kw)
    return kernels.paged_attn(**a)


def prompt(**kw):
    a = dict(q=dev(7, 4, 64), k=dev(7, 2, 64), v=dev(7, 2, 64), starts=i32(3))
    a.update(kw)
    return kernels.prompt_attn(**a)


@pytest.mark.parametrize("call,error,match", [
    (lambda: grow(tables=torch.zeros(3, 4, dtype=torch.int32)), ValueError, "device tensors"),
    (lambda: grow(tables=dev(3, 4, dtype=torch.int64)), TypeError, "tables must be int32"),
    (lambda: grow(tables=i32(4, 3).t()), ValueError, "contiguous rows"),
    (lambda: grow(lens=i32(2)), ValueError, "lens must hold 3"),
    (lambda: grow(new=dev(3, dtype=torch.int64)), TypeError, "new must be Int"),
    (lambda: grow(top=i32(2)), ValueError, "top must hold 1"),
    (lambda: grow(status=i32(0)), ValueError, "status must hold 1"),
    (lambda: grow(free=i32(3, 3)), ValueError, "free must be a contiguous vector"),
    (lambda: grow(tokens=-1), ValueError, "tokens"),
    (lambda: grow(lens_out=i32(4)), ValueError, "lens_out must hold 3"),
    (lambda: release(done=i32(3)), TypeError, "done must be Bool"),
    (lambda: release(lens=i32(6)[::2]), ValueError, "contiguous vector"),
    (lambda: append(k=dev(5, 2, 64, dtype=torch.float16)), TypeError, "k must be bf16"),
    (lambda: append(v=dev(5, 3, 64)), ValueError, "for pools"),
    (lambda: append(k_pool=dev(3, 16, 2, 64, dtype=torch.float32)), TypeError, "bf16 or e4m3"),
    (lambda: append(v_pool=dev(4, 16, 2, 64)), ValueError, "share shape and dtype"),
    (lambda: append(k_scales=dev(3, 16, 2, dtype=torch.float32)), ValueError, "bf16 pools have no scales"),
    (lambda: append(k_pool=dev(3, 16, 2, 64, dtype=torch.uint8), v_pool=dev(3, 16, 2, 64, dtype=torch.uint8)),
     ValueError, "need float32 scales"),
    (lambda: append(slots=i32(5)), TypeError, "slots must be Long"),
    (lambda: append(slots=dev(4, dtype=torch.int64)), ValueError, "slots must hold 5"),
    (lambda: token(q=dev(3, 3, 64)), ValueError, "multiple of the key heads"),
    (lambda: token(q=dev(2, 4, 64)), ValueError, "for pools"),
    (lambda: token(q=dev(3, 4, 128)), ValueError, "for pools"),
    (lambda: token(lens=dev(3, dtype=torch.int64)), TypeError, "lens must be Int"),
    (lambda: token(lse=dev(4, 3, dtype=torch.float32)), ValueError, "lse"),
    (lambda: token(out=dev(3, 4, 64, dtype=torch.float32)), TypeError, "out must be bf16"),
    (lambda: token(out=dev(3, 4, 32)), ValueError, "out"),
    (lambda: token(k_pool=dev(9, 16, 64, 2).transpose(2, 3)), ValueError, "contiguous D"),
    (lambda: prompt(k=dev(7, 3, 64)), ValueError, "multiple of the key heads"),
    (lambda: prompt(starts=i32(0)), ValueError, "one more value"),
    (lambda: prompt(k_starts=i32(4)), ValueError, "k_starts must hold 3"),
    (lambda: prompt(q=dev(7, 64, 4).transpose(1, 2)), ValueError, "contiguous D"),
    (lambda: prompt(lse=dev(7, 4, dtype=torch.float32)), ValueError, "lse"),
    (lambda: prompt(out=dev(7, 1, 64).expand(7, 4, 64)), ValueError, "rows of out overlap"),
    (lambda: prompt(out=dev(7 * 4 * 64).as_strided((7, 4, 64), (64, 64, 1))), ValueError, "rows of out overlap"),
    (lambda: token(out=dev(1, 4, 64).expand(3, 4, 64)), ValueError, "rows of out overlap"),
    (lambda: append(k_pool=dev(1, 16, 2, 64).expand(3, 16, 2, 64)), ValueError, "rows of a pool overlap"),
    (lambda: append(v_pool=dev(3 * 16 * 2 * 64).as_strided((3, 16, 2, 64), (1024, 64, 512, 1))), ValueError,
     "rows of a pool overlap"),
    (lambda: prompt(q=dev(7, 4, 64).requires_grad_()), RuntimeError, "computes no gradients"),
    (lambda: token(k_pool=dev(9, 16, 2, 64).requires_grad_()), RuntimeError, "computes no gradients"),
    (lambda: append(k=dev(5, 2, 64).requires_grad_()), RuntimeError, "computes no gradients"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


P = 1 << 20   # an address that no refused call reads


def raw(name, **kw):
    sig = {
        "ltx_kv_block_grow": dict(B=1, width=4, block=16, tables=P, t_bs=4, lens=P, fresh=P, free=P, n_free=9, top=P,
                                  status=P, tokens=5, lens_out=P, top_out=P, starts=P, slots=P, positions=P, stream=None),
        "ltx_paged_attn": dict(kv=1, B=1, Hk=1, G=1, D=64, q=P, q_bs=64, q_hs=64, k=P, k_ps=1024, k_ts=64, k_hs=64, v=P,
                               v_ps=1024, v_ts=64, v_hs=64, ks=None, vs=None, sc_ps=0, sc_hs=0, n=9, block=16, tables=P,
                               t_bs=4, width=4, lens=P, out=P, o_bs=64, o_hs=64, lse=None, scale=0.0, ws=None, wsb=0,
                               stream=None),
        "ltx_prompt_attn": dict(B=1, Tq=8, Tk=8, Hk=1, G=1, D=64, q=P, q_ls=64, q_hs=64, k=P, k_ls=64, k_hs=64, v=P,
                                v_ls=64, v_hs=64, qs=P, ks=P, causal=1, out=P, o_ls=64, o_hs=64, zt=0, lse=None,
                                scale=0.0, ws=None, wsb=0, stream=None),
        "ltx_kv_paged_append": dict(kv=1, T=4, H=1, D=64, k=P, k_ls=64, k_hs=64, v=P, v_ls=64, v_hs=64, kp=P, kp_ps=1024,
                                    kp_ts=64, kp_hs=64, vp=P, vp_ps=1024, vp_ts=64, vp_hs=64, ks=None, a=0, b=0, c=0,
                                    vs=None, d=0, e=0, f=0, n=9, block=16, slots=P, stream=None),
    }[name]
    assert set(kw) <= set(sig)
    return _native.call(name, *{**sig, **kw}.values())


@pytest.mark.parametrize("name,kw,match", [
    ("ltx_kv_block_grow", dict(block=24), "block of 24"), ("ltx_kv_block_grow", dict(block=8), "block of 8"),
    ("ltx_kv_block_grow", dict(B=4097), "at most 4096"), ("ltx_kv_block_grow", dict(width=1 << 28), "2\\^31"),
    ("ltx_kv_block_grow", dict(B=2, t_bs=3), "rows overlap"), ("ltx_kv_block_grow", dict(top=None), "null"),
    ("ltx_paged_attn", dict(D=96), "head layout"), ("ltx_paged_attn", dict(block=512), "block of 512"),
    ("ltx_paged_attn", dict(n=0), "at least one block"), ("ltx_paged_attn", dict(width=0), "table row"),
    ("ltx_paged_attn", dict(width=1 << 27), "table row"), ("ltx_paged_attn", dict(q=P + 8), "16-byte"),
    ("ltx_paged_attn", dict(k_ts=68), "16-byte"), ("ltx_paged_attn", dict(kv=2), "null"),
    ("ltx_paged_attn", dict(kv=2, ks=P + 4, vs=P), "scales"), ("ltx_paged_attn", dict(width=4096), "workspace"),
    ("ltx_paged_attn", dict(kv=0), "bf16 or e4m3"), ("ltx_paged_attn", dict(k_ts=-64), "token stride"),
    ("ltx_prompt_attn", dict(D=32), "head layout"), ("ltx_prompt_attn", dict(v_ls=60), "16-byte"),
    ("ltx_prompt_attn", dict(k_ls=32), "overlap"), ("ltx_prompt_attn", dict(v_ls=1 << 24), "too far"),
    ("ltx_prompt_attn", dict(B=5000), "at most 4096"),
    ("ltx_prompt_attn", dict(Tq=1 << 30, G=64), "one launch"), ("ltx_kv_paged_append", dict(T=1 << 40), "too many tokens"), ("ltx_prompt_attn", dict(Tq=1 << 31), "2\\^30"),
    ("ltx_prompt_attn", dict(k=None), "null"), ("ltx_prompt_attn", dict(Tk=1024), "workspace"), ("ltx_prompt_attn", dict(out=P + 8), "16-byte"),
    ("ltx_kv_paged_append", dict(D=256), "D 64 or 128"), ("ltx_kv_paged_append", dict(block=0), "block of 0"),
    ("ltx_kv_paged_append", dict(kp_ts=66), "pools"), ("ltx_kv_paged_append", dict(k=P + 4), "rows of k and v"),
    ("ltx_kv_paged_append", dict(kv=2), "null"),
])
def test_refusals_of_the_library(name, kw, match):
    with pytest.raises(_native.NativeCallError, match=match):
        raw(name, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(dim_head=32), "dim_head"), (dict(block_size=24), "block_size"), (dict(kv_dtype="fp16"), "kv_dtype"),
    (dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(blocks=0), "positive"),
    (dict(max_tokens=0), "positive"),
])
def test_cache_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        PagedKVCache(**{**dict(layers=1, requests=2, blocks=4, heads=1, dim_head=64, max_tokens=64, device="cpu"), **kw})


def test_cache_layout():
    c = PagedKVCache(layers=3, requests=2, blocks=5, heads=2, dim_head=64, max_tokens=100, block_size=32, kv_dtype="fp8",
                     device="cpu")
    k, v, ks, vs = c.pool(1)
    assert k.shape == v.shape == (5, 32, 2, 64) and ks.shape == vs.shape == (5, 32, 2)
    assert k.stride() == (2 * 32 * 64, 64, 32 * 64, 1) and ks.stride() == (64, 1, 32)
    assert k.data_ptr() + 5 * 2 * 32 * 64 == v.data_ptr() and c.tables.shape == (2, 4)
    assert sorted(c.free.tolist()) == list(range(5)) and c.top.item() == 5
    with pytest.raises(ValueError, match="device tensors"):
        c.grow([1, 2], 3)


def test_workspace_of_the_split():
    n = ctypes.c_int64()
    size = lambda *a: (_native.call("ltx_paged_attn_workspace_size", *a, ctypes.byref(n)), n.value)[1]  # noqa: E731
    part = 2 * 4 * 130 * 4
    assert size(64, 8, 4, 128, 64, 16) == 0                  # tables of 1024 tokens: a workgroup a request
    assert size(64, 8, 4, 128, 65, 16) == 64 * (8 * part + 16)
    assert size(8, 8, 4, 128, 32, 16) == 0                   # 512 tokens of a few requests
    assert size(8, 8, 4, 128, 33, 16) == 32 * (8 * part + 16)
    assert size(1, 8, 4, 128, 65, 16) == 9 * (8 * part + 16)
    assert size(1, 600, 1, 128, 65, 16) == 0                 # heads enough
    rows = lambda *a: (_native.call("ltx_prompt_attn_workspace_size", *a, ctypes.byref(n)), n.value)[1]  # noqa: E731
    part = 128 * 130 * 4
    assert rows(1, 128, 767, 8, 4, 128) == 0                 # too few keys to share
    assert rows(1, 128, 768, 8, 4, 128) == 32 * 16 * part
    assert rows(2, 128, 1535, 8, 4, 128) == 0 and rows(8, 1024, 16384, 8, 4, 128) == 0
    assert rows(1, 512, 2047, 8, 4, 128) == 0 and rows(1, 512, 2048, 8, 4, 128) == 128 * 4 * part
    assert rows(1, 1024, 8192, 8, 4, 128) == 0               # half of the resident workgroups
    # up to 32 rows a prompt
    assert rows(4, 128, 1023, 8, 4, 128) == 0 and rows(4, 128, 1024, 8, 4, 128) == 128 * 4 * part
    assert rows(8, 8, 2048, 8, 4, 128) == 256 * 2 * part and rows(9, 9, 4096, 8, 4, 128) == 0
    assert rows(2, 64, 767, 8, 4, 128) == 0 and rows(2, 64, 768, 8, 4, 128) == 64 * 8 * part


@pytest.mark.parametrize("call", [token, prompt])
@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e39, 3e38, 1e-60])
def test_scales_that_are_no_positive_float32_are_refused(call, scale):
    with pytest.raises(ValueError, match="scale must be a finite float32 above 0"):
        call(scale=scale)


@pytest.mark.parametrize("call", [grow, release])
@pytest.mark.parametrize("kw", [dict(lens_out=i32(2, 2, 2, 2, 2, 2)), dict(top_out=i32(2, 2, 2, 2, 2, 2)),
                                dict(lens_out=i32(3), top_out=i32(2, 2, 2, 2, 2, 2))])
def test_results_of_table_calls_are_vectors(call, kw):
    with pytest.raises(ValueError, match="_out must be a contiguous vector"):
        call(**kw)
