"""Block tables, paged append, attention over prompts and of single tokens, against float64 and plain loops."""
import math
import random

import pytest
import torch

from taomate_amd import KVArenaFull, PagedKVCache, kernels
from taomate_amd import _native as N

from .paged_reference import (BF, E4, Cache, assert_attention_close, assert_lse_close, grow_reference, ints,
                              prompt_reference, starts_of)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ tables
def _table_state(dev, lens, block, width, blocks, seed=0):
    rng = random.Random(seed)
    ids = list(range(blocks))
    rng.shuffle(ids)
    tables, at = [], 0
    for n in lens:
        held = -(-n // block)
        tables.append(ids[at:at + held] + [-9] * (width - held))
        at += held
    free = ids[at:] + [0] * at
    top = blocks - at
    return tables, free, top


@pytest.mark.parametrize("B,hi,new_hi,block,pad,in_place", [
    (1, 0, 1, 16, 0, False), (1, 100, 5000, 16, 3, True), (7, 40, 60, 16, 11, False), (64, 500, 1, 32, 0, True),
    (300, 300, 90, 64, 100, False), (300, 300, 90, 64, 100, True), (1025, 70, 3, 128, 5, False), (4096, 20, 2, 256, 0, True),
    (5, 0, 0, 16, 4, False),
])
def test_grow(dev, B, hi, new_hi, block, pad, in_place):
    rng = random.Random(B)
    lens = [rng.randint(0, hi) for _ in range(B)]
    new = [rng.randint(0, new_hi) for _ in range(B)]
    width = max(-(-(a + b) // block) for a, b in zip(lens, new)) + 1
    blocks = sum(-(-(a + b) // block) for a, b in zip(lens, new)) + 2
    tables, free, top = _table_state(dev, lens, block, width, blocks)
    T = sum(new) + pad
    want = grow_reference(tables, lens, new, free, top, block, T)
    t, le, fr, tp = ints(tables, dev), ints(lens, dev), ints(free, dev), ints([top], dev)
    status = ints([0], dev)
    plan = kernels.kv_block_grow(t, le, ints(new, dev), fr, tp, status, block, T, le if in_place else None,
                                 tp if in_place else None)
    assert status.item() == 0
    assert t.tolist() == want[0] and plan.slots.tolist() == want[1] and plan.positions.tolist() == want[2]
    assert plan.starts.tolist() == want[3] and plan.lens.tolist() == want[4] and plan.top.tolist() == [want[5]]
    assert fr.tolist() == free
    assert (le.tolist(), tp.tolist()) == ((want[4], [want[5]]) if in_place else (lens, [top]))


@pytest.mark.parametrize("why,code", [("free", N.BLOCKS_FREE), ("width", N.BLOCKS_WIDTH), ("tokens", N.BLOCKS_TOKENS),
                                      ("new", N.BLOCKS_LENGTH), ("len", N.BLOCKS_LENGTH), ("top", N.BLOCKS_FREE)])
@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_grow_that_does_not_fit_gives_nothing(dev, why, code, big, in_place):
    block, lens, new = 16, [5, 0, 33, 16], [20, 3000 if big else 1, 0, 1]
    T = sum(new)
    width, blocks = 200, 250
    tables, free, top = _table_state(dev, lens, block, width, blocks)
    if why == "free":
        top = 2
    if why == "top":
        top = blocks + 1
    if why == "width":
        width = 2 if not big else 100
        tables = [r[:width] for r in tables]
        lens = [5, 0, 30 if not big else 33, 16]
    if why == "tokens":
        T -= 1
    if why == "new":
        new[2] = -1
    if why == "len":
        lens[3] = -5
    if why == "width" and not big:
        new[0] = 30
        T = sum(new)
    t, le, tp, status = ints(tables, dev), ints(lens, dev), ints([top], dev), ints([0], dev)
    plan = kernels.kv_block_grow(t, le, ints(new, dev), ints(free, dev), tp, status, block, T, le if in_place else None,
                                 tp if in_place else None)
    assert status.item() & code
    assert t.tolist() == tables and plan.lens.tolist() == lens and plan.top.tolist() == [top]
    assert plan.starts.tolist() == [0] * 5 and plan.slots.tolist() == [-1] * T and plan.positions.tolist() == [0] * T


def test_tables_in_wide_rows_lie_apart_from_the_other_operands(dev):
    memory = torch.zeros(8, 100, dtype=torch.int32, device=dev)
    inside = memory[7, 4:]   # behind the first 8 * 20 elements, within the last row's
    new, free, top, status = ints([0] * 8, dev), ints([0, 1], dev), ints([2], dev), ints([0], dev)
    done = torch.zeros(8, dtype=torch.bool, device=dev)
    for lens, stack in ((inside[:8], free), (ints([0] * 8, dev), inside[:2])):
        with pytest.raises(ValueError, match="overlaps"):
            kernels.kv_block_grow(memory[:, :20], lens, new, stack, top, status, 16, 4)
    with pytest.raises(ValueError, match="free overlaps"):
        kernels.kv_block_release(memory[:, :20], new, done, inside[:2], top, status, 16)
    assert int(memory.abs().sum()) == 0 and status.item() == 0


@pytest.mark.parametrize("B,hi,block,in_place", [(1, 30, 16, False), (9, 100, 16, True), (513, 4000, 16, False),
                                                 (513, 4000, 16, True), (3, 0, 32, False)])
def test_release(dev, B, hi, block, in_place):
    rng = random.Random(B)
    lens = [rng.randint(0, hi) for _ in range(B)]
    width = max(1, max(-(-n // block) for n in lens))
    blocks = sum(-(-n // block) for n in lens) + 4
    tables, free, top = _table_state(dev, lens, block, width, blocks)
    done = [rng.random() < 0.5 for _ in range(B)]
    want_free, want_top = list(free), top
    for b in range(B):
        for j in range(-(-lens[b] // block) if done[b] else 0):
            want_free[want_top] = tables[b][j]
            want_top += 1
    t, le, fr, tp, status = ints(tables, dev), ints(lens, dev), ints(free, dev), ints([top], dev), ints([0], dev)
    out, top_out = kernels.kv_block_release(t, le, torch.tensor(done, device=dev), fr, tp, status, block,
                                            le if in_place else None, tp if in_place else None)
    assert status.item() == 0 and fr.tolist() == want_free and top_out.tolist() == [want_top]
    assert out.tolist() == [0 if d else n for n, d in zip(lens, done)] and t.tolist() == tables


def test_release_of_more_than_the_stack_holds(dev):
    t, le = ints([[0, 1], [2, 3]], dev), ints([32, 20], dev)
    fr, status = ints([0, 1, 2, 3], dev), ints([0], dev)
    out, top = kernels.kv_block_release(t, le, torch.tensor([True, True], device=dev), fr, ints([1], dev), status, 16)
    assert status.item() == N.BLOCKS_FREE and out.tolist() == [32, 20] and top.tolist() == [1]
    assert fr.tolist() == [0, 1, 2, 3]


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("T,Hk,D,block,kv,layout", [
    (1, 1, 64, 16, "bf16", "heads"), (77, 8, 128, 16, "bf16", "tokens"), (77, 8, 128, 16, "fp8", "heads"),
    (130, 3, 64, 32, "fp8", "tokens"), (500, 2, 128, 256, "bf16", "heads"), (0, 2, 64, 16, "bf16", "heads"),
])
def test_append(dev, T, Hk, D, block, kv, layout):
    g = torch.Generator().manual_seed(T)
    c = Cache([max(T, 1)], Hk, D, block, kv, dev, layout=layout)
    x = (torch.randn(T, 2 * Hk, D, generator=g) * 3).to(BF).to(dev)
    k, v = x[:, :Hk], x[:, Hk:]                       # strided rows of one projection
    slots = torch.randperm(c.n * block, generator=g)[:T].to(dev)
    if T > 10:
        slots[3], slots[7] = -1, c.n * block          # no slot; past the pool
        k[5] = 0.0
    pools = [c.k.clone(), c.v.clone()]
    scales = [None if s is None else s.clone() for s in (c.k_scales, c.v_scales)]
    kernels.kv_paged_append(k, v, c.k, c.v, slots, c.k_scales, c.v_scales)
    ok = (slots >= 0) & (slots < c.n * block)
    i, o = slots[ok] // block, slots[ok] % block
    for src, pool, sc, got, got_sc in ((k, pools[0], scales[0], c.k, c.k_scales), (v, pools[1], scales[1], c.v, c.v_scales)):
        x = src[ok]
        if kv == "bf16":
            pool[i, o] = x
            assert torch.equal(got, pool)
            continue
        # float32 quotients by way of float64, whose double rounding is harmless (53 >= 2 * 24 + 2 bits); torch
        # divides by a number as a product with its rounded reciprocal
        top = x.double().abs().amax(-1)
        s = torch.where(top > 0, top / 448, torch.ones_like(top)).float()
        pool.view(torch.uint8)[i, o] = (x.double() / s.double()[..., None]).float().to(E4).view(torch.uint8)
        sc[i, o] = s
        assert torch.equal(got_sc, sc) and torch.equal(got.view(torch.uint8), pool.view(torch.uint8))


def test_append_refuses_one_memory_for_both(dev):
    c = Cache([16], 1, 64, 16, "bf16", dev)
    x = torch.zeros(1, 1, 64, dtype=BF, device=dev)
    with pytest.raises(ValueError, match="same memory"):
        kernels.kv_paged_append(x, x, c.k, c.k, torch.zeros(1, dtype=torch.int64, device=dev))


def test_append_refuses_one_memory_for_both_scales(dev):
    c = Cache([16], 1, 64, 16, "fp8", dev)
    x = torch.zeros(1, 1, 64, dtype=BF, device=dev)
    with pytest.raises(ValueError, match="k_scales and v_scales are the same memory"):
        kernels.kv_paged_append(x, x, c.k, c.v, torch.zeros(1, dtype=torch.int64, device=dev), c.k_scales, c.k_scales)


def test_results_in_the_queries_memory(dev):
    """out may be q itself, whole and shared among workgroups."""
    c = Cache([300, 0, 2000], 2, 64, 16, "bf16", dev)
    q = torch.randn(3, 4, 64, device=dev).to(BF)
    want = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t)
    kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, out=q)
    assert torch.equal(q, want)
    for rows, keys in (([200, 50], [200, 50]), ([40], [3000])):
        q = torch.randn(sum(rows), 4, 64, device=dev).to(BF)
        k = torch.randn(sum(keys), 2, 64, device=dev).to(BF)
        want = kernels.prompt_attn(q, k, k, starts_of(rows, dev), starts_of(keys, dev))
        kernels.prompt_attn(q, k, k, starts_of(rows, dev), starts_of(keys, dev), out=q)
        assert torch.equal(q, want)


def test_append_of_values_that_are_not_finite(dev):
    c = Cache([16], 1, 64, 16, "fp8", dev)
    k = torch.ones(2, 1, 64, dtype=BF, device=dev)
    k[0, 0, 3], k[0, 0, 4], k[1] = math.inf, math.nan, math.nan
    kernels.kv_paged_append(k, k, c.k, c.v, torch.tensor([1, 2], device=dev), c.k_scales, c.v_scales)
    got = c.k.view(torch.uint8)[0, 1:3, 0].view(E4).float()
    assert got[0].isnan().nonzero().flatten().tolist() == [3, 4] and (got[0][[0, 63]] == 448).all()
    assert got[1].isnan().all() and c.k_scales[0, 1:3, 0].tolist() == [torch.tensor(1 / 448, dtype=torch.float32).item(), 1.0]


def test_append_of_tiny_and_large_rows(dev):
    """Maxima from the smallest bf16 to its largest: scales as far as float32 goes, codes of the exact quotients."""
    powers = torch.tensor([-133, -126, -110, -97, -96, -95, -20, 0, 60, 119], dtype=torch.float64)
    x = (torch.randn(10, 1, 64, generator=torch.Generator().manual_seed(1)).double() * 2.0 ** powers[:, None, None])
    x = x.to(BF).to(dev)
    c = Cache([16], 1, 64, 16, "fp8", dev, spare=0)
    kernels.kv_paged_append(x, x, c.k, c.v, torch.arange(10, device=dev), c.k_scales, c.v_scales)
    top = x.double().abs().amax(-1)
    s = torch.where(top > 0, top / 448, torch.ones_like(top)).float()
    want = (x.double() / s.double()[..., None]).float().to(E4)
    for pool, scales in ((c.k, c.k_scales), (c.v, c.v_scales)):
        assert torch.equal(scales[0, :10], s)
        assert torch.equal(pool.view(torch.uint8)[0, :10], want.view(torch.uint8))


# ------------------------------------------------------------------ prompts
PROMPTS = [
    # rows, keys, heads, key heads, D
    ([1], [1], 1, 1, 64), ([1], [300], 4, 2, 128), ([77], [77], 8, 8, 64), ([128], [128], 2, 1, 128),
    ([129, 1, 0, 64], [129, 1, 0, 64], 6, 2, 128), ([5, 200, 63, 65], [105, 200, 64, 1000], 4, 4, 64),
    ([300], [300], 7, 1, 64), ([40, 130], [20, 100], 4, 2, 128), ([10, 10], [0, 5], 2, 2, 64),
    ([257] * 5, [257] * 5, 16, 2, 128), ([1] * 70, list(range(70)), 3, 3, 64), ([640], [640], 24, 8, 128),
    ([300, 20, 700, 0, 128, 129, 1, 555], [300, 520, 700, 3, 128, 100, 1, 600], 32, 4, 64),
    # few rows over many keys: shared among workgroups
    ([5], [3100], 8, 2, 128), ([130, 1], [2500, 4000], 4, 4, 64), ([60], [1100], 3, 1, 128),
    ([1, 2, 3], [20, 9000, 1], 2, 1, 64), ([300, 10, 0], [200, 4500, 70], 2, 2, 128),
    ([8, 0, 3, 1], [900, 0, 30, 400], 8, 1, 64),
    ([1, 0, 3, 2] * 250, [5, 2, 3, 1] * 250, 1, 1, 64),
]


@pytest.mark.parametrize("rows,keys,H,Hk,D", PROMPTS)
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(dev, rows, keys, H, Hk, D, causal):
    g = torch.Generator().manual_seed(sum(rows))
    q = (torch.randn(sum(rows), H, D, generator=g) * 1.5).to(BF).to(dev)
    k, v = (torch.randn(sum(keys), Hk, D, generator=g).to(BF).to(dev) for _ in range(2))
    ref, mag, lse_ref = prompt_reference(q, k, v, rows, keys, causal)
    lse = torch.empty(H, sum(rows), device=dev)
    out = kernels.prompt_attn(q, k, v, starts_of(rows, dev), starts_of(keys, dev), causal=causal, lse=lse)
    assert_attention_close(out, ref, mag)
    assert_lse_close(lse, lse_ref)


def test_prompt_rows_of_a_packed_projection_and_the_rows_behind(dev):
    """q, k, v as columns of one [T, (H + 2 Hk) D] projection; 50 rows behind the prompts; out strided."""
    H, Hk, D, rows, T = 4, 2, 128, [70, 190], 310
    g = torch.Generator().manual_seed(3)
    x = torch.randn(T, H + 2 * Hk, D, generator=g).to(BF).to(dev)
    x[260:] = math.nan
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    ref, mag, _ = prompt_reference(q[:260], k[:260], v[:260], rows, rows, True)
    starts = starts_of(rows, dev)
    out = kernels.prompt_attn(q, k, v, starts)
    assert_attention_close(out[:260], ref, mag)
    assert (out[260:] == 0).all()
    wide = torch.full((T, H, 2 * D), 7.0, dtype=BF, device=dev)
    lse = torch.full((H, T), 5.0, device=dev)
    assert kernels.prompt_attn(q, k, v, starts, out=wide[..., :D], lse=lse).data_ptr() == wide.data_ptr()
    assert torch.equal(wide[:260, :, :D], out[:260]) and (wide[260:] == 7).all() and (wide[..., D:] == 7).all()
    assert (lse[:, 260:] == 5).all()


def test_prompt_keys_that_are_not_finite_and_lowest_scores(dev):
    """K of a later key, and K and V of another prompt and behind the last, hold NaN and infinities; scores of
    the first tiles are the lowest that float32 takes."""
    D, rows = 64, [200, 100]
    g = torch.Generator().manual_seed(4)
    q = torch.ones(300, 1, D, dtype=BF, device=dev)
    k, v = (torch.randn(320, 1, D, generator=g).to(BF).to(dev) for _ in range(2))
    k[:150] = -2.0e36                                    # 64 products: scores of -1.6e37
    k[199] = math.nan
    k[300:], v[300:] = math.inf, math.nan
    k[200:], v[250:300] = math.inf, math.inf
    ref, mag, _ = prompt_reference(q[:199], k[:199], v[:199], [199], [199], True)
    out = kernels.prompt_attn(q, k, v, starts_of(rows, dev))
    assert_attention_close(out[:199], ref, mag)
    assert out[199].isnan().all()


@pytest.mark.parametrize("past", [0, 10, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_values_that_are_not_finite_stay_within_their_128_rows(dev, past, D):
    n = 300
    g = torch.Generator().manual_seed(past)
    q = torch.randn(n, 2, D, generator=g).to(BF).to(dev)
    k, v = (torch.randn(n + past, 1, D, generator=g).to(BF).to(dev) for _ in range(2))
    starts, k_starts = starts_of([n], dev), starts_of([n + past], dev)
    want = kernels.prompt_attn(q, k, v, starts, k_starts)
    v[past + 128:past + 256] = math.nan               # the keys of rows 128 to 255
    v[past + 270] = math.inf
    got = kernels.prompt_attn(q, k, v, starts, k_starts)
    assert torch.equal(got[:128], want[:128]) and got[128:].isnan().any(-1).all()


def test_prompt_starts_outside_the_tensors_are_cut(dev):
    q = torch.randn(64, 1, 64, device=dev).to(BF)
    out = kernels.prompt_attn(q, q, q, ints([-5, 40, 30, 9999], dev))
    ref, mag, _ = prompt_reference(q[:40], q[:40], q[:40], [40], [40], True)
    assert_attention_close(out[:30], ref[:30], mag[:30])
    assert torch.isfinite(out).all()
    assert torch.equal(kernels.prompt_attn(q, q, q, ints([-5, 40], dev))[:30], out[:30])
    assert (kernels.prompt_attn(q, q, q, ints([0, 0], dev)) == 0).all()
    assert (kernels.prompt_attn(q, q, q, ints([50, 20], dev)) == 0)[50:].all()
    assert (kernels.prompt_attn(q, q, q, ints([0], dev)) == 0).all()


# ------------------------------------------------------------------ single tokens
TOKENS = [
    # lens, heads, key heads, D, block
    ([1], 1, 1, 64, 16), ([333], 8, 8, 64, 32), ([0, 1, 15, 16, 17, 31, 32, 33], 4, 2, 128, 16),
    ([128, 129, 127, 0, 640], 12, 4, 128, 64), ([5000], 8, 2, 64, 16), ([2000, 3, 0, 7000, 129], 32, 8, 128, 128),
    ([3100, 1500], 20, 1, 128, 16), ([900, 1100], 33, 1, 64, 256), ([40] * 300, 2, 2, 64, 16),
    ([1] * 9 + [20000], 7, 7, 128, 32), ([4096] * 3, 16, 1, 64, 16),
    # tables that could hold more than the last-level cache, in both forms
    ([33] * 120, 8, 4, 128, 16), ([1] * 129 + [1024], 8, 4, 128, 16),
    # a wave a request and key head
    ([0, 1, 31, 32, 33, 128, 127, 65] * 17, 12, 4, 64, 16), ([256, 0, 200, 129] * 64, 24, 8, 128, 32),
]


@pytest.mark.parametrize("lens,H,Hk,D,block", TOKENS)
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("width", ["tight", "wide"])
def test_tokens(dev, lens, H, Hk, D, block, kv, width):
    """``wide``: tables that could hold far more, so that the work is cut into ranges and joined."""
    w = None if width == "tight" else max(-(-max(lens) // block), 5000 // block) + 3
    c = Cache(lens, Hk, D, block, kv, dev, seed=len(lens), layout="tokens" if len(lens) == 2 else "heads", width=w)
    q = (torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(1)) * 1.5).to(BF).to(dev)
    ref, mag, lse_ref = c.reference(q)
    lse = torch.empty(len(lens), H, device=dev)
    out = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales, lse=lse)
    assert_attention_close(out, ref, mag, weight=2 ** -16)
    assert_lse_close(lse, lse_ref)
    again = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales)
    assert torch.equal(out, again)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("wide", [0, 400])
def test_token_blocks_hold_anything_behind_the_last_token(dev, kv, wide):
    lens, block = [0, 5, 16, 45, 100], 16
    c = Cache(lens, 2, 128, block, kv, dev, width=7 + wide)
    q = torch.randn(5, 4, 128, device=dev).to(BF)
    want = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales)
    used = torch.zeros(c.n, block, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            used[c.tables[b, p // block].item(), p % block] = True
    used = used.to(dev)
    for pool in (c.k, c.v):
        if kv == "bf16":
            pool[~used] = math.nan
        else:
            pool.view(torch.uint8)[~used] = 0x7F   # NaN
    for s in (c.k_scales, c.v_scales):
        if s is not None:
            s[~used] = math.inf
    got = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales)
    assert torch.equal(got, want) and (got[0] == 0).all()


def test_token_entries_outside_the_pool_take_no_part(dev):
    c = Cache([100, 64], 2, 64, 16, "bf16", dev)
    c.tables[0, 2], c.tables[0, 4], c.tables[1, 0] = -1, c.n, 1 << 30
    q = torch.randn(2, 2, 64, device=dev).to(BF)
    ref, mag, _ = c.reference(q)
    assert_attention_close(kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t), ref, mag)


def test_token_lengths_past_the_table_and_negative_are_cut(dev):
    c = Cache([64, 64], 1, 64, 16, "bf16", dev)
    q = torch.randn(2, 1, 64, device=dev).to(BF)
    out = kernels.paged_attn(q, c.k, c.v, c.tables, ints([1 << 30, -3], dev))
    want = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t)
    assert torch.equal(out[0], want[0]) and (out[1] == 0).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_token_scores_of_any_size(dev, kv):
    """The first keys' scores are near the lowest number of float32, all alike: they share the weight, and have
    none once there are others."""
    lens = [150, 260]
    c = Cache(lens, 1, 64, 16, kv, dev)
    for b in range(2):
        for p in range(150):
            i, o = c.tables[b, p // 16].item(), p % 16
            if kv == "bf16":
                c.k[i, o] = -2.0e36
            else:
                c.k.view(torch.uint8)[i, o] = 0xB8           # -1
                c.k_scales[i, o] = 2.0e36
    q = torch.ones(2, 1, 64, dtype=BF, device=dev)
    ref, mag, _ = c.reference(q)
    assert_attention_close(kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales), ref, mag)


def test_token_offsets_past_32_bits(dev):
    """Blocks whose distance from the pool's start passes 2^32 bytes."""
    block, D, Hk = 256, 128, 1
    n = (1 << 32) // (block * D * 2) + 40
    k = torch.zeros(n, block, Hk, D, dtype=BF, device=dev)
    v = torch.zeros_like(k)
    x = torch.randn(300, Hk, D, device=dev).to(BF)
    slots = torch.arange(300, device=dev) + (n - 3) * block
    kernels.kv_paged_append(x, x, k, v, slots)
    q = torch.randn(1, 2, D, device=dev).to(BF)
    tables = ints([[n - 3, n - 2, 0, 0, 0, 0, 0, 0]], dev)
    out = kernels.paged_attn(q, k, v, tables, ints([300], dev))
    ref, mag, _ = prompt_reference(q, x, x, [1], [300], True)
    assert_attention_close(out, ref, mag)


# ------------------------------------------------------------------ together
def test_prompts_then_tokens_under_a_graph(dev):
    """Prompts admitted and attended, then tokens one at a time (a captured step, replayed), against attention
    over everything so far; half of the requests released at the end."""
    H, Hk, D, block, lens = 4, 2, 128, 16, [5, 31, 0, 64]
    B, steps, width, blocks = len(lens), 20, 8, 40
    g = torch.Generator().manual_seed(9)
    hist = [[torch.zeros(0, Hk, D, dtype=BF, device=dev)] * 2 for _ in lens]
    pools = [torch.full((blocks, Hk, block, D), math.nan, dtype=BF, device=dev).permute(0, 2, 1, 3) for _ in range(2)]
    tables = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(blocks, generator=g).int().to(dev)
    top, status, held = ints([blocks], dev), ints([0], dev), ints([0] * B, dev)

    def rows(T):
        return [torch.randn(T, h, D, generator=g).to(BF).to(dev) for h in (H, Hk, Hk)]

    q, k, v = rows(sum(lens) + 6)
    plan = kernels.kv_block_grow(tables, held, ints(lens, dev), free, top, status, block, q.shape[0], held, top)
    kernels.kv_paged_append(k, v, *pools, plan.slots)
    out = kernels.prompt_attn(q, k, v, plan.starts)
    ref, mag, _ = prompt_reference(q[:sum(lens)], k, v, lens, lens, True)
    assert_attention_close(out[:sum(lens)], ref, mag)
    at = 0
    for b, n in enumerate(lens):
        hist[b] = [k[at:at + n], v[at:at + n]]
        at += n

    one = ints([1] * B, dev)
    sq, sk, sv = (torch.zeros(B, h, D, dtype=BF, device=dev) for h in (H, Hk, Hk))

    def step():
        p = kernels.kv_block_grow(tables, held, one, free, top, status, block, B, held, top)
        kernels.kv_paged_append(sk, sv, *pools, p.slots)
        return kernels.paged_attn(sq, *pools, tables, held)

    graph, warm = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    save = [t.clone() for t in (tables, held, top)]
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    for t, s in zip((tables, held, top), save):
        t.copy_(s)
    with torch.cuda.graph(graph):
        out = step()
    for i in range(steps):
        for dst, src in zip((sq, sk, sv), rows(B)):
            dst.copy_(src)
        graph.replay()
        for b in range(B):
            hist[b] = [torch.cat([hist[b][0], sk[b:b + 1]]), torch.cat([hist[b][1], sv[b:b + 1]])]
            ref, mag, _ = prompt_reference(sq[b:b + 1], *hist[b], [1], [lens[b] + i + 1], True)
            assert_attention_close(out[b:b + 1], ref, mag, f"step {i} request {b}")
        torch.cuda.synchronize()
    assert status.item() == 0 and held.tolist() == [n + steps for n in lens]
    done = torch.tensor([True, False, True, False], device=dev)
    kernels.kv_block_release(tables, held, done, free, top, status, block, held, top)
    assert held.tolist() == [0, lens[1] + steps, 0, lens[3] + steps]
    in_use = [tables[b, j].item() for b in (1, 3) for j in range(-(-held[b].item() // block))]
    assert sorted(free[:top.item()].tolist() + in_use) == list(range(blocks)) and status.item() == 0


def test_two_graphs_and_eager_calls_have_workspaces_of_their_own(dev):
    """Calls that share keys among workgroups, captured twice with other inputs, replayed side by side on two
    streams with eager calls between."""
    c = Cache([3000, 20, 700], 2, 128, 16, "bf16", dev)
    rows, keys = [20, 3], [2500, 1800]
    starts, k_starts = starts_of(rows, dev), starts_of(keys, dev)
    g = torch.Generator().manual_seed(5)
    sets = []
    for _ in range(3):
        q1 = torch.randn(3, 8, 128, generator=g).to(BF).to(dev)
        q2, k, v = (torch.randn(n, h, 128, generator=g).to(BF).to(dev) for n, h in ((23, 4), (4300, 2), (4300, 2)))
        sets.append((q1, q2, k, v))

    def call(q1, q2, k, v):
        return (kernels.paged_attn(q1, c.k, c.v, c.tables, c.lens_t), kernels.prompt_attn(q2, k, v, starts, k_starts))

    want = [[t.clone() for t in call(*s)] for s in sets]
    ref, mag, _ = c.reference(sets[0][0])
    assert_attention_close(want[0][0], ref, mag, weight=2 ** -16)
    torch.cuda.synchronize()
    graphs = []
    for s in sets[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*s)
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(4):
        for _, out, _ in graphs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = call(*sets[2])
        torch.cuda.synchronize()
        for got, w in zip([graphs[0][1], graphs[1][1], eager], want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_on_another_stream(dev):
    c = Cache([3000, 500], 2, 128, 16, "bf16", dev)
    q = torch.randn(2, 8, 128, device=dev).to(BF)
    want = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for outs in got for o in outs)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_cache_object(dev, kv):
    """Prompts, continued prompts and single tokens of two layers through one cache, some requests released and
    their blocks used again; every result against attention over the request's history as the cache holds it."""
    H, Hk, D, R = 4, 2, 64, 5
    c = PagedKVCache(layers=2, requests=R, blocks=21, heads=Hk, dim_head=D, max_tokens=130, block_size=16, kv_dtype=kv)
    g = torch.Generator().manual_seed(2)
    held = [0] * R
    hist = [[[torch.zeros(0, Hk, D, dtype=torch.float64, device=dev)] * 2 for _ in range(R)] for _ in range(2)]

    def stored(x):
        """What the cache holds of bf16 rows."""
        if kv == "bf16":
            return x.double()
        s = (x.double().abs().amax(-1, keepdim=True) / 448).float()
        return (x.double() / s.double()).float().to(E4).double() * s.double()

    def run(new, kind, behind=0):
        T = sum(new) + behind
        plan = c.grow(new, T)
        for b in range(R):
            held[b] += new[b]
        for layer in range(2):
            q, k, v = (torch.randn(T, h, D, generator=g).to(BF).to(dev) for h in (H, Hk, Hk))
            c.append(layer, k, v, plan)
            out = c.attend(layer, q) if kind == "token" else c.attend_prompts(layer, q, k, v, plan, kind == "continued")
            at = 0
            for b, n in enumerate(new):
                own = [x[at:at + n] for x in (k, v)]
                hist[layer][b] = [torch.cat([old, stored(x)]) for old, x in zip(hist[layer][b], own)]
                keys = [x.double() for x in own] if kind == "prompt" else hist[layer][b]
                ref, mag, _ = prompt_reference(q[at:at + n], *keys, [n], [keys[0].shape[0]], True)
                assert_attention_close(out[at:at + n], ref, mag, f"{kind} {layer} {b}")
                at += n
            assert (out[at:] == 0).all()
        assert c.lens.tolist() == held

    run([33, 5, 0, 70, 16], "prompt", behind=3)
    run([1] * R, "token")
    run([7, 0, 20, 1, 15], "continued", behind=2)
    c.release([True, False, False, True, False])
    for b in (0, 3):
        held[b], hist[0][b], hist[1][b] = 0, [x[:0] for x in hist[0][b]], [x[:0] for x in hist[1][b]]
    run([100, 0, 0, 40, 0], "prompt")
    run([1] * R, "token")
    c.check()
    before = [t.clone() for t in (c.tables, c.lens, c.top)]
    c.grow([0, 0, 0, 100, 0], 100)          # 141 tokens fit a row of 144, but 6 more blocks are not there: 16 of 21 are taken
    with pytest.raises(KVArenaFull, match="blocks were free"):
        c.check()
    c.grow([50, 0, 0, 0, 0], 50)
    with pytest.raises(KVArenaFull, match="outgrew 144"):
        c.check()
    c.grow([2, 0, 0, 0, 0], 1)
    with pytest.raises(ValueError, match="more tokens than rows"):
        c.check()
    assert all(torch.equal(a, b) for a, b in zip((c.tables, c.lens, c.top), before))
    c.check()


@pytest.mark.parametrize("first,rows,keys", [(50, [14], None), (300, [200, 0, 30], None), (64, [20], [3000]),
                                             (17, [], None), (40, [3] * 70, None)])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_rows_before_the_first_prompt(dev, first, rows, keys, D):
    """A call over some of the prompts: the rows of the others are zero in a new result, and left in one given."""
    T = first + sum(rows) + 9
    g = torch.Generator().manual_seed(first)
    q = torch.randn(T, 4, D, generator=g).to(BF).to(dev)
    k, v = (torch.randn(sum(keys or rows) + first, 2, D, generator=g).to(BF).to(dev) for _ in range(2))
    starts = starts_of(rows, dev) + first
    k_starts = starts_of(keys or rows, dev) + first
    mine = slice(first, first + sum(rows))
    ref, mag, lse_ref = prompt_reference(q[mine], k[first:], v[first:], rows, keys or rows, True)
    given = torch.full_like(q, 3.0)
    kernels.prompt_attn(q, k, v, starts, k_starts, out=given)
    lse = torch.full((4, T), 5.0, device=dev)
    dirty = torch.full_like(q, math.nan)
    at = dirty.data_ptr()
    del dirty                                            # the new result takes this memory
    out = kernels.prompt_attn(q, k, v, starts, k_starts, lse=lse)
    assert out.data_ptr() == at
    assert_attention_close(out[mine], ref, mag)
    assert_lse_close(lse[:, mine], lse_ref)
    rest = torch.ones(T, dtype=torch.bool, device=dev)
    rest[mine] = False
    assert (out[rest] == 0).all() and (lse[:, rest] == -math.inf).all()
    assert torch.equal(given[mine], out[mine]) and (given[rest] == 3).all()


def _share(a, b):
    """Whether two views of one storage have an element in common."""
    def elements(t):
        at = torch.tensor([t.storage_offset()])
        for n, step in zip(t.shape, t.stride()):
            at = (at[:, None] + torch.arange(n) * step).flatten()
        return set(at.tolist())
    return bool(elements(a) & elements(b))


def test_append_refuses_pools_that_overlap_and_takes_pools_that_take_turns(dev):
    """No rows, so nothing is launched: whether K's and V's pools share memory, against their elements."""
    none, slots = torch.empty(0, 2, 64, dtype=BF, device=dev), torch.empty(0, dtype=torch.int64, device=dev)
    memory = torch.empty(1 << 16, dtype=BF, device=dev)
    rng = random.Random(3)
    refused = 0
    for _ in range(300):
        sizes = {"n": rng.choice([1, 2, 3]), "t": 16, "h": 2}
        order = rng.sample(["n", "t", "h", "pair"], 4)     # from the innermost dimension; "pair": K, then V
        step, strides = 64, {}
        for d in order:
            strides[d] = step
            step = step * sizes.get(d, 2) + rng.choice([0, 0, 8])
        at = strides["pair"] if rng.random() < 0.5 else 8 * rng.randint(1, step // 4)
        shape, st = (sizes["n"], 16, 2, 64), (strides["n"], strides["t"], strides["h"], 1)
        k, v = memory.as_strided(shape, st), memory.as_strided(shape, st, at)
        if _share(k, v):
            refused += 1
            with pytest.raises(ValueError, match="k_pool overlaps"):
                kernels.kv_paged_append(none, none, k, v, slots)
            with pytest.raises(ValueError, match="k_pool overlaps"):
                kernels.kv_paged_append(none, none, v, k, slots)
        else:
            kernels.kv_paged_append(none, none, k, v, slots)
            kernels.kv_paged_append(none, none, v, k, slots)
    assert 50 < refused < 250


def test_append_refuses_rows_and_scales_inside_the_pools(dev):
    c = Cache([40], 2, 64, 16, "fp8", dev, layout="tokens")
    x = torch.zeros(4, 2, 64, dtype=BF, device=dev)
    slots = torch.arange(4, device=dev)
    before = [t.view(torch.uint8).clone() for t in (c.k, c.v)]
    inside = c.k.view(torch.uint8).flatten()[:1024].view(BF).view(4, 2, 64)
    for k, v, match in ((inside, x, "k_pool overlaps"), (x, inside, "k_pool overlaps")):
        with pytest.raises(ValueError, match=match):
            kernels.kv_paged_append(k, v, c.k, c.v, slots, c.k_scales, c.v_scales)
    scales = c.k.view(torch.uint8).flatten().view(torch.float32)[:c.n * 32].view(c.n, 2, 16).permute(0, 2, 1)
    assert scales.data_ptr() == c.k.data_ptr()
    with pytest.raises(ValueError, match="k_pool overlaps"):
        kernels.kv_paged_append(x, x, c.k, c.v, slots, scales, c.v_scales)
    both = torch.empty(c.n * 32 + 16, device=dev)
    first, second = (both[o:o + c.n * 32].view(c.n, 2, 16).permute(0, 2, 1) for o in (0, 16))
    with pytest.raises(ValueError, match="k_scales overlaps"):
        kernels.kv_paged_append(x, x, c.k, c.v, slots, first, second)
    assert all(torch.equal(t.view(torch.uint8), b) for t, b in zip((c.k, c.v), before))


def test_append_into_pools_that_take_turns(dev):
    """K and V of a block, or of a token, side by side in one storage."""
    for shape, pair, dims in (((5, 2, 2, 16, 64), 1, (0, 2, 1, 3)), ((5, 16, 2, 2, 64), 2, (0, 1, 2, 3))):
        store = torch.zeros(shape, dtype=BF, device=dev)
        k_pool, v_pool = (store.select(pair, i).permute(dims) for i in (0, 1))
        x = torch.randn(20, 4, 64, device=dev).to(BF)
        slots = torch.randperm(80, device=dev)[:20]
        kernels.kv_paged_append(x[:, :2], x[:, 2:], k_pool, v_pool, slots)
        assert torch.equal(k_pool[slots // 16, slots % 16], x[:, :2])
        assert torch.equal(v_pool[slots // 16, slots % 16], x[:, 2:])


def test_results_over_what_the_call_reads_are_refused(dev):
    c = Cache([30, 5], 2, 64, 16, "fp8", dev, layout="tokens")
    q = torch.randn(2, 2, 64, device=dev).to(BF)

    def token(match, **kw):
        with pytest.raises(ValueError, match=match):
            kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales, **kw)

    in_pool = c.v.view(torch.uint8).flatten()
    token("out overlaps", out=in_pool[256:768].view(BF).view(2, 2, 64))
    token("lse overlaps", lse=in_pool[:16].view(torch.float32).view(2, 2))
    token("lse overlaps", lse=q.flatten()[:8].view(torch.float32).view(2, 2))
    wide = torch.zeros(3, 2, 64, device=dev, dtype=BF)
    q = wide[:2]
    token("out overlaps", out=wide[1:])                      # q's rows, one further
    token("out overlaps", out=wide.flatten()[:256].view(2, 2, 64).transpose(0, 1))
    out = torch.zeros(2, 2, 64, device=dev, dtype=BF)
    token("out overlaps", out=out, lse=out.flatten()[:8].view(torch.float32).view(2, 2))

    x = torch.randn(40, 4, 64, device=dev).to(BF)
    starts = starts_of([30, 10], dev)
    k, v = x[:, :2], x[:, 2:]

    def prompt(match, q, k, v, **kw):
        with pytest.raises(ValueError, match=match):
            kernels.prompt_attn(q, k, v, starts, **kw)

    q = torch.randn(40, 2, 64, device=dev).to(BF)
    prompt("out overlaps", q, k, v, out=x[:, 1:3])
    prompt("out overlaps", q, q, v, out=q)                    # the queries' memory, but the keys' as well
    prompt("out overlaps", q, k, v, out=x.flatten()[64:64 + 40 * 128].view(40, 2, 64))
    prompt("lse overlaps", q, k, v, lse=x.flatten()[:160].view(torch.float32).view(2, 40))


def test_results_between_what_the_call_reads(dev):
    """q, k, v and the result take turns in one storage, rows of one prompt among others."""
    T, D, rows = 150, 64, [100, 50]
    x = torch.randn(T, 10, D, generator=torch.Generator().manual_seed(1)).to(BF).to(dev)
    q, k, v, out = x[:, :4], x[:, 4:5], x[:, 5:6], x[:, 6:]
    starts = starts_of(rows, dev)
    want, kv = kernels.prompt_attn(q, k, v, starts), x[:, :6].clone()
    kernels.prompt_attn(q, k, v, starts, out=out)
    assert torch.equal(out, want) and torch.equal(x[:, :6], kv)
    kernels.prompt_attn(q, k, v, starts, out=q)
    assert torch.equal(q, want) and torch.equal(x[:, 4:6], kv[:, 4:])
    # one row over all keys: its result lies between the keys' rows
    one, at = ints([0, 1], dev), ints([0, T], dev)
    want = kernels.prompt_attn(q[70:71], k, v, one, at)
    kernels.prompt_attn(q[70:71], k, v, one, at, out=out[70:71])
    assert torch.equal(out[70:71], want) and torch.equal(x[:, 4:6], kv[:, 4:])


def test_continued_prompts_gather_the_tables_of_one_call_at_a_time(dev):
    """9000 rows of two requests with table rows of 4096 entries: 64 MiB of tables for each 4096 rows."""
    rows, H, D = [8000, 1000], 1, 64
    c = PagedKVCache(layers=1, requests=2, blocks=600, heads=1, dim_head=D, max_tokens=4096 * 16, block_size=16)
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(sum(rows) + 5, H, D, generator=g).to(BF).to(dev) for _ in range(3))
    plan = c.grow(rows, sum(rows) + 5)
    c.append(0, k, v, plan)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = c.attend_prompts(0, q, k, v, plan, continued=True)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 96 << 20
    ref, mag, _ = prompt_reference(q[:9000], k[:9000], v[:9000], rows, rows, True)
    assert_attention_close(out[:9000], ref, mag, weight=2 ** -16)
    assert (out[9000:] == 0).all()


EARLIER = 1 << 8   # a bit of the status word that an earlier call may have left


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"top": 2}, N.BLOCKS_FREE), ({"top": -1}, N.BLOCKS_FREE), ({"top": 251}, N.BLOCKS_FREE),
    ({"width": 2, "new": 30}, N.BLOCKS_WIDTH), ({"tokens": -1}, N.BLOCKS_TOKENS),
    ({"len": -5}, N.BLOCKS_LENGTH), ({"new": -1, "tokens": 100}, N.BLOCKS_LENGTH),
    ({"top": 1, "width": 2, "new": 30, "tokens": -1}, N.BLOCKS_FREE | N.BLOCKS_WIDTH | N.BLOCKS_TOKENS),
])
def test_grow_notes_every_reason_and_no_other(dev, change, code, big, in_place):
    block, lens, new = 16, [5, 0, 30, 16], [20, 1, 2, 1]
    if big:
        new[1] = 3000 if "width" not in change else 1
    new[0] = change.get("new", new[0])
    lens[3] = change.get("len", lens[3])
    T = sum(new) + change.get("tokens", 0) + (2000 if big and "width" in change and "tokens" not in change else 0)
    width, blocks = change.get("width", 200), 250
    tables, free, top = _table_state(dev, [max(n, 0) for n in lens], block, width, blocks)
    top = change.get("top", top)
    t, le, fr, tp, status = ints(tables, dev), ints(lens, dev), ints(free, dev), ints([top], dev), ints([EARLIER], dev)
    plan = kernels.kv_block_grow(t, le, ints(new, dev), fr, tp, status, block, T, le if in_place else None,
                                 tp if in_place else None)
    assert status.item() == EARLIER | code
    if code == 0:
        want = grow_reference(tables, lens, new, free, top, block, T)
        assert t.tolist() == want[0] and plan.slots.tolist() == want[1] and plan.top.tolist() == [want[5]]
        return
    assert t.tolist() == tables and plan.lens.tolist() == lens and plan.top.tolist() == [top] and fr.tolist() == free
    assert plan.starts.tolist() == [0] * 5 and plan.slots.tolist() == [-1] * T and plan.positions.tolist() == [0] * T


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"top": 2}, N.BLOCKS_FREE), ({"top": -1}, N.BLOCKS_FREE),
    ({"kept": 1 << 30}, 0),                                   # a row that is not released may hold anything
    ({"released": 16 * 5000}, N.BLOCKS_WIDTH | N.BLOCKS_FREE), ({"released": -1}, N.BLOCKS_LENGTH),
    ({"kept": -1}, N.BLOCKS_LENGTH), ({"released": 16 * 5000, "kept": -1, "top": 0},
                                      N.BLOCKS_WIDTH | N.BLOCKS_FREE | N.BLOCKS_LENGTH),
])
def test_release_notes_every_reason_and_no_other(dev, change, code, wide, in_place):
    """``wide``: tables and a stack of more than 1024 blocks, so that the books are kept by a second launch."""
    block, lens, done = 16, [40, 0, 17, 100], [True, True, False, True]
    width, blocks = (1000, 3000) if wide else (8, 16)
    tables, free, top = _table_state(dev, lens, block, width, blocks)
    if "top" in change:
        top = change["top"] if change["top"] <= 0 else blocks - change["top"]
    lens[0], lens[2] = change.get("released", lens[0]), change.get("kept", lens[2])
    t, le, fr, tp, status = ints(tables, dev), ints(lens, dev), ints(free, dev), ints([top], dev), ints([EARLIER], dev)
    out, top_out = kernels.kv_block_release(t, le, torch.tensor(done, device=dev), fr, tp, status, block,
                                            le if in_place else None, tp if in_place else None)
    assert status.item() == EARLIER | code and t.tolist() == tables
    if code == 0:
        back = [tables[b][j] for b in (0, 3) for j in range(-(-lens[b] // block))]
        assert out.tolist() == [0, 0, lens[2], 0] and top_out.tolist() == [top + len(back)]
        assert fr.tolist() == free[:top] + back + free[top + len(back):]
    else:
        assert out.tolist() == lens and top_out.tolist() == [top] and fr.tolist() == free


@pytest.mark.parametrize("kv,requests", [("bf16", 257), ("fp8", 514)])
def test_token_a_wave_a_request_of_tables_past_the_last_level_cache(dev, kv, requests):
    """Tables of 256 tokens a request, 8 heads x 128: just past 256 MiB."""
    rng = random.Random(requests)
    lens = [rng.choice([0, 1, 31, 32, 33, 64, 256, rng.randint(1, 60)]) for _ in range(requests)]
    c = Cache(lens, 8, 128, 16, kv, dev, width=16)
    q = (torch.randn(requests, 8, 128, generator=torch.Generator().manual_seed(1)) * 1.5).to(BF).to(dev)
    ref, mag, lse_ref = c.reference(q)
    lse = torch.empty(requests, 8, device=dev)
    out = kernels.paged_attn(q, c.k, c.v, c.tables, c.lens_t, c.k_scales, c.v_scales, lse=lse)
    assert_attention_close(out, ref, mag, weight=2 ** -16)
    assert_lse_close(lse, lse_ref)
